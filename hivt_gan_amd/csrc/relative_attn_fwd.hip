// Forward of the attention with a learned bias for each bucket of relative positions.
//
// One pass over the keys with the running maximum and sum of the softmax.  A workgroup of four waves owns 64 QB query
// rows of one (batch, head) and walks 64-key tiles; the tile after the one being worked on is already on its way into
// registers.  A wave owns 16 QB query rows: its scores, its statistics and its share of the output stay in registers
// (see relative_core.h for the layout), keys and values come from LDS.
//   * Tiles without any allowed key are not loaded; tiles beyond the causal limit are not walked.
//   * Rows of masked keys enter the LDS tile as zeros, so whatever they hold cannot reach a result.
//   * Few query rows and a long axis of keys: the keys are cut into `splits` ranges, each leaves its unnormalised sum,
//     maximum and sum of weights, and a second kernel joins them.  Query heads of a group then share the rows of a tile
//     (`pack`), so a key is read once for all of them.
#include "relative_core.h"

namespace hivt {
namespace rel {
namespace {

constexpr int kBN = 64;

// Two waves to a SIMD, so that one's matrix instructions run beside the other's exponentials, where the registers allow.
// Bound by issue: at heads of 128 the matrix cores are busy for a quarter and the vector units (bias, exponentials, their
// rounding) for 45 % of the time.  Measured, bf16: 2 x 4096 causal, 16 heads of 128: 282 us, 487 TFLOP/s; 8 x 1024 masked,
// 16 heads of 64: 75 us, 455 TFLOP/s; fp32 64 x 301, 8 heads of 16: 58 us.  One query behind 30000 keys, 8 sequences of
// 8 key heads of 128: 178 us, 5.5 TB/s, bound by memory.
template <typename T, int DP, int QB>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP >= 96 && QB == 2 ? 1 : 2) void fwd_kernel(const Args a) {
  using TL = Tile<T, DP>;
  constexpr int NB = DP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* const kt = reinterpret_cast<T*>(smem);
  T* const vt = kt + kBN * TL::PITCH;
  float* const bias = reinterpret_cast<float*>(vt + kBN * TL::PITCH);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
  const int group = a.pack ? a.rep : 1;                    // heads whose rows share a tile
  const int rows = a.M * group;
  const int qtiles = (rows + 64 * QB - 1) / (64 * QB);
  const int heads = a.H / group;
  int unit, inner;
  walk(blockIdx.x, a.B * heads, qtiles * a.splits, unit, inner);
  const int split = inner % a.splits;
  const int qtile = qtiles - 1 - inner / a.splits;          // the longest rows of a causal problem first
  const int b = unit / heads, h0 = (unit % heads) * group, g = h0 / a.rep;

  const int width = bias_width(a), hi = bias_hi(a);
  for (int e = tid; e < width; e += 256) {
    const int bucket = entry_bucket(a, e);
    for (int s = 0; s < group; ++s) bias[s * width + e] = bias2(a.table[(int64_t)bucket * a.H + h0 + s]);
  }

  // this wave's rows; a row past the last one repeats it and is not stored
  const int row0 = qtile * 64 * QB + wave * 16 * QB;
  const bool active = row0 < rows;
  int pos[QB], slot[QB];
  bool live[QB];
  Frag<T, TL::E> qf[QB][TL::KSTEPS];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = row0 + qb * 16 + (lane & 15);
    live[qb] = r < rows;
    const int rc = min(r, rows - 1);
    const int s = rc / group;
    slot[qb] = rc % group;
    pos[qb] = s + a.offset;
    const T* q = static_cast<const T*>(a.q) + b * a.q_st[0] + s * a.q_st[1] + (h0 + slot[qb]) * a.q_st[2];
#pragma unroll
    for (int ks = 0; ks < TL::KSTEPS; ++ks)
      qf[qb][ks] = load_frag<T, TL::E>(q, ks * TL::KS + quad * TL::E, a.d, a.q_align, live[qb]);
  }
  const int first = min(row0, rows - 1) / group + a.offset, last = min(row0 + 16 * QB, rows) - 1;
  const int pos_lo = first, pos_hi = max(last, 0) / group + a.offset;
  // the workgroup's range of tiles
  const int wg_last = (min((qtile + 1) * 64 * QB, rows) - 1) / group + a.offset;
  const int keys_end = a.causal ? min(a.seen, wg_last + 1) : a.seen;
  const int tiles = keys_end > 0 ? (keys_end + kBN - 1) / kBN : 0;
  const int t_begin = split * a.tiles_per_split, t_end = min(tiles, t_begin + a.tiles_per_split);

  f32x4 o[NB][QB];
  float m[QB], l[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m[qb] = -INFINITY;
    l[qb] = 0.0f;
#pragma unroll
    for (int n = 0; n < NB; ++n) o[n][qb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const T* const kbase = static_cast<const T*>(a.k) + b * a.k_st[0] + g * a.k_st[2];
  const T* const vbase = static_cast<const T*>(a.v) + b * a.v_st[0] + g * a.v_st[2];
  Loader<T, DP, kBN, 256> kl, vl;
  uint64_t bits = 0;
  int t = t_begin;
  auto seek = [&]() {  // to the next tile that holds an allowed key, and asks for it
    while (t < t_end && (bits = tile_keys(a, b, t * kBN, lane)) == 0) ++t;
    if (t < t_end) {
      const int64_t k0 = (int64_t)t * kBN;
      auto keep = [&](int row) { return (bits >> row & 1) != 0; };
      kl.load(kbase + k0 * a.k_st[1], a.k_st[1], a.d, a.k_align, tid, bits == ~0ull, keep);
      vl.load(vbase + k0 * a.v_st[1], a.v_st[1], a.d, a.v_align, tid, bits == ~0ull, keep);
    }
  };
  seek();
  while (t < t_end) {
    __syncthreads();  // the tile before has been read by every wave
    kl.store(kt, tid);
    vl.store(vt, tid);
    const int k0 = t * kBN;
    const uint64_t keys = bits;
    ++t;
    seek();
    __syncthreads();
    if (!active || (a.causal && k0 > pos_hi)) continue;

    // A block's operands are read while the block before is multiplied (left alone, the compiler reads each right before
    // its product, and two waves do not hide that).
    f32x4 s[4][QB];
    Frag<T, TL::E> kf[2][TL::KSTEPS];
#pragma unroll
    for (int ks = 0; ks < TL::KSTEPS; ++ks) kf[0][ks] = TL::rows(kt, 0, ks, lane);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      if (kb < 3) {
#pragma unroll
        for (int ks = 0; ks < TL::KSTEPS; ++ks) kf[(kb + 1) & 1][ks] = TL::rows(kt, (kb + 1) * 16, ks, lane);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) s[kb][qb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < TL::KSTEPS; ++ks)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) Frag<T, TL::E>::mma(kf[kb & 1][ks], qf[qb][ks], s[kb][qb]);
    }
    constexpr int RING = sizeof(T) == 2 ? 4 : 2;
    Frag<T, 8> vf[RING];  // and the first of the values' while the softmax runs
#pragma unroll
    for (int i = 0; i < RING && i < 2 * NB; ++i) vf[i] = TL::cols(vt, i / NB * 32, i % NB * 16, lane);
    // scores in base-2 exponent units, with the bias of their distance
    const int rel_hi = k0 + kBN - 1 - pos_lo, rel_lo = k0 - pos_hi;
    const bool far = rel_hi <= -a.sat || rel_lo >= hi;
    const bool whole = keys == ~0ull && (!a.causal || rel_hi <= 0);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const float* const tab = bias + slot[qb] * width;
      // Far, whole tiles: one bias for all pairs, which waits until the exponent.  (A huge one may not: added to the score
      // at once it takes the score's digits, and tiles have to agree on that.)  Other tiles put bias and mask into the
      // scores; both then take the same way, so that no registers are moved between two.
      float mul = a.scale2, add = tab[rel_hi <= -a.sat ? 0 : width - 1];
      if (!__all(far && whole && a.scale2 > 0.0f && fabsf(add) <= kPlainBias)) {
        if (far) {
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[kb][qb][r] = fmaf(s[kb][qb][r], a.scale2, add);
        } else {
          const float* const at = tab + k0 + quad * 4 - pos[qb] + a.sat + kMargin;
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[kb][qb][r] = fmaf(s[kb][qb][r], a.scale2, at[kb * 16 + r]);
        }
        mul = 1.0f;
        add = 0.0f;
        if (!whole) {
          const int lim = a.causal ? pos[qb] - k0 : kBN;  // keys of the tile up to here
#pragma unroll
          for (int kb = 0; kb < 4; ++kb) {
            const uint32_t nibble = (uint32_t)(keys >> (kb * 16 + quad * 4));
#pragma unroll
            for (int r = 0; r < 4; ++r)
              s[kb][qb][r] = !(nibble >> r & 1) || kb * 16 + quad * 4 + r > lim ? -INFINITY : s[kb][qb][r];
          }
        }
      }
      float top = s[0][qb][0];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[kb][qb][r]);
      const float m_new = fmaxf(m[qb], quad_max(fmaf(top, mul, add)));
      const float m_safe = m_new == -INFINITY ? 0.0f : m_new;  // a row without any allowed key so far
      const float shift = add - m_safe;
      float sum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[kb][qb][r] = fexp2(fmaf(s[kb][qb][r], mul, shift));
          sum += s[kb][qb][r];
        }
      const float alpha = fexp2(m[qb] - m_safe);
      m[qb] = m_new;
      l[qb] = fmaf(l[qb], alpha, sum);  // (this lane's keys; the four lanes of a query are added at the end)
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[n][qb][r] *= alpha;
      }
    }
    // o += v^T p: the weights are rounded to the operands' type, their sum above is not
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      Frag<T, 8> pf[QB];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) pf[qb] = pair_frag<T>(s[2 * kk][qb], s[2 * kk + 1][qb]);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int at = kk * NB + n;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) Frag<T, 8>::mma(vf[at % RING], pf[qb], o[n][qb]);
        if (at + RING < 2 * NB) vf[at % RING] = TL::cols(vt, (at + RING) / NB * 32, (at + RING) % NB * 16, lane);
      }
    }
  }
  if (!active) return;

#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float total = quad_sum(l[qb]);
    if (!live[qb]) continue;
    const int r = row0 + qb * 16 + (lane & 15);
    if (a.splits > 1) {
      const int64_t at = ((int64_t)unit * a.splits + split) * rows + r;
      float* po = a.partial + at * (a.d + 2);
      if (quad == 0) {
        po[a.d] = m[qb];
        po[a.d + 1] = total;
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n * 16 + quad * 4 + j < a.d) po[n * 16 + quad * 4 + j] = o[n][qb][j];
      continue;
    }
    const float inv = total > 0.0f ? 1.0f / total : 0.0f;  // a row without any allowed key is zero
    const float norm = total != total ? total : inv;       // (NaN scores stay NaN)
    const int s = r / group, h = h0 + slot[qb];
    T* out = static_cast<T*>(a.out) + b * a.o_st[0] + s * a.o_st[1] + h * a.o_st[2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      f32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = o[n][qb][j] * norm;
      store4(out, n * 16 + quad * 4, a.d, w);
    }
    if (a.stats != nullptr && quad == 0)
      a.stats[((int64_t)b * a.H + h) * a.M + s] = make_float2(m[qb] == -INFINITY ? 0.0f : m[qb], norm);
  }
}

// One wave joins the splits of one query row, in ascending order of the keys (8 us; 17 us after the 30000 keys above).
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
  const int lane = threadIdx.x & 63;
  const int group = a.pack ? a.rep : 1, rows = a.M * group, heads = a.H / group;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= (int64_t)a.B * heads * rows) return;
  const int unit = (int)(at / rows), r = (int)(at % rows);
  const int b = unit / heads, h = (unit % heads) * group + r % group, s = r / group;
  const float* const p0 = a.partial + ((int64_t)unit * a.splits * rows + r) * (a.d + 2);
  const int64_t step = (int64_t)rows * (a.d + 2);
  // at most 128 splits: a lane weighs two of them
  float ms[2], w[2], l = 0.0f, m = -INFINITY;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = lane + 64 * j;
    ms[j] = i < a.splits ? p0[i * step + a.d] : -INFINITY;
    w[j] = i < a.splits ? p0[i * step + a.d + 1] : 0.0f;
    m = fmaxf(m, ms[j]);
  }
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float m_safe = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float sum = w[j];
    w[j] = fexp2(ms[j] - m_safe);
    l += w[j] * sum;
  }
  l = wave_sum(l);
  float o0 = 0.0f, o1 = 0.0f;
#pragma unroll 8
  for (int i = 0; i < a.splits; ++i) {
    const float* p = p0 + i * step;
    const float wi = __shfl(i < 64 ? w[0] : w[1], i & 63, 64);
    if (lane < a.d) o0 += wi * p[lane];
    if (lane + 64 < a.d) o1 += wi * p[lane + 64];
  }
  const float norm = l != l ? l : l > 0.0f ? 1.0f / l : 0.0f;
  T* out = static_cast<T*>(a.out) + b * a.o_st[0] + s * a.o_st[1] + h * a.o_st[2];
  if (lane < a.d) out[lane] = (T)(o0 * norm);
  if (lane + 64 < a.d) out[lane + 64] = (T)(o1 * norm);
  if (a.stats != nullptr && lane == 0) a.stats[((int64_t)b * a.H + h) * a.M + s] = make_float2(m_safe, norm);
}

template <typename T, int DP, int QB>
int launch_tile(const Args& a, hipStream_t stream) {
  using TL = Tile<T, DP>;
  const int group = a.pack ? a.rep : 1;
  const int64_t qtiles = ((int64_t)a.M * group + 64 * QB - 1) / (64 * QB);
  const int64_t blocks = (int64_t)a.B * (a.H / group) * qtiles * a.splits;
  HIVT_REQUIRE(blocks < ((int64_t)1 << 31), HIVT_ERR_ARG, "hivt_relative_attn_fwd: %lld workgroups", (long long)blocks);
  const size_t lds = (size_t)2 * kBN * TL::PITCH * sizeof(T) + (size_t)group * bias_width(a) * sizeof(float);
  if (lds > 48 * 1024)
    HIVT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&fwd_kernel<T, DP, QB>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), "hivt_relative_attn_fwd");
  hipLaunchKernelGGL((fwd_kernel<T, DP, QB>), dim3((unsigned)blocks), dim3(256), lds, stream, a);
  HIVT_CHECK_LAUNCH("hivt_relative_attn_fwd");
  if (a.splits > 1) {
    const int64_t joined = ((int64_t)a.B * a.H * a.M + 3) / 4;
    hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)joined), dim3(256), 0, stream, a);
    HIVT_CHECK_LAUNCH("hivt_relative_attn_fwd (join)");
  }
  return HIVT_OK;
}

template <typename T, int DP>
int launch_width(const Args& a, hipStream_t stream) {
  const int rows = a.M * (a.pack ? a.rep : 1);
  return rows <= 64 ? launch_tile<T, DP, 1>(a, stream) : launch_tile<T, DP, 2>(a, stream);
}

template <typename T>
int launch_type(const Args& a, hipStream_t stream) {
  if (a.d <= 16) return launch_width<T, 16>(a, stream);
  if (a.d <= 32) return launch_width<T, 32>(a, stream);
  if (a.d <= 64) return launch_width<T, 64>(a, stream);
  if (a.d <= 96) return launch_width<T, 96>(a, stream);
  return launch_width<T, 128>(a, stream);
}

// How the work is cut: `pack` where all rows of a group fit one 64-row tile (the bias tables of the group have to fit
// LDS beside the key and value tiles), and the keys split where the workgroups would leave the 256 compute units idle.
void plan(Args& a) {
  a.pack = a.rep > 1 && (int64_t)a.M * a.rep <= 64 && (int64_t)a.rep * bias_width(a) <= 8192 ? 1 : 0;
  const int group = a.pack ? a.rep : 1;
  const int64_t rows = (int64_t)a.M * group;
  const int64_t qtiles = rows <= 64 ? 1 : (rows + 127) / 128;
  const int64_t work = (int64_t)a.B * (a.H / group) * qtiles;
  const int tiles = (a.seen + kBN - 1) / kBN;
  // at least four tiles to a split: shorter ones spend their time on the start of a workgroup and on the join
  int64_t splits = work >= 512 ? 1 : 1024 / work;
  if (splits > tiles / 4) splits = tiles / 4;
  if (splits > 128) splits = 128;
  if (splits < 1) splits = 1;
  a.tiles_per_split = (int)((tiles + splits - 1) / splits);
  a.splits = a.tiles_per_split > 0 ? (tiles + a.tiles_per_split - 1) / a.tiles_per_split : 1;
  if (a.splits < 1) a.splits = 1;
}

}  // namespace

}  // namespace rel
}  // namespace hivt

using namespace hivt;
using namespace hivt::rel;

static size_t split_bytes(const Args& a) {
  return a.splits > 1 ? (size_t)a.splits * a.B * a.H * a.M * (a.d + 2) * sizeof(float) : 0;
}

extern "C" size_t hivt_relative_attn_fwd_workspace_bytes(const hivt_relative_attn* p, const int32_t* starts) {
  Args a;
  if (from_public("hivt_relative_attn_fwd", p, starts, 1.0f, a) != HIVT_OK || a.B == 0 || a.M == 0) return 0;
  if (short_fwd_route(a)) return 0;
  plan(a);
  return align_up(split_bytes(a), 256);
}

extern "C" int hivt_relative_attn_fwd(const hivt_relative_attn* p, const int32_t* starts, float scale, void* workspace,
                                      size_t workspace_bytes, hivt_stream_t stream) {
  const char* what = "hivt_relative_attn_fwd";
  Args a;
  const int rc = from_public(what, p, starts, scale, a);
  if (rc != HIVT_OK || a.B == 0 || a.M == 0) return rc;
  const bool is_short = short_fwd_route(a);
  if (!is_short) plan(a);
  const size_t need = split_bytes(a);
  HIVT_REQUIRE(a.q && a.table && a.out && (a.N == 0 || (a.k && a.v)), HIVT_ERR_ARG, "%s: null pointer", what);
  HIVT_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), HIVT_ERR_WORKSPACE,
               "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  if (is_short) return short_fwd(a, (int)p->dtype, (hipStream_t)stream);
  a.partial = static_cast<float*>(workspace);
  switch (p->dtype) {
    case HIVT_F32: return launch_type<float>(a, (hipStream_t)stream);
    case HIVT_BF16: return launch_type<__bf16>(a, (hipStream_t)stream);
    default: return launch_type<_Float16>(a, (hipStream_t)stream);
  }
}

// ---- arguments --------------------------------------------------------------------------------------------------------
namespace hivt {
namespace rel {

// The widest load that the base address and all strides of a tensor allow (bytes), as far as the head width needs it.
static int align_of(const void* p, const int64_t* st, const int64_t* extent, int d, int size) {
  int align = 16;
  auto limit = [&](uint64_t bytes) {
    while (align > size && bytes % align != 0) align /= 2;
  };
  limit(reinterpret_cast<uint64_t>(p));
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1) limit((uint64_t)(st[i] < 0 ? -st[i] : st[i]) * size);
  limit((uint64_t)d * size);
  return align;
}

int from_public(const char* what, const hivt_relative_attn* p, const int32_t* starts, float scale, Args& a) {
  HIVT_REQUIRE(p != nullptr, HIVT_ERR_ARG, "%s: null argument block", what);
  const int64_t big = (int64_t)1 << 31;
  HIVT_REQUIRE(p->dtype == HIVT_F32 || p->dtype == HIVT_BF16 || p->dtype == HIVT_F16, HIVT_ERR_UNSUPPORTED,
               "%s: element type %d", what, (int)p->dtype);
  HIVT_REQUIRE(p->batch >= 0 && p->q_len >= 0 && p->k_len >= 0 && p->heads >= 1 && p->kv_heads >= 1 &&
               p->batch < big && p->q_len < big / 128 && p->k_len < big / 2 && p->heads < 65536 &&
               p->batch * p->heads < big, HIVT_ERR_ARG, "%s: bad sizes", what);
  HIVT_REQUIRE(p->heads % p->kv_heads == 0, HIVT_ERR_ARG, "%s: %d query heads are no multiple of %d key heads", what,
               (int)p->heads, (int)p->kv_heads);
  HIVT_REQUIRE(p->head_dim >= 1 && p->head_dim <= 128, HIVT_ERR_UNSUPPORTED, "%s: head width %d not in [1,128]", what,
               (int)p->head_dim);
  HIVT_REQUIRE(p->q_offset > -(big / 2) && p->q_offset < big / 2 - p->q_len, HIVT_ERR_ARG, "%s: query offset out of range",
               what);
  const int64_t side = p->bidirectional ? p->buckets / 2 : p->buckets;
  HIVT_REQUIRE(p->buckets >= 2 && p->exact >= 1 && p->exact < big && p->starts >= 0 && p->starts <= kMaxStarts &&
               side * (p->bidirectional ? 2 : 1) == p->buckets && p->exact + p->starts + 1 == side,
               HIVT_ERR_ARG, "%s: %d buckets of which %d single and %d border distances do not belong together", what,
               (int)p->buckets, (int)p->exact, (int)p->starts);
  HIVT_REQUIRE(p->starts == 0 || starts != nullptr, HIVT_ERR_ARG, "%s: no border distances", what);
  memset(&a, 0, sizeof(a));
  int32_t before = (int32_t)p->exact;
  for (int i = 0; i < (int)p->starts; ++i) {
    HIVT_REQUIRE(starts[i] >= before, HIVT_ERR_ARG, "%s: border distances must ascend", what);
    before = a.starts[i] = starts[i];
  }
  a.sat = before;  // from here on every distance lies in the last bucket
  HIVT_REQUIRE(a.sat <= kMaxSat, HIVT_ERR_UNSUPPORTED, "%s: the last bucket starts at distance %d, beyond %d", what, a.sat,
               kMaxSat);
  a.q = reinterpret_cast<const void*>(p->q);
  a.k = reinterpret_cast<const void*>(p->k);
  a.v = reinterpret_cast<const void*>(p->v);
  a.table = reinterpret_cast<const float*>(p->table);
  a.mask = reinterpret_cast<const uint8_t*>(p->key_mask);
  a.mask_sb = p->mask_stride;
  a.out = reinterpret_cast<void*>(p->out);
  a.stats = reinterpret_cast<float2*>(p->stats);
  a.d_out = reinterpret_cast<const void*>(p->d_out);
  a.dq = reinterpret_cast<void*>(p->dq);
  a.dk = reinterpret_cast<void*>(p->dk);
  a.dv = reinterpret_cast<void*>(p->dv);
  a.d_table = reinterpret_cast<float*>(p->d_table);
  a.want_table = a.d_table != nullptr;
  const int64_t* from[8] = {p->q_stride, p->k_stride, p->v_stride, p->out_stride, p->d_out_stride, p->dq_stride,
                            p->dk_stride, p->dv_stride};
  int64_t* to[8] = {a.q_st, a.k_st, a.v_st, a.o_st, a.do_st, a.dq_st, a.dk_st, a.dv_st};
  for (int i = 0; i < 8; ++i)
    for (int j = 0; j < 3; ++j) to[i][j] = from[i][j];
  a.B = (int32_t)p->batch;
  a.M = (int32_t)p->q_len;
  a.N = (int32_t)p->k_len;
  a.H = (int32_t)p->heads;
  a.G = (int32_t)p->kv_heads;
  a.d = (int32_t)p->head_dim;
  a.rep = a.H / a.G;
  a.offset = (int32_t)p->q_offset;
  a.causal = p->causal != 0;
  const int64_t reach = p->q_len + p->q_offset;  // (a cache's unwritten end may hold anything)
  a.seen = !a.causal || reach >= p->k_len ? a.N : reach > 0 ? (int32_t)reach : 0;
  a.bidirectional = p->bidirectional != 0;
  a.buckets = (int32_t)p->buckets;
  a.exact = (int32_t)p->exact;
  a.nstarts = (int32_t)p->starts;
  const int size = p->dtype == HIVT_F32 ? 4 : 2;
  const int64_t qe[3] = {p->batch, p->q_len, p->heads}, ke[3] = {p->batch, p->k_len, p->kv_heads};
  a.q_align = align_of(a.q, a.q_st, qe, a.d, size);
  a.k_align = align_of(a.k, a.k_st, ke, a.d, size);
  a.v_align = align_of(a.v, a.v_st, ke, a.d, size);
  a.do_align = align_of(a.d_out, a.do_st, qe, a.d, size);
  a.o_align = align_of(a.out, a.o_st, qe, a.d, size);
  a.scale = scale;
  a.scale2 = scale * kLog2e;
  a.splits = 1;
  return HIVT_OK;
}

}  // namespace rel
}  // namespace hivt
