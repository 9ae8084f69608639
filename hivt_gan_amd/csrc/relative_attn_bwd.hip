// Backward of the attention with a learned bias for each bucket of relative positions.
//
// No atomics, so equal calls give equal bits.  Three passes recompute the weights from the saved statistics:
//   dq_kernel    a workgroup owns query rows and walks the keys: dq, and what each row's ds sum up to;
//   dkv_kernel   a workgroup owns keys and walks the query rows of every head of the group: dk, dv;
//   bias_kernel  a wave owns query rows and walks the keys nearer than the last bucket: sums of ds along diagonals.
//
// The bias gradient needs more care than the others.  Each row of ds sums to zero, so a bucket that holds most keys of
// most rows is left with the small rest of that cancellation, and an error of delta_i (it comes from an output that is
// rounded, and whose weights were rounded for the matrix cores) enters it once per row, all with one sign for a row.
// dq_kernel therefore adds up r_i = sum_j ds_ij in fp32, which is that error (the weights of a row sum to one), writes
// delta_i + r_i for the passes behind it, and corrects its own sums over the far keys by r_i times their weights.
#include "relative_core.h"

namespace hivt {
namespace rel {
namespace {

constexpr int kBN = 64;

// d_out . out of a lane's share of a row
template <typename T, int E>
__device__ __forceinline__ float dot(const Frag<T, E>& a, const Frag<T, E>& b) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < E; ++j) s = fmaf((float)a.v[j], (float)b.v[j], s);
  return s;
}

// Waves to a SIMD: two where the registers allow, so that one's matrix instructions run beside the other's exponentials.
// Bound by issue and latency, as the forward: bf16 2 x 4096 causal, 16 heads of 128: 359 us, 575 TFLOP/s; 8 x 1024, 16
// heads of 64: 88 us, 585 TFLOP/s; fp32 64 x 301, 8 heads of 16: 75 us.
// The widest 16-bit heads need two LDS buffers for that (`paired`): keys are on their way to the other one during the
// first half of a tile and values during the second, in the same registers (505 -> 359 us).
template <typename T, int DP, int QB>
__host__ __device__ constexpr bool paired() { return sizeof(T) == 2 && DP > 96 && QB == 2; }
template <typename T, int DP, int QB>
__host__ __device__ constexpr int waves_per_simd() {
  if (sizeof(T) == 2) return 2;
  return QB == 1 ? (DP >= 128 ? 1 : 2) : DP <= 32 ? 2 : 1;
}
template <typename T, int DP, int QB>
__global__ __launch_bounds__(256, (waves_per_simd<T, DP, QB>())) void dq_kernel(const Args a, float2* __restrict__ far_sums) {
  using TL = Tile<T, DP>;
  constexpr int NB = DP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* const kt = reinterpret_cast<T*>(smem);
  T* const vt = kt + kBN * TL::PITCH;
  constexpr bool PAIRED = paired<T, DP, QB>();
  constexpr int BUFFER = 2 * kBN * TL::PITCH;
  float* const bias = reinterpret_cast<float*>(kt + (PAIRED ? 2 : 1) * BUFFER);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
  const int qtiles = (a.M + 64 * QB - 1) / (64 * QB);
  int unit, inner;
  walk(blockIdx.x, a.B * a.H, qtiles, unit, inner);
  const int qtile = qtiles - 1 - inner;
  const int b = unit / a.H, h = unit % a.H, g = h / a.rep;
  const int width = bias_width(a), hi = bias_hi(a);
  for (int e = tid; e < width; e += 256) bias[e] = bias2(a.table[(int64_t)entry_bucket(a, e) * a.H + h]);

  const int row0 = qtile * 64 * QB + wave * 16 * QB;
  const bool active = row0 < a.M;
  int pos[QB];
  bool live[QB];
  float m[QB], il[QB], delta[QB], rsum[QB];
  Frag<T, TL::E> qf[QB][TL::KSTEPS], of[QB][TL::KSTEPS];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = row0 + qb * 16 + (lane & 15);
    live[qb] = r < a.M;
    const int s = min(r, a.M - 1);
    pos[qb] = s + a.offset;
    const T* q = static_cast<const T*>(a.q) + b * a.q_st[0] + s * a.q_st[1] + h * a.q_st[2];
    const T* go = static_cast<const T*>(a.d_out) + b * a.do_st[0] + s * a.do_st[1] + h * a.do_st[2];
    const T* out = static_cast<const T*>(a.out) + b * a.o_st[0] + s * a.o_st[1] + h * a.o_st[2];
    float part = 0.0f;
#pragma unroll
    for (int ks = 0; ks < TL::KSTEPS; ++ks) {
      const int col = ks * TL::KS + quad * TL::E;
      qf[qb][ks] = load_frag<T, TL::E>(q, col, a.d, a.q_align, live[qb]);
      of[qb][ks] = load_frag<T, TL::E>(go, col, a.d, a.do_align, live[qb]);
      part += dot(of[qb][ks], load_frag<T, TL::E>(out, col, a.d, a.o_align, live[qb]));
    }
    delta[qb] = quad_sum(part);
    const float2 st = live[qb] ? a.stats[((int64_t)b * a.H + h) * a.M + s] : make_float2(0.0f, 0.0f);
    m[qb] = st.x;
    il[qb] = st.y;
    rsum[qb] = 0.0f;
  }
  const int pos_lo = min(row0, a.M - 1) + a.offset, pos_hi = max(min(row0 + 16 * QB, a.M) - 1, 0) + a.offset;
  const int wg_last = min((qtile + 1) * 64 * QB, a.M) - 1 + a.offset;
  const int keys_end = a.causal ? min(a.seen, wg_last + 1) : a.seen;
  const int t_end = keys_end > 0 ? (keys_end + kBN - 1) / kBN : 0;

  f32x4 dq[NB][QB];
  float far_l[QB], far_r[QB], w_l[QB], w_r[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    far_l[qb] = far_r[qb] = w_l[qb] = w_r[qb] = 0.0f;
#pragma unroll
    for (int n = 0; n < NB; ++n) dq[n][qb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const T* const kbase = static_cast<const T*>(a.k) + b * a.k_st[0] + g * a.k_st[2];
  const T* const vbase = static_cast<const T*>(a.v) + b * a.v_st[0] + g * a.v_st[2];
  // half a tile: two 16-key blocks, what the reduction over the keys takes
  int k0 = 0;
  uint64_t keys = 0;
  auto half = [&](int kk, const T* kt, const T* vt) __attribute__((always_inline)) {
    if (!active || (a.causal && k0 > pos_hi)) return;
    const int rel_hi = k0 + kBN - 1 - pos_lo, rel_lo = k0 - pos_hi;
    const bool left = rel_hi <= -a.sat, right = rel_lo >= hi, far = left || right;
    const bool whole = keys == ~0ull && (!a.causal || rel_hi <= 0);
    const float c = bias[left ? 0 : width - 1];
    const bool plain = far && whole && fabsf(c) <= kPlainBias;  // (see the forward)
    f32x4 s[2][QB], dp[2][QB];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) s[i][qb] = dp[i][qb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < TL::KSTEPS; ++ks) {
        const Frag<T, TL::E> kf = TL::rows(kt, (2 * kk + i) * 16, ks, lane), vf = TL::rows(vt, (2 * kk + i) * 16, ks, lane);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          Frag<T, TL::E>::mma(kf, qf[qb][ks], s[i][qb]);
          Frag<T, TL::E>::mma(vf, of[qb][ks], dp[i][qb]);
        }
      }
    }
    Frag<T, 8> df[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float mul = a.scale2, add = c;  // (see the forward)
      if (!plain) {
        if (far) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[i][qb][r] = fmaf(s[i][qb][r], a.scale2, c);
        } else {
          const float* const at = bias + k0 + kk * 32 + quad * 4 - pos[qb] + a.sat + kMargin;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[i][qb][r] = fmaf(s[i][qb][r], a.scale2, at[i * 16 + r]);
        }
        mul = 1.0f;
        add = 0.0f;
        if (!whole) {
          const int lim = a.causal ? pos[qb] - k0 : kBN;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t nibble = (uint32_t)(keys >> (kk * 32 + i * 16 + quad * 4));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool out = !(nibble >> r & 1) || kk * 32 + i * 16 + quad * 4 + r > lim;
              s[i][qb][r] = out ? -INFINITY : s[i][qb][r];
              dp[i][qb][r] = out ? 0.0f : dp[i][qb][r];
            }
          }
        }
      }
      const float shift = add - m[qb];
      float sum_ds = 0.0f, sum_p = 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = fexp2(fmaf(s[i][qb][r], mul, shift)) * il[qb];
          dp[i][qb][r] = p * (dp[i][qb][r] - delta[qb]);
          sum_ds += dp[i][qb][r];
          sum_p += p;
        }
      rsum[qb] += sum_ds;
      if (left) { far_l[qb] += sum_ds; w_l[qb] += sum_p; }
      else if (right) { far_r[qb] += sum_ds; w_r[qb] += sum_p; }
      df[qb] = pair_frag<T>(dp[0][qb], dp[1][qb]);
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const Frag<T, 8> kf = TL::cols(kt, kk * 32, n * 16, lane);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) Frag<T, 8>::mma(kf, df[qb], dq[n][qb]);
    }
  };

  int t = 0;
  uint64_t bits = 0;
  auto seek = [&]() {  // to the next tile that holds an allowed key
    while (t < t_end && (bits = tile_keys(a, b, t * kBN, lane)) == 0) ++t;
  };
  Loader<T, DP, kBN, 256> kl, vl;
  auto load = [&](Loader<T, DP, kBN, 256>& l, const T* base, const int64_t* st, int align) {
    auto keep = [&](int row) { return (bits >> row & 1) != 0; };
    l.load(base + (int64_t)t * kBN * st[1], st[1], a.d, align, tid, bits == ~0ull, keep);
  };
  seek();
  if constexpr (PAIRED) {
    int at = 0;
    if (t < t_end) {
      load(kl, kbase, a.k_st, a.k_align);
      load(vl, vbase, a.v_st, a.v_align);
      kl.store(kt, tid);
      vl.store(vt, tid);
    }
    while (t < t_end) {
      __syncthreads();  // this buffer has been filled, the other one read by every wave
      k0 = t * kBN;
      keys = bits;
      ++t;
      seek();
      if (t < t_end) load(kl, kbase, a.k_st, a.k_align);
      half(0, kt + at, vt + at);
      if (t < t_end) {
        kl.store(kt + (BUFFER - at), tid);
        load(kl, vbase, a.v_st, a.v_align);
      }
      half(1, kt + at, vt + at);
      if (t < t_end) kl.store(vt + (BUFFER - at), tid);
      at = BUFFER - at;
    }
  } else {
    if (t < t_end) {
      load(kl, kbase, a.k_st, a.k_align);
      load(vl, vbase, a.v_st, a.v_align);
    }
    while (t < t_end) {
      __syncthreads();
      kl.store(kt, tid);
      vl.store(vt, tid);
      k0 = t * kBN;
      keys = bits;
      ++t;
      seek();
      if (t < t_end) {
        load(kl, kbase, a.k_st, a.k_align);
        load(vl, vbase, a.v_st, a.v_align);
      }
      __syncthreads();
      half(0, kt, vt);
      half(1, kt, vt);
    }
  }
  if (!active) return;

  float sum_l = 0.0f, sum_r = 0.0f;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float r = quad_sum(rsum[qb]);
    sum_l += quad_sum(far_l[qb]) - r * quad_sum(w_l[qb]);
    sum_r += quad_sum(far_r[qb]) - r * quad_sum(w_r[qb]);
    if (!live[qb]) continue;
    const int s = row0 + qb * 16 + (lane & 15);
    if (quad == 0) a.delta[((int64_t)b * a.H + h) * a.M + s] = delta[qb] + r;
    T* out = static_cast<T*>(a.dq) + b * a.dq_st[0] + s * a.dq_st[1] + h * a.dq_st[2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      f32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = dq[n][qb][j] * a.scale;
      store4(out, n * 16 + quad * 4, a.d, w);
    }
  }
  if (far_sums != nullptr) {
    sum_l = group_sum<16>(sum_l);
    sum_r = group_sum<16>(sum_r);
    const int groups = (a.M + 16 * QB - 1) / (16 * QB);
    if (lane == 0) far_sums[(int64_t)unit * groups + row0 / (16 * QB)] = make_float2(sum_l, sum_r);
  }
}

// BQ query rows a step; a wave owns 16 KB keys, a workgroup has WAVES of them.  Four products to dq_kernel's three, bound
// by the same; in the order of its cases: 475 us, 579 TFLOP/s; 124 us, 554 TFLOP/s; 92 us.  (Two LDS buffers, as in
// dq_kernel, cost registers and gained nothing here: 1.18 -> 1.20 ms for the whole of the first case.)
template <typename T, int DP, int KB, int BQ, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 ? 2 : 1) void dkv_kernel(const Args a) {
  using TL = Tile<T, DP>;
  constexpr int NB = DP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* const qt = reinterpret_cast<T*>(smem);
  T* const ot = qt + BQ * TL::PITCH;
  float4* const rowst = reinterpret_cast<float4*>(ot + BQ * TL::PITCH);  // m, 1 / l, delta of a row
  float* const bias = reinterpret_cast<float*>(rowst + BQ);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
  const int ktiles = (a.N + 16 * WAVES * KB - 1) / (16 * WAVES * KB);
  // One query head to a workgroup, or (a.splits == 1) all of the group: their shares of dk and dv are then added by
  // another kernel.
  const int parts = a.splits, heads = a.rep / parts;
  int unit, inner;
  walk(blockIdx.x, a.B * a.G, ktiles * parts, unit, inner);
  const int ktile = inner / parts, part = inner % parts;
  const int b = unit / a.G, g = unit % a.G;
  const int width = bias_width(a), hi = bias_hi(a);

  const int key0 = ktile * 16 * WAVES * KB + wave * 16 * KB;
  bool keep[KB];
  int key[KB];
  Frag<T, TL::E> kf[KB][TL::KSTEPS], vf[KB][TL::KSTEPS];
  bool any = false;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    key[kb] = key0 + kb * 16 + (lane & 15);
    keep[kb] = key[kb] < a.seen && (a.mask == nullptr || a.mask[(int64_t)b * a.mask_sb + key[kb]] == 0);
    any = any || keep[kb];
    const int64_t kc = min(key[kb], a.N - 1);
    const T* k = static_cast<const T*>(a.k) + b * a.k_st[0] + kc * a.k_st[1] + g * a.k_st[2];
    const T* v = static_cast<const T*>(a.v) + b * a.v_st[0] + kc * a.v_st[1] + g * a.v_st[2];
#pragma unroll
    for (int ks = 0; ks < TL::KSTEPS; ++ks) {
      const int col = ks * TL::KS + quad * TL::E;
      kf[kb][ks] = load_frag<T, TL::E>(k, col, a.d, a.k_align, keep[kb]);
      vf[kb][ks] = load_frag<T, TL::E>(v, col, a.d, a.v_align, keep[kb]);
    }
  }
  const bool active = __any(any);
  const bool all = __all([&]() { bool x = true;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) x = x && keep[kb];
    return x; }());
  const int key_hi = min(key0 + 16 * KB, a.N) - 1;

  f32x4 dk[NB][KB], dv[NB][KB];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) dk[n][kb] = dv[n][kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int qsteps = (a.M + BQ - 1) / BQ;
  const int first = a.causal ? max(0, ktile * 16 * WAVES * KB - a.offset) / BQ : 0;  // rows before it see none of these keys
  Loader<T, DP, BQ, 64 * WAVES> ql, ol;
  for (int hr = 0; hr < heads; ++hr) {
    const int h = g * a.rep + part * heads + hr;
    __syncthreads();  // the head before has been finished by every wave
    for (int e = tid; e < width; e += 64 * WAVES) bias[e] = bias2(a.table[(int64_t)entry_bucket(a, e) * a.H + h]);
    const T* const qbase = static_cast<const T*>(a.q) + b * a.q_st[0] + h * a.q_st[2];
    const T* const obase = static_cast<const T*>(a.d_out) + b * a.do_st[0] + h * a.do_st[2];
    const int64_t rowbase = ((int64_t)b * a.H + h) * a.M;
    float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto fetch = [&](int step) {
      const int s0 = step * BQ;
      auto in = [&](int row) { return s0 + row < a.M; };
      ql.load(qbase + (int64_t)s0 * a.q_st[1], a.q_st[1], a.d, a.q_align, tid, s0 + BQ <= a.M, in);
      ol.load(obase + (int64_t)s0 * a.do_st[1], a.do_st[1], a.d, a.do_align, tid, s0 + BQ <= a.M, in);
      if (tid < BQ) {
        st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (s0 + tid < a.M) {
          const float2 s2 = a.stats[rowbase + s0 + tid];
          st = make_float4(s2.x, s2.y, a.delta[rowbase + s0 + tid], 0.0f);
        }
      }
    };
    if (first < qsteps) fetch(first);
    for (int step = first; step < qsteps; ++step) {
      __syncthreads();
      ql.store(qt, tid);
      ol.store(ot, tid);
      if (tid < BQ) rowst[tid] = st;
      if (step + 1 < qsteps) fetch(step + 1);
      __syncthreads();
      const int s0 = step * BQ, pos0 = s0 + a.offset;
      const int pos_last = min(s0 + BQ, a.M) - 1 + a.offset;
      if (!active || (a.causal && key0 > pos_last)) continue;
      const int rel_hi = key_hi - pos0, rel_lo = key0 - pos_last;
      const bool left = rel_hi <= -a.sat, far = left || rel_lo >= hi;
      const bool whole = all && s0 + BQ <= a.M && (!a.causal || rel_hi <= 0);
      const float c = bias[left ? 0 : width - 1];
      const bool plain = far && whole && fabsf(c) <= kPlainBias;  // (see the forward)
#pragma unroll
      for (int qq = 0; qq < BQ / 32; ++qq) {
        f32x4 p[2][KB], ds[2][KB];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) p[i][kb] = ds[i][kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int ks = 0; ks < TL::KSTEPS; ++ks) {
            const Frag<T, TL::E> qf = TL::rows(qt, qq * 32 + i * 16, ks, lane), of = TL::rows(ot, qq * 32 + i * 16, ks, lane);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              Frag<T, TL::E>::mma(qf, kf[kb][ks], p[i][kb]);
              Frag<T, TL::E>::mma(of, vf[kb][ks], ds[i][kb]);
            }
          }
        }
        // (two ways with registers moved between them: put together as in the other kernels, the rows' statistics are read
        // twice, which cost more: 122 -> 149 us for the encoder layer of 1024 positions)
        if (plain) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float4 rs = rowst[qq * 32 + i * 16 + quad * 4 + r];
              const float shift = c - rs.x;
#pragma unroll
              for (int kb = 0; kb < KB; ++kb) {
                const float w = fexp2(fmaf(p[i][kb][r], a.scale2, shift)) * rs.y;
                p[i][kb][r] = w;
                ds[i][kb][r] = w * (ds[i][kb][r] - rs.z);
              }
            }
        } else {  // (one loop, clamped: bias and mask in loops of their own, as in the other kernels, took a quarter more)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int row = qq * 32 + i * 16 + quad * 4 + r;
              const float4 rs = rowst[row];
#pragma unroll
              for (int kb = 0; kb < KB; ++kb) {
                const int rel = key[kb] - pos0 - row;
                const float add = bias[min(max(rel + a.sat + kMargin, 0), width - 1)];
                float w = fexp2(fmaf(p[i][kb][r], a.scale2, add) - rs.x) * rs.y;
                float dp = ds[i][kb][r];
                if (!keep[kb] || s0 + row >= a.M || (a.causal && rel > 0)) w = dp = 0.0f;
                p[i][kb][r] = w;
                ds[i][kb][r] = w * (dp - rs.z);
              }
            }
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const Frag<T, 8> pf = pair_frag<T>(p[0][kb], p[1][kb]), df = pair_frag<T>(ds[0][kb], ds[1][kb]);
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            Frag<T, 8>::mma(TL::cols(ot, qq * 32, n * 16, lane), pf, dv[n][kb]);
            Frag<T, 8>::mma(TL::cols(qt, qq * 32, n * 16, lane), df, dk[n][kb]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    if (key[kb] >= a.N) continue;
    if (parts > 1) {  // [part][batch, key, key head][dk, dv][d]
      float* const share = a.partial + ((((int64_t)part * a.B + b) * a.N + key[kb]) * a.G + g) * 2 * a.d;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        f32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = keep[kb] ? dk[n][kb][j] * a.scale : 0.0f;
        store4(share, n * 16 + quad * 4, a.d, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = keep[kb] ? dv[n][kb][j] : 0.0f;
        store4(share + a.d, n * 16 + quad * 4, a.d, w);
      }
      continue;
    }
    T* ok = static_cast<T*>(a.dk) + b * a.dk_st[0] + key[kb] * a.dk_st[1] + g * a.dk_st[2];
    T* ov = static_cast<T*>(a.dv) + b * a.dv_st[0] + key[kb] * a.dv_st[1] + g * a.dv_st[2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      f32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = keep[kb] ? dk[n][kb][j] * a.scale : 0.0f;
      store4(ok, n * 16 + quad * 4, a.d, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = keep[kb] ? dv[n][kb][j] : 0.0f;
      store4(ov, n * 16 + quad * 4, a.d, w);
    }
  }
}

// dk, dv = the sums of the query heads' shares, in ascending order of the heads; bound by memory (2 x 4096, 4 of 16 heads
// of 128: 151 MB in 43 us, 3.5 TB/s)
template <typename T>
__global__ __launch_bounds__(256) void group_kernel(const Args a) {
  const int64_t rows = (int64_t)a.B * a.N * a.G, total = rows * 2 * a.d;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    float s = 0.0f;
    for (int p = 0; p < a.splits; ++p) s += a.partial[p * total + i];
    const int64_t row = i / (2 * a.d);
    const int c = (int)(i % (2 * a.d)), g = (int)(row % a.G);
    const int64_t key = row / a.G % a.N, b = row / a.G / a.N;
    if (c < a.d) static_cast<T*>(a.dk)[b * a.dk_st[0] + key * a.dk_st[1] + g * a.dk_st[2] + c] = (T)s;
    else static_cast<T*>(a.dv)[b * a.dv_st[0] + key * a.dv_st[1] + g * a.dv_st[2] + c - a.d] = (T)s;
  }
}

// Sums of ds over the buckets, for 16 QB query rows of one (batch, head): the tiles that dq_kernel did not count as far.
// The tile of ds passes through LDS so that a lane can add along a diagonal; diagonals add up in LDS (one lane each, no
// conflicts), distances beyond the last border in registers.  A chain of small products, LDS and waits, one wave to a tile:
// 86, 58 and 50 us in the cases of dq_kernel.
template <typename T, int DP, int QB>
__global__ __launch_bounds__(64) void bias_kernel(const Args a, const float2* __restrict__ far_sums,
                                                  float* __restrict__ partial) {
  using TL = Tile<T, DP>;
  // sixteen rows at a time, each between margins of zeros, so that every diagonal has sixteen elements
  constexpr int ROWS = 16 * QB, LEFT = 16, PITCH = LEFT + kBN + 16 + 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* const skew = reinterpret_cast<float*>(smem);
  float* const bias = skew + 16 * PITCH;
  const int hi = bias_hi(a);
  float* const diag = bias + bias_width(a);

  const int lane = threadIdx.x, quad = lane >> 4;
  const int groups = (a.M + ROWS - 1) / ROWS;
  int unit, group;
  walk(blockIdx.x, a.B * a.H, groups, unit, group);
  const int b = unit / a.H, h = unit % a.H, g = h / a.rep;
  for (int e = lane; e < bias_width(a); e += 64) bias[e] = bias2(a.table[(int64_t)entry_bucket(a, e) * a.H + h]);
  for (int e = lane; e < core_width(a); e += 64) diag[e] = 0.0f;
  for (int e = lane; e < 16 * PITCH; e += 64) skew[e] = 0.0f;
  __syncthreads();
  const int row0 = group * ROWS;
  int pos[QB];
  float m[QB], il[QB], delta[QB];
  Frag<T, TL::E> qf[QB][TL::KSTEPS], of[QB][TL::KSTEPS];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = row0 + qb * 16 + (lane & 15);
    const bool live = r < a.M;
    const int s = min(r, a.M - 1);
    pos[qb] = r + a.offset;
    const T* q = static_cast<const T*>(a.q) + b * a.q_st[0] + s * a.q_st[1] + h * a.q_st[2];
    const T* go = static_cast<const T*>(a.d_out) + b * a.do_st[0] + s * a.do_st[1] + h * a.do_st[2];
#pragma unroll
    for (int ks = 0; ks < TL::KSTEPS; ++ks) {
      qf[qb][ks] = load_frag<T, TL::E>(q, ks * TL::KS + quad * TL::E, a.d, a.q_align, live);
      of[qb][ks] = load_frag<T, TL::E>(go, ks * TL::KS + quad * TL::E, a.d, a.do_align, live);
    }
    const int64_t at = ((int64_t)b * a.H + h) * a.M + s;
    const float2 st = live ? a.stats[at] : make_float2(0.0f, 0.0f);
    m[qb] = st.x;
    il[qb] = st.y;
    delta[qb] = live ? a.delta[at] : 0.0f;
  }
  const int pos_lo = row0 + a.offset, pos_hi = min(row0 + ROWS, a.M) - 1 + a.offset;
  const int keys_end = a.causal ? min(a.seen, pos_hi + 1) : a.seen;
  // the tiles that are not far: rel_hi > -sat and rel_lo < hi
  const int t_begin = max(0, pos_lo - a.sat) / kBN;
  const int t_end = min(keys_end > 0 ? (keys_end + kBN - 1) / kBN : 0, max(0, (pos_hi + hi + kBN - 1) / kBN + 1));
  const T* const kbase = static_cast<const T*>(a.k) + b * a.k_st[0] + g * a.k_st[2];
  const T* const vbase = static_cast<const T*>(a.v) + b * a.v_st[0] + g * a.v_st[2];
  float acc_l = 0.0f, acc_r = 0.0f;
  for (int t = t_begin; t < t_end; ++t) {
    const int k0 = t * kBN;
    const int rel_hi = k0 + kBN - 1 - pos_lo, rel_lo = k0 - pos_hi;
    if (rel_hi <= -a.sat || rel_lo >= hi) continue;
    const uint64_t keys = tile_keys(a, b, k0, lane);
    if (keys == 0) continue;
    f32x4 ds[4][QB];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const int key = k0 + kb * 16 + (lane & 15);
      const bool keep = (keys >> (kb * 16 + (lane & 15)) & 1) != 0;
      const int64_t kc = min(key, a.N - 1);
      f32x4 s[QB], dp[QB];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) s[qb] = dp[qb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < TL::KSTEPS; ++ks) {
        const int col = ks * TL::KS + quad * TL::E;
        const Frag<T, TL::E> kf = load_frag<T, TL::E>(kbase + kc * a.k_st[1], col, a.d, a.k_align, keep);
        const Frag<T, TL::E> vf = load_frag<T, TL::E>(vbase + kc * a.v_st[1], col, a.d, a.v_align, keep);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          Frag<T, TL::E>::mma(kf, qf[qb][ks], s[qb]);
          Frag<T, TL::E>::mma(vf, of[qb][ks], dp[qb]);
        }
      }
      const uint32_t nibble = (uint32_t)(keys >> (kb * 16 + quad * 4));
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const int rel0 = k0 + kb * 16 + quad * 4 - pos[qb];
        const float* const at = bias + rel0 + a.sat + kMargin;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = fexp2(fmaf(s[qb][r], a.scale2, at[r]) - m[qb]) * il[qb];
          const bool out = !(nibble >> r & 1) || (a.causal && rel0 + r > 0) || pos[qb] > pos_hi;
          ds[kb][qb][r] = out ? 0.0f : p * (dp[qb][r] - delta[qb]);
        }
      }
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
        *reinterpret_cast<f32x4*>(skew + (lane & 15) * PITCH + LEFT + kb * 16 + quad * 4) = ds[kb][qb];
      __syncthreads();
      // diagonal c: key - row = c - 15 within the sixteen rows
#pragma unroll
      for (int c0 = 0; c0 < kBN + 15; c0 += 64) {
        const int c = c0 + lane;
        const int rel = k0 - (pos_lo + qb * 16) + c - 15;
        const float* const from = skew + LEFT - 15 + min(c, kBN + 15);
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += from[r * (PITCH + 1)];
        if (c < kBN + 15) {
          if (rel <= -a.sat) acc_l += sum;
          else if (rel >= hi) acc_r += sum;
          else diag[rel + a.sat] += sum;
        }
        __syncthreads();
      }
    }
  }
  const float2 fs = far_sums[(int64_t)unit * groups + group];
  acc_l = wave_sum(acc_l) + fs.x;
  acc_r = wave_sum(acc_r) + fs.y;
  if (lane == 0) {
    diag[0] += acc_l;
    diag[core_width(a) - 1] += acc_r;
  }
  __syncthreads();
  const int side = a.bidirectional ? a.buckets / 2 : a.buckets;
  for (int bucket = lane; bucket < a.buckets; bucket += 64) {
    const bool behind = bucket >= side;  // keys behind the query
    const int sb = behind ? bucket - side : bucket;
    int from = sb < a.exact ? sb : sb == a.exact ? a.exact : a.starts[sb - a.exact - 1];
    const int to = sb < a.exact ? sb + 1 : sb - a.exact < a.nstarts ? a.starts[sb - a.exact] : a.sat + 1;
    if (behind && from == 0) from = 1;  // distance 0 belongs to the other side
    float sum = 0.0f;
    for (int n = from; n < to; ++n) sum += diag[behind ? a.sat + n : a.sat - n];
    partial[(((int64_t)b * groups + group) * a.H + h) * a.buckets + bucket] = sum;
  }
}

// d_table[bucket][h] = sum over the rows of partial [rows][H][buckets]: a workgroup takes 64 columns and cuts the rows into
// 16 slices, each added in ascending order, then the slices; in 64 bits.  5 us, its launch.
__global__ __launch_bounds__(1024) void table_kernel(const float* __restrict__ partial, int64_t rows, int H, int buckets,
                                                     float* __restrict__ d_table) {
  __shared__ double sums[16][64];
  const int slice = threadIdx.x >> 6;
  const int64_t cols = (int64_t)H * buckets, col = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  double s = 0.0;
  if (col < cols) {
    const int64_t end = rows * (slice + 1) / 16;
    int64_t i = rows * slice / 16;
    const float* p = partial + i * cols + col;
    for (; i + 8 <= end; i += 8, p += 8 * cols) {  // eight loads on their way at once
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = p[j * cols];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; i < end; ++i, p += cols) s += *p;
  }
  sums[slice][threadIdx.x & 63] = s;
  __syncthreads();
  if (slice == 0 && col < cols) {
    for (int i = 1; i < 16; ++i) s += sums[i][threadIdx.x];
    d_table[col % buckets * H + col / buckets] = (float)s;
  }
}
int launch_table(const Args& a, const float* partial, int64_t rows, hipStream_t stream) {
  const int64_t cols = (int64_t)a.H * a.buckets;
  hipLaunchKernelGGL(table_kernel, dim3((unsigned)((cols + 63) / 64)), dim3(1024), 0, stream, partial, rows, a.H, a.buckets,
                     a.d_table);
  HIVT_CHECK_LAUNCH("hivt_relative_attn_bwd");
  return HIVT_OK;
}

constexpr int rows_per_group(int M) { return M <= 64 ? 16 : 32; }

struct Work {
  size_t delta, far, partial, shares, total;
  int groups, parts;
};

// Query heads of a group in workgroups of their own: where the key tiles alone leave compute units idle, or a causal
// problem, whose first keys are seen by all rows and whose last by few, would wait for its longest workgroup.
int parts_of(const Args& a) {
  if (a.rep == 1) return 1;
  const int64_t tiles = (int64_t)a.B * a.G * ((a.N + 63) / 64);
  return tiles < 2048 ? a.rep : 1;
}
Work work_of(const Args& a) {
  Work w;
  if (short_bwd_route(a)) {
    w.groups = short_slots(a);
    w.delta = w.far = w.partial = w.shares = 0;
    w.parts = 1;
    w.total = a.want_table ? align_up((size_t)w.groups * a.H * a.buckets * sizeof(float), 256) : 0;
    return w;
  }
  w.groups = (a.M + rows_per_group(a.M) - 1) / rows_per_group(a.M);
  w.delta = 0;
  w.far = align_up((size_t)a.B * a.H * a.M * sizeof(float), 256);
  w.partial = w.far + (a.want_table ? align_up((size_t)a.B * a.H * w.groups * sizeof(float2), 256) : 0);
  w.shares = w.partial + (a.want_table ? align_up((size_t)a.B * a.H * w.groups * a.buckets * sizeof(float), 256) : 0);
  w.parts = parts_of(a);
  w.total = w.shares + (w.parts > 1 ? align_up((size_t)w.parts * a.B * a.N * a.G * 2 * a.d * sizeof(float), 256) : 0);
  return w;
}

template <typename T, int DP, int QB>
int launch_rows(const Args& a, char* ws, const Work& w, hipStream_t stream) {
  using TL = Tile<T, DP>;
  const char* what = "hivt_relative_attn_bwd";
  const size_t table = (size_t)bias_width(a) * sizeof(float);
  float2* const far_sums = a.want_table ? reinterpret_cast<float2*>(ws + w.far) : nullptr;
  const int64_t blocks = (int64_t)a.B * a.H * ((a.M + 64 * QB - 1) / (64 * QB));
  const size_t lds = (size_t)(paired<T, DP, QB>() ? 4 : 2) * kBN * TL::PITCH * sizeof(T) + table;
  HIVT_REQUIRE(blocks < ((int64_t)1 << 31) && (int64_t)a.B * a.H * w.groups < ((int64_t)1 << 31), HIVT_ERR_ARG,
               "%s: too many workgroups", what);
  if (lds > 48 * 1024)
    HIVT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&dq_kernel<T, DP, QB>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), what);
  hipLaunchKernelGGL((dq_kernel<T, DP, QB>), dim3((unsigned)blocks), dim3(256), lds, stream, a, far_sums);
  HIVT_CHECK_LAUNCH(what);
  if (a.want_table) {
    const size_t lb = (size_t)16 * (kBN + 36) * sizeof(float) + table + (size_t)core_width(a) * sizeof(float);
    float* const partial = reinterpret_cast<float*>(ws + w.partial);
    if (lb > 48 * 1024)
      HIVT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&bias_kernel<T, DP, QB>),
                                         hipFuncAttributeMaxDynamicSharedMemorySize, (int)lb), what);
    hipLaunchKernelGGL((bias_kernel<T, DP, QB>), dim3((unsigned)((int64_t)a.B * a.H * w.groups)), dim3(64), lb, stream, a,
                       far_sums, partial);
    HIVT_CHECK_LAUNCH(what);
    return launch_table(a, partial, (int64_t)a.B * w.groups, stream);
  }
  return HIVT_OK;
}

template <typename T, int DP>
int launch_width(const Args& a, char* ws, const Work& w, hipStream_t stream) {
  using TL = Tile<T, DP>;
  // 32 keys to a wave where that leaves two waves per SIMD, 16 for the widest heads (bf16, decoder layer of 4096 positions:
  // 32 keys in workgroups of two waves, one to a SIMD, 529 us, 16 keys in workgroups of four 475 us).  fp32 from 64 wide on
  // has one wave per SIMD either way; its workgroups are of two waves: two of them share a compute unit, and twice as many
  // of half the length even out the causal ones.
  constexpr bool FP32 = sizeof(T) == 4;
  constexpr int KB = DP >= 96 ? 1 : 2, BQ = 32, WAVES = FP32 && DP > 32 ? 2 : 4;
  const char* what = "hivt_relative_attn_bwd";
  const int rc = rows_per_group(a.M) == 16 ? launch_rows<T, DP, 1>(a, ws, w, stream) : launch_rows<T, DP, 2>(a, ws, w, stream);
  if (rc != HIVT_OK || a.N == 0) return rc;
  Args b = a;
  b.splits = w.parts;
  b.partial = reinterpret_cast<float*>(ws + w.shares);
  const int64_t blocks = (int64_t)a.B * a.G * w.parts * ((a.N + 16 * WAVES * KB - 1) / (16 * WAVES * KB));
  const size_t lds = (size_t)2 * BQ * TL::PITCH * sizeof(T) + BQ * sizeof(float4) + (size_t)bias_width(a) * sizeof(float);
  HIVT_REQUIRE(blocks < ((int64_t)1 << 31), HIVT_ERR_ARG, "%s: too many workgroups", what);
  if (lds > 48 * 1024)
    HIVT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&dkv_kernel<T, DP, KB, BQ, WAVES>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), what);
  hipLaunchKernelGGL((dkv_kernel<T, DP, KB, BQ, WAVES>), dim3((unsigned)blocks), dim3(64 * WAVES), lds, stream, b);
  HIVT_CHECK_LAUNCH(what);
  if (w.parts > 1) {
    const int64_t pieces = ((int64_t)a.B * a.N * a.G * 2 * a.d + 255) / 256;
    hipLaunchKernelGGL(group_kernel<T>, dim3((unsigned)(pieces < 65536 ? pieces : 65536)), dim3(256), 0, stream, b);
    HIVT_CHECK_LAUNCH(what);
  }
  return HIVT_OK;
}

template <typename T>
int launch_type(const Args& a, char* ws, const Work& w, hipStream_t stream) {
  if (a.d <= 16) return launch_width<T, 16>(a, ws, w, stream);
  if (a.d <= 32) return launch_width<T, 32>(a, ws, w, stream);
  if (a.d <= 64) return launch_width<T, 64>(a, ws, w, stream);
  if (a.d <= 96) return launch_width<T, 96>(a, ws, w, stream);
  return launch_width<T, 128>(a, ws, w, stream);
}

}  // namespace

}  // namespace rel
}  // namespace hivt

using namespace hivt;
using namespace hivt::rel;

extern "C" size_t hivt_relative_attn_bwd_workspace_bytes(const hivt_relative_attn* p, const int32_t* starts) {
  Args a;
  if (from_public("hivt_relative_attn_bwd", p, starts, 1.0f, a) != HIVT_OK) return 0;
  return work_of(a).total;
}

extern "C" int hivt_relative_attn_bwd(const hivt_relative_attn* p, const int32_t* starts, float scale, void* workspace,
                                      size_t workspace_bytes, hivt_stream_t stream) {
  const char* what = "hivt_relative_attn_bwd";
  Args a;
  const int rc = from_public(what, p, starts, scale, a);
  if (rc != HIVT_OK) return rc;
  HIVT_REQUIRE(a.B == 0 || a.M == 0 || (a.q && a.table && a.out && a.stats && a.d_out && a.dq), HIVT_ERR_ARG,
               "%s: null pointer", what);
  HIVT_REQUIRE(a.B == 0 || a.N == 0 || (a.k && a.v && a.dk && a.dv), HIVT_ERR_ARG, "%s: null pointer", what);
  HIVT_REQUIRE(a.B > 0 && a.M > 0, HIVT_ERR_ARG, "%s: no query rows: the gradients are zero", what);
  const Work w = work_of(a);
  HIVT_REQUIRE(w.total == 0 || (workspace != nullptr && workspace_bytes >= w.total), HIVT_ERR_WORKSPACE,
               "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, w.total);
  if (short_bwd_route(a)) {
    float* const partial = a.want_table ? static_cast<float*>(workspace) : nullptr;
    const int rs = short_bwd(a, (int)p->dtype, w.groups, partial, (hipStream_t)stream);
    return rs == HIVT_OK && a.want_table ? launch_table(a, partial, w.groups, (hipStream_t)stream) : rs;
  }
  char* const ws = static_cast<char*>(workspace);
  a.delta = reinterpret_cast<float*>(ws + w.delta);
  switch (p->dtype) {
    case HIVT_F32: return launch_type<float>(a, ws, w, (hipStream_t)stream);
    case HIVT_BF16: return launch_type<__bf16>(a, ws, w, (hipStream_t)stream);
    default: return launch_type<_Float16>(a, ws, w, (hipStream_t)stream);
  }
}
