// Short sequences: one wave to a (batch, head).  Forward: at most 64 queries and 32 keys, or 64 keys with heads of at most
// 32.  Backward: at most 32 queries and keys, heads of at most 64 (more does not fit the registers twice).
//
// At 21 positions with heads of 16 the pass is bound by memory (300 MB forward and backward for 2560 sequences of 8 heads)
// and the general kernels' tiles of 64 keys and 64 rows are mostly padding.  Here every score of a (batch, head) fits the
// registers of one wave: operands come straight from memory in the lanes' layout (64-byte rows of neighbouring heads,
// taken by neighbouring waves, share cache lines), there is no LDS tile and no barrier.
// The backward computes the softmax again, from its definition: delta is sum_j p_ij dp_ij itself, neither the output nor
// saved statistics are read.  The product that is reduced over the queries needs p and ds with the queries as its
// reduction index; the scores are simply computed a second time with the operands exchanged, at width 16 one matrix
// instruction per block, instead of moving them between lanes.
// Waves keep to one head and walk over the batch, so ds adds up over the batch in registers, score by score (the relative
// positions are the same in every sequence), and its diagonals are summed once per wave.
#include "relative_core.h"

namespace hivt {
namespace rel {
namespace {

constexpr int64_t kMaxStride = 1 << 23;  // elements between positions: 64 of them stay within 2^31 bytes
// relative positions of at most 64 queries and 64 keys (127), with room for the rows behind the last query of a block
constexpr int kFirst = 64, kRel = 192;

// 32 rows of a tile in memory as reduction index, columns col0 + (lane & 15) as output index: see Tile::cols
// (offsets within a sequence are 32-bit: see route)
template <typename T>
__device__ __forceinline__ Frag<T, 8> cols_from(const T* base, int stride, int row0, uint64_t keep, int col0, int d, int lane) {
  Frag<T, 8> f;
  const int col = col0 + (lane & 15), quad = lane >> 4;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = row0 + 16 * i + 4 * quad + j;
      f.v[4 * i + j] = col < d && (keep >> row & 1) ? base[row * stride + col] : (T)0.0f;
    }
  return f;
}

__device__ __forceinline__ uint64_t first_bits(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1; }

// The bias of every relative position -(M - 1) .. N - 1 (key index - query index) from entry kFirst on, in base-2 exponent
// units, zero elsewhere.
__device__ __forceinline__ void fill_bias(const Args& a, int h, float* bias, int lane) {
  for (int i = lane; i < kRel; i += 64) {
    const int e = i - kFirst;
    const int rel = min(max(e - (a.M - 1) - a.offset, -a.sat), bias_hi(a));
    bias[i] = e >= 0 && e < a.M + a.N - 1 ? bias2(a.table[(int64_t)rel_bucket(a, rel) * a.H + h]) : 0.0f;
  }
}

// Weights of 32 queries from row q0 on, transposed (rows = keys): scores, softmax.  p is normalised.
template <typename T, int DP, int KB>
__device__ __forceinline__ void weights(const Args& a, const Frag<T, Tile<T, DP>::E> (&qf)[2][Tile<T, DP>::KSTEPS],
                                        const Frag<T, Tile<T, DP>::E> (&kf)[KB][Tile<T, DP>::KSTEPS], const float* bias, int q0,
                                        uint64_t keys, int lane, f32x4 (&p)[KB][2], float (&m)[2], float (&il)[2]) {
  using TL = Tile<T, DP>;
  const int quad = lane >> 4;
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int q = q0 + qb * 16 + (lane & 15);
    const int lim = a.causal ? q + a.offset : a.N;
    const float* const at = bias + kFirst + quad * 4 - q + a.M - 1;
    float top = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      f32x4 s = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < TL::KSTEPS; ++ks) Frag<T, TL::E>::mma(kf[kb][ks], qf[qb][ks], s);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = kb * 16 + quad * 4 + r;
        const bool ok = (keys >> key & 1) && key <= lim;
        s[r] = ok ? fmaf(s[r], a.scale2, at[kb * 16 + r]) : -INFINITY;
        top = fmaxf(top, s[r]);
      }
      p[kb][qb] = s;
    }
    top = quad_max(top);
    m[qb] = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[kb][qb][r] = fexp2(p[kb][qb][r] - m[qb]);
        sum += p[kb][qb][r];
      }
    sum = quad_sum(sum);
    il[qb] = sum != sum ? sum : sum > 0.0f ? 1.0f / sum : 0.0f;
  }
}

// fp32, 2560 sequences of 21 positions and 8 heads of 16: 36 us, 3.1 TB/s, short of memory's 4.9 by the latency of a wave's
// few loads; one query of 20 sequences: 7.5 us
template <typename T, int DP, int KB>
__global__ __launch_bounds__(256) void short_fwd_kernel(const Args a) {
  using TL = Tile<T, DP>;
  constexpr int NB = DP / 16;
  __shared__ float bias_all[4][kRel];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quad = lane >> 4;
  float* const bias = bias_all[wave];
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  if (unit >= (int64_t)a.B * a.H) return;
  const int b = (int)(unit / a.H), h = (int)(unit % a.H), g = h / a.rep;
  const uint64_t keys = tile_keys(a, b, 0, lane);
  const T* const kbase = static_cast<const T*>(a.k) + b * a.k_st[0] + g * a.k_st[2];
  const T* const vbase = static_cast<const T*>(a.v) + b * a.v_st[0] + g * a.v_st[2];
  Frag<T, TL::E> kf[KB][TL::KSTEPS];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int key = kb * 16 + (lane & 15);
    const bool keep = (keys >> key & 1) != 0;
#pragma unroll
    for (int ks = 0; ks < TL::KSTEPS; ++ks)
      kf[kb][ks] = load_frag<T, TL::E>(kbase + (keep ? key : 0) * (int)a.k_st[1], ks * TL::KS + quad * TL::E, a.d, a.k_align, keep);
  }
  fill_bias(a, h, bias, lane);
  __builtin_amdgcn_wave_barrier();  // the wave's own LDS stores come before its loads; the compiler keeps the order too
  for (int q0 = 0; q0 < a.M; q0 += 32) {
    Frag<T, TL::E> qf[2][TL::KSTEPS];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      const int s = q0 + qb * 16 + (lane & 15);
      const T* q = static_cast<const T*>(a.q) + b * a.q_st[0] + h * a.q_st[2] + min(s, a.M - 1) * (int)a.q_st[1];
#pragma unroll
      for (int ks = 0; ks < TL::KSTEPS; ++ks)
        qf[qb][ks] = load_frag<T, TL::E>(q, ks * TL::KS + quad * TL::E, a.d, a.q_align, s < a.M);
    }
    f32x4 p[KB][2];
    float m[2], il[2];
    weights<T, DP, KB>(a, qf, kf, bias, q0, keys, lane, p, m, il);
    Frag<T, 8> pf[KB / 2][2];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb)
#pragma unroll
      for (int kk = 0; kk < KB / 2; ++kk) pf[kk][qb] = pair_frag<T>(p[2 * kk][qb], p[2 * kk + 1][qb]);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      f32x4 o[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
      for (int kk = 0; kk < KB / 2; ++kk) {
        const Frag<T, 8> vf = cols_from<T>(vbase, (int)a.v_st[1], kk * 32, keys, n * 16, a.d, lane);
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) Frag<T, 8>::mma(vf, pf[kk][qb], o[qb]);
      }
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        const int s = q0 + qb * 16 + (lane & 15);
        if (s >= a.M) continue;
        f32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = o[qb][j] * il[qb];
        store4(static_cast<T*>(a.out) + b * a.o_st[0] + h * a.o_st[2] + s * (int)a.o_st[1], n * 16 + quad * 4, a.d, w);
      }
    }
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      const int s = q0 + qb * 16 + (lane & 15);
      if (a.stats != nullptr && quad == 0 && s < a.M) a.stats[unit * a.M + s] = make_float2(m[qb], il[qb]);
    }
  }
}

// One head to a wave, its sequences b = slot, slot + slots, ...; two waves to a SIMD, so that one computes while the
// other waits for its rows.  The same sequences: 126 us, 1.5 TB/s, bound by the instructions of a wave (scores twice, padded
// from 21 to 32 both ways)
template <typename T, int DP>
__global__ __launch_bounds__(256, DP == 16 ? 3 : DP == 32 ? 2 : 1) void short_bwd_kernel(const Args a, int slots, float* __restrict__ partial) {
  using TL = Tile<T, DP>;
  constexpr int KB = 2, QQ = 1, NB = DP / 16, PITCH = KB * 16 + 1;
  __shared__ float bias_all[4][kRel];
  __shared__ float skew_all[4][32 * PITCH];
  const int self = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float* const bias = bias_all[wave];
  const int w = blockIdx.x * 4 + wave;
  if (w >= slots * a.H) return;
  const int h = w % a.H, slot = w / a.H;
  fill_bias(a, h, bias, self);
  __builtin_amdgcn_wave_barrier();

  f32x4 total[QQ][KB][2];  // ds over the batch
#pragma unroll
  for (int qq = 0; qq < QQ; ++qq)
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) total[qq][kb][0] = total[qq][kb][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  for (int b = slot; b < a.B; b += slots) {
    // The biases of the lane's 32 pairs and its rows' offsets are the same in every sequence; kept in registers over the
    // loop they cost two waves per SIMD, so the compiler is kept from knowing that this is the same lane.
    int lane = self;
    asm volatile("" : "+v"(lane));
    const int quad = lane >> 4;
    const uint64_t keys = tile_keys(a, b, 0, lane), queries = first_bits(a.M);
    const T* const qbase = static_cast<const T*>(a.q) + b * a.q_st[0] + h * a.q_st[2];
    const T* const obase = static_cast<const T*>(a.d_out) + b * a.do_st[0] + h * a.do_st[2];
    const T* const kbase = static_cast<const T*>(a.k) + b * a.k_st[0] + h * a.k_st[2];
    const T* const vbase = static_cast<const T*>(a.v) + b * a.v_st[0] + h * a.v_st[2];
    Frag<T, TL::E> kf[KB][TL::KSTEPS], vf[KB][TL::KSTEPS];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int key = kb * 16 + (lane & 15);
      const bool keep = (keys >> key & 1) != 0;
#pragma unroll
      for (int ks = 0; ks < TL::KSTEPS; ++ks) {
        const int col = ks * TL::KS + quad * TL::E;
        kf[kb][ks] = load_frag<T, TL::E>(kbase + (keep ? key : 0) * (int)a.k_st[1], col, a.d, a.k_align, keep);
        vf[kb][ks] = load_frag<T, TL::E>(vbase + (keep ? key : 0) * (int)a.v_st[1], col, a.d, a.v_align, keep);
      }
    }
    f32x4 dk[KB][NB], dv[KB][NB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int n = 0; n < NB; ++n) dk[kb][n] = dv[kb][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int qq = 0; qq < QQ; ++qq) {
      const int q0 = qq * 32;
      Frag<T, TL::E> qf[2][TL::KSTEPS], of[2][TL::KSTEPS];
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        const int s = q0 + qb * 16 + (lane & 15), sc = min(s, a.M - 1);
#pragma unroll
        for (int ks = 0; ks < TL::KSTEPS; ++ks) {
          const int col = ks * TL::KS + quad * TL::E;
          qf[qb][ks] = load_frag<T, TL::E>(qbase + sc * (int)a.q_st[1], col, a.d, a.q_align, s < a.M);
          of[qb][ks] = load_frag<T, TL::E>(obase + sc * (int)a.do_st[1], col, a.d, a.do_align, s < a.M);
        }
      }
      f32x4 p[KB][2];
      float m[2], il[2], delta[2];
      weights<T, DP, KB>(a, qf, kf, bias, q0, keys, lane, p, m, il);
      // transposed: dp, delta, ds
      Frag<T, 8> df[KB / 2][2];
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        const bool row = q0 + qb * 16 + (lane & 15) < a.M;
        f32x4 dp[KB];
        float part = 0.0f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          dp[kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int ks = 0; ks < TL::KSTEPS; ++ks) Frag<T, TL::E>::mma(vf[kb][ks], of[qb][ks], dp[kb]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = kb * 16 + quad * 4 + r;
            // (a later value that is not finite must not meet a weight of zero)
            const bool ok = (keys >> key & 1) && (!a.causal || key <= q0 + qb * 16 + (lane & 15) + a.offset);
            p[kb][qb][r] *= il[qb];
            if (!ok) dp[kb][r] = p[kb][qb][r] = 0.0f;
            part = fmaf(p[kb][qb][r], dp[kb][r], part);
          }
        }
        delta[qb] = quad_sum(part);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            dp[kb][r] = p[kb][qb][r] * (dp[kb][r] - delta[qb]);
            if (row) total[qq][kb][qb][r] += dp[kb][r];
          }
#pragma unroll
        for (int kk = 0; kk < KB / 2; ++kk) df[kk][qb] = pair_frag<T>(dp[2 * kk], dp[2 * kk + 1]);
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        f32x4 dq[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int kk = 0; kk < KB / 2; ++kk) {
          const Frag<T, 8> kc = cols_from<T>(kbase, (int)a.k_st[1], kk * 32, keys, n * 16, a.d, lane);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) Frag<T, 8>::mma(kc, df[kk][qb], dq[qb]);
        }
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          const int s = q0 + qb * 16 + (lane & 15);
          if (s >= a.M) continue;
          f32x4 x;
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = dq[qb][j] * a.scale;
          store4(static_cast<T*>(a.dq) + b * a.dq_st[0] + h * a.dq_st[2] + s * (int)a.dq_st[1], n * 16 + quad * 4, a.d, x);
        }
      }
      // rows = queries, columns = keys: p and ds as operands that are reduced over the queries
      float mr[2][4], ir[2][4], dr[2][4];
#pragma unroll
      for (int qb = 0; qb < 2; ++qb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          mr[qb][r] = __shfl(m[qb], quad * 4 + r, 64);
          ir[qb][r] = __shfl(il[qb], quad * 4 + r, 64);
          dr[qb][r] = __shfl(delta[qb], quad * 4 + r, 64);
        }
      Frag<T, 8> pf[KB], sf[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int key = kb * 16 + (lane & 15);
        const bool keep = (keys >> key & 1) != 0;
        const float* const at = bias + kFirst + key - q0 - quad * 4 + a.M - 1;
        f32x4 pr[2], ds[2];
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          pr[qb] = ds[qb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int ks = 0; ks < TL::KSTEPS; ++ks) {
            Frag<T, TL::E>::mma(qf[qb][ks], kf[kb][ks], pr[qb]);
            Frag<T, TL::E>::mma(of[qb][ks], vf[kb][ks], ds[qb]);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int q = q0 + qb * 16 + quad * 4 + r;
            const bool ok = keep && q < a.M && (!a.causal || key <= q + a.offset);
            const float x = ok ? fexp2(fmaf(pr[qb][r], a.scale2, at[-qb * 16 - r]) - mr[qb][r]) * ir[qb][r] : 0.0f;
            pr[qb][r] = x;
            ds[qb][r] = ok ? x * (ds[qb][r] - dr[qb][r]) : 0.0f;
          }
        }
        pf[kb] = pair_frag<T>(pr[0], pr[1]);
        sf[kb] = pair_frag<T>(ds[0], ds[1]);
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const Frag<T, 8> oc = cols_from<T>(obase, (int)a.do_st[1], q0, queries, n * 16, a.d, lane);
        const Frag<T, 8> qc = cols_from<T>(qbase, (int)a.q_st[1], q0, queries, n * 16, a.d, lane);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          Frag<T, 8>::mma(oc, pf[kb], dv[kb][n]);
          Frag<T, 8>::mma(qc, sf[kb], dk[kb][n]);
        }
      }
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int key = kb * 16 + (lane & 15);
      if (key >= a.N) continue;
      T* ok = static_cast<T*>(a.dk) + b * a.dk_st[0] + h * a.dk_st[2] + key * (int)a.dk_st[1];
      T* ov = static_cast<T*>(a.dv) + b * a.dv_st[0] + h * a.dv_st[2] + key * (int)a.dv_st[1];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        f32x4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = dk[kb][n][j] * a.scale;
        store4(ok, n * 16 + quad * 4, a.d, x);
        store4(ov, n * 16 + quad * 4, a.d, dv[kb][n]);
      }
    }
  }
  if (partial == nullptr) return;
  const int lane = self, quad = lane >> 4;

  // diagonals of the summed ds, through the wave's LDS, into the entries of the bias table; then the buckets
  float* const skew = skew_all[wave];
  float* const diag = bias;
  __builtin_amdgcn_wave_barrier();
  for (int e = lane; e < kRel; e += 64) diag[e] = 0.0f;
#pragma unroll
  for (int qq = 0; qq < QQ; ++qq) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int qb = 0; qb < 2; ++qb)
#pragma unroll
        for (int r = 0; r < 4; ++r) skew[(qb * 16 + (lane & 15)) * PITCH + kb * 16 + quad * 4 + r] = total[qq][kb][qb][r];
    __builtin_amdgcn_wave_barrier();
    for (int c = lane; c < KB * 16 + 31; c += 64) {  // key - row = c - 31
      float sum = 0.0f;
      for (int r = 0; r < 32; ++r) {
        const int key = c - 31 + r;
        if (key >= 0 && key < KB * 16) sum += skew[r * PITCH + key];
      }
      const int e = c - 31 - qq * 32 + a.M - 1;
      if (e >= 0 && e < a.M + a.N - 1) diag[e] += sum;  // (outside: rows and keys that are not there, zero)
    }
  }
  __builtin_amdgcn_wave_barrier();
  for (int bucket = lane; bucket < a.buckets; bucket += 64) {
    float sum = 0.0f;
    for (int e = 0; e < a.M + a.N - 1; ++e) {
      const int rel = min(max(e - (a.M - 1) - a.offset, -a.sat), bias_hi(a));
      if (rel_bucket(a, rel) == bucket) sum += diag[e];
    }
    partial[(int64_t)w * a.buckets + bucket] = sum;
  }
}

template <typename T, int DP, int KB>
int launch_fwd(const Args& a, hipStream_t stream) {
  const int64_t blocks = ((int64_t)a.B * a.H + 3) / 4;
  hipLaunchKernelGGL((short_fwd_kernel<T, DP, KB>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  HIVT_CHECK_LAUNCH("hivt_relative_attn_fwd");
  return HIVT_OK;
}

template <typename T, int DP>
int launch_bwd(const Args& a, int slots, float* partial, hipStream_t stream) {
  const unsigned blocks = (unsigned)(((int64_t)slots * a.H + 3) / 4);
  hipLaunchKernelGGL((short_bwd_kernel<T, DP>), dim3(blocks), dim3(256), 0, stream, a, slots, partial);
  HIVT_CHECK_LAUNCH("hivt_relative_attn_bwd");
  return HIVT_OK;
}

template <typename T>
int type_fwd(const Args& a, hipStream_t stream) {
  if (a.N <= 32) {
    if (a.d <= 16) return launch_fwd<T, 16, 2>(a, stream);
    if (a.d <= 32) return launch_fwd<T, 32, 2>(a, stream);
    if (a.d <= 64) return launch_fwd<T, 64, 2>(a, stream);
    return launch_fwd<T, 128, 2>(a, stream);
  }
  return a.d <= 16 ? launch_fwd<T, 16, 4>(a, stream) : launch_fwd<T, 32, 4>(a, stream);
}

template <typename T>
int type_bwd(const Args& a, int slots, float* partial, hipStream_t stream) {
  if (a.d <= 16) return launch_bwd<T, 16>(a, slots, partial, stream);
  if (a.d <= 32) return launch_bwd<T, 32>(a, slots, partial, stream);
  return launch_bwd<T, 64>(a, slots, partial, stream);
}

bool near(const int64_t* st) { return st[1] >= 0 && st[1] < kMaxStride; }

}  // namespace

bool short_fwd_route(const Args& a) {
  return a.M <= 64 && a.N >= 1 && (a.N <= 32 || (a.N <= 64 && a.d <= 32)) && near(a.q_st) && near(a.k_st) && near(a.v_st) &&
         near(a.o_st);
}
bool short_bwd_route(const Args& a) {
  return a.M <= 32 && a.N >= 1 && a.N <= 32 && a.rep == 1 && a.d <= 64 && near(a.q_st) && near(a.k_st) && near(a.v_st) &&
         near(a.do_st) && near(a.dq_st) && near(a.dk_st) && near(a.dv_st);
}
// Sequences of a head are dealt to this many waves: 4096 waves fill the compute units, and the bias gradient has that
// many rows to add up.
int short_slots(const Args& a) {
  const int slots = 4096 / a.H;
  return slots < 1 ? 1 : slots > a.B ? a.B : slots;
}

int short_fwd(const Args& a, int dtype, hipStream_t stream) {
  if (dtype == HIVT_F32) return type_fwd<float>(a, stream);
  return dtype == HIVT_BF16 ? type_fwd<__bf16>(a, stream) : type_fwd<_Float16>(a, stream);
}
int short_bwd(const Args& a, int dtype, int slots, float* partial, hipStream_t stream) {
  if (dtype == HIVT_F32) return type_bwd<float>(a, slots, partial, stream);
  return dtype == HIVT_BF16 ? type_bwd<__bf16>(a, slots, partial, stream) : type_bwd<_Float16>(a, slots, partial, stream);
}

}  // namespace rel
}  // namespace hivt
