// Root-mean-square norm of every head of the queries and keys, and the rotation of its first components by position.
//
//   y = R(pos) (w * x r),  r = 1 / sqrt(mean x^2 + eps);  pair i of the first `rotary` components turns by pos * rate_i
//   (pairs (i, i + rotary / 2), or (2 i, 2 i + 1) when interleaved)
//   backward, b = R(-pos) dy, n = x r:  dw = sum b n,  dx = r (w b - n mean(w b n));  r is computed again, not kept.
//
// Bound by memory: a row is read once and written once.  A workgroup takes a few positions with all their heads.  The
// sines of a position are computed once for all heads, into LDS: the angle in turns as a 64-bit product, its whole
// turns dropped there, so that far positions keep their fraction (a 32-bit product at position 10^6 is off by 0.06).
// A row is spread over a power of two of lanes; a lane holds both members of its pairs, as two pieces of V elements that
// are loaded and stored whole.
#include "common.h"

#include <math.h>
#include <string.h>

namespace hivt {
namespace {

constexpr int kMaxDim = 256;
constexpr int kMaxTokens = 32;       // positions of a workgroup
constexpr int kTable = 2048;         // (cos, sin) pairs of a workgroup in LDS
constexpr int kGradBlocks = 1024;    // workgroups of the backward: as many partial rows for the gains' gradients

struct Side {  // the queries or the keys
  const void *x, *dy;
  void *y, *dx;
  const float* w;
  int64_t x_st[3], dy_st[3], y_st[3], dx_st[3];  // batch, position, head; in elements
  int32_t heads;
};

struct RotArgs {
  Side side[2];
  const void* positions;
  int64_t pos_sb, pos_ss;
  int32_t pos_bytes;      // 4 or 8; 0: the position is the row's index
  int32_t B, S, d, rotary, interleaved, lanes, tokens;
  float eps;
  float* partial;         // [workgroups][2][d]
  double turns[kMaxDim / 2];  // rate_i / (2 pi)
};

template <typename T, int V> struct alignas(V * sizeof(T)) Piece { T e[V]; };

__device__ __forceinline__ float group_sum_of(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// One unit of a row: elements p0 .. p0 + V - 1 in a, p1 .. p1 + V - 1 in b.
template <typename T, int V>
struct Unit {
  float a[V], b[V];
  __device__ __forceinline__ void load(const T* row, int p0, int p1) {
    const Piece<T, V> x = *reinterpret_cast<const Piece<T, V>*>(row + p0), y = *reinterpret_cast<const Piece<T, V>*>(row + p1);
#pragma unroll
    for (int i = 0; i < V; ++i) { a[i] = (float)x.e[i]; b[i] = (float)y.e[i]; }
  }
  __device__ __forceinline__ void store(T* row, int p0, int p1) const {
    Piece<T, V> x, y;
#pragma unroll
    for (int i = 0; i < V; ++i) { x.e[i] = (T)a[i]; y.e[i] = (T)b[i]; }
    *reinterpret_cast<Piece<T, V>*>(row + p0) = x;
    *reinterpret_cast<Piece<T, V>*>(row + p1) = y;
  }
  // turns the pairs of the unit; cs: the position's (cos, sin), `first` the unit's first pair, `pairs` how many turn
  __device__ __forceinline__ void turn(const float2* cs, int first, int pairs, bool interleaved, float sign) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (first + i >= pairs) break;
      const float2 t = cs[first + i];
      const float c = t.x, s = t.y * sign;
      if (!interleaved) {
        const float u = a[i], v = b[i];
        a[i] = u * c - v * s;
        b[i] = u * s + v * c;
      } else {  // (the 2 V elements of the unit stand in a row: its pair i is 2 i, 2 i + 1)
        float& x = 2 * i < V ? a[2 * i < V ? 2 * i : 0] : b[2 * i >= V ? 2 * i - V : 0];
        float& y = 2 * i + 1 < V ? a[2 * i + 1 < V ? 2 * i + 1 : 0] : b[2 * i + 1 >= V ? 2 * i + 1 - V : 0];
        const float u = x, v = y;
        x = u * c - v * s;
        y = u * s + v * c;
      }
    }
  }
};

// Measured: bf16 4 x 4096 positions, 32 + 8 heads of 128: forward 69 us, 4.8 TB/s, backward 137 us, 3.7 TB/s (three rows at
// a time, and the gains' sums); fp32 2560 x 21, 8 + 8 heads of 16: 22 and 35 us, 5.0 and 4.8 TB/s.
template <typename T, int V, int UPL, bool BWD>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs a) {
  __shared__ float2 table[kTable];
  __shared__ float red[BWD ? 256 * 2 * V * UPL : 1];
  const int tid = threadIdx.x;
  const int lane = tid & (a.lanes - 1), group = tid / a.lanes, groups = 256 / a.lanes;
  const int units = a.d / (2 * V), half = a.rotary / 2;
  const int turning = a.interleaved ? units : half / V;  // units that hold pairs to turn
  const int64_t total = (int64_t)a.B * a.S;
  const int64_t blocks = (total + a.tokens - 1) / a.tokens;
  int p0[UPL], p1[UPL], first[UPL];
  bool on[UPL];
#pragma unroll
  for (int u = 0; u < UPL; ++u) {
    const int unit = lane + u * a.lanes;
    on[u] = unit < units;
    const int at = on[u] ? unit : 0;
    if (a.interleaved || at >= turning) {
      p0[u] = a.interleaved ? at * 2 * V : a.rotary + (at - turning) * 2 * V;
      p1[u] = p0[u] + V;
    } else {
      p0[u] = at * V;
      p1[u] = half + at * V;
    }
    first[u] = at < turning ? at * V : half;  // (a unit without pairs starts behind the last)
  }
  float grad[2][UPL][2 * V];
  if constexpr (BWD) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int u = 0; u < UPL; ++u)
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) grad[w][u][i] = 0.0f;
  }

  for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    const int64_t t0 = block * a.tokens;
    const int tokens = (int)(total - t0 < a.tokens ? total - t0 : a.tokens);
    __syncthreads();  // the table of the block before has been read
    for (int i = tid; i < tokens * half; i += 256) {
      const int64_t token = t0 + i / half;
      const int64_t b = token / a.S, s = token % a.S;
      int64_t pos = s;
      if (a.pos_bytes == 8) pos = static_cast<const int64_t*>(a.positions)[b * a.pos_sb + s * a.pos_ss];
      else if (a.pos_bytes == 4) pos = static_cast<const int32_t*>(a.positions)[b * a.pos_sb + s * a.pos_ss];
      const double turns = (double)pos * a.turns[i % half];
      float sn, cs;
      sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
      table[i] = make_float2(cs, sn);
    }
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const Side& sd = a.side[which];
      float gain[UPL][2 * V];
#pragma unroll
      for (int u = 0; u < UPL; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          gain[u][i] = on[u] ? sd.w[p0[u] + i] : 0.0f;
          gain[u][V + i] = on[u] ? sd.w[p1[u] + i] : 0.0f;
        }
      const int rows = tokens * sd.heads;
      for (int r = group; r < rows; r += groups) {
        const int token = r / sd.heads, h = r % sd.heads;
        const int64_t b = (t0 + token) / a.S, s = (t0 + token) % a.S;
        const T* x = static_cast<const T*>(sd.x) + b * sd.x_st[0] + s * sd.x_st[1] + h * sd.x_st[2];
        Unit<T, V> n[UPL], g[UPL];
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < UPL; ++u) {
          if (on[u]) {
            n[u].load(x, p0[u], p1[u]);
            if constexpr (BWD)
              g[u].load(static_cast<const T*>(sd.dy) + b * sd.dy_st[0] + s * sd.dy_st[1] + h * sd.dy_st[2], p0[u], p1[u]);
          } else {
#pragma unroll
            for (int i = 0; i < V; ++i) n[u].a[i] = n[u].b[i] = g[u].a[i] = g[u].b[i] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < V; ++i) sum += n[u].a[i] * n[u].a[i] + n[u].b[i] * n[u].b[i];
        }
        sum = group_sum_of(sum, a.lanes);
        const float inv = 1.0f / sqrtf(sum / (float)a.d + a.eps);
        const float2* cs = table + token * half;
        if constexpr (!BWD) {
          T* y = static_cast<T*>(sd.y) + b * sd.y_st[0] + s * sd.y_st[1] + h * sd.y_st[2];
#pragma unroll
          for (int u = 0; u < UPL; ++u) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              n[u].a[i] *= inv * gain[u][i];
              n[u].b[i] *= inv * gain[u][V + i];
            }
            n[u].turn(cs, first[u], half, a.interleaved != 0, 1.0f);
            if (on[u]) n[u].store(y, p0[u], p1[u]);
          }
        } else {
          float mean = 0.0f;
#pragma unroll
          for (int u = 0; u < UPL; ++u) {
            g[u].turn(cs, first[u], half, a.interleaved != 0, -1.0f);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              n[u].a[i] *= inv;
              n[u].b[i] *= inv;
              grad[which][u][i] += g[u].a[i] * n[u].a[i];
              grad[which][u][V + i] += g[u].b[i] * n[u].b[i];
              g[u].a[i] *= gain[u][i];
              g[u].b[i] *= gain[u][V + i];
              mean += g[u].a[i] * n[u].a[i] + g[u].b[i] * n[u].b[i];
            }
          }
          mean = group_sum_of(mean, a.lanes) / (float)a.d;
          T* dx = static_cast<T*>(sd.dx) + b * sd.dx_st[0] + s * sd.dx_st[1] + h * sd.dx_st[2];
#pragma unroll
          for (int u = 0; u < UPL; ++u) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              g[u].a[i] = (g[u].a[i] - n[u].a[i] * mean) * inv;
              g[u].b[i] = (g[u].b[i] - n[u].b[i] * mean) * inv;
            }
            if (on[u]) g[u].store(dx, p0[u], p1[u]);
          }
        }
      }
    }
  }
  if constexpr (BWD) {  // the groups' shares of the gains' gradients, in ascending order of the groups
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < UPL; ++u)
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) red[(u * 2 * V + i) * 256 + tid] = grad[which][u][i];
      __syncthreads();
      for (int j = tid; j < a.lanes * UPL * 2 * V; j += 256) {
        const int l = j % a.lanes, i = j / a.lanes % (2 * V), u = j / a.lanes / (2 * V);
        const int unit = l + u * a.lanes;
        if (unit >= units) continue;
        float s = 0.0f;
        for (int gr = 0; gr < groups; ++gr) s += red[(u * 2 * V + i) * 256 + gr * a.lanes + l];
        int at;
        if (a.interleaved || unit >= turning) at = (a.interleaved ? unit * 2 * V : a.rotary + (unit - turning) * 2 * V) + i;
        else at = i < V ? unit * V + i : half + unit * V + i - V;
        a.partial[((int64_t)blockIdx.x * 2 + which) * a.d + at] = s;
      }
    }
  }
}

// column sums of partial [rows][2 d]: sixteen slices of the rows in ascending order, then the slices; in 64 bits
// (5 us)
__global__ __launch_bounds__(1024) void gain_kernel(const float* __restrict__ partial, int rows, int d, float* __restrict__ dwq,
                                                    float* __restrict__ dwk) {
  __shared__ double sums[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
  double s = 0.0;
  if (col < 2 * d) {
    int r = rows * slice / 16;
    const int end = rows * (slice + 1) / 16;
    const float* p = partial + (int64_t)r * 2 * d + col;
    for (; r + 8 <= end; r += 8, p += 16 * d) {  // eight loads on their way at once
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = p[j * 2 * d];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; r < end; ++r, p += 2 * d) s += *p;
  }
  sums[slice][threadIdx.x & 63] = s;
  __syncthreads();
  if (slice == 0 && col < 2 * d) {
    for (int i = 1; i < 16; ++i) s += sums[i][threadIdx.x];
    (col < d ? dwq : dwk)[col < d ? col : col - d] = (float)s;
  }
}

// Pieces of V elements: the tensors' addresses and strides, the head and the turning part are multiples of them.
int piece_of(const RotArgs& a, int size, bool backward) {
  int v = 16 / size;
  auto limit = [&](uint64_t elements) {
    while (v > 1 && elements % v != 0) v /= 2;
  };
  while (v > 1 && (a.d % (2 * v) != 0 || (!a.interleaved && a.rotary % (2 * v) != 0))) v /= 2;
  for (int w = 0; w < 2; ++w) {
    const Side& s = a.side[w];
    const void* ptr[4] = {s.x, backward ? s.dx : s.y, s.dy, nullptr};
    const int64_t* st[3] = {s.x_st, backward ? s.dx_st : s.y_st, s.dy_st};
    const int64_t extent[3] = {a.B, a.S, s.heads};
    for (int t = 0; t < (backward ? 3 : 2); ++t) {
      limit(reinterpret_cast<uint64_t>(ptr[t]) / size);
      for (int j = 0; j < 3; ++j)
        if (extent[j] > 1) limit((uint64_t)(st[t][j] < 0 ? -st[t][j] : st[t][j]));
    }
  }
  return v;
}

int64_t blocks_of(const RotArgs& a) { return ((int64_t)a.B * a.S + a.tokens - 1) / a.tokens; }

template <typename T, int V, bool BWD>
int launch(RotArgs& a, hipStream_t stream) {
  const int units = a.d / (2 * V);
  int lanes = 1;
  while (lanes < units && lanes < 64) lanes *= 2;
  a.lanes = lanes;
  const int64_t blocks = blocks_of(a);
  const char* what = BWD ? "hivt_qk_norm_rotary_bwd" : "hivt_qk_norm_rotary_fwd";
  HIVT_REQUIRE(blocks < ((int64_t)1 << 31), HIVT_ERR_ARG, "%s: too many rows", what);
  const unsigned grid = (unsigned)(BWD && blocks > kGradBlocks ? kGradBlocks : blocks);
  // (a head is at most 256 wide: only pieces of one element make more than 64 units of it)
  if constexpr (V == 1) {
    if (units > 64) {
      hipLaunchKernelGGL((rotary_kernel<T, V, 2, BWD>), dim3(grid), dim3(256), 0, stream, a);
      HIVT_CHECK_LAUNCH(what);
      return HIVT_OK;
    }
  }
  hipLaunchKernelGGL((rotary_kernel<T, V, 1, BWD>), dim3(grid), dim3(256), 0, stream, a);
  HIVT_CHECK_LAUNCH(what);
  return HIVT_OK;
}

template <typename T, bool BWD>
int launch_type(RotArgs& a, hipStream_t stream) {
  const int v = piece_of(a, (int)sizeof(T), BWD);
  if constexpr (sizeof(T) == 2)
    if (v == 8) return launch<T, 8, BWD>(a, stream);
  if (v == 4) return launch<T, 4, BWD>(a, stream);
  if (v == 2) return launch<T, 2, BWD>(a, stream);
  return launch<T, 1, BWD>(a, stream);
}

int from_public(const char* what, const hivt_qk_norm_rotary* p, const double* rates, float eps, bool backward, RotArgs& a) {
  HIVT_REQUIRE(p != nullptr, HIVT_ERR_ARG, "%s: null argument block", what);
  HIVT_REQUIRE(p->dtype == HIVT_F32 || p->dtype == HIVT_BF16 || p->dtype == HIVT_F16, HIVT_ERR_UNSUPPORTED,
               "%s: element type %d", what, (int)p->dtype);
  const int64_t big = (int64_t)1 << 31;
  HIVT_REQUIRE(p->batch >= 0 && p->length >= 0 && p->batch < big && p->length < big && p->heads >= 1 && p->kv_heads >= 1 &&
               p->heads < 65536 && p->kv_heads < 65536, HIVT_ERR_ARG, "%s: bad sizes", what);
  HIVT_REQUIRE(p->head_dim >= 2 && p->head_dim <= kMaxDim && p->head_dim % 2 == 0, HIVT_ERR_UNSUPPORTED,
               "%s: head width %d (even, 2 to %d)", what, (int)p->head_dim, kMaxDim);
  HIVT_REQUIRE(p->rotary_dim >= 0 && p->rotary_dim <= p->head_dim && p->rotary_dim % 2 == 0, HIVT_ERR_ARG,
               "%s: %d turning components of %d", what, (int)p->rotary_dim, (int)p->head_dim);
  HIVT_REQUIRE(p->rotary_dim == 0 || rates != nullptr, HIVT_ERR_ARG, "%s: no rates", what);
  HIVT_REQUIRE(eps > 0.0f, HIVT_ERR_ARG, "%s: eps must be positive", what);
  HIVT_REQUIRE(p->position_bytes == 0 || ((p->position_bytes == 4 || p->position_bytes == 8) && p->positions), HIVT_ERR_ARG,
               "%s: positions of %d bytes", what, (int)p->position_bytes);
  memset(&a, 0, sizeof(a));
  const int64_t heads[2] = {p->heads, p->kv_heads};
  const int64_t x[2] = {p->q, p->k}, y[2] = {p->q_out, p->k_out}, dy[2] = {p->d_q_out, p->d_k_out}, dx[2] = {p->dq, p->dk},
                w[2] = {p->q_weight, p->k_weight};
  const int64_t* st[2][4] = {{p->q_stride, p->q_out_stride, p->d_q_out_stride, p->dq_stride},
                             {p->k_stride, p->k_out_stride, p->d_k_out_stride, p->dk_stride}};
  for (int i = 0; i < 2; ++i) {
    Side& s = a.side[i];
    s.heads = (int32_t)heads[i];
    s.x = reinterpret_cast<const void*>(x[i]);
    s.y = reinterpret_cast<void*>(y[i]);
    s.dy = reinterpret_cast<const void*>(dy[i]);
    s.dx = reinterpret_cast<void*>(dx[i]);
    s.w = reinterpret_cast<const float*>(w[i]);
    int64_t* to[4] = {s.x_st, s.y_st, s.dy_st, s.dx_st};
    for (int t = 0; t < 4; ++t)
      for (int j = 0; j < 3; ++j) to[t][j] = st[i][t][j];
    HIVT_REQUIRE(p->batch * p->length == 0 || (s.x && s.w && (backward ? s.dy && s.dx : s.y != nullptr)),
                 HIVT_ERR_ARG, "%s: null pointer", what);
  }
  a.positions = reinterpret_cast<const void*>(p->positions);
  a.pos_sb = p->position_stride[0];
  a.pos_ss = p->position_stride[1];
  a.pos_bytes = (int32_t)p->position_bytes;
  a.B = (int32_t)p->batch;
  a.S = (int32_t)p->length;
  a.d = (int32_t)p->head_dim;
  a.rotary = (int32_t)p->rotary_dim;
  a.interleaved = p->interleaved != 0;
  a.eps = eps;
  for (int i = 0; i < a.rotary / 2; ++i) a.turns[i] = rates[i] / 6.283185307179586476925;
  // positions of a workgroup: more share one computation of the sines, fewer fill the compute units
  int64_t tokens = (int64_t)a.B * a.S / 2048;
  if (tokens > kMaxTokens) tokens = kMaxTokens;
  if (a.rotary > 0 && tokens > 2 * kTable / a.rotary) tokens = 2 * kTable / a.rotary;
  a.tokens = tokens < 1 ? 1 : (int32_t)tokens;
  return HIVT_OK;
}

}  // namespace
}  // namespace hivt

using namespace hivt;

extern "C" int hivt_qk_norm_rotary_fwd(const hivt_qk_norm_rotary* p, const double* rates, float eps, hivt_stream_t stream) {
  RotArgs a;
  const int rc = from_public("hivt_qk_norm_rotary_fwd", p, rates, eps, false, a);
  if (rc != HIVT_OK || a.B == 0 || a.S == 0) return rc;
  switch (p->dtype) {
    case HIVT_F32: return launch_type<float, false>(a, (hipStream_t)stream);
    case HIVT_BF16: return launch_type<__bf16, false>(a, (hipStream_t)stream);
    default: return launch_type<_Float16, false>(a, (hipStream_t)stream);
  }
}

extern "C" size_t hivt_qk_norm_rotary_bwd_workspace_bytes(int64_t head_dim) {
  return (size_t)kGradBlocks * 2 * (head_dim > 0 ? head_dim : 0) * sizeof(float);
}

extern "C" int hivt_qk_norm_rotary_bwd(const hivt_qk_norm_rotary* p, const double* rates, float eps, void* workspace,
                                       size_t workspace_bytes, hivt_stream_t stream) {
  const char* what = "hivt_qk_norm_rotary_bwd";
  RotArgs a;
  int rc = from_public(what, p, rates, eps, true, a);
  if (rc != HIVT_OK) return rc;
  HIVT_REQUIRE(a.B > 0 && a.S > 0, HIVT_ERR_ARG, "%s: no rows: the gradients are zero", what);
  HIVT_REQUIRE(p->dq_weight && p->dk_weight, HIVT_ERR_ARG, "%s: null pointer", what);
  HIVT_REQUIRE(workspace && workspace_bytes >= hivt_qk_norm_rotary_bwd_workspace_bytes(a.d), HIVT_ERR_WORKSPACE,
               "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, hivt_qk_norm_rotary_bwd_workspace_bytes(a.d));
  a.partial = static_cast<float*>(workspace);
  switch (p->dtype) {
    case HIVT_F32: rc = launch_type<float, true>(a, (hipStream_t)stream); break;
    case HIVT_BF16: rc = launch_type<__bf16, true>(a, (hipStream_t)stream); break;
    default: rc = launch_type<_Float16, true>(a, (hipStream_t)stream);
  }
  if (rc != HIVT_OK) return rc;
  const int64_t blocks = blocks_of(a);
  hipLaunchKernelGGL(gain_kernel, dim3((unsigned)((2 * a.d + 63) / 64)), dim3(1024), 0, (hipStream_t)stream, a.partial,
                     (int)(blocks > kGradBlocks ? kGradBlocks : blocks), a.d, reinterpret_cast<float*>(p->dq_weight),
                     reinterpret_cast<float*>(p->dk_weight));
  HIVT_CHECK_LAUNCH(what);
  return HIVT_OK;
}
