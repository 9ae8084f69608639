// Orthogonalised updates: five steps of a quintic Newton-Schulz iteration on X / |X|, for a list of matrices.
//
//   X <- a X + (b G + c G^2) X,  G = X X'   (X with rows <= columns; a taller matrix enters transposed)
//
// Every factor in front of X is a polynomial of G, and polynomials of one symmetric matrix commute, so a phase of several
// steps can be taken on the small side alone:
//   P = a + b G + c G^2,  Q <- P Q,  G <- P G P   per step, and X <- Q X once at the end of the phase.
// With X m x n that costs 3 m^2 n per phase and 5 m^3 or fewer per step (symmetric products at half, only the tiles on and
// below the diagonal are computed) instead of 3 m^2 n + m^3 per step.  A phase forms G from the rounded X of the phase
// before: what the squares of small singular values lose in G comes back only there.  Hence the phases' lengths: single
// steps for matrices that are not wide, where that costs little more or the same (20 m^3 for square ones) and is the most
// accurate (a 64 x 64 one with columns falling to 1e-3: 3e-7 off instead of 4e-6 with 2 + 3); 1 + 2 + 2 for wide fp32 ones
// (47 instead of 65 m^3 at n = 4 m), 2 + 3 for wide 16-bit ones (38 m^3; 128 x 20 of low rank: 3.0e-6 off, fp32 products by
// the definition 1.8e-6).  Wide is n >= 2.5 m and n > 256 for fp32 (60 x 128: 2.2e-6 off in phases, by the definition
// 1.2e-6), n >= 1.5 m for 16 bits.  One phase of five would save more, but is 5e-3 off on matrices of low rank, even for
// 16-bit results too much.
//
// Bound by the matrix cores.  fp32 ones are eight times slower than 16-bit ones, so a value x is kept as two fp16 numbers
// (hi = fp16(s x), lo = fp16(s x - hi)) and a product is hi hi + hi lo + lo hi with fp32 sums: 2^-24 of the value per
// operand, as fp32, at three matrix instructions.  bfloat16 halves would keep 16 bits only.  fp16's range is no concern:
// the iteration keeps all singular values below 1.21, so the scale s is known beforehand.  (One fp16 product alone is
// not enough even for 16-bit results: 5e-2 on matrices of low rank, whose small singular values the iteration lifts.)
//
// Every product takes both operands with the reduction index innermost, which X X' and the symmetric products have
// anyway; for Q X the transposed X is kept as well (written by the same epilogue).  Operands are stored as the products
// read them: blocks of 64 rows by 32 of the reduction index, hi then lo, 8 KB in a piece, in the order of the LDS image.
// (Row-major planes cost a factor of six at 4096 columns: rows 8 KB apart meet on one memory channel.)  Sides are padded
// to multiples of 64 with zeros.
#include "common.h"

#include <math.h>
#include <string.h>

namespace hivt {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMats = 64;        // matrices per launch (descriptors travel in the argument block)
constexpr int kPad = 64;
constexpr int kSumChunk = 8192;  // elements of a workgroup of the norm
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;

struct Mat {
  const void* in;
  void* out;
  int64_t ws;        // byte offset of this matrix's workspace
  int32_t rows, cols;
};
struct Group {
  Mat mats[kMats];
  int32_t first[kMats];  // first workgroup of a matrix in the launch
  int32_t count, dtype;
  char* base;
  float eps;
};

// Workspace of a matrix: scalars, partial sums, planes.  A plane pair is [rows padded][columns padded] fp16 twice.
struct Layout {
  int32_t m, n, mp, np;    // small side, large side, padded
  int64_t big, small;      // bytes of a plane pair: X or its transpose; a square one
  int64_t sums, x, xt0, sq0, total;
  __host__ __device__ int64_t xt(int i) const { return xt0 + i * big; }
  __host__ __device__ int64_t sq(int i) const { return sq0 + i * small; }
};
__host__ __device__ inline int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
__host__ __device__ inline Layout layout_of(int32_t rows, int32_t cols) {
  Layout l;
  l.m = rows < cols ? rows : cols;
  l.n = rows < cols ? cols : rows;
  l.mp = (int32_t)up(l.m, kPad);
  l.np = (int32_t)up(l.n, kPad);
  l.big = (int64_t)l.mp * l.np * 4;
  l.small = (int64_t)l.mp * l.mp * 4;
  l.sums = 256;
  const int64_t at = l.sums + up(((int64_t)rows * cols + kSumChunk - 1) / kSumChunk * 8, 256);
  l.x = at;
  l.xt0 = at + l.big;
  l.sq0 = l.xt0 + 2 * l.big;
  l.total = up(l.sq0 + 5 * l.small, 256);
  return l;
}

// the matrix that a workgroup works for: every lane looks at one
__device__ __forceinline__ int which(const Group& g, int block) {
  const int lane = threadIdx.x & 63;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < g.count && g.first[lane] <= block)) - 1);
}

// matrices whose steps are taken in phases (see above)
__host__ __device__ inline bool is_wide(int64_t rows, int64_t cols, int dtype) {
  const int64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return dtype == HIVT_F32 ? 2 * n >= 5 * m && n > 256 : 2 * n >= 3 * m;
}

// sums of squares, in 64 bits: squares of small or large gradients leave the range of fp32
// (fp32 4096 x 4096: 14 us, 4.7 TB/s)
__global__ __launch_bounds__(256) void sum_kernel(const Group g) {
  __shared__ double red[4];
  const int i = which(g, blockIdx.x);
  const Mat& a = g.mats[i];
  const int64_t total = (int64_t)a.rows * a.cols, from = (int64_t)(blockIdx.x - g.first[i]) * kSumChunk;
  const int left = (int)(total - from < kSumChunk ? total - from : kSumChunk);
  float v[kSumChunk / 256];  // all on their way at once
  auto load = [&](auto* in) {
#pragma unroll
    for (int j = 0; j < kSumChunk / 256; ++j) {
      const int at = threadIdx.x + j * 256;
      v[j] = at < left ? (float)in[from + at] : 0.0f;
    }
  };
  if (g.dtype == HIVT_F32) load(static_cast<const float*>(a.in));
  else if (g.dtype == HIVT_BF16) load(static_cast<const __bf16*>(a.in));
  else load(static_cast<const _Float16*>(a.in));
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < kSumChunk / 256; ++j) s += (double)v[j] * v[j];
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double* sums = reinterpret_cast<double*>(g.base + a.ws + layout_of(a.rows, a.cols).sums);
    sums[blockIdx.x - g.first[i]] = red[0] + red[1] + red[2] + red[3];
  }
}

// Exponent of the scale of X's planes after `taken` steps: the spectral norm is at most 1.21, and at most x0 a^taken
// where |X| / (|X| + eps) = x0 is small (a matrix near or below eps keeps its relative precision).
__device__ __forceinline__ int x_exponent(float x0, int taken) {
  float bound = x0;
  for (int i = 0; i < taken; ++i) bound = fminf(bound * kA, 1.0f);
  if (!(bound > 0.0f)) return 14;
  const int k = -(int)floorf(log2f(bound)) - 1;
  return 14 + (k > 0 ? (k < 100 ? k : 100) : 0);
}

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// Rows of 32 halves; the four 16-byte pieces of a row trade places by the row's bits 2-3, so that sixteen consecutive
// rows read at one column start on sixteen groups of four banks.
constexpr int kBlock = 64 * 32;
__device__ __forceinline__ int lds_at(int row, int piece) { return row * 32 + (((piece ^ (row >> 2)) & 3) << 3); }
// element (row, k) of an operand with K (a multiple of 64) columns; the lo half is kBlock further
__device__ __forceinline__ int64_t at_of(int row, int k, int K) {
  return ((int64_t)(row >> 6) * (K >> 5) + (k >> 5)) * (2 * kBlock) + lds_at(row & 63, k >> 3 & 3) + (k & 7);
}

// x / (|x| + eps) into the planes of X and of its transpose, a 64 x 64 tile per workgroup (fp32 4096 x 4096: 35 us,
// 5.7 TB/s, 128 MB of it written and mostly still in the cache that the next product reads)
__global__ __launch_bounds__(256) void convert_kernel(const Group g) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int i = which(g, blockIdx.x);
  const Mat& a = g.mats[i];
  const Layout l = layout_of(a.rows, a.cols);
  char* const ws = g.base + a.ws;
  const double* sums = reinterpret_cast<const double*>(ws + l.sums);
  const int parts = (int)(((int64_t)a.rows * a.cols + kSumChunk - 1) / kSumChunk);
  double s = 0.0;
  for (int j = threadIdx.x; j < parts; j += 256) s += sums[j];
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const double norm = sqrt(red[0] + red[1] + red[2] + red[3]);
  const float x0 = (float)(norm / (norm + g.eps));
  const int block = blockIdx.x - g.first[i];
  if (block == 0 && threadIdx.x == 0) *reinterpret_cast<float*>(ws) = x0;
  const double factor = ldexp(1.0 / (norm + g.eps), x_exponent(x0, 0));
  const bool flip = a.rows > a.cols;
  const int tc = l.np / 64, i0 = block / tc * 64, j0 = block % tc * 64;  // of the small x large form
  // read along the rows of the matrix as it lies
  float in[16];
  auto load = [&](auto* from) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int row = (flip ? j0 : i0) + j * 4 + (threadIdx.x >> 6), col = (flip ? i0 : j0) + (threadIdx.x & 63);
      in[j] = row < a.rows && col < a.cols ? (float)from[(int64_t)row * a.cols + col] : 0.0f;
    }
  };
  if (g.dtype == HIVT_F32) load(static_cast<const float*>(a.in));
  else if (g.dtype == HIVT_BF16) load(static_cast<const __bf16*>(a.in));
  else load(static_cast<const _Float16*>(a.in));
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int r = j * 4 + (threadIdx.x >> 6), c = threadIdx.x & 63;
    tile[flip ? c : r][flip ? r : c] = (float)(in[j] * factor);
  }
  __syncthreads();
  _Float16* const x = reinterpret_cast<_Float16*>(ws + l.x);
  _Float16* const xt = reinterpret_cast<_Float16*>(ws + l.xt(0));
  for (int e = threadIdx.x; e < 1024; e += 256) {  // four elements at a time
    const int r = e >> 4, c = (e & 15) * 4;
    f16x4 hi, lo, hit, lot;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      _Float16 u, v;
      split(tile[r][c + j], u, v);
      hi[j] = u;
      lo[j] = v;
      split(tile[c + j][r], u, v);
      hit[j] = u;
      lot[j] = v;
    }
    int64_t at = at_of(i0 + r, j0 + c, l.np);
    *reinterpret_cast<f16x4*>(x + at) = hi;
    *reinterpret_cast<f16x4*>(x + at + kBlock) = lo;
    at = at_of(j0 + r, i0 + c, l.mp);
    *reinterpret_cast<f16x4*>(xt + at) = hit;
    *reinterpret_cast<f16x4*>(xt + at + kBlock) = lot;
  }
}

// One product for every matrix of the group: dst = alpha A B' + beta R + diag I, all as planes; A, B with the reduction
// index contiguous.
enum Shape : int { SHAPE_GRAM, SHAPE_SQUARE, SHAPE_APPLY };  // X X';  small x small;  Q X (as Q Xt')
struct Product {
  int32_t shape;
  int32_t a, b, dst;     // SQUARE: which of the five square planes; GRAM: dst; APPLY: a
  int32_t from, to;      // APPLY / GRAM: which transposed planes hold X / get the result
  int32_t r;             // SQUARE: the planes added with beta, or -1
  int32_t ea, eb, ed, er;  // exponents of the planes' scales (of square planes)
  int32_t taken, taken_after;  // steps that X has taken before / after (its scale)
  int32_t last;          // APPLY: the result is the output
  int32_t base, quarters;  // the launch's first tile; tiles of 128 are worked on as four of 64
  float alpha, beta, diag;
};

// A workgroup's square of results.  Its loop is bound by latency if nothing is done about it: a step of 32 takes 200 to
// 800 clocks of matrix work and its operands, just written by another kernel, over 2000 to arrive.  So AHEAD steps are on
// their way into registers (variables of their own: an indexed ring goes to scratch memory, which made the loop four
// times slower) and two in LDS.  Rates at fp32 4096 x 4096, three fp16 products counted: 1155 TFLOP/s in tiles of 256
// (357 us for Q X), 1020 in tiles of 128 (195 us for the tiles of a symmetric product), what a library's fp16 product
// reaches (1170).  The smaller ones are bound by latency (1024 x 1024: 15 us, 0.2 of that rate).  The smallest tile, which is taken where there are few, has four groups of waves that take
// every fourth step each and add their sums at the end (a bf16 1024 x 4096: 392 us with one group, 382 with two, 368 with
// four; two groups for the middle tile: 4.91 instead of 4.65 ms for fp32 4096 x 4096).
template <int BM_> struct Cfg {
  static constexpr int BM = BM_, BK = 32;
  static constexpr int WAVES = BM == 256 ? 8 : 4;  // that share a step
  static constexpr int GROUPS = BM == 64 ? 4 : 1;  // of them, that take the steps in turn
  static constexpr int THREADS = GROUPS * WAVES * 64;
  static constexpr int AHEAD = BM == 256 ? 1 : 2;
  static constexpr int WM = BM / (BM == 256 ? 4 : 2), WN = BM / 2;  // a wave's rows and columns
  static constexpr int TM = WM / 32, TN = WN / 32;                  // 32 x 32 blocks of them
  static constexpr int TILE = BM / 64 * 2 * kBlock;                 // halves of an operand's step in LDS
  static constexpr size_t LDS = (size_t)GROUPS * 4 * TILE * sizeof(_Float16);
  static constexpr int NPT = TILE * 2 / 16 / (WAVES * 64);          // 16-byte pieces of it per thread
};

template <int BM, bool SUMS>
__global__ __launch_bounds__(Cfg<BM>::THREADS) void product_kernel(const Group g, const Product p) {
  using C = Cfg<BM>;
  extern __shared__ __attribute__((aligned(16))) _Float16 lds_everyone[];  // [GROUPS][2][A, B][TILE]
  const bool quarters = BM == 64 && p.quarters;
  const int tile = p.base + (quarters ? blockIdx.x >> 2 : blockIdx.x), size = quarters ? 128 : BM;
  const int gi = which(g, tile);
  const Mat& mat = g.mats[gi];
  const Layout l = layout_of(mat.rows, mat.cols);
  char* const ws = g.base + mat.ws;
  const int block = tile - g.first[gi];
  const int lane = threadIdx.x & 63, wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int turns = wave_all / C::WAVES, wave = wave_all % C::WAVES, tid = wave * 64 + lane;
  _Float16* const lds_all = lds_everyone + turns * 4 * C::TILE;
  const float x0 = *reinterpret_cast<const float*>(ws);

  const bool apply = p.shape == SHAPE_APPLY, gram = p.shape == SHAPE_GRAM;
  const int M = l.mp, N = apply ? l.np : l.mp, K = gram ? l.np : l.mp;
  int ti, tj;
  if (apply) {
    const int tiles = (N + size - 1) / size;
    ti = block / tiles;
    tj = block % tiles;
  } else {  // tiles on and below the diagonal
    ti = (int)((sqrtf(8.0f * (float)block + 1.0f) - 1.0f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= block) ++ti;
    while (ti * (ti + 1) / 2 > block) --ti;
    tj = block - ti * (ti + 1) / 2;
  }
  if (quarters) {
    ti = ti * 2 + (blockIdx.x >> 1 & 1);
    tj = tj * 2 + (blockIdx.x & 1);
    if (ti * BM >= M || tj * BM >= N || (!apply && tj > ti)) return;
  }
  const int i0 = ti * BM, j0 = tj * BM;
  const _Float16* A = reinterpret_cast<const _Float16*>(ws + (gram ? l.x : l.sq(p.a)));
  const _Float16* B = reinterpret_cast<const _Float16*>(ws + (gram ? l.x : apply ? l.xt(p.from) : l.sq(p.b)));
  // (a 128-row tile may reach past an operand, which is padded to 64 rows: it reads the last block again and does not
  // store those results)
  const int steps = K / C::BK, rounds = (steps + C::GROUPS - 1) / C::GROUPS;
  struct Step { u32x4 a[C::NPT], b[C::NPT]; };
  auto fetch = [&](Step& r, int round) {
    const int step = min(round * C::GROUPS + turns, steps - 1);
#pragma unroll
    for (int i = 0; i < C::NPT; ++i) {
      const int idx = tid + i * C::WAVES * 64, sub = idx / (2 * kBlock / 8), in = idx % (2 * kBlock / 8) * 8;
      const int64_t ra = (int64_t)min((i0 >> 6) + sub, (M >> 6) - 1) * (K >> 5) + step;
      const int64_t rb = (int64_t)min((j0 >> 6) + sub, (N >> 6) - 1) * (K >> 5) + step;
      r.a[i] = *reinterpret_cast<const u32x4*>(A + ra * (2 * kBlock) + in);
      r.b[i] = *reinterpret_cast<const u32x4*>(B + rb * (2 * kBlock) + in);
    }
  };
  auto put = [&](const Step& r, int buf) {
#pragma unroll
    for (int i = 0; i < C::NPT; ++i) {
      _Float16* const at = lds_all + buf * 2 * C::TILE + (tid + i * C::WAVES * 64) * 8;
      *reinterpret_cast<u32x4*>(at) = r.a[i];
      *reinterpret_cast<u32x4*>(at + C::TILE) = r.b[i];
    }
  };

  f32x16 acc[C::TM][C::TN];
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
  const int wi = (wave >> 1) * C::WM, wj = (wave & 1) * C::WN;
  auto compute = [&](int buf, f32x16 (&acc)[C::TM][C::TN]) {
    const _Float16* const la = lds_all + buf * 2 * C::TILE;
    const _Float16* const lb = la + C::TILE;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      f16x8 fa[2][C::TM], fb[2][C::TN];
      const int piece = ks * 2 + (lane >> 5);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
          const int r = wi + i * 32 + (lane & 31);
          fa[q][i] = *reinterpret_cast<const f16x8*>(la + ((r >> 6) * 2 + q) * kBlock + lds_at(r & 63, piece));
        }
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
          const int r = wj + j * 32 + (lane & 31);
          fb[q][j] = *reinterpret_cast<const f16x8*>(lb + ((r >> 6) * 2 + q) * kBlock + lds_at(r & 63, piece));
        }
      }
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0][i], fb[0][j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0][i], fb[1][j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[1][i], fb[0][j], acc[i][j], 0, 0, 0);
        }
    }
  };

  // one step: its products, then the next one's operands into the other buffer (whose readers passed the barrier of the
  // step before) and a later one's on their way.  The steps are an even number: sides are padded to 64.
  // SUMS (fp32 in the smallest tile): each step has a sum of its own, as for the small matrices (200 x 1000: 2.4e-6 instead
  // of 4.1e-6 off, by the definition 2.6e-6; 16 bits round coarser than either, and a bf16 1024 x 4096 takes 394 us without
  // and 448 us with it)
  auto turn = [&](int round, int buf, Step& r, int later) {
    if (C::GROUPS > 1 && round * C::GROUPS + turns >= steps) {
    } else if constexpr (SUMS) {
      f32x16 part[C::TM][C::TN];
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) part[i][j][e] = 0.0f;
      compute(buf, part);
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] += part[i][j][e];
    } else {
      compute(buf, acc);
    }
    put(r, buf ^ 1);
    fetch(r, later);
    __syncthreads();
  };
  if constexpr (C::AHEAD == 1) {  // (two would not fit the registers of two waves per SIMD)
    Step r0;
    fetch(r0, 0);
    put(r0, 0);
    fetch(r0, 1);
    __syncthreads();
    for (int s = 0; s < rounds; s += 2) {
      turn(s, 0, r0, s + 2);
      turn(s + 1, 1, r0, s + 3);
    }
  } else {
    Step r0, r1;
    fetch(r0, 0);
    fetch(r1, 1);
    put(r0, 0);
    fetch(r0, 2);
    __syncthreads();
    for (int s = 0; s < rounds; s += 2) {
      turn(s, 0, r1, s + 3);
      turn(s + 1, 1, r0, s + 4);
    }
  }
  // The groups' sums, added in their order; each group then finishes its share of every block's rows.
  constexpr int SHARE = 4 / C::GROUPS;
  f32x4 sums[C::TM][C::TN][SHARE];
  if constexpr (C::GROUPS > 1) {
    f32x4* const all = reinterpret_cast<f32x4*>(lds_everyone) + wave * C::TM * C::TN * 4 * 64 + lane;
    constexpr int GROUP = C::WAVES * C::TM * C::TN * 4 * 64;
#pragma unroll
    for (int bi = 0; bi < C::TM; ++bi)
#pragma unroll
      for (int bj = 0; bj < C::TN; ++bj)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4)
          all[turns * GROUP + ((bi * C::TN + bj) * 4 + e4) * 64] =
              f32x4{acc[bi][bj][e4 * 4], acc[bi][bj][e4 * 4 + 1], acc[bi][bj][e4 * 4 + 2], acc[bi][bj][e4 * 4 + 3]};
    __syncthreads();
#pragma unroll
    for (int bi = 0; bi < C::TM; ++bi)
#pragma unroll
      for (int bj = 0; bj < C::TN; ++bj)
#pragma unroll
        for (int i = 0; i < SHARE; ++i) {
          const int at = ((bi * C::TN + bj) * 4 + turns * SHARE + i) * 64;
          f32x4 v = all[at];
#pragma unroll
          for (int q = 1; q < C::GROUPS; ++q) v += all[q * GROUP + at];
          sums[bi][bj][i] = v;
        }
  } else {
#pragma unroll
    for (int bi = 0; bi < C::TM; ++bi)
#pragma unroll
      for (int bj = 0; bj < C::TN; ++bj)
#pragma unroll
        for (int e = 0; e < 16; ++e) sums[bi][bj][e / 4][e % 4] = acc[bi][bj][e];
  }

  // results: column = lane & 31, rows 8 (e / 4) + 4 (lane >> 5) + e % 4 of a 32 x 32 block
  const int ex = x_exponent(x0, p.taken), ex_after = x_exponent(x0, p.taken_after);
  const int down = gram ? 2 * ex : apply ? p.ea + ex : p.ea + p.eb;
  const float unscale = ldexpf(p.alpha, -down);
  const int ed = apply ? ex_after : p.ed;
  const _Float16* R = p.r >= 0 ? reinterpret_cast<const _Float16*>(ws + l.sq(p.r)) : nullptr;
  const float rscale = ldexpf(p.beta, -p.er);
#pragma unroll
  for (int bi = 0; bi < C::TM; ++bi)
#pragma unroll
    for (int bj = 0; bj < C::TN; ++bj)
#pragma unroll
      for (int share = 0; share < SHARE; ++share) {
        const int e4 = turns * SHARE + share;
        const int row = i0 + wi + bi * 32 + e4 * 8 + (lane >> 5) * 4, col = j0 + wj + bj * 32 + (lane & 31);
        if (row >= M || col >= N) continue;
        float v[4];
        f16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = sums[bi][bj][share][e] * unscale;
          if (!apply) {
            if (R != nullptr) {
              const int64_t at = at_of(row + e, col, l.mp);
              v[e] += rscale * ((float)R[at] + (float)R[at + kBlock]);
            }
            if (row + e == col) v[e] += p.diag;
          }
          const bool in = row + e < l.m && col < (apply ? l.n : l.m);
          if (!in) v[e] = 0.0f;
        }
        if (apply && p.last) {
          const bool flip = mat.rows > mat.cols;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (row + e >= l.m || col >= l.n) continue;
            const int64_t at = flip ? (int64_t)col * l.m + row + e : (int64_t)(row + e) * l.n + col;
            if (g.dtype == HIVT_F32) static_cast<float*>(mat.out)[at] = v[e];
            else if (g.dtype == HIVT_BF16) static_cast<__bf16*>(mat.out)[at] = (__bf16)v[e];
            else static_cast<_Float16*>(mat.out)[at] = (_Float16)v[e];
          }
          continue;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          _Float16 h, o;
          split(ldexpf(v[e], ed), h, o);
          hi[e] = h;
          lo[e] = o;
        }
        // as it stands, and transposed (the square results are symmetric: the tile above the diagonal)
        _Float16* dst = reinterpret_cast<_Float16*>(ws + (apply ? l.x : l.sq(p.dst)));
        _Float16* dt = reinterpret_cast<_Float16*>(ws + (apply ? l.xt(p.to) : l.sq(p.dst)));
        const int ld = apply ? l.np : l.mp;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t at = at_of(row + e, col, ld);
          dst[at] = hi[e];
          dst[at + kBlock] = lo[e];
        }
        if (apply || ti != tj) {
          const int64_t at = at_of(col, row, l.mp);
          *reinterpret_cast<f16x4*>(dt + at) = hi;
          *reinterpret_cast<f16x4*>(dt + at + kBlock) = lo;
        }
      }
}

// ---- small matrices: all steps in one workgroup ---------------------------------------------------------------------------
// With the smaller side at most 128 a product is a few microseconds of one compute unit, less than the launch in between:
// a workgroup takes a matrix through all phases.  G and the polynomials stay in LDS (two square operands: a phase has at
// most two steps), X comes through a staging buffer of 32 of the reduction index and goes back to the workspace.  A result
// is symmetric, or wanted transposed as well, so four consecutive rows of a lane are stored as one piece of a row.
// 62 matrices of the 128-wide model: 2 + 1 launches instead of 37; 217 us, the time of a 512 x 128 one (bound by the latency
// of its chain; most compute units are idle).
template <int MP> struct Small {
  static constexpr int THREADS = MP == 128 ? 512 : 256;
  static constexpr int TN = MP / 64;                        // 32 x 32 blocks of a wave along the columns (one along the rows)
  static constexpr int SQUARE = MP * MP * 2;                // halves of a square operand
  static constexpr int STAGE = MP * 32 * 2;                 // halves of a staged step
  static constexpr int NPT = STAGE * 2 / 16 / THREADS;
  static constexpr size_t LDS = (size_t)(2 * SQUARE + STAGE) * sizeof(_Float16);
};

template <int MP>
__global__ __launch_bounds__(Small<MP>::THREADS) void small_kernel(const Group g, int steps_wanted) {
  using C = Small<MP>;
  extern __shared__ __attribute__((aligned(16))) _Float16 lds_all[];
  _Float16* const s0 = lds_all;
  _Float16* const s1 = s0 + C::SQUARE;
  _Float16* const stage = s1 + C::SQUARE;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Mat& mat = g.mats[blockIdx.x];
  const Layout l = layout_of(mat.rows, mat.cols);
  char* const ws = g.base + mat.ws;
  const float x0 = *reinterpret_cast<const float*>(ws);
  _Float16* const X = reinterpret_cast<_Float16*>(ws + l.x);
  _Float16* const Xt = reinterpret_cast<_Float16*>(ws + l.xt(0));
  const int wi = (wave >> 1) * 32, wj = (wave & 1) * (MP / 2);
  const int mb = l.mp >> 6;  // blocks of 64 rows that exist (1 or 2)

  f32x16 acc[C::TN], turned[C::TN];
  auto clear = [&](f32x16 (&acc)[C::TN]) {
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][e] = 0.0f;
  };
  // 32 of the reduction index: A and B in blocks, `stride` blocks apart per 64 rows.  Every step has a sum of its own, added
  // to the whole in fp32: a matrix instruction cuts what it adds to a large sum short, and one chain over 512 is 3.3e-6 off
  // in the result where this is 2.1e-6 (fp32 products by the definition: 1.9e-6).
  auto multiply = [&](f32x16 (&acc)[C::TN], const _Float16* A, int sa, const _Float16* B, int sb) {
    f32x16 part[C::TN];
    clear(part);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int piece = ks * 2 + (lane >> 5);
      const int ra = wi + (lane & 31);
      f16x8 fa[2], fb[2][C::TN];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        fa[q] = *reinterpret_cast<const f16x8*>(A + ((ra >> 6) * sa * 2 + q) * kBlock + lds_at(ra & 63, piece));
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
          const int rb = wj + j * 32 + (lane & 31);
          fb[q][j] = *reinterpret_cast<const f16x8*>(B + ((rb >> 6) * sb * 2 + q) * kBlock + lds_at(rb & 63, piece));
        }
      }
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        part[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0], fb[0][j], part[j], 0, 0, 0);
        part[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0], fb[1][j], part[j], 0, 0, 0);
        part[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[1], fb[0][j], part[j], 0, 0, 0);
      }
    }
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][e] += part[j][e];
  };
  constexpr int KB = MP / 32;  // steps of a square operand
  auto square = [&](const _Float16* A, const _Float16* B) {
    clear(acc);
#pragma unroll 1
    for (int kb = 0; kb < KB; ++kb) multiply(acc, A + kb * 2 * kBlock, KB, B + kb * 2 * kBlock, KB);
  };
  // the lane's number, anew: offsets that the compiler would otherwise hold over all phases, for want of registers in memory
  auto anew = [](int x) {
    asm volatile("" : "+v"(x));
    return x;
  };
  // acc * 2^-down (+ b G + a I) as a square operand of scale 2^ed; G: the operand it was made from (scale 2^14)
  auto keep = [&](_Float16* dst, int down, int ed, float alpha, const _Float16* G) {
    const float unscale = ldexpf(alpha, -down), gscale = ldexpf(kB, -14);
    const int ln = anew(lane);
    float v[C::TN][16];
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int row = wi + e4 * 8 + (ln >> 5) * 4, col = wj + j * 32 + (ln & 31);
        f16x4 gh, gl;
        if (G != nullptr) {  // (symmetric: row `col`, four columns)
          const int64_t at = at_of(col, row, MP);
          gh = *reinterpret_cast<const f16x4*>(G + at);
          gl = *reinterpret_cast<const f16x4*>(G + at + kBlock);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = acc[j][e4 * 4 + e] * unscale;
          if (G != nullptr) {
            x += gscale * ((float)gh[e] + (float)gl[e]);
            if (row + e == col) x += kA;
          }
          v[j][e4 * 4 + e] = row + e < l.m && col < l.m ? ldexpf(x, ed) : 0.0f;
        }
      }
    __syncthreads();  // every wave has read its operands
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int row = wi + e4 * 8 + (ln >> 5) * 4, col = wj + j * 32 + (ln & 31);
        f16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          _Float16 h, o;
          split(v[j][e4 * 4 + e], h, o);
          hi[e] = h;
          lo[e] = o;
        }
        const int64_t at = at_of(col, row, MP);
        *reinterpret_cast<f16x4*>(dst + at) = hi;
        *reinterpret_cast<f16x4*>(dst + at + kBlock) = lo;
      }
    __syncthreads();
  };
  // a step of a staged operand: `blocks` blocks of 64 rows from `src` on, `stride` blocks apart; rows that are not there
  // repeat the last
  struct Step { u32x4 r[C::NPT]; };
  Step r0, r1, r2, r3;  // four steps on their way: a step computes a tenth of the time that its operands take to arrive
  auto fetch = [&](Step& r, const _Float16* src, int stride, int blocks) {
    const int id = anew(tid);
#pragma unroll
    for (int i = 0; i < C::NPT; ++i) {
      const int idx = id + i * C::THREADS, sub = idx / (2 * kBlock / 8), in = idx % (2 * kBlock / 8) * 8;
      r.r[i] = *reinterpret_cast<const u32x4*>(src + (int64_t)min(sub, blocks - 1) * stride * (2 * kBlock) + in);
    }
  };
  auto put = [&](const Step& r) {
#pragma unroll
    for (int i = 0; i < C::NPT; ++i) *reinterpret_cast<u32x4*>(stage + (tid + i * C::THREADS) * 8) = r.r[i];
  };

  const int kn = l.np >> 5, km = l.mp >> 5, nb = l.np >> 6;
  constexpr int CB = MP / 64;  // blocks of 64 columns of X at a time
  auto fetch_x = [&](Step& r, int k) { fetch(r, X + (int64_t)min(k, kn - 1) * 2 * kBlock, kn, mb); };
  auto fetch_xt = [&](Step& r, int c, int k) {
    c = min(c, nb - 1);
    fetch(r, Xt + ((int64_t)c * km + min(k, km - 1)) * 2 * kBlock, km, min(CB, nb - c));
  };

  const int at_once = is_wide(mat.rows, mat.cols, g.dtype) ? 2 : 1;
  int taken = 0;
  while (taken < steps_wanted) {
    const int steps = (steps_wanted - taken) % at_once != 0 ? 1 : at_once;
    const bool last = taken + steps == steps_wanted;
    const int ex = x_exponent(x0, taken), ex_after = x_exponent(x0, taken + steps);
    // G = X X'
    clear(acc);
    fetch_x(r0, 0);
    fetch_x(r1, 1);
    fetch_x(r2, 2);
    fetch_x(r3, 3);
    auto gram = [&](Step& r, int later) {
      __syncthreads();
      put(r);
      fetch_x(r, later);
      __syncthreads();
      multiply(acc, stage, 1, stage, 1);
    };
    for (int k = 0;; k += 4) {  // (an even number of steps)
      gram(r0, k + 4);
      gram(r1, k + 5);
      if (k + 2 >= kn) break;
      gram(r2, k + 6);
      gram(r3, k + 7);
      if (k + 4 >= kn) break;
    }
    fetch_xt(r0, 0, 0);
    fetch_xt(r1, 0, 1);
    fetch_xt(r2, 0, 2);
    fetch_xt(r3, 0, 3);
    keep(s0, 2 * ex, 14, 1.0f, nullptr);
    // the polynomial in front of X: into s0
    int eq = 14;
    if (steps == 1) {
      square(s0, s0);
      keep(s0, 28, 14, kC, s0);
    } else {
      square(s0, s0);
      keep(s1, 28, 14, kC, s0);      // P
      square(s1, s0);
      keep(s0, 28, 14, 1.0f, nullptr);  // P G
      square(s0, s1);
      keep(s0, 28, 14, 1.0f, nullptr);  // P G P
      square(s0, s0);
      keep(s0, 28, 14, kC, s0);      // the second P
      square(s0, s1);
      eq = 12;
      keep(s0, 28, eq, 1.0f, nullptr);
    }
    // X <- Q X, MP columns at a time.  Both the result and its transpose are stored with the reduction index of a later
    // product innermost, four of which a lane holds in a row only in the product with the operands exchanged: it is
    // computed twice.  Pieces of 8 bytes go to 64 cache lines a store (13 000 clocks for 128 x 128); they are put together
    // in LDS, in the free square operand, and leave it in whole lines.
    const float unscale = ldexpf(1.0f, -(eq + ex));
    for (int c = 0; c < nb; c += CB) {
      clear(acc);
      clear(turned);
      auto apply = [&](Step& r, int k) {
        __syncthreads();
        put(r);
        fetch_xt(r, c + CB, k);
        __syncthreads();
        multiply(acc, s0 + k * 2 * kBlock, KB, stage, 1);
        if (!last) multiply(turned, stage, 1, s0 + k * 2 * kBlock, KB);
      };
      apply(r0, 0);
      apply(r1, 1);
      if (km == 4) {
        apply(r2, 2);
        apply(r3, 3);
      }
      // (these columns of Xt have been read; the rest of them belongs to other columns of X)
      const int ln = anew(lane);
      if (last) {
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int row = wi + (e >> 2) * 8 + (ln >> 5) * 4 + (e & 3), col = c * 64 + wj + j * 32 + (ln & 31);
            if (row >= l.m || col >= l.n) continue;
            const float x = acc[j][e] * unscale;
            const int64_t at = mat.rows > mat.cols ? (int64_t)col * l.m + row : (int64_t)row * l.n + col;
            if (g.dtype == HIVT_F32) static_cast<float*>(mat.out)[at] = x;
            else if (g.dtype == HIVT_BF16) static_cast<__bf16*>(mat.out)[at] = (__bf16)x;
            else static_cast<_Float16*>(mat.out)[at] = (_Float16)x;
          }
        continue;
      }
      // four elements of row `to` from element `from` on, into the image of a square operand
      auto piece = [&](int to, int from, const f32x16& v, int e4, bool in, int limit) {
        f16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          _Float16 h, o;
          split(in && from + e < limit ? ldexpf(v[e4 * 4 + e] * unscale, ex_after) : 0.0f, h, o);
          hi[e] = h;
          lo[e] = o;
        }
        const int64_t at = at_of(to, from, MP);
        *reinterpret_cast<f16x4*>(s1 + at) = hi;
        *reinterpret_cast<f16x4*>(s1 + at + kBlock) = lo;
      };
      // blocks [rows][steps] of the image to memory, `stride` blocks apart per 64 rows
      auto leave = [&](_Float16* dst, int rows, int steps, int stride) {
        const int id = anew(tid);
        for (int i = id; i < MP / 64 * KB * (2 * kBlock / 8); i += C::THREADS) {
          const int block = i / (2 * kBlock / 8), in = i % (2 * kBlock / 8) * 8, rb = block / KB, kb = block % KB;
          if (rb < rows && kb < steps)
            *reinterpret_cast<u32x4*>(dst + ((int64_t)rb * stride + kb) * (2 * kBlock) + in) =
                *reinterpret_cast<const u32x4*>(s1 + block * 2 * kBlock + in);
        }
      };
      const int there = min(CB, nb - c);  // blocks of 64 columns
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {  // rows of X down, columns across
          const int down = wi + e4 * 8 + (ln >> 5) * 4, across = wj + j * 32 + (ln & 31);
          piece(across, down, acc[j], e4, c * 64 + across < l.n, l.m);
        }
      __syncthreads();
      leave(Xt + (int64_t)c * km * 2 * kBlock, there, km, km);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {  // columns of X down, rows across
          const int down = wi + e4 * 8 + (ln >> 5) * 4, across = wj + j * 32 + (ln & 31);
          piece(across, down, turned[j], e4, across < l.m, l.n - c * 64);
        }
      __syncthreads();
      leave(X + (int64_t)c * 2 * 2 * kBlock, mb, there * 2, kn);
    }
    taken += steps;
    __threadfence();  // what this workgroup wrote to memory it reads again
    __syncthreads();
  }
}

int64_t tiles_of(const Mat& a, int shape, int bm) {
  const Layout l = layout_of(a.rows, a.cols);
  const int64_t tm = (l.mp + bm - 1) / bm, tn = (l.np + bm - 1) / bm;
  return shape == SHAPE_APPLY ? tm * tn : tm * (tm + 1) / 2;
}

// tiles `begin` to `end` of a product in tiles of `size` (BM, or in quarters); g.first holds the matrices' first tiles
template <int BM, bool SUMS = false>
int launch_tiles(const Group& g, Product p, int size, int64_t begin, int64_t end, hipStream_t stream) {
  using C = Cfg<BM>;
  const char* what = "hivt_orthogonalize";
  p.base = (int32_t)begin;
  p.quarters = size != BM;
  if (C::LDS > 48 * 1024)
    HIVT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&product_kernel<BM, SUMS>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)C::LDS), what);
  hipLaunchKernelGGL((product_kernel<BM, SUMS>), dim3((unsigned)((end - begin) * (p.quarters ? 4 : 1))), dim3(C::THREADS),
                     C::LDS, stream, g, p);
  HIVT_CHECK_LAUNCH(what);
  return HIVT_OK;
}

// The largest tile that still gives every compute unit one.  Tiles of 128 run two to a compute unit; up to 64 that would
// be left for a last turn are worked on in quarters, one to a compute unit, by another launch (fp32 4096 x 4096, 528
// tiles: 290 us a product without, 195 + 34 us with it).
int launch_product(Group& g, const Product& p, hipStream_t stream) {
  constexpr int64_t kUnits = 256;
  const char* what = "hivt_orthogonalize";
  auto count = [&](int size) {
    int64_t tiles = 0;
    for (int i = 0; i < g.count; ++i) {
      g.first[i] = (int32_t)tiles;
      tiles += tiles_of(g.mats[i], p.shape, size);
      if (tiles >= (int64_t)1 << 29) return (int64_t)-1;
    }
    return tiles;
  };
  int64_t tiles = count(64);
  HIVT_REQUIRE(tiles >= 0, HIVT_ERR_ARG, "%s: too many workgroups", what);
  tiles = count(256);
  if (tiles >= kUnits) return launch_tiles<256>(g, p, 256, 0, tiles, stream);
  tiles = count(128);
  auto smallest = [&](int size, int64_t begin, int64_t end) {
    return g.dtype == HIVT_F32 ? launch_tiles<64, true>(g, p, size, begin, end, stream)
                               : launch_tiles<64>(g, p, size, begin, end, stream);
  };
  if (tiles < kUnits) {
    tiles = count(64);
    return smallest(64, 0, tiles);
  }
  const int64_t left = tiles > 2 * kUnits && tiles % (2 * kUnits) <= 64 ? tiles % (2 * kUnits) : 0;
  const int rc = launch_tiles<128>(g, p, 128, 0, tiles - left, stream);
  return rc != HIVT_OK || left == 0 ? rc : smallest(128, tiles - left, tiles);
}

// exponent of the scale of a product of k factors P (each at most 3.45)
int q_exponent(int k) { return 16 - 2 * k; }

template <int MP>
int launch_small(const Group& g, int steps, hipStream_t stream) {
  using C = Small<MP>;
  const char* what = "hivt_orthogonalize";
  if (C::LDS > 48 * 1024)
    HIVT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&small_kernel<MP>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)C::LDS), what);
  hipLaunchKernelGGL(small_kernel<MP>, dim3((unsigned)g.count), dim3(C::THREADS), C::LDS, stream, g, steps);
  HIVT_CHECK_LAUNCH(what);
  return HIVT_OK;
}

struct Phases { int32_t count, steps[16]; };

// one workgroup to a matrix of this shape: 0 (no), or the smaller side that its kernel is made for
int small_side(int64_t rows, int64_t cols) {
  const int64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return m > 128 || n > 1024 ? 0 : m > 64 ? 128 : 64;
}

// small: one workgroup to a matrix, through all steps
int run_group(Group& g, const Phases& list, bool small, int steps, hipStream_t stream) {
  const char* what = "hivt_orthogonalize";
  const int32_t* const phases = list.steps;
  const int nphases = list.count;
  int64_t blocks = 0;
  for (int i = 0; i < g.count; ++i) {
    g.first[i] = (int32_t)blocks;
    blocks += ((int64_t)g.mats[i].rows * g.mats[i].cols + kSumChunk - 1) / kSumChunk;
  }
  HIVT_REQUIRE(blocks < ((int64_t)1 << 31), HIVT_ERR_ARG, "%s: too many workgroups", what);
  hipLaunchKernelGGL(sum_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, g);
  HIVT_CHECK_LAUNCH(what);
  blocks = 0;
  for (int i = 0; i < g.count; ++i) {
    g.first[i] = (int32_t)blocks;
    const Layout l = layout_of(g.mats[i].rows, g.mats[i].cols);
    blocks += (int64_t)(l.mp / 64) * (l.np / 64);
  }
  HIVT_REQUIRE(blocks < ((int64_t)1 << 31), HIVT_ERR_ARG, "%s: too many workgroups", what);
  hipLaunchKernelGGL(convert_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, g);
  HIVT_CHECK_LAUNCH(what);

  if (small) {
    // (a matrix of up to 64 gives the same bits in either kernel: the larger one adds zeros)
    int side = 0;
    for (int i = 0; i < g.count; ++i) side = max(side, small_side(g.mats[i].rows, g.mats[i].cols));
    return side == 64 ? launch_small<64>(g, steps, stream) : launch_small<128>(g, steps, stream);
  }
  int taken = 0, at = 0;
  for (int f = 0; f < nphases; ++f) {
    // square planes: 0 G, 1 P G, 2 P, and 3 / 4 in turn Q
    Product p;
    memset(&p, 0, sizeof(p));
    p.r = -1;
    p.alpha = 1.0f;
    p.shape = SHAPE_GRAM;
    p.taken = p.taken_after = taken;
    p.dst = 0;
    p.ed = 14;
    int rc = launch_product(g, p, stream);
    if (rc != HIVT_OK) return rc;
    p.shape = SHAPE_SQUARE;
    int q = 3;
    for (int s = 0; s < phases[f]; ++s) {
      auto square = [&](int a, int ea, int b, int eb, int dst, int ed, float alpha, int r, float beta, float diag) {
        p.a = a; p.ea = ea; p.b = b; p.eb = eb; p.dst = dst; p.ed = ed;
        p.alpha = alpha; p.r = r; p.er = 14; p.beta = beta; p.diag = diag;
        return launch_product(g, p, stream);
      };
      const int poly = s == 0 ? q : 2;
      if ((rc = square(0, 14, 0, 14, poly, 14, kC, 0, kB, kA)) != HIVT_OK) return rc;
      if (s > 0) {
        if ((rc = square(poly, 14, q, q_exponent(s), 7 - q, q_exponent(s + 1), 1.0f, -1, 0.0f, 0.0f)) != HIVT_OK) return rc;
        q = 7 - q;
      }
      if (s + 1 < phases[f]) {
        if ((rc = square(poly, 14, 0, 14, 1, 14, 1.0f, -1, 0.0f, 0.0f)) != HIVT_OK) return rc;
        if ((rc = square(1, 14, poly, 14, 0, 14, 1.0f, -1, 0.0f, 0.0f)) != HIVT_OK) return rc;
      }
    }
    memset(&p, 0, sizeof(p));
    p.r = -1;
    p.alpha = 1.0f;
    p.shape = SHAPE_APPLY;
    p.a = q;
    p.ea = q_exponent(phases[f]);
    p.from = at;
    p.to = at ^ 1;
    p.taken = taken;
    p.taken_after = taken + phases[f];
    p.last = f + 1 == nphases;
    if ((rc = launch_product(g, p, stream)) != HIVT_OK) return rc;
    taken += phases[f];
    at ^= 1;
  }
  return HIVT_OK;
}

int check(const char* what, const hivt_matrix* list, int32_t count, int32_t dtype, int32_t steps) {
  HIVT_REQUIRE(count >= 0 && (count == 0 || list != nullptr), HIVT_ERR_ARG, "%s: bad list", what);
  HIVT_REQUIRE(dtype == HIVT_F32 || dtype == HIVT_BF16 || dtype == HIVT_F16, HIVT_ERR_UNSUPPORTED, "%s: element type %d",
               what, (int)dtype);
  HIVT_REQUIRE(steps >= 1 && steps <= 16, HIVT_ERR_ARG, "%s: %d steps (1 to 16)", what, (int)steps);
  for (int32_t i = 0; i < count; ++i)
    HIVT_REQUIRE(list[i].rows >= 0 && list[i].cols >= 0 && list[i].rows <= 65536 && list[i].cols <= 65536, HIVT_ERR_ARG,
                 "%s: matrix %d is %lld x %lld (at most 65536)", what, (int)i, (long long)list[i].rows, (long long)list[i].cols);
  return HIVT_OK;
}

}  // namespace
}  // namespace hivt

using namespace hivt;

extern "C" size_t hivt_orthogonalize_workspace_bytes(const hivt_matrix* list, int32_t count) {
  if (check("hivt_orthogonalize", list, count, HIVT_F32, 1) != HIVT_OK) return 0;
  int64_t total = 0;
  for (int32_t i = 0; i < count; ++i)
    if (list[i].rows > 0 && list[i].cols > 0) total += layout_of((int32_t)list[i].rows, (int32_t)list[i].cols).total;
  return (size_t)total;
}

extern "C" int hivt_orthogonalize(const hivt_matrix* list, int32_t count, int32_t dtype, int32_t steps, float eps,
                                  void* workspace, size_t workspace_bytes, hivt_stream_t stream) {
  const char* what = "hivt_orthogonalize";
  int rc = check(what, list, count, dtype, steps);
  if (rc != HIVT_OK) return rc;
  HIVT_REQUIRE(eps > 0.0f, HIVT_ERR_ARG, "%s: eps must be positive", what);
  const size_t need = hivt_orthogonalize_workspace_bytes(list, count);
  HIVT_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), HIVT_ERR_WORKSPACE,
               "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  for (int32_t i = 0; i < count; ++i)
    HIVT_REQUIRE(list[i].rows * list[i].cols == 0 || (list[i].in && list[i].out), HIVT_ERR_ARG, "%s: null pointer", what);
  // nearly square matrices, wide ones (with phases of up to two or three steps), small ones
  int64_t at = 0;
  for (int kind = 0; kind < 3; ++kind) {
    Phases phases;
    phases.count = 0;
    int left = steps;
    const int most = kind == 0 ? 1 : dtype == HIVT_F32 ? 2 : 3;
    if (left % most != 0) { phases.steps[phases.count++] = left % most; left -= left % most; }
    for (; left > 0; left -= most) phases.steps[phases.count++] = most;
    Group g;
    memset(&g, 0, sizeof(g));
    g.dtype = dtype;
    g.base = static_cast<char*>(workspace);
    g.eps = eps;
    for (int32_t i = 0; i <= count; ++i) {
      if (i < count) {
        const int64_t r = list[i].rows, c = list[i].cols;
        if (r * c == 0) continue;
        if ((small_side(r, c) ? 2 : is_wide(r, c, dtype) ? 1 : 0) != kind) continue;
        Mat& m = g.mats[g.count++];
        m.in = reinterpret_cast<const void*>(list[i].in);
        m.out = reinterpret_cast<void*>(list[i].out);
        m.rows = (int32_t)r;
        m.cols = (int32_t)c;
        m.ws = at;
        at += layout_of(m.rows, m.cols).total;
      }
      if (g.count > 0 && (i == count || g.count == kMats)) {
        rc = run_group(g, phases, kind == 2, steps, (hipStream_t)stream);
        if (rc != HIVT_OK) return rc;
        g.count = 0;
      }
    }
  }
  return HIVT_OK;
}
