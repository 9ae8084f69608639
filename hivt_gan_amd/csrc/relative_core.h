// What the forward and backward kernels of the relative-position attention share: operand types, the tile staging,
// the matrix-core products and the bias of a pair of positions.
//
// Mathematics, for one (batch, head); queries i at position i + offset, keys j at position j:
//   s_ij = scale q_i . k_j + T[bucket(j - (i + offset))][h]          (allowed pairs only: causal rule, key mask)
//   p_ij = exp(s_ij - m_i) / l_i,  o_i = sum_j p_ij v_j
//   delta_i = sum_j p_ij (do_i . v_j),  ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i,  dT[b][h] = sum ds_ij over b
// A bucket depends on the distance alone and does not change beyond distance `sat`, so a tile of keys that lies wholly
// beyond it adds one constant; nearer tiles read the bias of each pair from a table of 2 sat + 1 entries in LDS.
//
// Layout of the products: v_mfma_f32_16x16x{32,16} on 16-bit operands, v_mfma_f32_16x16x4 on fp32 ones, the latter
// issued once per element of the same fragments (the order of the reduction index is free as long as both operands
// agree).  The score tile is computed transposed (rows = keys, columns = queries): a lane then holds four consecutive
// keys of ONE query per 16 x 16 block, so the softmax statistics are per lane and two such blocks are, without any
// movement between lanes, the second operand of the product that reduces over the keys.
#pragma once

#include "common.h"

#include <math.h>
#include <string.h>

namespace hivt {
namespace rel {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxStarts = 127;  // wide buckets of one side
constexpr float kPlainBias = 4096.0f;  // scores keep twelve digits behind the point beside it
constexpr int kMaxSat = 4096;    // distances with an LDS entry of their own, per side

// Arguments of the kernels; strides in elements.
struct Args {
  const void *q, *k, *v, *d_out;
  const float* table;    // [buckets][H]
  const uint8_t* mask;   // [B][N], nonzero: the key is left out; null: none
  void *out, *dq, *dk, *dv;
  float* d_table;        // [buckets][H]
  float2* stats;         // [B * H][M]: (m in the exponent's base-2 units, 1 / l)
  float* delta;          // [B * H][M]
  float* partial;        // forward: split sums; backward: bias-gradient partials
  int64_t q_st[3], k_st[3], v_st[3], o_st[3], do_st[3], dq_st[3], dk_st[3], dv_st[3];  // batch, position, head
  int64_t mask_sb;
  int32_t B, M, N, H, G, d, rep;  // rep = H / G query heads to a key head
  int32_t offset;                 // position of query 0
  int32_t seen;                   // keys that the last query may look at by position: those behind are not read
  int32_t causal, bidirectional;
  int32_t buckets, exact, nstarts, sat;
  int32_t pack;                   // rows of a tile run over (position, head of the group) instead of positions
  int32_t splits, tiles_per_split;
  int32_t q_align, k_align, v_align, do_align, o_align;  // bytes of the widest load the tensor allows (2 .. 16)
  int32_t want_table;
  float scale, scale2;            // scale2 = scale * log2(e)
  int32_t starts[kMaxStarts];
};

// bucket of a distance n >= 0 on one side
__device__ __forceinline__ int side_bucket(const Args& a, int n) {
  if (n < a.exact) return n;
  int b = a.exact;
  for (int t = 0; t < a.nstarts; ++t) b += n >= a.starts[t] ? 1 : 0;
  return b;
}
// bucket of a relative position (key - query); n is clamped by the caller
__device__ __forceinline__ int rel_bucket(const Args& a, int rel) {
  if (!a.bidirectional) return side_bucket(a, rel < 0 ? -rel : 0);
  return rel > 0 ? a.buckets / 2 + side_bucket(a, rel) : side_bucket(a, -rel);
}

// The LDS bias table of one head: relative positions -sat .. hi, and kMargin more on either side that repeat the ends, so
// that a tile that is not wholly beyond them (at most 64 keys and 32 rows, or the reverse) needs no clamping.
constexpr int kMargin = 96;
__host__ __device__ __forceinline__ int bias_hi(const Args& a) { return a.bidirectional ? a.sat : 0; }
__host__ __device__ __forceinline__ int core_width(const Args& a) { return a.sat + 1 + bias_hi(a); }
__host__ __device__ __forceinline__ int bias_width(const Args& a) { return core_width(a) + 2 * kMargin; }
// bucket of entry e of the table
__device__ __forceinline__ int entry_bucket(const Args& a, int e) {
  return rel_bucket(a, min(max(e - kMargin - a.sat, -a.sat), bias_hi(a)));
}

// bias in base-2 exponent units; the type's lowest value stays finite (a row of such biases is a row of equal ones)
__device__ __forceinline__ float bias2(float b) {
  const float x = b * kLog2e;
  return isinf(b) ? b : fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f);
}

__device__ __forceinline__ float fexp2(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- matrix-core products ----------------------------------------------------------------------------------------
// Frag<T, E>: the E reduction elements of a lane (E = 8: reduction length 32, E = 4: 16); acc += A B.
template <typename T, int E> struct Frag;
template <> struct Frag<__bf16, 8> {
  bf16x8 v;
  __device__ __forceinline__ static void mma(const Frag& a, const Frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
  }
};
template <> struct Frag<_Float16, 8> {
  f16x8 v;
  __device__ __forceinline__ static void mma(const Frag& a, const Frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0);
  }
};
template <> struct Frag<__bf16, 4> {
  bf16x4 v;
  __device__ __forceinline__ static void mma(const Frag& a, const Frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a.v), __builtin_bit_cast(s16x4, b.v), c, 0, 0, 0);
  }
};
template <> struct Frag<_Float16, 4> {
  f16x4 v;
  __device__ __forceinline__ static void mma(const Frag& a, const Frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x16f16(a.v, b.v, c, 0, 0, 0);
  }
};
template <int E> struct Frag<float, E> {
  float v __attribute__((ext_vector_type(E)));
  __device__ __forceinline__ static void mma(const Frag& a, const Frag& b, f32x4& c) {
#pragma unroll
    for (int j = 0; j < E; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
  }
};

// ---- tiles in LDS ------------------------------------------------------------------------------------------------
// [row][DP] with 16 bytes of padding: sixteen rows' 16-byte pieces at one column start on sixteen distinct groups of
// four banks.
template <typename T, int DP> struct Tile {
  static constexpr int CH = 16 / (int)sizeof(T);   // elements of a 16-byte piece
  static constexpr int PITCH = DP + CH;
  static constexpr int KS = DP >= 32 ? 32 : 16;    // reduction length of one product over the head width
  static constexpr int E = KS / 4;                 // elements of a lane
  static constexpr int KSTEPS = DP / KS;

  // operand with rows of the tile as output index, head width as reduction: row0 + (lane & 15)
  __device__ static __forceinline__ Frag<T, E> rows(const T* lds, int row0, int ks, int lane) {
    const T* p = lds + (row0 + (lane & 15)) * PITCH + ks * KS + (lane >> 4) * E;
    Frag<T, E> f;
    if constexpr (sizeof(T) * E == 32) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) { f.v[j] = lo[j]; f.v[4 + j] = hi[j]; }
    } else {
      f.v = *reinterpret_cast<const decltype(f.v)*>(p);
    }
    return f;
  }
  // operand with the head width as output index (col0 + (lane & 15)) and 32 rows of the tile as reduction, in the order
  // that two 16 x 16 result blocks hold them: rows row0 + 4 quad + j and row0 + 16 + 4 quad + j, j < 4.
  // 16-bit: the LDS's transposing read delivers four rows of a column per lane; lane l of a group of 16 names the
  // address of row (l >> 2), columns 4 (l & 3) .. + 3.
  __device__ static __forceinline__ Frag<T, 8> cols(const T* lds, int row0, int col0, int lane) {
    Frag<T, 8> f;
    const int quad = lane >> 4, l = lane & 15;
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const T* p = lds + (row0 + 4 * quad + (l >> 2)) * PITCH + col0 + 4 * (l & 3);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 16 * PITCH));
      typedef T t4 __attribute__((ext_vector_type(4)));
      const t4 a = __builtin_bit_cast(t4, lo), b = __builtin_bit_cast(t4, hi);
      f.v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const T* p = lds + (row0 + 4 * quad) * PITCH + col0 + l;
#pragma unroll
      for (int j = 0; j < 4; ++j) { f.v[j] = p[j * PITCH]; f.v[4 + j] = p[(16 + j) * PITCH]; }
    }
    return f;
  }
};

// two 16 x 16 result blocks as the operand that is reduced over their rows, rounded to the operands' type (nearest even)
template <typename T>
__device__ __forceinline__ Frag<T, 8> pair_frag(const f32x4& lo, const f32x4& hi) {
  Frag<T, 8> f;
#pragma unroll
  for (int j = 0; j < 4; ++j) { f.v[j] = (T)lo[j]; f.v[4 + j] = (T)hi[j]; }
  return f;
}

// `n` elements (n * sizeof(T) = 16 bytes) of a row from memory that allows loads of `align` bytes; columns from `left`
// on are zero.
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T* p, int left, int align) {
  uint4 r = make_uint4(0, 0, 0, 0);
  constexpr int CH = 16 / (int)sizeof(T);
  if (align == 16) {
    if (left > 0) r = *reinterpret_cast<const uint4*>(p);  // (the width is a multiple of the piece)
    return r;
  }
  if (align >= 8) {
    uint2 x = make_uint2(0, 0), y = make_uint2(0, 0);
    if (left > 0) x = *reinterpret_cast<const uint2*>(p);
    if (left > CH / 2) y = *reinterpret_cast<const uint2*>(p + CH / 2);
    return make_uint4(x.x, x.y, y.x, y.y);
  }
  if (align >= 4) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (left > i * CH / 4) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  uint32_t w[4] = {0, 0, 0, 0};
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (left > i) w[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A tile of ROWS rows on its way from memory to LDS through registers: NT threads, NPT 16-byte pieces each.
template <typename T, int DP, int ROWS, int NT>
struct Loader {
  static constexpr int CH = 16 / (int)sizeof(T);
  static constexpr int CPR = DP / CH;
  static constexpr int TOTAL = ROWS * CPR;
  static constexpr int NPT = (TOTAL + NT - 1) / NT;
  uint4 r[NPT];

  // keep(row): whether the row of the tile is loaded (zero otherwise), whole: all of them; base: row 0 of the tile.
  // The usual tile, whole and aligned, has a path without a single question per piece (decoder layer of 4096
  // positions: forward 320 -> 311 us, dk and dv 560 -> 523 us).
  template <typename Keep>
  __device__ __forceinline__ void load(const T* base, int64_t stride, int d, int align, int tid, bool whole, Keep keep) {
    if (whole && align == 16 && d == DP) {
#pragma unroll
      for (int i = 0; i < NPT; ++i) {
        const int idx = tid + i * NT;
        if (TOTAL % NT == 0 || idx < TOTAL) r[i] = *reinterpret_cast<const uint4*>(base + (idx / CPR) * stride + (idx % CPR) * CH);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int idx = tid + i * NT;
      const int row = idx / CPR, col = (idx % CPR) * CH;
      r[i] = make_uint4(0, 0, 0, 0);
      if ((TOTAL % NT == 0 || idx < TOTAL) && col < d && keep(row)) r[i] = load_piece(base + row * stride + col, d - col, align);
    }
  }
  __device__ __forceinline__ void store(T* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int idx = tid + i * NT;
      if (TOTAL % NT == 0 || idx < TOTAL)
        *reinterpret_cast<uint4*>(lds + (idx / CPR) * (DP + CH) + (idx % CPR) * CH) = r[i];
    }
  }
};

// operand of a lane straight from memory: `E` consecutive elements of a row, zero beyond the head width
template <typename T, int E>
__device__ __forceinline__ Frag<T, E> load_frag(const T* row, int col, int d, int align, bool keep) {
  Frag<T, E> f;
  constexpr int BYTES = E * (int)sizeof(T);
  if constexpr (BYTES >= 16) {
    uint4 w[BYTES / 16];
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const int c = col + i * (16 / (int)sizeof(T));
      w[i] = keep && c < d ? load_piece(row + c, d - c, align) : make_uint4(0, 0, 0, 0);
    }
    __builtin_memcpy(&f.v, w, BYTES);
  } else {  // four 16-bit elements
    T e[E];
#pragma unroll
    for (int j = 0; j < E; ++j) e[j] = keep && col + j < d ? row[col + j] : (T)0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) f.v[j] = e[j];
  }
  return f;
}

// four consecutive columns of a result row
template <typename T>
__device__ __forceinline__ void store4(T* row, int col, int d, const f32x4& v) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  if ((d & 3) == 0 && ((reinterpret_cast<uintptr_t>(row) & (4 * sizeof(T) - 1)) == 0)) {
    if (col < d) {
      t4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (T)v[j];
      *reinterpret_cast<t4*>(row + col) = w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (col + j < d) row[col + j] = (T)v[j];
}

// Keys of a tile of 64 that may be looked at: bit j = key k0 + j is seen by some position and not masked.  Uniform over the wave.
__device__ __forceinline__ uint64_t tile_keys(const Args& a, int b, int k0, int lane) {
  const int key = k0 + lane;
  bool ok = key < a.seen;
  if (ok && a.mask != nullptr) ok = a.mask[(int64_t)b * a.mask_sb + key] == 0;
  return __ballot(ok);
}

// maximum / sum over the four lanes that hold one query of a transposed score tile
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// Workgroups of one outer unit (a batch and head: its tiles read the same keys) share an XCD's L2: ids are dealt
// round-robin over eight XCDs, so eight outer units are walked together.
__device__ __forceinline__ void walk(int linear, int outer_count, int inner_count, int& outer, int& inner) {
  const int grouped = outer_count / 8 * 8 * inner_count;
  if (linear < grouped) {
    const int rem = linear % (8 * inner_count);
    outer = linear / (8 * inner_count) * 8 + rem % 8;
    inner = rem / 8;
  } else {
    outer = outer_count / 8 * 8 + (linear - grouped) / inner_count;
    inner = (linear - grouped) % inner_count;
  }
}

// relative_attn_short.hip: which problems it takes, and its launches
bool short_fwd_route(const Args& a);
bool short_bwd_route(const Args& a);
int short_slots(const Args& a);
int short_fwd(const Args& a, int dtype, hipStream_t stream);
int short_bwd(const Args& a, int dtype, int slots, float* partial, hipStream_t stream);

// relative_attn_fwd.hip: the checked arguments of an entry point
int from_public(const char* what, const hivt_relative_attn* p, const int32_t* starts, float scale, Args& a);

}  // namespace rel
}  // namespace hivt
