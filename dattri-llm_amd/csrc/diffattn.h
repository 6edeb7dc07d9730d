// What the kernels of difference attention share: rows, tiles in LDS, operands of the
// matrix instructions.
//
// The G query heads of one key head are read as one matrix of rows r = t G + g, so that a
// tile of keys is read once for all of them, and a single new token fills G rows of a tile.
#pragma once

#include <type_traits>

#include "common.h"

namespace da {
namespace diff {

constexpr int kTile = 32;  // rows or keys of a tile: one 32 x 32 matrix instruction
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLowest = -3.4028234663852886e38f;

struct Args {
  const char *q, *k, *v;
  const void* lam;
  int lam_dtype;
  int64_t lam_stride;
  const uint8_t *mask, *q_mask;  // keys (batch, S), queries (batch, T)
  int64_t q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h;  // elements
  int64_t m_b, m_k, qm_b, qm_t;
  int batch, T, S, Hk, G, D, Dv;
  int causal;
  int64_t q_start;
  float scale;
  char* out;      // (batch, T, Hk G, Dv)
  char* second;   // like out: the second map's values, for the backward pass; NULL: none
  float* lse;     // (batch, Hk, 2, T G): log2 of the exponentials' sums; +inf for a row that sees nothing
  int splits, split_keys, row_blocks;
  float* part;    // (splits, batch, Hk, T G, 2, DVP + 2): values, maximum, sum of each part
  // backward
  const char* g;
  int64_t g_b, g_t, g_h;
  float* delta;   // (batch, Hk, 2, T G): g . o_m
  float* most;    // largest |g| of the call (16-bit floats of five exponent bits), NULL: not needed
  char *dq, *dk, *dv;
  float* lam_part;  // (batch, heads, chunks)
  int chunk, chunks;
};

template <int DT>
struct Type {
  static constexpr int ES = Elem<DT>::kBytes, V = Elem<DT>::kVec;
  static constexpr int kStep = 2 * V;             // contracted entries of one pair of chunks
  static constexpr int kChunks = kTile / kStep;   // chunks of a tile contracted over its rows
};

__device__ __forceinline__ float lam_of(const Args& a, int h) {
  const int64_t at = h * a.lam_stride;
  return a.lam_dtype == DA_F32 ? Elem<DA_F32>::load(a.lam, at)
         : a.lam_dtype == DA_BF16 ? Elem<DA_BF16>::load(a.lam, at) : Elem<DA_F16>::load(a.lam, at);
}

// Entries e0 .. e0 + V of a row of d entries, from any address; zeros past its end, not read.
template <int DT>
__device__ __forceinline__ u32x4 load_run(const char* row, int e0, int d) {
  constexpr int ES = Type<DT>::ES, V = Type<DT>::V;
  if (e0 + V <= d) return ld16_any<ES>(row + e0 * ES);
  u32x4 v = {0, 0, 0, 0};
  if (e0 >= d) return v;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (e0 + e >= d) continue;
    if constexpr (ES == 4) v[e] = *(const uint32_t*)(row + (e0 + e) * 4);
    else v[e / 2] |= (uint32_t)(*(const uint16_t*)(row + (e0 + e) * 2)) << (16 * (e % 2));
  }
  return v;
}

// Four entries e0 .. e0 + 3 of a row of d, rounded once.
template <int DT>
__device__ __forceinline__ void store4(char* row, int e0, int d, float f0, float f1, float f2, float f3) {
  constexpr int ES = Type<DT>::ES;
  if (e0 >= d) return;
  if (e0 + 4 <= d) {
    if constexpr (ES == 4) {
      st16_any<4>(row + e0 * 4, u32x4{__float_as_uint(f0), __float_as_uint(f1), __float_as_uint(f2), __float_as_uint(f3)});
    } else {
      typedef uint32_t u32x2_at2 __attribute__((ext_vector_type(2), aligned(2)));
      *(u32x2_at2*)(row + e0 * 2) = u32x2_at2{pack2<DT>(f0, f1), pack2<DT>(f2, f3)};
    }
    return;
  }
  Elem<DT>::store(row, e0, f0);
  if (e0 + 1 < d) Elem<DT>::store(row, e0 + 1, f1);
  if (e0 + 2 < d) Elem<DT>::store(row, e0 + 2, f2);
}

// Chunk (16 bytes) c of row r of a tile lies at place c ^ swizzle(r) of its row.  Read by
// rows (32 rows, one chunk each) and transposed (4 rows, 64 bytes each), either way the
// lanes that are served together use every bank once.
template <int kRowBytes>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (kRowBytes >= 256) return (r & 3) << 2 | (r >> 2 & 3);
  else if constexpr (kRowBytes == 128) return (r >> 1 & 1) << 2 | (r >> 2 & 3);
  else return r >> 2 & 3;
}

// A tile of kTile rows of W entries on its way from memory to LDS, over NT threads.
template <int DT, int W, int NT>
struct Tile {
  static constexpr int kRow = W * Type<DT>::ES, kPer = kRow / 16, kBytes = kTile * kRow;
  static constexpr int N = kTile * kPer / NT;
  static_assert(N * NT == kTile * kPer, "whole chunks a thread");
  u32x4 r[N];
  // row(i): where row i starts, NULL: a row of zeros
  template <class F>
  __device__ __forceinline__ void fetch(F row, int d) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + i * NT;
      const char* p = row(at / kPer);
      r[i] = p ? load_run<DT>(p, at % kPer * Type<DT>::V, d) : u32x4{0, 0, 0, 0};
    }
  }
  // `live`: a bit a row; the others are stored as zeros, whatever was read
  __device__ __forceinline__ void put(char* lds, uint32_t live) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + i * NT, row = at / kPer, c = at % kPer;
      const uint32_t keep = (live >> row & 1) ? ~0u : 0u;
      st16(lds + row * kRow + ((c ^ swizzle<kRow>(row)) << 4), r[i] & u32x4{keep, keep, keep, keep});
    }
  }
};

// Operand chunk kk of a tile read by rows: lane l has row l % 32, the entries of its half.
template <int DT, int W>
__device__ __forceinline__ u32x4 by_rows(const char* lds, int kk, int lane) {
  constexpr int kRow = W * Type<DT>::ES;
  const int row = lane & 31, c = 2 * kk + (lane >> 5);
  return ld16(lds + row * kRow + ((c ^ swizzle<kRow>(row)) << 4));
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Operand chunk j of a tile read transposed: lane l has column 32 block + l % 32, at the
// rows that registers of an accumulator hold in the same half: those of chunk j.
template <int DT, int W>
__device__ __forceinline__ u32x4 by_columns(const char* lds, int block, int j, int lane) {
  constexpr int kRow = W * Type<DT>::ES;
  const int half = lane >> 5;
  if constexpr (DT == DA_F32) {
    const int col = 32 * block + (lane & 31), c = col >> 2;
    u32x4 v;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int row = 8 * j + 4 * half + s;
      v[s] = *(const uint32_t*)(lds + row * kRow + ((c ^ swizzle<kRow>(row)) << 4) + (col & 3) * 4);
    }
    return v;
  } else {
    // ds_read_b64_tr_b16: of 16 lanes, lane i addresses four columns (i % 4) of row i / 4
    // and receives four rows of column i.
    const int i = lane & 15, c = 4 * block + (lane >> 4 & 1) * 2 + (i & 3) / 2;
    u32x2 part[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int row = 16 * j + 8 * s + 4 * half + i / 4;
      const char* p = lds + row * kRow + ((c ^ swizzle<kRow>(row)) << 4) + (i & 1) * 8;
      part[s] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(const lds_char*)p));
    }
    return u32x4{part[0][0], part[0][1], part[1][0], part[1][1]};
  }
}

// Operand chunk j from an accumulator's registers: the other operand of by_columns.
template <int DT>
__device__ __forceinline__ u32x4 from_acc(const f32x16& x, int j) {
  u32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (DT == DA_F32) v[k] = __float_as_uint(x[4 * j + k]);
    else v[k] = pack2<DT>(x[8 * j + 2 * k], x[8 * j + 2 * k + 1]);
  }
  return v;
}

// Row r of an accumulator's registers within its tile.
__device__ __forceinline__ int acc_at(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

__device__ __forceinline__ f32x16 zeros() {
  f32x16 v;
#pragma unroll
  for (int r = 0; r < 16; ++r) v[r] = 0.f;
  return v;
}

// Bits of the live keys among k0 .. k0 + 31, the same in every wave.
__device__ __forceinline__ int key_byte(const Args& a, int b, int k0, int end, int lane) {
  const int key = k0 + (lane & 31);
  return key < end ? (a.mask ? a.mask[b * a.m_b + key * a.m_k] : 1) : 0;
}
__device__ __forceinline__ uint32_t key_word(int byte) { return (uint32_t)__ballot(byte != 0); }

// The last key that row r sees (-1: none, also for a row that takes no part).
__device__ __forceinline__ int last_key(const Args& a, int b, int t) {
  if (t >= a.T || (a.q_mask && !a.q_mask[b * a.qm_b + t * a.qm_t])) return -1;
  if (!a.causal) return a.S - 1;
  const int64_t last = t + a.q_start;
  return last < -1 ? -1 : last >= a.S ? a.S - 1 : (int)last;
}

// ---------------------------------------------------------------------------
// Host side (defined in diffattn.hip).
// ---------------------------------------------------------------------------
int check_sizes(const char* what, int dtype, int64_t batch, int64_t T, int64_t S, int64_t heads, int64_t k_heads,
                int64_t D, int64_t Dv, int64_t q_start);
int fill_args(Args& a, const char* what, const da_diff_inputs* in, int64_t batch, int64_t T, int64_t S, int64_t heads,
              int64_t k_heads, int64_t D, int64_t Dv, float scale, int causal, int64_t q_start);
// Dynamic LDS past 64 KB has to be asked for.
int allow_lds(const void* kernel, int bytes);
// The least kernel widths that hold D and Dv: an index of by_widths.
int widths(int64_t D, int64_t Dv);

template <class F>
int by_widths(int dtype, int w, F f) {
#define DA_W(DT)                                                                                         \
  switch (w) {                                                                                           \
    case 0: return f(std::integral_constant<int, DT>{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 64>{});    \
    case 1: return f(std::integral_constant<int, DT>{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 128>{});   \
    case 2: return f(std::integral_constant<int, DT>{}, std::integral_constant<int, 128>{}, std::integral_constant<int, 128>{});  \
    default: return f(std::integral_constant<int, DT>{}, std::integral_constant<int, 128>{}, std::integral_constant<int, 256>{}); \
  }
  if (dtype == DA_BF16) DA_W(DA_BF16)
  if (dtype == DA_F16) DA_W(DA_F16)
  DA_W(DA_F32)
#undef DA_W
}

}  // namespace diff
}  // namespace da
