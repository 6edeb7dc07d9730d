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
  uint32_t g_factor;  // r / G = r g_factor >> g_shift for 0 <= r < 2^31
  int g_shift;
  char* out;      // (batch, T, Hk G, Dv)
  char* second;   // like out: the second map's values, for the backward pass; NULL: none
  // (2, batch, Hk, 2, T G): log2 of the sums of 2^((score - top) c), +inf for a row that sees
  // nothing; then top, the largest scores (as products of q and k, not scaled).
  float* lse;
  int blocks;     // workgroups of one (batch, key head), apart from splits
  int splits, each;  // the other side's entries of a split (a whole number of tiles)
  float* part;    // sums of each split, joined by a second launch
  // backward
  const char* g;
  int64_t g_b, g_t, g_h;
  float* delta;   // (batch, Hk, 2, T G): g . o_m
  int row_splits;
  char* records;  // (batch, Hk, T G): lse and delta of both maps as diff_grad_keys reads them
  uint8_t* takes_part;  // (batch, Hk, T G): 1 where the row sees a key, 3 where its scores are large besides
  float* off;     // 16 bits: (row splits, batch, Hk, 2, T G): how far delta was off, in parts
  float* most;    // fp16: (batch, Hk, 2): largest norms of g's rows and of v's, squared
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

// Which of n groups (batch, key head, split) and of their `blocks` a workgroup takes: block 0
// has the most work.  A group's workgroups run on one die where the groups can be dealt out
// evenly, the heaviest blocks of all its groups first, every other round of a die's 32 CUs
// backwards: two workgroups that share a CU then have a heavy block and a light one.
__device__ __forceinline__ void deal(int n, int blocks, int* group, int* block) {
  const bool even = n % kXcds == 0;
  const int id = blockIdx.x, die = even ? id % kXcds : 0, per = even ? n / kXcds : n;
  const int slots = even ? 32 : 256, all = per * blocks;
  int i = even ? id / kXcds : id;
  const int round = i / slots;
  if (round & 1) i = round * slots + min((round + 1) * slots, all) - 1 - i;
  *block = i / per;
  *group = die * per + (i - *block * per);
}

__device__ __forceinline__ int token_of(const Args& a, int r) {
  return (int)((uint64_t)(uint32_t)r * a.g_factor >> a.g_shift);
}

// Largest scores `top` and the rest apart, as a difference of large numbers is formed before it is
// rounded: of maps that are one key, or a few with equal scores, nothing else would be left.
__device__ __forceinline__ int64_t tops_at(const Args& a) { return (int64_t)a.batch * a.Hk * 2 * a.T * a.G; }

__device__ __forceinline__ float lam_of(const Args& a, int h) {
  const int64_t at = h * a.lam_stride;
  return a.lam_dtype == DA_F32 ? Elem<DA_F32>::load(a.lam, at)
         : a.lam_dtype == DA_BF16 ? Elem<DA_BF16>::load(a.lam, at) : Elem<DA_F16>::load(a.lam, at);
}

// Entries e0 .. e0 + V of a row of d entries, d a multiple of V.
template <int DT>
__device__ __forceinline__ u32x4 load_run(const char* row, int e0, int d) {
  return e0 < d ? ld16(row + e0 * Type<DT>::ES) : u32x4{0, 0, 0, 0};
}

// Four entries e0 .. e0 + 3 of a row of d, a multiple of four, rounded once.
template <int DT>
__device__ __forceinline__ void store4(char* row, int e0, int d, float f0, float f1, float f2, float f3) {
  if (e0 >= d) return;
  if constexpr (DT == DA_F32) *(f32x4*)(row + e0 * 4) = f32x4{f0, f1, f2, f3};
  else *(u32x2*)(row + e0 * 2) = u32x2{pack2<DT>(f0, f1), pack2<DT>(f2, f3)};
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

// A tile of kTile rows of W entries, read straight into LDS by NT threads: 16 bytes a lane,
// nothing in registers on the way.  A lane's place in LDS is fixed, so the swizzle is in what
// it reads; a row that takes no part, and entries past d, read as zeros and touch no memory.
constexpr uint32_t kOutside = 0x80000000u;  // past the range of any buffer here

template <int DT, int W, int NT>
struct Tile {
  static constexpr int kRow = W * Type<DT>::ES, kPer = kRow / 16, kBytes = kTile * kRow;
  static constexpr int N = kTile * kPer / NT;
  static_assert(N * NT == kTile * kPer, "whole chunks a thread");
  __device__ __forceinline__ static int row(int i) { return (threadIdx.x + i * NT) / kPer; }
  __device__ __forceinline__ static uint32_t column(int i, int d) {  // in bytes
    const int at = threadIdx.x + i * NT, c = (at % kPer) ^ swizzle<kRow>(at / kPer);
    return c * Type<DT>::V < d ? c * 16 : kOutside;
  }
  __device__ __forceinline__ static void issue(u32x4 rsrc, uint32_t lds, int i, uint32_t offset) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63u);
    dma16(rsrc, lds + (wave + i * NT) * 16, offset);
  }
};

// Tiles of consecutive rows (keys): a lane's offsets are the same in every tile.
template <int DT, int W, int NT>
struct Keys : Tile<DT, W, NT> {
  using T = Tile<DT, W, NT>;
  uint32_t at[T::N];
  __device__ __forceinline__ Keys(int64_t stride, int d) {
#pragma unroll
    for (int i = 0; i < T::N; ++i) {
      const uint32_t c = T::column(i, d);
      at[i] = c == kOutside ? kOutside : (uint32_t)(T::row(i) * stride * Type<DT>::ES) + c;
    }
  }
  // `base`: the tile's first row; `live`: a bit a row
  __device__ __forceinline__ void fetch(const char* base, uint32_t lds, uint32_t live) const {
    const u32x4 rsrc = uniform4(make_rsrc(base, kOutside - 1));
#pragma unroll
    for (int i = 0; i < T::N; ++i)
      T::issue(rsrc, lds, i, (live >> T::row(i) & 1) ? at[i] : kOutside);
  }
};

// Tiles of rows r = t G + g: heads of one token are `head` apart, tokens `token` (bytes).
// Where G divides a tile, a lane's offsets from the tile's first token are the same in every
// tile that starts at a whole one.
template <int DT, int W, int NT>
struct Rows : Tile<DT, W, NT> {
  using T = Tile<DT, W, NT>;
  __device__ __forceinline__ static void place(const Args& a, int r0, uint32_t token, uint32_t head, int d,
                                               uint32_t* at) {
    const int t0 = token_of(a, r0);
#pragma unroll
    for (int i = 0; i < T::N; ++i) {
      const int r = r0 + T::row(i), t = token_of(a, r);
      const uint32_t c = T::column(i, d);
      at[i] = c == kOutside ? kOutside : (uint32_t)(t - t0) * token + (uint32_t)(r - t * a.G) * head + c;
    }
  }
  // `base`: the first head of the tile's first token; `thread`: the thread's number
  __device__ __forceinline__ static void fetch(const char* base, uint32_t lds, const uint32_t* at, uint32_t live,
                                               int thread) {
    const u32x4 rsrc = uniform4(make_rsrc(base, kOutside - 1));
#pragma unroll
    for (int i = 0; i < T::N; ++i)
      T::issue(rsrc, lds, i, live >> ((thread + i * NT) / T::kPer) & 1 ? at[i] : kOutside);
  }
};

// A barrier that the tiles under way have to reach first: the compiler does not count their
// loads, and its own barrier waits for none of them.
__device__ __forceinline__ void tiles_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ uint32_t lds_address(const char* p) { return (uint32_t)(uintptr_t)(const lds_char*)p; }
__device__ __forceinline__ u32x4 lds16(uint32_t at) {
  return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)at;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Where a lane reads tiles of W entries.  A chunk's place is its number xor the row's
// swizzle, so that of all chunks which one lane reads differ from one register by a constant:
// xor in the bits that are swizzled (16 .. 240 bytes), else added.
template <int DT, int W>
struct Reader {
  static constexpr int kRow = W * Type<DT>::ES;
  uint32_t of_rows, of_columns;
  __device__ __forceinline__ Reader(const char* lds, int lane) {
    const uint32_t base = lds_address(lds), half = lane >> 5;
    const int row = lane & 31;
    of_rows = base + row * kRow + ((half ^ swizzle<kRow>(row)) << 4);
    if constexpr (DT == DA_F32) {
      const int col = lane & 31;
      of_columns = base + 4 * half * kRow + (((col >> 2) ^ half) << 4) + (col & 3) * 4;
    } else {
      const int i = lane & 15, r = 4 * half + i / 4, c = (lane >> 4 & 1) * 2 + (i & 3) / 2;
      of_columns = base + r * kRow + ((c ^ swizzle<kRow>(r)) << 4) + (i & 1) * 8;
    }
  }
  // The registers as they stand in the tile of `key`: else sums with every constant are kept
  // over the loop instead, and fill the registers.
  __device__ __forceinline__ Reader fresh(int key) const {
    Reader r = *this;
    asm("" : "+v"(r.of_rows) : "s"(key));
    asm("" : "+v"(r.of_columns) : "s"(key));
    return r;
  }
  // Operand chunk kk of the tile `skip` bytes on, by rows: lane l has row l % 32, the entries of
  // its half.
  __device__ __forceinline__ u32x4 rows(int skip, int kk) const {
    const uint32_t c = kk << 5;
    return lds16((of_rows ^ (c & 0xf0)) + (c & ~0xf0u) + skip);
  }
  // Operand chunk j transposed: lane l has column 32 n + l % 32, at the rows that registers of
  // an accumulator hold in the same half, those of chunk j.
  __device__ __forceinline__ u32x4 columns(int skip, int n, int j) const {
    if constexpr (DT == DA_F32) {
      u32x4 v;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t c = n << 7 ^ s << 6 ^ (j & 1) << 5;
        v[s] = *(const __attribute__((address_space(3))) uint32_t*)(uintptr_t)(
            (of_columns ^ (c & 0xf0)) + (c & ~0xf0u) + skip + (8 * j + s) * kRow);
      }
      return v;
    } else {
      // ds_read_b64_tr_b16: of 16 lanes, lane i addresses four columns (i % 4) of row i / 4
      // and receives four rows of column i.
      u32x2 part[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t c = n << 6 ^ s << 5;
        part[s] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(uintptr_t)(
                (of_columns ^ (c & 0xf0)) + (c & ~0xf0u) + skip + (16 * j + 8 * s) * kRow)));
      }
      return u32x4{part[0][0], part[0][1], part[1][0], part[1][1]};
    }
  }
};

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

// What rounding to operand chunk j left, rounded in turn.
template <int DT>
__device__ __forceinline__ u32x4 rest_of(const f32x16& x, int j, u32x4 p) {
  u32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    v[k] = pack2<DT>(x[8 * j + 2 * k] - Elem<DT>::from_bits(p[k] & 0xffffu),
                     x[8 * j + 2 * k + 1] - Elem<DT>::from_bits(p[k] >> 16));
  return v;
}

// The other half's value: lane l's of lane l ^ 32.
__device__ __forceinline__ float other_half(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(__lane_id() < 32 ? x[1] : x[0]);
}

// Over an accumulator's registers, in a tree.
template <class Op>
__device__ __forceinline__ float over_acc(const f32x16& x, Op op) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = op(x[i], x[i + 8]);
#pragma unroll
  for (int n = 4; n > 0; n /= 2)
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = op(v[i], v[i + n]);
  return v[0];
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

// Of a tile's live keys, a bit each, those up to `last`: shifted so that the lane's half has
// its row x at bit acc_at(x, 0).
__device__ __forceinline__ uint32_t seen_of(uint32_t word, int key, int last, int half) {
  const int n = last - key;  // the last one seen
  const uint32_t upto = n >= 31 ? ~0u : n < 0 ? 0u : (2u << n) - 1u;
  return (word & upto) >> (4 * half);
}

// Goes over the tiles that have a live key: their first key, and a bit a key (0: no more).
struct Live {
  int key, byte;
  uint32_t word;
  __device__ __forceinline__ Live(const Args& a, int b, int first, int end, int lane) {
    key = first - kTile;
    byte = key_byte(a, b, first, end, lane);
    next(a, b, end, lane);
  }
  __device__ __forceinline__ void next(const Args& a, int b, int end, int lane) {
    do {
      key += kTile;
      word = key < end ? key_word(byte) : 0;
      byte = key_byte(a, b, key + kTile, end, lane);
    } while (!word && key < end);
  }
};

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
int fill_args(Args& a, const char* what, int dtype, const da_diff_inputs* in, int64_t batch, int64_t T, int64_t S, int64_t heads,
              int64_t k_heads, int64_t D, int64_t Dv, float scale, int causal, int64_t q_start);
// Whether one operand's rows can be read as the kernels do.
int check_side(const char* what, const char* name, const void* x, int es, int64_t width, int64_t tokens, int64_t heads,
               int64_t bs, int64_t ts, int64_t hs);
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
