// A learned relative position bias by buckets, and its per-sample gradient.
//
//   bias[h,i,j] = table[bucket(j - i - start), h]
//   dtable[b,v,h] = sum of g[b,h,i,j] over the live (i, j) with bucket(j - i - start) = v
//
// The bucket depends on the offset o = j - i - start alone: with r = |o|
// (bidirectional) or max(-o, 0), it is the last x whose least distance edges[x]
// is at most r, plus n (the buckets of one side) where bidirectional and o > 0.
// The edges are integers worked out by the caller, so that no logarithm decides
// which side of a border a distance falls on.  With `causal`, keys after their
// query are no part of the attention: the bias is -inf there, and whatever g holds
// there adds nothing.
#include <algorithm>

#include "common.h"

namespace da {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBuckets = 256;

struct Edges {
  int n;      // buckets of one side
  int both;   // bidirectional
  int32_t least[kMaxBuckets];
};

__device__ __forceinline__ int bucket_of(const int* least, int n, int both, int o) {
  const int r = o < 0 ? -o : both ? o : 0;
  int lo = 0, hi = n;  // least[lo] <= r < least[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (least[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo + (both && o > 0 ? n : 0);
}

// With V entries in 16 bytes, rows and columns are taken in blocks of V: the square
// of row block r and column block c holds the offsets of diagonal block k = c - r,
// whatever r.  All accesses are aligned runs of 16 bytes.
//
// Rows need not be aligned: entry j of row i is at address mis + i stride + j
// (modulo V; mis that of the plane's first entry), so with R = stride mod V the
// aligned run of row rV + e in column block c starts at column c V - mis -
// shift(e), shift(e) = e R mod V, and 3V - 2 offsets k V - mis + [-2 (V - 1), V - 1]
// cover a diagonal block for every R.  In the backward pass R is a template
// argument: all indices into a lane's sums are constants.
template <int V, int R>
struct Walk {
  __host__ __device__ static constexpr int shift(int e) { return e * R % V; }
  __host__ __device__ static constexpr int at(int e, int x) { return x - e - shift(e) + 2 * (V - 1); }
  __host__ __device__ static constexpr int end(bool last) {
    int t = last ? 0 : 3 * V;
    for (int e = 0; e < V; ++e) {
      const int u = at(e, last ? V - 1 : 0);
      if (last ? u > t : u < t) t = u;
    }
    return t;
  }
  static constexpr int kFirst = end(false), kLast = end(true);  // the places in use
  // Bit x: a run may reach column first - (V - 1) + x (first: of an unshifted run).
  __host__ __device__ static constexpr int columns() {
    int bits = 0;
    for (int e = 0; e < V; ++e) bits |= ((1 << V) - 1) << (V - 1 - shift(e));
    return bits;
  }
};

// Offsets o that belong to a bucket: one range each.
__device__ __forceinline__ void bucket_range(const Edges& e, int x, int* lo, int* hi) {
  const int side = x < e.n ? 0 : 1, at = x - side * e.n;
  const int first = e.least[at], next = at + 1 < e.n ? e.least[at + 1] : 0x40000000;  // past every distance
  if (side) {
    *lo = max(first, 1);
    *hi = next - 1;
  } else {
    *lo = 1 - next;
    *hi = !e.both && first == 0 && next > 0 ? 0x3fffffff : -first;  // later offsets: the last bucket from 0 on
  }
}

struct BiasArgs {
  const char* table;
  char* out;
  int64_t q_len, k_len;
  int64_t t_b, t_h;  // table strides in elements
  int start, causal;
  int columns, windows, steps;  // column blocks, windows of kWave of them; row blocks of a workgroup
  int spread;                   // runs that a row may be ahead of its line: 7, or 0 where all rows start one
  uint32_t closed;              // bits of -inf
};

template <int ES>
__device__ __forceinline__ uint32_t load_bits(const char* p, int64_t i) {
  if constexpr (ES == 4) return ((const uint32_t*)p)[i];
  else return ((const uint16_t*)p)[i];
}
template <int ES>
__device__ __forceinline__ void store_bits(char* p, int64_t i, uint32_t v) {
  if constexpr (ES == 4) ((uint32_t*)p)[i] = v;
  else ((uint16_t*)p)[i] = (uint16_t)v;
}

// A workgroup writes one head's entries of up to 64 column blocks and `steps` row
// blocks.  The run of row rV + e in column block c depends on e and on c - r alone:
// the runs of all diagonal blocks lie ready in LDS, one array for each e, and a
// store is one 16-byte LDS read (neighbouring lanes read neighbours) and one
// aligned 16-byte write.  Each row's columns are shifted so that a wave's 64 runs
// are whole 128-byte lines: a line that two workgroups write in parts goes to memory
// twice (32 x 2047 x 2047 bf16: 84 us unshifted, 72 us so).  Runs that a row's end
// cuts are written entry by entry at the end.
//
// Bound by the writes: 32 x 2048 x 2048 bf16 takes 48 us into one buffer, 55 us into
// alternating ones (5.6 and 4.9 TB/s; a kernel that only fills memory 5.3 to 5.6).
// With the runs in the lanes' registers, lanes on fixed diagonals, it took 86 us: a
// wave's columns then start at any run, and every line is written in parts.
template <int ES>
__global__ __launch_bounds__(kThreads) void bias_forward(BiasArgs a, Edges e) {
  constexpr int V = 16 / ES;
  extern __shared__ u32x4 runs[];  // [V][blocks], then the line of single values
  __shared__ int least[kMaxBuckets];
  __shared__ uint32_t column[kMaxBuckets];
  const int tid = threadIdx.x;
  const int window = blockIdx.x % a.windows, r0 = blockIdx.x / a.windows * a.steps;
  const int64_t h = blockIdx.y;
  char* plane = a.out + h * a.q_len * a.k_len * ES;
  const int mis = (int)((uintptr_t)plane / ES % V);
  const int k_len = (int)a.k_len, i0 = r0 * V, rows = (int)min((int64_t)a.steps * V, a.q_len - i0);
  const int c0 = window * kWave, width = min(kWave, a.columns + a.spread - c0);
  // Diagonal blocks, the first of them: a row's column blocks start up to `spread` before c0.
  const int blocks = width + a.steps - 1 + a.spread, k0 = c0 - a.spread - (r0 + a.steps - 1);
  uint32_t* line = (uint32_t*)(runs + V * blocks);
  if (tid < e.n) least[tid] = e.least[tid];
  if (tid < (e.both ? 2 : 1) * e.n) column[tid] = load_bits<ES>(a.table, tid * a.t_b + h * a.t_h);
  __syncthreads();
  for (int p = tid; p < (blocks + 2) * V; p += kThreads) {
    const int o = k0 * V + p - 2 * (V - 1) - mis - a.start;
    line[p] = a.causal && o > 0 ? a.closed : column[bucket_of(least, e.n, e.both, o)];
  }
  __syncthreads();
  const int stride = k_len % V;
  // Runs from a line's start to column block 0 of row i (whole lines are a power of
  // two long: the product may wrap).
  const uint32_t base = (uint32_t)((uintptr_t)plane / 16);
  auto ahead = [&](int i, int shift) {
    return (int)((base + ((uint32_t)(i0 + i) * (uint32_t)k_len - (uint32_t)shift) / V) & (uint32_t)a.spread);
  };
  for (int n = tid; n < min(rows, V) * blocks; n += kThreads) {
    const int r = n / blocks, k = n - r * blocks;
    const uint32_t* at = line + k * V + 2 * (V - 1) - r - r * stride % V;
    u32x4 run;
#pragma unroll
    for (int q = 0; q < 4; ++q) run[q] = ES == 4 ? at[q] : at[2 * q] | at[2 * q + 1] << 16;
    runs[n] = run;
  }
  __syncthreads();
  const int together = kThreads / width;  // rows that the workgroup writes at once
  const int c = tid % width;
  if (tid < together * width)
    for (int i = tid / width; i < rows; i += together) {
      const int r = i % V, shift = r * stride % V, at = c - ahead(i, shift), j = (c0 + at) * V - mis - shift;
      if (j >= 0 && j + V <= k_len)
        st16(plane + ((int64_t)(i0 + i) * k_len + j) * ES, runs[r * blocks + at + a.spread + a.steps - 1 - i / V]);
    }
  if (stride == 0 && mis == 0) return;
  for (int n = tid; n < rows * 2 * V; n += kThreads) {  // the first and the last run of each row
    const int i = n / (2 * V), x = n % V, r = i % V, shift = r * stride % V;
    const int head = (mis + shift) / V, tail = (k_len - 1 + mis + shift) / V;  // their column blocks
    const bool second = n % (2 * V) >= V;
    if (second && tail == head) continue;  // one run is both
    const int at = (second ? tail : head) - c0, first = (c0 + at) * V - mis - shift, j = first + x;
    if (first >= 0 && first + V <= k_len) continue;  // a whole run
    const int c = at + ahead(i, shift);
    if (j >= 0 && j < k_len && c >= 0 && c < width)
      store_bits<ES>(plane, (int64_t)(i0 + i) * k_len + j,
                     line[(at + a.spread + a.steps - 1 - i / V) * V + 2 * (V - 1) - r - shift + x]);
  }
}

struct GradArgs {
  const char* g;
  const uint8_t* mask;  // (batch, k_len): query i is position i + start; NULL: all live
  float* partial;       // (batch, heads, blocks, buckets)
  float* out;           // (batch, buckets, heads)
  int64_t heads, q_len, k_len;
  int64_t g_b, g_h, g_i;  // elements
  int64_t mask_b, mask_k;
  int64_t blocks;  // workgroups of a plane
  int buckets, start, causal;
  int row_blocks, last_block;  // row blocks; the last diagonal block that counts
  int windows, steps;          // groups of column blocks; row blocks of a group
};

// Row blocks of a group of lanes at most: its sums lie in LDS.
__host__ __device__ constexpr int max_steps(int group) { return group == 64 ? 64 : 16; }

constexpr int kGroups = 4;  // of a team
// Row blocks whose loads are in flight.  Four instead of two: 27 us instead of 25 for
// 48 causal planes of 777 x 777 in fp32 (more registers, steps rounded up further).
constexpr int kAhead = 2;

__device__ const u32x4 kZeros = {0, 0, 0, 0};

// Whole-wave (kG 64) or row-of-16 shift by one lane: lane l takes lane l - 1's
// value, the first lane of a group zero.
template <int kG>
__device__ __forceinline__ float from_left(float v) {
  constexpr int kCtrl = kG == 64 ? 0x138 : 0x111;  // wave_shr:1, row_shr:1
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), kCtrl, 0xf, 0xf, false));
}

// A group of kG lanes owns kG column blocks and walks down `steps` row blocks of
// one plane.  A lane's column stays while its diagonal moves one block left with
// each row block, so its sums move one lane right: every load of the walk is
// whole lines, all lanes work, and all groups alike.  The sums of the diagonal
// block that leaves at the last lane go to its slot in LDS, at the end those of
// all lanes.  An offset lies in up to three slots of each group; their sums form a
// line, and sixteen lanes sum a bucket's range of it.  Four groups are a team: with
// groups of 16 (narrow planes) a wave is a team, and four heads share a workgroup.
//
// Bound by HBM where the planes are large: 256 planes of 1024 x 1024 bf16 take 87 us
// for 537 MB (6.2 TB/s; a kernel that only reads reaches 6.3, streamed 6.9) and 4 us
// to join.  A thread a diagonal took 4075 us; lanes on fixed diagonals 125, a third of
// them past the planes' corners.  Rows of any other length than a multiple of V need
// their ends masked: 1023 x 1023 122 us.  Small planes are bound by what a team does
// once (10 us: edges, slots, line, buckets): 512 of 128 x 128 take 11 us.
template <int DT, int R, int kG>
__global__ __launch_bounds__(kThreads) void bias_backward(GradArgs a, Edges e) {
  constexpr int V = Elem<DT>::kVec, ES = Elem<DT>::kBytes;
  constexpr int kTeam = kGroups * kG, kTeams = kThreads / kTeam;
  using W = Walk<V, R>;
  constexpr int kSums = W::kLast - W::kFirst + 1, kSlot = (kSums + 3) / 4 * 4;
  extern __shared__ __attribute__((aligned(16))) float shared[];
  __shared__ int ranges[kMaxBuckets][2];
  __shared__ uint8_t live_rows[kGroups * max_steps(kG)];
  const int tid = threadIdx.x, team = tid / kTeam, u = tid % kTeam, l = u % kG;
  const int group = kG == 64 ? __builtin_amdgcn_readfirstlane(u / kG) : u / kG;
  const int window = blockIdx.x % a.windows, split = blockIdx.x / a.windows;
  const int64_t own = (int64_t)blockIdx.y * kTeams + team, b = blockIdx.z;
  const int64_t h = min(own, a.heads - 1);  // a team past the heads only keeps step
  // A team's LDS: slots [kGroups][steps + kG][kSlot], then its line of offsets.
  const int line_at = kGroups * (a.steps + kG) * kSlot;
  float* slots = shared + team * (line_at + (kGroups * a.steps + kG + 1) * V);
  const char* plane = a.g + (b * a.g_b + h * a.g_h) * ES;
  const int mis = (int)((uintptr_t)plane / ES % V);
  const int k_len = (int)a.k_len, q_len = (int)a.q_len;
  const int c = window * kG + l;  // column block
  const int first = c * V - mis;  // column of its unshifted run
  const int begin = split * kGroups * a.steps;
  const int r0 = begin + group * a.steps, r1 = min(r0 + a.steps, a.row_blocks);
  auto store = [&](int x, float u) {
    if (own >= a.heads) return;
    if (a.blocks == 1) a.out[(b * a.buckets + x) * a.heads + h] = u;
    else a.partial[((b * a.heads + h) * a.blocks + blockIdx.x) * a.buckets + x] = u;
  };
  if (window * kG - a.last_block >= begin + kGroups * a.steps) {  // causal: all keys follow the queries
    for (int x = u; x < a.buckets; x += kTeam) store(x, 0.f);
    return;
  }
  float* mine = slots + group * (a.steps + kG) * kSlot;
  for (int p = l; p < a.steps * kSlot; p += kG) mine[p] = 0.f;
  if (tid < a.buckets) {
    bucket_range(e, tid, &ranges[tid][0], &ranges[tid][1]);
    if (a.causal) ranges[tid][1] = min(ranges[tid][1], 0);
  }
  // Bit x: column first - (V - 1) + x is there and live.
  constexpr int kAll = W::columns(), kRows = (1 << V) - 1;
  const int lo = min(max(V - 1 - first, 0), 2 * V - 1), hi = min(max(k_len - first + V - 1, 0), 2 * V - 1);
  int cols = ((1 << hi) - 1) & ~((1 << lo) - 1);
  bool dead_row = false;
  if (a.mask) {
    const uint8_t* m = a.mask + b * a.mask_b;
    uint8_t col[2 * V - 1];  // places past the ends read an end: cols has no bit there
#pragma unroll
    for (int x = 0; x < 2 * V - 1; ++x) col[x] = m[min(max(first - (V - 1) + x, 0), k_len - 1) * a.mask_k];
    for (int n = tid; n < kGroups * a.steps; n += kThreads) {
      int bits = 0;
#pragma unroll
      for (int x = 0; x < V; ++x) bits |= (m[(min((begin + n) * V + x, q_len - 1) + a.start) * a.mask_k] != 0) << x;
      live_rows[n] = (uint8_t)bits;
      dead_row |= bits != kRows;
    }
    int bits = 0;
#pragma unroll
    for (int x = 0; x < 2 * V - 1; ++x) bits |= (col[x] != 0) << x;
    cols &= bits;
  }
  dead_row = __syncthreads_or(dead_row);
  const int64_t plane_end = (int64_t)(q_len - 1) * a.g_i + k_len;

  float sum[kSlot];
#pragma unroll
  for (int t = 0; t < kSlot; ++t) sum[t] = 0.f;

  // The lane's runs of row block r: every entry there, live and counted. Read
  // once, and past the caches: 537 MB of scores take 91 us so and 102 us cached, 33
  // MB 15.7 and 14.8.
  auto load_whole = [&](u32x4 (&v)[V], int r) {
    const char* at = plane + ((int64_t)(r * V) * a.g_i + first) * ES;
#pragma unroll
    for (int x = 0; x < V; ++x)
      v[x] = __builtin_nontemporal_load((const u32x4*)(at + (x * a.g_i - W::shift(x)) * ES));
  };
  auto add_whole = [&](const u32x4 (&v)[V]) {
#pragma unroll
    for (int x = 0; x < V; ++x) {
      float f[V];
      unpack16<DT>(v[x], f);
#pragma unroll
      for (int q = 0; q < V; ++q) sum[W::at(x, q) - W::kFirst] += f[q];
    }
  };
  int runs = 0;  // bit x: the run of row x has a live entry
#pragma unroll
  for (int x = 0; x < V; ++x) runs |= ((cols >> (V - 1 - W::shift(x)) & kRows) != 0) << x;
  // Only a plane's first and last row block, or rows closer than two runs, have
  // runs that stick out of the plane (bit x): their entries are added one by one.
  auto torn_of = [&](int r) {
    int torn = 0;
    if (r > 0 && r < a.row_blocks - 1 && a.g_i >= 2 * V) return torn;
#pragma unroll
    for (int x = 0; x < V; ++x) {
      const int64_t at = ((int64_t)(r * V) + x) * a.g_i + first - W::shift(x);
      torn |= (at < 0 || at + V > plane_end) << x;
    }
    return torn;
  };
  // Any row block: a run without a live entry, or a torn one, reads zeros instead.
  auto rows_of = [&](int r) {
    int rows = r >= r1 || c - r > a.last_block ? 0 : q_len - r * V >= V ? kRows : (1 << (q_len - r * V)) - 1;
    if (a.mask && r < r1) rows &= live_rows[r - begin];
    return rows;
  };
  auto load_some = [&](u32x4 (&v)[V], int r) {
    const int need = rows_of(r) & runs & ~torn_of(r);
    const char* at = plane + ((int64_t)(r * V) * a.g_i + first) * ES;
#pragma unroll
    for (int x = 0; x < V; ++x)
      v[x] = *(need >> x & 1 ? (const u32x4*)(at + (x * a.g_i - W::shift(x)) * ES) : &kZeros);
  };
  auto add_some = [&](u32x4 (&v)[V], int r) {
    int keep_cols = cols;
    asm volatile("" : "+v"(keep_cols));  // its masks are made here, not held through the loop
#pragma unroll
    for (int x = 0; x < V; ++x)
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // entries that are not there, or dead, to zero bits
        const int at = V - 1 - W::shift(x) + q * 4 / ES;
        uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe(keep_cols, at, 1);
        if constexpr (ES == 2)
          keep = (keep & 0xffffu) | ((uint32_t)__builtin_amdgcn_sbfe(keep_cols, at + 1, 1) & 0xffff0000u);
        v[x][q] &= keep;
      }
    add_whole(v);
    const int torn = torn_of(r) & rows_of(r);
    if (!__any(torn)) return;
#pragma unroll
    for (int x = 0; x < V; ++x) {
      const int64_t at = ((int64_t)(r * V) + x) * a.g_i + first - W::shift(x);
#pragma unroll
      for (int q = 0; q < V; ++q)
        if (torn >> x & 1 && cols >> (V - 1 - W::shift(x) + q) & 1)
          sum[W::at(x, q) - W::kFirst] += Elem<DT>::load(plane, at + q);
    }
  };
  // On to row block r0 + step + 1.  Diagonal block c - r lies in slot l + steps - 1 - step.
  auto next = [&](int step) {
    if (l == kG - 1) {
      f32x4* out = (f32x4*)(mine + (a.steps - 1 - step + l) * kSlot);
#pragma unroll
      for (int t = 0; t < kSlot; t += 4) out[t / 4] = f32x4{sum[t], sum[t + 1], sum[t + 2], sum[t + 3]};
    }
#pragma unroll
    for (int t = 0; t < kSums; ++t) sum[t] = from_left<kG>(sum[t]);
  };

  // Row blocks whose diagonal blocks are all past the last are left out.
  const int count = (max(r1 - r0, 0) + kAhead - 1) / kAhead * kAhead;
  int step = min(max(window * kG - a.last_block - r0, 0) / kAhead * kAhead, count);
  const bool whole = !dead_row && __all((cols & kAll) == kAll && r1 * V <= q_len && count == r1 - r0 &&
                                        c - (r0 + step) <= a.last_block);
  for (int s = 0; s < step; ++s)  // slots that no row block reaches
    if (l == kG - 1)
#pragma unroll
      for (int t = 0; t < kSlot; ++t) mine[(a.steps - 1 - s + l) * kSlot + t] = 0.f;
  u32x4 v[kAhead][V];
  if (whole) {
    if (step < count)
#pragma unroll
      for (int k = 0; k < kAhead; ++k) load_whole(v[k], r0 + step + k);
    for (; step < count; step += kAhead)
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        add_whole(v[k]);
        next(step + k);
        if (step + kAhead < count) load_whole(v[k], r0 + step + kAhead + k);
      }
  } else {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) load_some(v[k], r0 + step + k);
    for (; step < count; step += kAhead)
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        add_some(v[k], r0 + step + k);
        next(step + k);
        load_some(v[k], r0 + step + kAhead + k);
      }
  }
  // Before row block r0 + count the lanes from 1 on hold diagonal blocks.
  if (l > 0 || count < a.steps) {
    float* out = mine + (a.steps - 1 - count + l) * kSlot;
#pragma unroll
    for (int t = 0; t < kSlot; ++t) out[t] = sum[t];
  }
  __syncthreads();

  // The team's line of offsets: block 0 is the last group's first slot.
  float* line = slots + line_at;
  const int used = a.steps + kG - 1, blocks = (kGroups - 1) * a.steps + used, length = (blocks - 1) * V + kSums;
  for (int p = u; p < length; p += kTeam) {
    const int k = p / V, t = p % V;
    float sum_p = 0.f;
#pragma unroll
    for (int back = 0; back < 3; ++back) {
      if (t + back * V >= kSums) continue;
      int at = k - back - (kGroups - 1) * a.steps;
#pragma unroll
      for (int g = 0; g < kGroups; ++g, at += a.steps)
        if (at >= 0 && at < used) sum_p += slots[(g * (a.steps + kG) + at) * kSlot + t + back * V];
    }
    line[p] = sum_p;
  }
  __syncthreads();
  const int lane = u & 15;
  const int o0 = (window * kG - (begin + kGroups * a.steps - 1)) * V + W::kFirst - 2 * (V - 1) - mis - a.start;
  for (int x = u >> 4; x < a.buckets; x += kTeam / 16) {
    const int from = max(ranges[x][0] - o0, 0), to = min(ranges[x][1] - o0, length - 1);
    float sum_x = 0.f;
    for (int p = from + lane; p <= to; p += 16) sum_x += line[p];
    sum_x = lanes_sum<16>(sum_x);
    if (lane == 0) store(x, sum_x);
  }
}

// A plane's buckets: its workgroups' sums, in groups of threads that stride over
// the workgroups, the groups in order.
__global__ __launch_bounds__(kThreads) void bias_join(GradArgs a) {
  __shared__ float sums[kThreads];
  const int tid = threadIdx.x;
  const int64_t h = blockIdx.x, b = blockIdx.y;
  int width = 1;
  while (width < a.buckets) width *= 2;
  const int groups = kThreads / width, x = tid % width;
  float v = 0.f;
  if (x < a.buckets) {
    const float* p = a.partial + (b * a.heads + h) * a.blocks * a.buckets + x;
    for (int64_t c = tid / width; c < a.blocks; c += groups) v += p[c * a.buckets];
  }
  sums[tid] = v;
  __syncthreads();
  if (tid < a.buckets) {
    for (int g = 1; g < groups; ++g) v += sums[g * width + tid];
    a.out[(b * a.buckets + tid) * a.heads + h] = v;
  }
}

int take_edges(const char* what, Edges& e, const int32_t* edges, int n, int bidirectional) {
  if (!edges || n < 1 || n * (bidirectional ? 2 : 1) > kMaxBuckets)
    return set_error(DA_ERR_UNSUPPORTED, "%s: 1 to %d buckets", what, kMaxBuckets);
  if (edges[0] != 0) return set_error(DA_ERR_INVALID, "%s: the first bucket's least distance must be 0", what);
  e.n = n;
  e.both = bidirectional ? 1 : 0;
  for (int x = 0; x < n; ++x) {
    if (x && edges[x] < edges[x - 1]) return set_error(DA_ERR_INVALID, "%s: the least distances must ascend", what);
    e.least[x] = std::min(edges[x], 1 << 30);  // further than any distance
  }
  return DA_OK;
}

// Every index into a line of offsets and every column fits 32 bits with room.
constexpr int64_t kMaxLen = (int64_t)1 << 26;

constexpr int64_t kWantBlocks = 1024;  // four workgroups for each CU

struct GradPlan {
  int group, row_blocks, last_block, windows, splits, steps;
};

// Column blocks go to groups of lanes, row blocks to the groups of a workgroup
// and, where the planes are few, to several workgroups.
GradPlan grad_plan(int v, bool aligned, int64_t planes, int64_t q_len, int64_t k_len, int64_t start, bool causal) {
  GradPlan p;
  p.row_blocks = (int)((q_len + v - 1) / v);
  const int64_t slack = aligned ? 0 : v - 1;
  int64_t last = kMaxLen, columns = (k_len - 1 + 2 * slack) / v + 1;
  if (causal) {
    last = std::max<int64_t>((start + v - 1 + 2 * slack) / v, -p.row_blocks);
    columns = std::max<int64_t>(std::min(columns, last + p.row_blocks), 1);
  }
  p.last_block = (int)last;
  // Groups of 16 where those of 64 would have half as many lanes again, idle ones: 512
  // planes of 513 x 513 take 94 us in groups of 16, 128 in groups of 64.  With fewer
  // idle lanes the longer lines of 64 count for more: 300 x 300 48 us against 67,
  // 1023 x 1023 122 against 133.
  const int64_t by16 = (columns + 15) / 16 * 16, by64 = (columns + 63) / 64 * 64;
  p.group = by16 * 3 <= by64 * 2 ? 16 : 64;
  p.windows = (int)((columns + p.group - 1) / p.group);
  const int teams = kThreads / (kGroups * p.group);
  int64_t steps = p.row_blocks * planes * p.windows / (kWantBlocks * kGroups * teams);
  steps = std::min<int64_t>(std::max<int64_t>(steps, 8), max_steps(p.group));
  steps = std::min<int64_t>(steps, (p.row_blocks + kGroups - 1) / kGroups);
  p.steps = (int)(steps + kAhead - 1) / kAhead * kAhead;
  p.splits = (p.row_blocks + kGroups * p.steps - 1) / (kGroups * p.steps);
  return p;
}

// Bytes of LDS of a team.
template <int DT, int R>
size_t team_lds(const GradPlan& p) {
  constexpr int V = 16 / (DT == DA_F32 ? 4 : 2);
  using W = Walk<V, R>;
  constexpr int kSlot = (W::kLast - W::kFirst + 1 + 3) / 4 * 4;
  return (size_t)(kGroups * (p.steps + p.group) * kSlot + (kGroups * p.steps + p.group + 1) * V) * sizeof(float);
}

int check_sizes(const char* what, int64_t batch, int64_t heads, int64_t q_len, int64_t k_len, int64_t start) {
  if (batch < 0 || heads < 0 || q_len < 0 || k_len < 0) return set_error(DA_ERR_INVALID, "%s: negative size", what);
  if (q_len > kMaxLen || k_len > kMaxLen || start > kMaxLen || start < -kMaxLen || heads > 65535 || batch > 65535)
    return set_error(DA_ERR_UNSUPPORTED, "%s: lengths up to 2^26, batch and heads up to 65535", what);
  return DA_OK;
}

}  // namespace
}  // namespace da

using namespace da;

extern "C" {

int da_relative_bias(const void* table, int dtype, int64_t table_bstride, int64_t table_hstride, int64_t heads,
                     int64_t q_len, int64_t k_len, int64_t q_start, const int32_t* edges, int side_buckets,
                     int bidirectional, int causal, void* out, void* stream) {
  const char* what = "da_relative_bias";
  if (!valid_dtype(dtype)) return set_error(DA_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  if (int rc = check_sizes(what, 1, heads, q_len, k_len, q_start)) return rc;
  Edges e{};
  if (int rc = take_edges(what, e, edges, side_buckets, bidirectional)) return rc;
  if (!heads || !q_len || !k_len) return DA_OK;
  if (!table || !out) return set_error(DA_ERR_INVALID, "%s: NULL pointer", what);
  const int es = (int)elem_bytes(dtype), v = 16 / es;
  const bool aligned = (uintptr_t)out % 16 == 0 && k_len % v == 0;
  const int64_t row_blocks = (q_len + v - 1) / v;
  BiasArgs a{};
  a.table = (const char*)table, a.out = (char*)out, a.q_len = q_len, a.k_len = k_len, a.t_b = table_bstride;
  a.t_h = table_hstride, a.start = (int)q_start, a.causal = causal;
  // A row's first run may start up to 2 (v - 1) entries before it.
  a.columns = (int)((k_len - 1 + (aligned ? 0 : 2 * (v - 1))) / v + 1);
  a.spread = (uintptr_t)out % 128 == 0 && k_len * es % 128 == 0 ? 0 : 7;
  a.windows = (a.columns + a.spread + kWave - 1) / kWave;
  // Row blocks of a workgroup: 4 to 32, so that there are kWantBlocks workgroups.
  a.steps = (int)std::min<int64_t>(std::max<int64_t>(row_blocks * a.windows * heads / kWantBlocks, 4), 32);
  a.steps = (int)std::min<int64_t>(a.steps, row_blocks);
  a.closed = dtype == DA_F32 ? 0xff800000u : dtype == DA_BF16 ? 0xff80u : 0xfc00u;
  hipStream_t st = (hipStream_t)stream;
  const int64_t grid_x = a.windows * ((row_blocks + a.steps - 1) / a.steps);
  if (grid_x > 0x7fffffff) return set_error(DA_ERR_UNSUPPORTED, "%s: too many entries", what);
  const dim3 grid((unsigned)grid_x, (unsigned)heads);
  const int blocks = std::min<int>(kWave, a.columns + a.spread) + a.steps - 1 + a.spread;
  const size_t lds = (size_t)v * blocks * 16 + (size_t)(blocks + 2) * v * 4;
  if (es == 2) bias_forward<2><<<grid, kThreads, lds, st>>>(a, e);
  else bias_forward<4><<<grid, kThreads, lds, st>>>(a, e);
  return check_launch(what);
}

int da_relative_bias_grad_workspace(int dtype, int64_t batch, int64_t heads, int64_t q_len, int64_t k_len,
                                    int64_t q_start, int buckets, int causal, size_t* bytes) {
  const char* what = "da_relative_bias_grad_workspace";
  if (!bytes) return set_error(DA_ERR_INVALID, "%s: NULL bytes", what);
  if (!valid_dtype(dtype)) return set_error(DA_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  if (int rc = check_sizes(what, batch, heads, q_len, k_len, q_start)) return rc;
  *bytes = 0;
  if (!batch || !heads || !q_len || !k_len) return DA_OK;
  for (int aligned = 0; aligned < 2; ++aligned) {
    const GradPlan p = grad_plan(dtype == DA_F32 ? 4 : 8, aligned, batch * heads, q_len, k_len, q_start, causal);
    const int64_t blocks = (int64_t)p.windows * p.splits;
    if (blocks > 1) *bytes = std::max(*bytes, (size_t)(blocks * batch * heads * buckets) * sizeof(float));
  }
  return DA_OK;
}

int da_relative_bias_grad(const void* g, int dtype, int64_t batch, int64_t heads, int64_t q_len, int64_t k_len,
                          int64_t g_bstride, int64_t g_hstride, int64_t g_istride, int64_t q_start,
                          const int32_t* edges, int side_buckets, int bidirectional, int causal, const uint8_t* mask,
                          int64_t mask_bstride, int64_t mask_kstride, float* out, void* workspace,
                          size_t workspace_bytes, void* stream) {
  const char* what = "da_relative_bias_grad";
  if (!valid_dtype(dtype)) return set_error(DA_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  if (int rc = check_sizes(what, batch, heads, q_len, k_len, q_start)) return rc;
  Edges e{};
  if (int rc = take_edges(what, e, edges, side_buckets, bidirectional)) return rc;
  const int buckets = side_buckets * (bidirectional ? 2 : 1);
  if (!batch || !heads) return DA_OK;
  if (!out) return set_error(DA_ERR_INVALID, "%s: NULL out", what);
  hipStream_t st = (hipStream_t)stream;
  if (!q_len || !k_len) return zero_f32_2d(out, 1, batch * heads * buckets, batch * heads * buckets, st);
  if (!g) return set_error(DA_ERR_INVALID, "%s: NULL g", what);
  if (g_bstride < 0 || g_hstride < 0 || g_istride < 0)
    return set_error(DA_ERR_INVALID, "%s: negative stride", what);
  if (mask && (q_start < 0 || q_start + q_len > k_len))
    return set_error(DA_ERR_INVALID, "%s: a mask over the keys needs every query's position among them", what);
  const int v = dtype == DA_F32 ? 4 : 8;
  const bool aligned = (uintptr_t)g % 16 == 0 && g_istride % v == 0 && (heads == 1 || g_hstride % v == 0) &&
                       (batch == 1 || g_bstride % v == 0);
  const GradPlan p = grad_plan(v, aligned, batch * heads, q_len, k_len, q_start, causal);
  GradArgs a{};
  a.g = (const char*)g, a.mask = mask, a.out = out, a.heads = heads, a.q_len = q_len, a.k_len = k_len;
  a.start = (int)q_start, a.g_b = g_bstride, a.g_h = g_hstride, a.g_i = g_istride, a.mask_b = mask_bstride;
  a.mask_k = mask_kstride, a.buckets = buckets, a.causal = causal, a.row_blocks = p.row_blocks;
  a.last_block = p.last_block, a.windows = p.windows, a.steps = p.steps;
  a.blocks = (int64_t)p.windows * p.splits;
  const size_t need = a.blocks > 1 ? (size_t)(a.blocks * batch * heads * buckets) * sizeof(float) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  if (a.blocks > 0x7fffffff) return set_error(DA_ERR_UNSUPPORTED, "%s: too many entries", what);
  a.partial = (float*)workspace;
  const int teams = kThreads / (kGroups * p.group);
  const dim3 grid((unsigned)a.blocks, (unsigned)((heads + teams - 1) / teams), (unsigned)batch);
#define DA_BWD(DT, R)                                                                 \
  case R:                                                                             \
    if (p.group == 16)                                                                \
      bias_backward<DT, R, 16><<<grid, kThreads, team_lds<DT, R>(p) * teams, st>>>(a, e); \
    else bias_backward<DT, R, 64><<<grid, kThreads, team_lds<DT, R>(p), st>>>(a, e);  \
    break;
#define DA_BWD8(DT)                                                                                    \
  switch (g_istride % 8) {                                                                             \
    DA_BWD(DT, 0) DA_BWD(DT, 1) DA_BWD(DT, 2) DA_BWD(DT, 3) DA_BWD(DT, 4) DA_BWD(DT, 5) DA_BWD(DT, 6) \
    DA_BWD(DT, 7)                                                                                      \
  }
  if (dtype == DA_BF16) {
    DA_BWD8(DA_BF16)
  } else if (dtype == DA_F16) {
    DA_BWD8(DA_F16)
  } else {
    switch (g_istride % 4) { DA_BWD(DA_F32, 0) DA_BWD(DA_F32, 1) DA_BWD(DA_F32, 2) DA_BWD(DA_F32, 3) }
  }
#undef DA_BWD8
#undef DA_BWD
  if (int rc = check_launch(what)) return rc;
  if (a.blocks == 1) return DA_OK;
  bias_join<<<dim3((unsigned)heads, (unsigned)batch), kThreads, 0, st>>>(a);
  return check_launch(what);
}

}  // extern "C"
