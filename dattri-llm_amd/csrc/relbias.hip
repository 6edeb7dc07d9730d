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
// query are no part of the attention: the bias is -inf there and g is not read.
#include <algorithm>

#include "common.h"

namespace da {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxBuckets = 256;

struct Edges {
  int n;      // buckets of one side
  int both;   // bidirectional
  int32_t least[kMaxBuckets];
};

__device__ __forceinline__ int bucket_of(const Edges& e, int64_t o) {
  const int64_t away = e.both ? (o < 0 ? -o : o) : (o < 0 ? -o : 0);
  const int32_t r = (int32_t)min(away, (int64_t)0x7fffffff);
  int lo = 0, hi = e.n;  // least[lo] <= r < least[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (e.least[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo + (e.both && o > 0 ? e.n : 0);
}

// A square of scores is walked along its diagonals.  With V entries in 16 bytes,
// a lane owns diagonal block k: in row block r (rows rV .. rV + V - 1) its
// columns are those of column block r + k, so that from one row block to the
// next it meets the same 2V - 1 offsets j - i again: they stay in registers for
// the whole walk -- as sums in the backward pass, as packed 16-byte values in the
// forward pass -- while every access is one aligned 16 bytes and the lanes of a
// wave are neighbours in the row.
//
// Rows need not be aligned: entry j of row i is at address mis + i stride + j
// (modulo V; mis that of the plane's first entry), so with R = stride mod V the
// aligned run of row rV + e starts at column (r + k) V - mis - shift(e), shift(e)
// = e R mod V.  R is a template argument, all indices into the registers are
// constants, and 3V - 2 offsets cover every R.
template <int V, int R>
struct Walk {
  static constexpr int kLine = (kWave + 2) * V;  // offsets of a wave's 64 diagonal blocks
  __host__ __device__ static constexpr int shift(int e) { return e * R % V; }
  __host__ __device__ static constexpr int at(int e, int x) { return x - e - shift(e) + 2 * (V - 1); }
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
    *hi = !e.both && first == 0 ? 0x3fffffff : -first;
  }
}

struct BiasArgs {
  const char* table;
  char* out;
  int64_t q_len, k_len;
  int64_t t_b, t_h;  // table strides in elements
  int start, causal;
  int row_blocks, first_block;  // row blocks; the least diagonal block
  int windows, splits, steps;   // waves of diagonal blocks; parts of the rows, row blocks of each
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

// A workgroup writes one head's entries of 64 diagonal blocks in a part of the
// rows: the offsets' values go to LDS once, each lane packs the V runs of its
// block and then only stores.  Runs that a row's end cuts are left to the
// workgroup of the first window, entry by entry.
template <int ES, int R>
__global__ __launch_bounds__(kThreads) void bias_forward(BiasArgs a, Edges e) {
  constexpr int V = 16 / ES;
  using W = Walk<V, R>;
  __shared__ uint32_t line[W::kLine];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int window = blockIdx.x % a.windows, split = blockIdx.x / a.windows;
  const int64_t h = blockIdx.y;
  char* plane = a.out + h * a.q_len * a.k_len * ES;
  const int mis = (int)((uintptr_t)plane / ES % V);
  const int k0 = a.first_block + window * kWave, k = k0 + lane;
  const char* column = a.table + h * a.t_h * ES;
  for (int p = tid; p < W::kLine; p += kThreads) {
    const int o = k0 * V + p - 2 * (V - 1) - mis - a.start;
    line[p] = a.causal && o > 0 ? a.closed : load_bits<ES>(column, bucket_of(e, o) * a.t_b);
  }
  __syncthreads();
  u32x4 run[V];
#pragma unroll
  for (int r = 0; r < V; ++r)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (ES == 4) run[r][q] = line[lane * V + W::at(r, q)];
      else run[r][q] = line[lane * V + W::at(r, 2 * q)] | line[lane * V + W::at(r, 2 * q + 1)] << 16;
    }
  const int r0 = split * a.steps, r1 = min(r0 + a.steps, a.row_blocks);
  const int k_len = (int)a.k_len, q_len = (int)a.q_len;
  const int last = min(r1, (k_len + mis + 2 * V - 2) / V - k0);
  for (int r = max(r0, 1 - kWave - k0) + wave; r < last; r += kWaves) {
    const int first = (r + k) * V - mis;  // column of an unshifted run
#pragma unroll
    for (int x = 0; x < V; ++x) {
      const int i = r * V + x, j = first - W::shift(x);
      if (i < q_len && j >= 0 && j + V <= k_len) st16(plane + ((int64_t)i * k_len + j) * ES, run[x]);
    }
  }
  if (window == 0 && (R != 0 || mis != 0 || k_len % V != 0)) {
    const int rows = min(r1 * V, q_len) - r0 * V;
    for (int n = tid; n < rows * 2 * V; n += kThreads) {
      const int i = r0 * V + n / (2 * V), x = n % (2 * V);
      const int lead = (int)((V - (mis + (int64_t)i * k_len) % V) % V);  // entries before the first whole run
      const int tail = k_len < lead ? 0 : (k_len - lead) % V;
      int j;
      if (x < V) {
        if (x >= min(lead, k_len)) continue;
        j = x;
      } else {
        if (x - V >= tail) continue;
        j = k_len - tail + x - V;
      }
      const int o = j - i - a.start;
      store_bits<ES>(plane, (int64_t)i * k_len + j,
                     a.causal && o > 0 ? a.closed : load_bits<ES>(column, bucket_of(e, o) * a.t_b));
    }
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
  int row_blocks, first_block, last_block;
  int windows, splits, steps;
};

constexpr int kMaxSteps = 512;  // row blocks of a workgroup at most: its mask bits lie in LDS

// A workgroup sums 64 diagonal blocks of one plane over a part of its rows; its
// waves take row blocks in turn.  Their 3V - 2 sums a lane meet in LDS, lane by
// lane in three steps (a lane's offsets overlap its neighbours'), and each
// bucket's range of offsets is then summed by one wave.
template <int DT, int R>
__global__ __launch_bounds__(kThreads) void bias_backward(GradArgs a, Edges e) {
  constexpr int V = Elem<DT>::kVec, ES = Elem<DT>::kBytes;
  using W = Walk<V, R>;
  __shared__ float line[kWaves][W::kLine];
  __shared__ uint8_t live_cols[kMaxSteps + kWave + 1], live_rows[kMaxSteps];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int window = blockIdx.x % a.windows, split = blockIdx.x / a.windows;
  const int64_t h = blockIdx.y, b = blockIdx.z;
  const char* plane = a.g + (b * a.g_b + h * a.g_h) * ES;
  const int mis = (int)((uintptr_t)plane / ES % V);
  const int k0 = a.first_block + window * kWave, k = k0 + lane;
  const int k_len = (int)a.k_len, q_len = (int)a.q_len;
  // Row blocks where some lane's column block holds an entry of a row.
  const int r0 = max(split * a.steps, 1 - kWave - k0);
  const int r1 = min(min((split + 1) * a.steps, a.row_blocks), (k_len + mis + 2 * V - 2) / V - k0);
  if (a.mask) {
    const uint8_t* m = a.mask + b * a.mask_b;
    for (int n = tid; n < r1 - r0 + kWave; n += kThreads) {  // column blocks r0 + k0 - 1 ...
      const int64_t j0 = (int64_t)(r0 + k0 - 1 + n) * V - mis;
      int bits = 0;
      for (int x = 0; x < V; ++x)
        if (j0 + x >= 0 && j0 + x < k_len && m[(j0 + x) * a.mask_k]) bits |= 1 << x;
      live_cols[n] = (uint8_t)bits;
    }
    for (int n = tid; n < r1 - r0; n += kThreads) {
      int bits = 0;
      for (int x = 0; x < V; ++x) {
        const int64_t i = (int64_t)(r0 + n) * V + x;
        if (i < q_len && m[(i + a.start) * a.mask_k]) bits |= 1 << x;
      }
      live_rows[n] = (uint8_t)bits;
    }
    __syncthreads();
  }
  float sum[3 * V - 2];
#pragma unroll
  for (int t = 0; t < 3 * V - 2; ++t) sum[t] = 0.f;
  const int64_t plane_end = (int64_t)(q_len - 1) * a.g_i + k_len;
  for (int r = r0 + wave; r < r1; r += kWaves) {
    const int first = (r + k) * V - mis;
    int rows = q_len - r * V >= V ? (1 << V) - 1 : (1 << (q_len - r * V)) - 1;
    // Bit x of cols: column first - (V - 1) + x is there (and live).
    constexpr int kAll = (1 << (2 * V - 1)) - 1;
    int cols = 0;
    if (k <= a.last_block) {
      const int lo = min(max(V - 1 - first, 0), 2 * V - 1), hi = min(max(k_len - first + V - 1, 0), 2 * V - 1);
      cols = ((1 << hi) - 1) & ~((1 << lo) - 1);
      if (a.mask) cols &= (live_cols[r - r0 + lane] | live_cols[r - r0 + lane + 1] << V) >> 1;
    }
    if (a.mask) rows = __builtin_amdgcn_readfirstlane(live_rows[r - r0]);
    if (!__any(cols) || !rows) continue;
    u32x4 v[V];
#pragma unroll
    for (int x = 0; x < V; ++x) {
      v[x] = u32x4{0, 0, 0, 0};
      if (!(rows >> x & 1)) continue;
      const int64_t at = (int64_t)(r * V + x) * a.g_i + first - W::shift(x);
      const int here = cols >> (V - 1 - W::shift(x)) & ((1 << V) - 1);  // the run's live entries
      if (here) {
        if (at >= 0 && at + V <= plane_end) v[x] = ld16(plane + at * ES);
        else {  // the plane's first or last run sticks out of it
#pragma unroll
          for (int q = 0; q < V; ++q)
            if (here >> q & 1) v[x][q * ES / 4] |= load_bits<ES>(plane, at + q) << (ES == 2 ? q % 2 * 16 : 0);
        }
      }
    }
    if (__all(cols == kAll)) {
#pragma unroll
      for (int x = 0; x < V; ++x) {
        float f[V];
        unpack16<DT>(v[x], f);
#pragma unroll
        for (int q = 0; q < V; ++q) sum[W::at(x, q)] += f[q];
      }
    } else {
#pragma unroll
      for (int x = 0; x < V; ++x) {
        float f[V];
        unpack16<DT>(v[x], f);
#pragma unroll
        for (int q = 0; q < V; ++q) sum[W::at(x, q)] += cols >> (V - 1 - W::shift(x) + q) & 1 ? f[q] : 0.f;
      }
    }
  }
  float* mine = line[wave];
#pragma unroll
  for (int step = 0; step < 3; ++step) {
#pragma unroll
    for (int x = 0; x < V; ++x) {
      const int t = step * V + x;
      const float u = t < 3 * V - 2 ? sum[t < 3 * V - 2 ? t : 0] : 0.f;
      const int p = (lane + step) * V + x;
      // The last `step` blocks of the line are met for the first time.
      mine[p] = step == 0 || lane == kWave - 1 ? u : mine[p] + u;
    }
    __syncthreads();
  }
  for (int p = tid; p < W::kLine; p += kThreads) {
    float u = line[0][p];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) u += line[w][p];
    line[0][p] = u;
  }
  __syncthreads();
  const int o0 = k0 * V - 2 * (V - 1) - mis - a.start;  // the line's first offset
  for (int x = wave; x < a.buckets; x += kWaves) {
    int lo, hi;
    bucket_range(e, x, &lo, &hi);
    if (a.causal) hi = min(hi, 0);
    lo = max(lo - o0, 0);
    hi = min(hi - o0, W::kLine - 1);
    float u = 0.f;
    if (lo <= hi) {
      for (int p = lo + lane; p <= hi; p += kWave) u += line[0][p];
      u = wave_sum(u);
    }
    if (lane == 0) {
      if (a.blocks == 1) a.out[(b * a.buckets + x) * a.heads + h] = u;
      else a.partial[((b * a.heads + h) * a.blocks + blockIdx.x) * a.buckets + x] = u;
    }
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

struct Plan {
  int row_blocks, first_block, last_block, windows, splits, steps;
};

// Diagonal blocks run from the first column block against the last row block to
// the last column block against the first (with `causal` to the last that holds
// an offset up to 0), whatever the plane's misalignment.  The rows are split
// until `planes` of them fill the card with `want` workgroups, each of at least
// four row blocks a wave.
Plan make_plan(int v, bool aligned, int64_t planes, int64_t q_len, int64_t k_len, int64_t start, bool causal) {
  Plan p;
  p.row_blocks = (int)((q_len + v - 1) / v);
  p.first_block = 1 - p.row_blocks;
  const int64_t slack = aligned ? 0 : v - 1;  // most that mis, and that a row's shift, can be
  int64_t last = (k_len - 1 + 2 * slack) / v;
  if (causal) last = std::min(last, std::max<int64_t>((start + v - 1 + 2 * slack) / v, p.first_block));
  p.last_block = (int)last;
  p.windows = (int)((last - p.first_block + kWave) / kWave);
  int64_t splits = (kWantBlocks + planes * p.windows - 1) / (planes * p.windows);
  splits = std::min<int64_t>(splits, (p.row_blocks + 4 * kWaves - 1) / (4 * kWaves));
  splits = std::max<int64_t>(splits, (p.row_blocks + kMaxSteps - 1) / kMaxSteps);
  p.steps = (int)((p.row_blocks + splits - 1) / splits);
  p.splits = (p.row_blocks + p.steps - 1) / p.steps;
  return p;
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
  // Every column block of a row is written: no diagonal block is left out.
  const bool aligned = (uintptr_t)out % 16 == 0 && k_len % v == 0;
  const Plan p = make_plan(v, aligned, heads, q_len, k_len, q_start, false);
  BiasArgs a{};
  a.table = (const char*)table, a.out = (char*)out, a.q_len = q_len, a.k_len = k_len, a.t_b = table_bstride;
  a.t_h = table_hstride, a.start = (int)q_start, a.causal = causal, a.row_blocks = p.row_blocks;
  a.first_block = p.first_block, a.windows = p.windows, a.splits = p.splits, a.steps = p.steps;
  a.closed = dtype == DA_F32 ? 0xff800000u : dtype == DA_BF16 ? 0xff80u : 0xfc00u;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(p.windows * p.splits), (unsigned)heads);
#define DA_FWD(ES, R) \
  case R: bias_forward<ES, R><<<grid, kThreads, 0, st>>>(a, e); break;
  if (es == 2) {
    switch (k_len % 8) {
      DA_FWD(2, 0) DA_FWD(2, 1) DA_FWD(2, 2) DA_FWD(2, 3) DA_FWD(2, 4) DA_FWD(2, 5) DA_FWD(2, 6) DA_FWD(2, 7)
    }
  } else {
    switch (k_len % 4) { DA_FWD(4, 0) DA_FWD(4, 1) DA_FWD(4, 2) DA_FWD(4, 3) }
  }
#undef DA_FWD
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
    const Plan p = make_plan(dtype == DA_F32 ? 4 : 8, aligned, batch * heads, q_len, k_len, q_start, causal);
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
  const Plan p = make_plan(v, aligned, batch * heads, q_len, k_len, q_start, causal);
  GradArgs a{};
  a.g = (const char*)g, a.mask = mask, a.out = out, a.heads = heads, a.q_len = q_len, a.k_len = k_len;
  a.start = (int)q_start, a.g_b = g_bstride, a.g_h = g_hstride, a.g_i = g_istride, a.mask_b = mask_bstride;
  a.mask_k = mask_kstride, a.buckets = buckets, a.causal = causal, a.row_blocks = p.row_blocks;
  a.first_block = p.first_block, a.last_block = p.last_block, a.windows = p.windows, a.splits = p.splits;
  a.steps = p.steps, a.blocks = (int64_t)p.windows * p.splits;
  const size_t need = a.blocks > 1 ? (size_t)(a.blocks * batch * heads * buckets) * sizeof(float) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  a.partial = (float*)workspace;
  const dim3 grid((unsigned)a.blocks, (unsigned)heads, (unsigned)batch);
#define DA_BWD(DT, R) \
  case R: bias_backward<DT, R><<<grid, kThreads, 0, st>>>(a, e); break;
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
