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

struct BiasArgs {
  const char* table;
  char* out;
  int64_t heads, q_len, k_len, start;
  int64_t t_b, t_h;  // table strides in elements
  int causal;
};

template <int DT>
__global__ __launch_bounds__(kThreads) void bias_forward(BiasArgs a, Edges e) {
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= a.heads * a.q_len * a.k_len) return;
  const int64_t row = at / a.k_len, j = at - row * a.k_len;
  const int64_t h = row / a.q_len, i = row - h * a.q_len;
  const int64_t o = j - i - a.start;
  const float v = a.causal && o > 0 ? -__builtin_inff() : Elem<DT>::load(a.table, bucket_of(e, o) * a.t_b + h * a.t_h);
  Elem<DT>::store(a.out, at, v);
}

struct GradArgs {
  const char* g;
  const uint8_t* mask;  // (batch, k_len): query i is position i + start; NULL: all live
  float* partial;       // (blocks, batch, buckets, heads)
  float* out;           // (batch, buckets, heads)
  int64_t batch, heads, q_len, k_len, start;
  int64_t g_b, g_h, g_i;  // elements
  int64_t mask_b, mask_k;
  int64_t blocks;
  int buckets, causal;
};

// A thread owns one offset and walks its diagonal; its workgroup's 256 sums
// then go to their buckets in order.
template <int DT>
__global__ __launch_bounds__(kThreads) void bias_backward(GradArgs a, Edges e) {
  __shared__ float sums[kThreads];
  __shared__ int bins[kThreads];
  const int tid = threadIdx.x;
  const int64_t h = blockIdx.y, b = blockIdx.z;
  const int64_t line = (int64_t)blockIdx.x * kThreads + tid;  // j - i + q_len - 1
  const int64_t shift = line - (a.q_len - 1);                 // j - i
  const int64_t o = shift - a.start;
  const bool in = line < a.q_len + a.k_len - 1 && !(a.causal && o > 0);
  float v = 0.f;
  if (in) {
    const int64_t i0 = max((int64_t)0, -shift), i1 = min(a.q_len, a.k_len - shift);
    for (int64_t i = i0; i < i1; ++i) {
      const int64_t j = i + shift;
      const bool live = !a.mask || (a.mask[b * a.mask_b + (i + a.start) * a.mask_k] && a.mask[b * a.mask_b + j * a.mask_k]);
      if (live) v += Elem<DT>::load(a.g, b * a.g_b + h * a.g_h + i * a.g_i + j);
    }
  }
  sums[tid] = v;
  bins[tid] = in ? bucket_of(e, o) : -1;
  __syncthreads();
  for (int x = tid; x < a.buckets; x += kThreads) {
    float t = 0.f;
    for (int k = 0; k < kThreads; ++k) t += bins[k] == x ? sums[k] : 0.f;
    a.partial[((blockIdx.x * a.batch + b) * a.buckets + x) * a.heads + h] = t;
  }
}

__global__ __launch_bounds__(kThreads) void bias_join(GradArgs a) {
  const int64_t n = a.batch * a.buckets * a.heads;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= n) return;
  float v = 0.f;
  for (int64_t c = 0; c < a.blocks; ++c) v += a.partial[c * n + at];
  a.out[at] = v;
}

int take_edges(const char* what, Edges& e, const int32_t* edges, int n, int bidirectional) {
  if (!edges || n < 1 || n * (bidirectional ? 2 : 1) > kMaxBuckets)
    return set_error(DA_ERR_UNSUPPORTED, "%s: 1 to %d buckets", what, kMaxBuckets);
  if (edges[0] != 0) return set_error(DA_ERR_INVALID, "%s: the first bucket's least distance must be 0", what);
  e.n = n;
  e.both = bidirectional ? 1 : 0;
  for (int x = 0; x < n; ++x) {
    if (x && edges[x] < edges[x - 1]) return set_error(DA_ERR_INVALID, "%s: the least distances must ascend", what);
    e.least[x] = edges[x];
  }
  return DA_OK;
}

int64_t grad_blocks(int64_t q_len, int64_t k_len) { return (q_len + k_len - 1 + kThreads - 1) / kThreads; }

constexpr int64_t kMaxLen = (int64_t)1 << 30;

int check_sizes(const char* what, int64_t batch, int64_t heads, int64_t q_len, int64_t k_len, int64_t start) {
  if (batch < 0 || heads < 0 || q_len < 0 || k_len < 0) return set_error(DA_ERR_INVALID, "%s: negative size", what);
  if (q_len > kMaxLen || k_len > kMaxLen || start > kMaxLen || start < -kMaxLen || heads > 65535 || batch > 65535)
    return set_error(DA_ERR_UNSUPPORTED, "%s: lengths up to 2^30, batch and heads up to 65535", what);
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
  const int64_t n = heads * q_len * k_len;
  if (!n) return DA_OK;
  if (!table || !out) return set_error(DA_ERR_INVALID, "%s: NULL pointer", what);
  BiasArgs a{(const char*)table, (char*)out, heads, q_len, k_len, q_start, table_bstride, table_hstride, causal};
  hipStream_t st = (hipStream_t)stream;
  const int64_t blocks = (n + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) return set_error(DA_ERR_UNSUPPORTED, "%s: too many entries", what);
  if (dtype == DA_BF16) bias_forward<DA_BF16><<<(unsigned)blocks, kThreads, 0, st>>>(a, e);
  else if (dtype == DA_F16) bias_forward<DA_F16><<<(unsigned)blocks, kThreads, 0, st>>>(a, e);
  else bias_forward<DA_F32><<<(unsigned)blocks, kThreads, 0, st>>>(a, e);
  return check_launch(what);
}

int da_relative_bias_grad_workspace(int64_t batch, int64_t heads, int64_t q_len, int64_t k_len, int buckets,
                                    size_t* bytes) {
  const char* what = "da_relative_bias_grad_workspace";
  if (!bytes) return set_error(DA_ERR_INVALID, "%s: NULL bytes", what);
  if (int rc = check_sizes(what, batch, heads, q_len, k_len, 0)) return rc;
  *bytes = (size_t)(grad_blocks(q_len, k_len) * batch * heads * buckets) * sizeof(float);
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
  if (mask && (q_start < 0 || q_start + q_len > k_len))
    return set_error(DA_ERR_INVALID, "%s: a mask over the keys needs every query's position among them", what);
  GradArgs a{};
  a.g = (const char*)g, a.mask = mask, a.out = out, a.batch = batch, a.heads = heads, a.q_len = q_len, a.k_len = k_len;
  a.start = q_start, a.g_b = g_bstride, a.g_h = g_hstride, a.g_i = g_istride, a.mask_b = mask_bstride;
  a.mask_k = mask_kstride, a.buckets = buckets, a.causal = causal;
  a.blocks = grad_blocks(q_len, k_len);
  const size_t need = (size_t)(a.blocks * batch * heads * buckets) * sizeof(float);
  if (!workspace || workspace_bytes < need)
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  a.partial = (float*)workspace;
  const dim3 grid((unsigned)a.blocks, (unsigned)heads, (unsigned)batch);
  if (dtype == DA_BF16) bias_backward<DA_BF16><<<grid, kThreads, 0, st>>>(a, e);
  else if (dtype == DA_F16) bias_backward<DA_F16><<<grid, kThreads, 0, st>>>(a, e);
  else bias_backward<DA_F32><<<grid, kThreads, 0, st>>>(a, e);
  if (int rc = check_launch(what)) return rc;
  bias_join<<<(unsigned)((batch * heads * buckets + kThreads - 1) / kThreads), kThreads, 0, st>>>(a);
  return check_launch(what);
}

}  // extern "C"
