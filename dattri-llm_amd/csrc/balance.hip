// Router balance and z losses with per-expert counts, and the logits' gradient.
//
// Per sample b with n live tokens, p = softmax(logits of a token), c_e the
// choices of expert e among the live tokens, f = c / n:
//
//   loss = E sum_e f_e mean(p_e),   z = mean(logsumexp^2)
//   dlogit_e = up (E / n) p_e (f_e - sum f p) + up_z (2 / n) logsumexp p_e
//
// (n = 0: zeros).  The counts carry no gradient.  A choice outside the experts
// (a dropped one) counts for none.
//
// kL lanes share a token, each with S runs of V experts (16 bytes where the rows
// allow it), and a wave takes 64 / kL tokens at once: the softmax is two butterflies
// over kL lanes, a lane adds its experts' probabilities up in registers, and no
// probability goes to memory.  A workgroup sums a chunk of one sample's tokens; a
// sample of one chunk is finished there, else a second launch joins its chunks in
// order.  Counts are whole numbers: their LDS atomics have no order to keep.
//
// 32 x 4096 tokens, 128 experts, top-8, bf16 (42 MB read forward, 67 MB read and
// written backward): 13.0 + 4.7 us forward, 17.1 us backward; one wave a token, from
// memory to the losses, 132 us for both.  By counters the vector ALU is active for 8.3
// and 10.5 us of that (exponentials, butterflies), and waves wait for 47% and 58% of
// their time: a token's mask is read before its logits, one step ahead.  Small layers
// are bound by their launches: 16 x 256 tokens of 8 experts 5.6 and 3.6 us.
#include <algorithm>

#include "common.h"

namespace da {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kJoinThreads = 512;
constexpr int kMaxExperts = 1024;
constexpr float kLog2e = 1.44269504088896341f;

struct BalArgs {
  const char* logits;
  const int64_t* index;
  const uint8_t* mask;
  int64_t tokens, batch;
  int64_t row, mask_b, mask_t;  // elements
  int experts, top;
  float* p;        // (batch, chunks, experts): sums of the probabilities
  int32_t* seen;   // (batch, chunks, experts): choices
  float* z;        // (batch, chunks): sums of logsumexp^2
  int32_t* n;      // (batch, chunks): live tokens
  int64_t chunk, chunks;
  float* loss;
  float* z_loss;
  int64_t* counts;
  int64_t* live;
  const float* up;
  const float* up_z;
  char* grad;
  int64_t grad_row;
};

// ---------------------------------------------------------------------------
// One token's logits: lane l of its kL holds runs l, l + kL, ... of V experts.
// ---------------------------------------------------------------------------
template <int DT, int V, int kL, int S>
struct Token {
  static constexpr int ES = Elem<DT>::kBytes;
  u32x4 raw[V == 1 ? (S + 3) / 4 : S];  // V == 1: one value a word

  // Runs past the experts hold -inf: no weight in the largest logit or the sum.  A
  // token without a part holds zeros: its softmax is finite, and not used.
  __device__ void load(const char* row, int experts, int l, bool live) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int e = (l + i * kL) * V;
      const uint32_t none = e < experts ? 0u : DT == DA_F32 ? 0xff800000u : DT == DA_BF16 ? 0xff80ff80u : 0xfc00fc00u;
      if constexpr (V == 1) {
        uint32_t w = ES == 4 ? none : none & 0xffffu;
        if (live && e < experts) w = ES == 4 ? *(const uint32_t*)(row + e * ES) : *(const uint16_t*)(row + e * ES);
        raw[i / 4][i % 4] = w;
      } else {
        raw[i] = u32x4{none, none, none, none};
        if (live && e < experts) raw[i] = ld16(row + e * ES);
      }
    }
  }
  // p = exp(logit - largest); inv = 1 / their sum; returns the logits' logsumexp.
  // The difference is taken first: equal logits of any size, a type's lowest value
  // among them, leave zeros.
  __device__ float softmax(float (&p)[S][V], float& inv) const {
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < S; ++i) {
      if constexpr (V == 1) p[i][0] = Elem<DT>::from_bits(raw[i / 4][i % 4]);
      else unpack16<DT>(raw[i], p[i]);
#pragma unroll
      for (int e = 0; e < V; ++e) top = fmaxf(top, p[i][e]);
    }
    top = lanes_max<kL>(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // All -inf: inf - inf is NaN here, as in a softmax.
        p[i][e] = __builtin_amdgcn_exp2f((p[i][e] - top) * kLog2e);
        sum += p[i][e];
      }
    sum = lanes_sum<kL>(sum);
    inv = __builtin_amdgcn_rcpf(sum);
    return top + __builtin_amdgcn_logf(sum) * 0.69314718055994531f;  // base 2 to natural
  }
};

// A sample's losses from its sums in LDS; every thread of the workgroup calls.
template <int kN>
__device__ void finish(const BalArgs& a, int64_t b, const float* p, const int32_t* seen, float z, int n) {
  __shared__ float terms[kN / kWave];
  const float inv = n ? 1.f / (float)n : 0.f;
  float term = 0.f;
  for (int e = threadIdx.x; e < a.experts; e += kN) {
    a.counts[b * a.experts + e] = seen[e];
    term += ((float)seen[e] * inv) * (p[e] * inv);
  }
  term = wave_sum(term);
  if (threadIdx.x % kWave == 0) terms[threadIdx.x / kWave] = term;
  __syncthreads();
  if (threadIdx.x == 0) {
    float sum = 0.f;
    for (int w = 0; w < kN / kWave; ++w) sum += terms[w];
    a.loss[b] = (float)a.experts * sum;
    a.z_loss[b] = z * inv;
    a.live[b] = n;
  }
}

template <int DT, int V, int kL, int S>
__global__ __launch_bounds__(kThreads) void balance_forward(BalArgs a) {
  constexpr int kTokens = kWave / kL, kStep = kWaves * kTokens;  // tokens of a wave, of a workgroup's step
  extern __shared__ char lds[];
  float* sums = (float*)lds;                            // [kWaves][experts]
  int32_t* seen = (int32_t*)(sums + kWaves * a.experts);  // [experts]
  __shared__ float z_sums[kWaves];
  __shared__ int n_sums[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = lane % kL, sub = lane / kL;
  const int64_t b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  for (int e = tid; e < a.experts; e += kThreads) seen[e] = 0;
  __syncthreads();
  const int64_t t0 = chunk * a.chunk, t1 = min(t0 + a.chunk, a.tokens);
  const uint8_t* mask = a.mask ? a.mask + b * a.mask_b : nullptr;
  float p[S][V], z = 0.f;
  int n = 0;
#pragma unroll
  for (int i = 0; i < S; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) p[i][e] = 0.f;
  int64_t t = t0 + wave * kTokens + sub;
  const char* row = a.logits + (b * a.tokens + t) * a.row * Elem<DT>::kBytes;
  Token<DT, V, kL, S> x;
  bool live = t < t1 && (!mask || mask[t * a.mask_t]);
  x.load(row, a.experts, l, live);
  // The choices meanwhile: one entry a thread.
  const int64_t* index = a.index + (b * a.tokens + t0) * a.top;
  const int entries = (int)(t1 - t0) * a.top;
  for (int at0 = tid; at0 < entries; at0 += 4 * kThreads) {
    int64_t e[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) e[k] = index[min(at0 + k * kThreads, entries - 1)];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int at = at0 + k * kThreads;
      if (at < entries && e[k] >= 0 && e[k] < a.experts && (!mask || mask[(t0 + at / a.top) * a.mask_t]))
        atomicAdd(&seen[e[k]], 1);
    }
  }
  for (int64_t first = t0; first < t1; first += kStep) {
    const Token<DT, V, kL, S> now = x;
    const bool counts = live;
    t += kStep;
    row += kStep * a.row * Elem<DT>::kBytes;
    live = t < t1 && (!mask || mask[t * a.mask_t]);
    x.load(row, a.experts, l, live);
    float q[S][V], inv;
    const float lse = now.softmax(q, inv);
    inv = counts ? inv : 0.f;  // a token without a part reads zeros: finite
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) p[i][e] += q[i][e] * inv;
    z += counts ? lse * lse : 0.f;
    n += counts;
  }
  // The wave's tokens, then the waves.
#pragma unroll
  for (int i = 0; i < S; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
      for (int off = kL; off < kWave; off <<= 1) p[i][e] += __shfl_xor(p[i][e], off, kWave);
      const int at = (l + i * kL) * V + e;
      if (sub == 0 && at < a.experts) sums[wave * a.experts + at] = p[i][e];
    }
#pragma unroll
  for (int off = kL; off < kWave; off <<= 1) {
    z += __shfl_xor(z, off, kWave);
    n += __shfl_xor(n, off, kWave);
  }
  if (lane == 0) z_sums[wave] = z, n_sums[wave] = n;
  __syncthreads();
  z = 0.f, n = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) z += z_sums[w], n += n_sums[w];
  const bool alone = a.chunks == 1;
  for (int e = tid; e < a.experts; e += kThreads) {
    float v = sums[e];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w * a.experts + e];
    if (alone) sums[e] = v;
    else {
      a.p[(int64_t)blockIdx.x * a.experts + e] = v;
      a.seen[(int64_t)blockIdx.x * a.experts + e] = seen[e];
    }
  }
  if (alone) finish<kThreads>(a, b, sums, seen, z, n);  // each thread reads the entries it wrote
  else if (tid == 0) {
    a.z[blockIdx.x] = z;
    a.n[blockIdx.x] = n;
  }
}

// A sample's chunks in order: groups of threads stride over them, then the groups.
__global__ __launch_bounds__(kJoinThreads) void balance_join(BalArgs a) {
  __shared__ float p[kMaxExperts], parts[kJoinThreads];
  __shared__ int32_t seen[kMaxExperts], seen_parts[kJoinThreads];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x, first = b * a.chunks;
  int width = 1;
  while (width < a.experts && width < kJoinThreads) width *= 2;
  const int groups = kJoinThreads / width, x = tid % width;
  for (int e0 = 0; e0 < a.experts; e0 += width) {
    float v = 0.f;
    int32_t k = 0;
    if (e0 + x < a.experts)
#pragma unroll 4
      for (int64_t c = tid / width; c < a.chunks; c += groups) {
        v += a.p[(first + c) * a.experts + e0 + x];
        k += a.seen[(first + c) * a.experts + e0 + x];
      }
    __syncthreads();
    parts[tid] = v;
    seen_parts[tid] = k;
    __syncthreads();
    if (tid < width && e0 + tid < a.experts) {
      for (int g = 1; g < groups; ++g) v += parts[g * width + tid], k += seen_parts[g * width + tid];
      p[e0 + tid] = v;
      seen[e0 + tid] = k;
    }
  }
  float z = 0.f;
  int n = 0;
  for (int64_t c = tid; c < a.chunks; c += kJoinThreads) z += a.z[first + c], n += a.n[first + c];
  __syncthreads();
  parts[tid] = z;
  seen_parts[tid] = n;
  for (int off = kJoinThreads / 2; off > 0; off >>= 1) {
    __syncthreads();
    if (tid < off) parts[tid] += parts[tid + off], seen_parts[tid] += seen_parts[tid + off];
  }
  __syncthreads();
  finish<kJoinThreads>(a, b, p, seen, parts[0], seen_parts[0]);
}

template <int DT, int V, int kL, int S>
__global__ __launch_bounds__(kThreads) void balance_backward(BalArgs a) {
  constexpr int ES = Elem<DT>::kBytes, kTokens = kWave / kL, kStep = kWaves * kTokens;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = lane % kL, sub = lane / kL;
  const int64_t b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  const int64_t t0 = chunk * a.chunk, t1 = min(t0 + a.chunk, a.tokens);
  const uint8_t* mask = a.mask ? a.mask + b * a.mask_b : nullptr;
  int64_t t = t0 + wave * kTokens + sub;
  const char* row = a.logits + (b * a.tokens + t) * a.row * ES;
  char* out = a.grad + (b * a.tokens + t) * a.grad_row * ES;
  const int n = (int)a.live[b];
  Token<DT, V, kL, S> x;
  bool live = t < t1 && (!mask || mask[t * a.mask_t]);
  x.load(row, a.experts, l, live);
  const float inv = n ? 1.f / (float)n : 0.f;
  const float up = (a.up ? a.up[b] : 0.f) * (float)a.experts * inv, up_z = (a.up_z ? a.up_z[b] : 0.f) * 2.f * inv;
  float f[S][V];  // up f
#pragma unroll
  for (int i = 0; i < S; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int at = (l + i * kL) * V + e;
      f[i][e] = at < a.experts ? up * ((float)a.counts[b * a.experts + at] * inv) : 0.f;
    }
  for (int64_t first = t0; first < t1; first += kStep) {
    const Token<DT, V, kL, S> now = x;
    const bool there = t < t1, lives = live;
    char* to = out;
    t += kStep;
    row += kStep * a.row * ES;
    out += kStep * a.grad_row * ES;
    live = t < t1 && (!mask || mask[t * a.mask_t]);
    x.load(row, a.experts, l, live);
    float q[S][V], by, dot = 0.f;
    const float lse = now.softmax(q, by);
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) dot += f[i][e] * q[i][e];
    const float rest = up_z * lse - lanes_sum<kL>(dot) * by;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int e0 = (l + i * kL) * V;
      float g[V];
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = lives ? q[i][e] * by * (f[i][e] + rest) : 0.f;
      if (!there || e0 >= a.experts) continue;
      if constexpr (V == 1) Elem<DT>::store(to, e0, g[0]);
      else {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (DT == DA_F32) w[k] = __float_as_uint(g[k]);
          else w[k] = pack2<DT>(g[2 * k], g[2 * k + 1]);
        }
        st16(to + e0 * ES, w);
      }
    }
  }
}

int check_args(const char* what, int dtype, int64_t batch, int64_t tokens, int experts) {
  if (!valid_dtype(dtype)) return set_error(DA_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || tokens < 0) return set_error(DA_ERR_INVALID, "%s: negative size", what);
  if (experts < 1 || experts > kMaxExperts)
    return set_error(DA_ERR_UNSUPPORTED, "%s: 1 to %d experts, got %d", what, kMaxExperts, experts);
  return DA_OK;
}

// Experts of a run, lanes of a token, runs of a lane.
struct Shape {
  int v, lanes, runs;
};
Shape shape_of(int dtype, int experts, bool aligned) {
  Shape s;
  s.v = dtype == DA_F32 ? 4 : 8;
  if (!aligned || experts % s.v) s.v = 1;
  const int slots = (experts + s.v - 1) / s.v;
  s.lanes = 1;
  while (s.lanes < slots && s.lanes < 64) s.lanes *= 2;
  s.runs = (slots + s.lanes - 1) / s.lanes;
  return s;
}

// Tokens of a workgroup: `least` of its steps, more where the tokens fill `most`
// workgroups; a sample of up to twice
// that stays whole (the forward pass then needs no second launch).
void chunking(BalArgs& a, const Shape& s, int64_t least, int64_t most) {
  const int64_t step = kWaves * kWave / s.lanes;
  const int64_t steps = std::max<int64_t>(least, a.batch * a.tokens / (step * most));
  a.chunk = step * steps;
  if (a.tokens <= 2 * a.chunk) a.chunk = std::max<int64_t>(a.tokens, 1);
  a.chunks = std::max<int64_t>((a.tokens + a.chunk - 1) / a.chunk, 1);
}

size_t partial_bytes(const BalArgs& a) {
  return a.chunks > 1 ? (size_t)(a.batch * a.chunks * (a.experts + 1)) * 8 : 0;
}

// Launches the forward or the backward kernel for a type and a shape.
struct Launch {
  const BalArgs& a;
  bool grad;
  hipStream_t stream;

  template <int DT, int V, int kL, int S>
  void kernel() const {
    const unsigned blocks = (unsigned)(a.batch * a.chunks);
    if (grad) balance_backward<DT, V, kL, S><<<blocks, kThreads, 0, stream>>>(a);
    else balance_forward<DT, V, kL, S><<<blocks, kThreads, (size_t)a.experts * (kWaves + 1) * 4, stream>>>(a);
  }
  template <int DT, int V>
  void lanes(const Shape& s) const {
    if (s.lanes == 1) kernel<DT, V, 1, 1>();
    else if (s.lanes == 2) kernel<DT, V, 2, 1>();
    else if (s.lanes == 4) kernel<DT, V, 4, 1>();
    else if (s.lanes == 8) kernel<DT, V, 8, 1>();
    else if (s.lanes == 16) kernel<DT, V, 16, 1>();
    else if (s.lanes == 32) kernel<DT, V, 32, 1>();
    else if (s.runs == 1) kernel<DT, V, 64, 1>();
    else if (s.runs == 2) kernel<DT, V, 64, 2>();
    else if constexpr (V < 8) {
      if (s.runs <= 4) kernel<DT, V, 64, 4>();
      else if constexpr (V == 1) kernel<DT, V, 64, 16>();
    }
  }
  template <int DT>
  void runs(const Shape& s) const {
    if (s.v == 1) lanes<DT, 1>(s);
    else lanes<DT, 16 / Elem<DT>::kBytes>(s);
  }
  void operator()(int dtype, const Shape& s) const {
    if (dtype == DA_BF16) runs<DA_BF16>(s);
    else if (dtype == DA_F16) runs<DA_F16>(s);
    else runs<DA_F32>(s);
  }
};

// 32 x 4096 tokens of 128 experts: backward 22 us at 4096 workgroups, 17.7 at 2048,
// 19.8 at 512; forward 17.4 at 512, 14.5 at 1024, 13.7 at 2048.
constexpr int64_t kForwardSteps = 4, kForwardBlocks = 2048, kBackwardSteps = 1, kBackwardBlocks = 2048;

}  // namespace
}  // namespace da

using namespace da;

extern "C" {

int da_balance_loss_workspace(int dtype, int64_t batch, int64_t tokens, int experts, size_t* bytes) {
  const char* what = "da_balance_loss_workspace";
  if (!bytes) return set_error(DA_ERR_INVALID, "%s: NULL bytes", what);
  if (int rc = check_args(what, dtype, batch, tokens, experts)) return rc;
  *bytes = 0;
  for (int aligned = 0; aligned < 2; ++aligned) {
    BalArgs a{};
    a.batch = batch, a.tokens = tokens, a.experts = experts;
    chunking(a, shape_of(dtype, experts, aligned), kForwardSteps, kForwardBlocks);
    *bytes = std::max(*bytes, partial_bytes(a));
  }
  return DA_OK;
}

int da_balance_loss(const void* logits, int dtype, int64_t batch, int64_t tokens, int experts, int64_t row_stride,
                    const int64_t* index, int top, const uint8_t* mask, int64_t mask_bstride, int64_t mask_tstride,
                    float* loss, float* z_loss, int64_t* counts, int64_t* live, void* workspace,
                    size_t workspace_bytes, void* stream) {
  const char* what = "da_balance_loss";
  if (int rc = check_args(what, dtype, batch, tokens, experts)) return rc;
  if (top < 0) return set_error(DA_ERR_INVALID, "%s: negative size", what);
  if (!batch) return DA_OK;
  if (!loss || !z_loss || !counts || !live || (tokens && (!logits || (top && !index))))
    return set_error(DA_ERR_INVALID, "%s: NULL pointer", what);
  const int es = (int)elem_bytes(dtype);
  BalArgs a{};
  a.logits = (const char*)logits, a.index = index, a.mask = mask, a.tokens = tokens, a.batch = batch;
  a.row = row_stride, a.mask_b = mask_bstride, a.mask_t = mask_tstride, a.experts = experts, a.top = top;
  a.loss = loss, a.z_loss = z_loss, a.counts = counts, a.live = live;
  const Shape shape = shape_of(dtype, experts, (uintptr_t)logits % 16 == 0 && row_stride * es % 16 == 0);
  chunking(a, shape, kForwardSteps, kForwardBlocks);
  const size_t need = partial_bytes(a);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  // The choices' 32-bit index runs up to four strides past the last of them.
  if (batch * a.chunks > kMaxBlocks || a.chunk * top > 0x7fffffff - 4 * kThreads)
    return set_error(DA_ERR_UNSUPPORTED, "%s: too many tokens", what);
  const int64_t parts = batch * a.chunks;
  a.p = (float*)workspace;
  a.seen = (int32_t*)(a.p + parts * experts);
  a.z = (float*)(a.seen + parts * experts);
  a.n = (int32_t*)(a.z + parts);
  hipStream_t st = (hipStream_t)stream;
  Launch{a, false, st}(dtype, shape);
  if (int rc = check_launch(what)) return rc;
  if (a.chunks == 1) return DA_OK;
  balance_join<<<(unsigned)batch, kJoinThreads, 0, st>>>(a);
  return check_launch(what);
}

int da_balance_loss_grad(const float* up, const float* up_z, const void* logits, int dtype, int64_t batch,
                         int64_t tokens, int experts, int64_t row_stride, const int64_t* counts, const int64_t* live,
                         const uint8_t* mask, int64_t mask_bstride, int64_t mask_tstride, void* grad,
                         int64_t grad_row_stride, void* stream) {
  const char* what = "da_balance_loss_grad";
  if (int rc = check_args(what, dtype, batch, tokens, experts)) return rc;
  if (!batch || !tokens) return DA_OK;
  if (!logits || !counts || !live || !grad) return set_error(DA_ERR_INVALID, "%s: NULL pointer", what);
  const int es = (int)elem_bytes(dtype);
  BalArgs a{};
  a.up = up, a.up_z = up_z, a.logits = (const char*)logits, a.mask = mask, a.tokens = tokens, a.batch = batch;
  a.row = row_stride, a.mask_b = mask_bstride, a.mask_t = mask_tstride, a.experts = experts;
  a.counts = (int64_t*)counts, a.live = (int64_t*)live, a.grad = (char*)grad, a.grad_row = grad_row_stride;
  const bool aligned = ((uintptr_t)logits | (uintptr_t)grad) % 16 == 0 && (row_stride | grad_row_stride) * es % 16 == 0;
  const Shape shape = shape_of(dtype, experts, aligned);
  chunking(a, shape, kBackwardSteps, kBackwardBlocks);
  if (batch * a.chunks > kMaxBlocks) return set_error(DA_ERR_UNSUPPORTED, "%s: too many tokens", what);
  Launch{a, true, (hipStream_t)stream}(dtype, shape);
  return check_launch(what);
}

}  // extern "C"
