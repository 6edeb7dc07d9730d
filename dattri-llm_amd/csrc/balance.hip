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
#include "common.h"

namespace da {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxExperts = 1024;

struct BalArgs {
  const char* logits;
  const int64_t* index;
  const uint8_t* mask;
  int64_t tokens, batch;
  int64_t row, mask_b, mask_t;  // elements
  int experts, top;
  float* partial;      // (batch, chunks, experts + 1): sums of p, sum of logsumexp^2
  int32_t* part_live;  // (batch, chunks, experts + 1): counts, live tokens
  int64_t chunk, chunks;
  float* loss;
  float* z;
  int32_t* counts;
  int32_t* live;
  const float* up;
  const float* up_z;
  char* grad;
  int64_t grad_row;
};

// One token's logits in a wave: lane l holds experts l, l + 64, ...
template <int DT, int S>
struct Token {
  float p[S];
  float lse;
  __device__ void load(const char* row, int experts, int lane) {
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int e = lane + i * kWave;
      p[i] = e < experts ? Elem<DT>::load(row, e) : -__builtin_inff();
      top = fmaxf(top, p[i]);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int e = lane + i * kWave;
      p[i] = e < experts ? expf(p[i] - top) : 0.f;
      sum += p[i];
    }
    sum = wave_sum(sum);
    const float inv = 1.f / sum;
#pragma unroll
    for (int i = 0; i < S; ++i) p[i] *= inv;
    lse = top + logf(sum);
  }
};

template <int DT, int S>
__global__ __launch_bounds__(kThreads) void balance_partials(BalArgs a) {
  extern __shared__ char lds[];
  const int w = a.experts + 1;
  float* sums = (float*)lds;                // [kWaves][w]
  int32_t* seen = (int32_t*)(sums + kWaves * w);  // [w]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  for (int e = tid; e < w; e += kThreads) seen[e] = 0;
  __syncthreads();
  const int64_t t0 = chunk * a.chunk, t1 = min(t0 + a.chunk, a.tokens);
  float p[S], z = 0.f;
#pragma unroll
  for (int i = 0; i < S; ++i) p[i] = 0.f;
  for (int64_t t = t0 + wave; t < t1; t += kWaves) {
    if (a.mask && !a.mask[b * a.mask_b + t * a.mask_t]) continue;
    Token<DT, S> x;
    x.load(a.logits + (b * a.tokens + t) * a.row * Elem<DT>::kBytes, a.experts, lane);
#pragma unroll
    for (int i = 0; i < S; ++i) p[i] += x.p[i];
    z += x.lse * x.lse;
    for (int k = lane; k < a.top; k += kWave) {
      const int64_t e = a.index[(b * a.tokens + t) * a.top + k];
      if (e >= 0 && e < a.experts) atomicAdd(&seen[e], 1);
    }
    if (lane == 0) atomicAdd(&seen[a.experts], 1);
  }
#pragma unroll
  for (int i = 0; i < S; ++i)
    if (lane + i * kWave < a.experts) sums[wave * w + lane + i * kWave] = p[i];
  if (lane == 0) sums[wave * w + a.experts] = z;
  __syncthreads();
  for (int e = tid; e < w; e += kThreads) {
    float v = 0.f;
    for (int k = 0; k < kWaves; ++k) v += sums[k * w + e];
    a.partial[(int64_t)blockIdx.x * w + e] = v;
    a.part_live[(int64_t)blockIdx.x * w + e] = seen[e];
  }
}

__global__ __launch_bounds__(kThreads) void balance_join(BalArgs a) {
  __shared__ float terms[kThreads];
  const int w = a.experts + 1, tid = threadIdx.x;
  const int64_t b = blockIdx.x;
  int n = 0;
  for (int64_t c = 0; c < a.chunks; ++c) n += a.part_live[(b * a.chunks + c) * w + a.experts];
  const float inv = n ? 1.f / (float)n : 0.f;
  float term = 0.f;
  for (int e = tid; e < w; e += kThreads) {
    float v = 0.f;
    int32_t k = 0;
    for (int64_t c = 0; c < a.chunks; ++c) {
      v += a.partial[(b * a.chunks + c) * w + e];
      k += a.part_live[(b * a.chunks + c) * w + e];
    }
    if (e < a.experts) {
      a.counts[b * a.experts + e] = k;
      term += ((float)k * inv) * (v * inv);
    } else {
      a.z[b] = v * inv;
      a.live[b] = k;
    }
  }
  terms[tid] = term;
  __syncthreads();
  for (int off = kThreads / 2; off > 0; off >>= 1) {
    if (tid < off) terms[tid] += terms[tid + off];
    __syncthreads();
  }
  if (tid == 0) a.loss[b] = (float)a.experts * terms[0];
}

template <int DT, int S>
__global__ __launch_bounds__(kThreads) void balance_backward(BalArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t token = (int64_t)blockIdx.x * kWaves + wave;
  if (token >= a.batch * a.tokens) return;
  const int64_t b = token / a.tokens, t = token - b * a.tokens;
  const int n = a.live[b];
  const bool live = n > 0 && (!a.mask || a.mask[b * a.mask_b + t * a.mask_t]);
  char* out = a.grad + token * a.grad_row * Elem<DT>::kBytes;
  if (!live) {
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (lane + i * kWave < a.experts) Elem<DT>::store(out, lane + i * kWave, 0.f);
    return;
  }
  const float inv = 1.f / (float)n;
  Token<DT, S> x;
  x.load(a.logits + token * a.row * Elem<DT>::kBytes, a.experts, lane);
  float f[S], dot = 0.f;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int e = lane + i * kWave;
    f[i] = e < a.experts ? (float)a.counts[b * a.experts + e] * inv : 0.f;
    dot += f[i] * x.p[i];
  }
  dot = wave_sum(dot);
  const float up = (a.up ? a.up[b] : 0.f) * (float)a.experts * inv, up_z = (a.up_z ? a.up_z[b] : 0.f) * 2.f * inv * x.lse;
#pragma unroll
  for (int i = 0; i < S; ++i)
    if (lane + i * kWave < a.experts) Elem<DT>::store(out, lane + i * kWave, x.p[i] * (up * (f[i] - dot) + up_z));
}

int check_args(const char* what, int dtype, int64_t batch, int64_t tokens, int experts) {
  if (!valid_dtype(dtype)) return set_error(DA_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || tokens < 0) return set_error(DA_ERR_INVALID, "%s: negative size", what);
  if (experts < 1 || experts > kMaxExperts)
    return set_error(DA_ERR_UNSUPPORTED, "%s: 1 to %d experts, got %d", what, kMaxExperts, experts);
  return DA_OK;
}

void chunking(BalArgs& a) {
  a.chunk = 64;
  a.chunks = (a.tokens + a.chunk - 1) / a.chunk;
}

}  // namespace
}  // namespace da

using namespace da;

#define DA_BAL_SLOTS(CALL, DT)                       \
  if (experts <= 64) { CALL(DT, 1) }                 \
  else if (experts <= 128) { CALL(DT, 2) }           \
  else if (experts <= 256) { CALL(DT, 4) }           \
  else { CALL(DT, 16) }
#define DA_BAL_DISPATCH(CALL)                              \
  if (dtype == DA_BF16) { DA_BAL_SLOTS(CALL, DA_BF16) }    \
  else if (dtype == DA_F16) { DA_BAL_SLOTS(CALL, DA_F16) } \
  else { DA_BAL_SLOTS(CALL, DA_F32) }

extern "C" {

int da_balance_loss_workspace(int64_t batch, int64_t tokens, int experts, size_t* bytes) {
  if (!bytes) return set_error(DA_ERR_INVALID, "da_balance_loss_workspace: NULL bytes");
  if (int rc = check_args("da_balance_loss_workspace", DA_F32, batch, tokens, experts)) return rc;
  BalArgs a{};
  a.batch = batch, a.tokens = tokens;
  chunking(a);
  *bytes = (size_t)(batch * a.chunks * (experts + 1)) * 8;
  return DA_OK;
}

int da_balance_loss(const void* logits, int dtype, int64_t batch, int64_t tokens, int experts, int64_t row_stride,
                    const int64_t* index, int top, const uint8_t* mask, int64_t mask_bstride, int64_t mask_tstride,
                    float* loss, float* z_loss, int32_t* counts, int32_t* live, void* workspace,
                    size_t workspace_bytes, void* stream) {
  const char* what = "da_balance_loss";
  if (int rc = check_args(what, dtype, batch, tokens, experts)) return rc;
  if (top < 0) return set_error(DA_ERR_INVALID, "%s: negative size", what);
  if (!batch) return DA_OK;
  if (!loss || !z_loss || !counts || !live || (tokens && (!logits || (top && !index))))
    return set_error(DA_ERR_INVALID, "%s: NULL pointer", what);
  BalArgs a{};
  a.logits = (const char*)logits, a.index = index, a.mask = mask, a.tokens = tokens, a.batch = batch;
  a.row = row_stride, a.mask_b = mask_bstride, a.mask_t = mask_tstride, a.experts = experts, a.top = top;
  a.loss = loss, a.z = z_loss, a.counts = counts, a.live = live;
  chunking(a);
  const int64_t entries = batch * a.chunks * (experts + 1);
  if (entries && (!workspace || workspace_bytes < (size_t)entries * 8))
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, (size_t)entries * 8);
  if (batch * a.chunks > 0x7fffffff || batch > 0x7fffffff) return set_error(DA_ERR_UNSUPPORTED, "%s: too many tokens", what);
  a.partial = (float*)workspace;
  a.part_live = (int32_t*)(a.partial + entries);
  hipStream_t st = (hipStream_t)stream;
  if (entries) {
    const unsigned blocks = (unsigned)(batch * a.chunks);
    const size_t lds = (size_t)(experts + 1) * (kWaves + 1) * 4;
#define DA_BAL_FWD(DT, S) balance_partials<DT, S><<<blocks, kThreads, lds, st>>>(a);
    DA_BAL_DISPATCH(DA_BAL_FWD)
#undef DA_BAL_FWD
    if (int rc = check_launch(what)) return rc;
  }
  balance_join<<<(unsigned)batch, kThreads, 0, st>>>(a);
  return check_launch(what);
}

int da_balance_loss_grad(const float* up, const float* up_z, const void* logits, int dtype, int64_t batch,
                         int64_t tokens, int experts, int64_t row_stride, const int32_t* counts, const int32_t* live,
                         const uint8_t* mask, int64_t mask_bstride, int64_t mask_tstride, void* grad,
                         int64_t grad_row_stride, void* stream) {
  const char* what = "da_balance_loss_grad";
  if (int rc = check_args(what, dtype, batch, tokens, experts)) return rc;
  if (!batch || !tokens) return DA_OK;
  if (!logits || !counts || !live || !grad) return set_error(DA_ERR_INVALID, "%s: NULL pointer", what);
  BalArgs a{};
  a.up = up, a.up_z = up_z, a.logits = (const char*)logits, a.mask = mask, a.tokens = tokens, a.batch = batch;
  a.row = row_stride, a.mask_b = mask_bstride, a.mask_t = mask_tstride, a.experts = experts;
  a.counts = (int32_t*)counts, a.live = (int32_t*)live, a.grad = (char*)grad, a.grad_row = grad_row_stride;
  const int64_t blocks = (batch * tokens + kWaves - 1) / kWaves;
  if (blocks > 0x7fffffff) return set_error(DA_ERR_UNSUPPORTED, "%s: too many tokens", what);
  hipStream_t st = (hipStream_t)stream;
#define DA_BAL_BWD(DT, S) balance_backward<DT, S><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  DA_BAL_DISPATCH(DA_BAL_BWD)
#undef DA_BAL_BWD
  return check_launch(what);
}

}  // extern "C"
