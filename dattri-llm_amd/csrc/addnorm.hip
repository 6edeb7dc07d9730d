// The residual's addition with the RMS norm that follows it, and their gradients.
//
// Per live token, x and residual of d entries (a masked token's rows are zero and add
// nothing to a gradient):
//
//   total = round(x + residual),   r = (mean(total^2) + eps)^(-1/2)
//   out_i = total_i w_i r
//
// The norm is that of total as it is returned, so that the backward pass, which has
// only total, differentiates the same function.  In 8 bits (e4m3) out is divided by a
// scale, the row's (or each 128 entries') largest |out_i| / 448.  Backward, with
// t_i = total_i r and h = g w:
//
//   dx = dresidual = r (h - t mean(h t)) + g_total,   dw[sample] = sum over tokens of g t
//
// A row is held in registers by one wave, four, eight or sixteen, S runs of 16 bytes a lane, so
// that every value is read once.  Weights stay in registers while the waves go over
// their rows, and the next row's loads are under way while one is computed.  The weight
// gradient adds up in registers too: a workgroup takes a chunk of one sample's tokens, and
// a second launch joins a sample's chunks in order.
//
// Everything between the loads and a result is in fp32 and rounded once: total, then out from
// total as rounded; dx; out in 8 bits from its fp32 value, not from a rounded one.  out is (total w)
// r: a product of two 16-bit values is exact in fp32, which leaves one rounding (8-bit values on the
// wrong side of a border: an error of 8.0e-4 in place of 8.9e-4 for (total r) w at the size below).
//
// HBM bounds both.  8 x 2048 rows of 4096 in bf16: 94 us forward (537 MB, 5.7 TB/s), 74 with
// out in 8 bits (470 MB, 6.4 TB/s), 101 backward (537 MB, 5.3 TB/s).
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace da {
namespace {

constexpr int kMaxRuns = 4096;        // runs of 16 bytes of a row
constexpr float kMost8 = 448.f;        // the largest e4m3 value
constexpr float kLeast8 = 0x1p-100f;   // runs below it become zeros with scale 1
constexpr int kRun8 = 128;             // entries of a scaled run

enum { kPlain = 0, kRowScale = 1, kRunScale = 2 };

struct AddNormArgs {
  const char* x;         // backward: the output's gradient
  const char* residual;  // backward: total's gradient; NULL: none
  const char* total_in;  // backward
  const char* weight;
  const uint8_t* mask;
  char* out;             // backward: dx
  char* total;
  float* scales;
  float* partial;        // (batch, chunks, d)
  int64_t tokens, rows;
  int64_t x_b, x_t, r_b, r_t, h_b, h_t, mask_b, mask_t;  // elements
  int64_t chunk, chunks;
  int64_t step_b, step_t;  // forward: the workgroups' rows in one step, as samples and tokens
  int d, runs;           // runs: scales of a row
  float eps;
};

// Entries e0 .. e0 + kVec of a row of d.  The run that holds a row's last entries is read
// from where it ends with the row, and brought to its place by settle() when it is used, so
// that no load has a branch behind it; runs past the end are zero.  kShort: rows of less than
// a run, entry by entry.
template <int DT, bool kStream, bool kShort>
__device__ __forceinline__ u32x4 load_run(const char* row, int e0, int d) {
  constexpr int ES = Elem<DT>::kBytes, V = Elem<DT>::kVec;
  u32x4 v = {0, 0, 0, 0};
  if constexpr (kShort) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (e0 + e >= d) continue;
      if constexpr (ES == 4) v[e] = *(const uint32_t*)(row + (e0 + e) * 4);
      else v[e / 2] |= (uint32_t)(*(const uint16_t*)(row + (e0 + e) * 2)) << (16 * (e % 2));
    }
  } else if (e0 < d) {
    const char* p = row + (int64_t)min(e0, d - V) * ES;
    v = kStream ? ld16_any_nt<ES>(p) : ld16_any<ES>(p);
  }
  return v;
}

template <int DT, bool kShort>
__device__ __forceinline__ u32x4 settle(u32x4 v, int e0, int d) {
  constexpr int ES = Elem<DT>::kBytes, V = Elem<DT>::kVec;
  const int skip = (V - d % V) % V;  // entries before the run's first
  if (kShort || skip == 0) return v;
  u32x4 w = v;
  if (skip * ES & 8) w = u32x4{w[2], w[3], 0, 0};
  if (skip * ES & 4) w = u32x4{w[1], w[2], w[3], 0};
  if (skip * ES & 2) w = u32x4{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16};
  return e0 < d && e0 + V > d ? w : v;
}

template <int DT, bool kStream = false>
__device__ __forceinline__ void store_run(char* row, int e0, int d, u32x4 v) {
  constexpr int ES = Elem<DT>::kBytes, V = Elem<DT>::kVec;
  if (e0 + V <= d) {
    if constexpr (kStream) st16_any_nt<ES>(row + (int64_t)e0 * ES, v);
    else st16_any<ES>(row + (int64_t)e0 * ES, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (e0 + e >= d) continue;
    if constexpr (ES == 4) *(uint32_t*)(row + (int64_t)(e0 + e) * 4) = v[e];
    else *(uint16_t*)(row + (int64_t)(e0 + e) * 2) = (uint16_t)(v[e / 2] >> (16 * (e % 2)));
  }
}

template <int DT>
__device__ __forceinline__ u32x4 pack16(const float* f) {
  u32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (DT == DA_F32) v[k] = __float_as_uint(f[k]);
    else v[k] = pack2<DT>(f[2 * k], f[2 * k + 1]);
  }
  return v;
}

// x / scale to the nearest: one step of Markstein's correction of a product with the nearest to
// 1 / scale.  That product alone is off by up to a unit more, and what lies half way between two
// 8-bit values goes to the wrong one.  (448 scale is the largest |x|, and scale 2^-109 and more: only
// quotients next to zero have a remainder that is not exact.)  Zeros keep their sign; with an
// infinite scale the finite are zero and the infinite NaN.
struct Quotient {
  float scale, by;
  __device__ __forceinline__ explicit Quotient(float s) : scale(s < __builtin_inff() ? s : 1.f), by(1.f / s) {}
  __device__ __forceinline__ float operator()(float x) const {
    const float q = x * by;
    return copysignf(fmaf(fmaf(-q, scale, x), by, q), x);
  }
};

// kVec entries of out in 8 bits.
template <int V>
__device__ __forceinline__ void store_run8(char* row, int e0, int d, const float* f) {
  typedef uint32_t u32_1 __attribute__((aligned(1)));
  typedef uint32_t u32x2_1 __attribute__((ext_vector_type(2), aligned(1)));
  uint32_t w[V / 4];
#pragma unroll
  for (int k = 0; k < V / 4; ++k) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k], f[4 * k + 1], 0, false);
    w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k + 2], f[4 * k + 3], p, true);
  }
  if (e0 + V <= d) {
    if constexpr (V == 8) *(u32x2_1*)(row + e0) = u32x2_1{w[0], w[1]};
    else *(u32_1*)(row + e0) = w[0];
    return;
  }
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (e0 + e < d) row[e0 + e] = (char)(w[e / 4] >> (8 * (e % 4)));
}

// Weights of a lane's runs, in the rows' type or in fp32.
template <int DT, bool kWide, int S, bool kShort>
struct Weights {
  static constexpr int V = Elem<DT>::kVec, N = kWide && DT != DA_F32 ? 2 : 1;
  u32x4 raw[S][N];
  __device__ void load(const char* w, int first, int step, int d) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int e0 = (first + i * step) * V;
      if constexpr (N == 2) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          raw[i][k] = settle<DA_F32, kShort>(load_run<DA_F32, false, kShort>(w, e0 + 4 * k, d), e0 + 4 * k, d);
      } else {
        raw[i][0] = settle<DT, kShort>(load_run<DT, false, kShort>(w, e0, d), e0, d);
      }
    }
  }
  __device__ void get(int i, float* f) const {
    if constexpr (N == 2) {
      unpack16<DA_F32>(raw[i][0], f);
      unpack16<DA_F32>(raw[i][1], f + 4);
    } else {
      unpack16<DT>(raw[i][0], f);
    }
  }
};

// Over the NW waves of a row, the result in all of them.  `slot` alternates, so that one
// barrier a call is enough: a slot is written again only past the next call's barrier.
template <int NW, class Op>
__device__ __forceinline__ float over_row(float v, float (*parts)[NW], int& slot, Op op) {
  v = over_lanes<64>(v, op);
  if constexpr (NW > 1) {
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) parts[slot][wave] = v;
    __syncthreads();
    v = parts[slot][0];
#pragma unroll
    for (int w = 1; w < NW; ++w) v = op(v, parts[slot][w]);
    slot ^= 1;
  }
  return v;
}
// Two sums at once.
template <int NW>
__device__ __forceinline__ void sums_over_row(float& u, float& v, float2 (*parts)[NW], int& slot) {
  u = lanes_sum<64>(u);
  v = lanes_sum<64>(v);
  if constexpr (NW > 1) {
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) parts[slot][wave] = float2{u, v};
    __syncthreads();
    u = parts[slot][0].x, v = parts[slot][0].y;
#pragma unroll
    for (int w = 1; w < NW; ++w) u += parts[slot][w].x, v += parts[slot][w].y;
    slot ^= 1;
  }
}
__device__ __forceinline__ float add_f(float a, float b) { return a + b; }
__device__ __forceinline__ float max_f(float a, float b) { return fmaxf(a, b); }

// ---------------------------------------------------------------------------
// Forward.  A workgroup is NW waves on one row, or four waves on a row each.
// ---------------------------------------------------------------------------
template <int DT, bool kWide, int NW, int S, int kOut, bool kStream, bool kShort>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * kWave) void add_norm_forward(AddNormArgs a) {
  constexpr int ES = Elem<DT>::kBytes, V = Elem<DT>::kVec, kStep = NW * kWave;
  constexpr int kRows = NW == 1 ? 4 : 1;  // rows of a workgroup
  __shared__ float parts[2][NW];
  const int at = NW == 1 ? threadIdx.x % kWave : threadIdx.x;
  int slot = 0;
  Weights<DT, kWide, S, kShort> w;
  w.load(a.weight, at, kStep, a.d);
  const int64_t stride = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + (NW == 1 ? threadIdx.x / kWave : 0);
  u32x4 x[S], r[S];
  bool live = false;
  int64_t b = row / a.tokens, t = row - b * a.tokens;
  auto fetch = [&](int64_t to) {
    live = to < a.rows && (!a.mask || a.mask[b * a.mask_b + t * a.mask_t]);
    const char* xr = a.x + (b * a.x_b + t * a.x_t) * ES;
    const char* rr = a.residual + (b * a.r_b + t * a.r_t) * ES;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      x[i] = r[i] = u32x4{0, 0, 0, 0};
      if (live) x[i] = load_run<DT, kStream, kShort>(xr, (at + i * kStep) * V, a.d);
    }
    if (a.residual && live)
#pragma unroll
      for (int i = 0; i < S; ++i) r[i] = load_run<DT, kStream, kShort>(rr, (at + i * kStep) * V, a.d);
    b += a.step_b;
    t += a.step_t;
    if (t >= a.tokens) t -= a.tokens, ++b;
  };
  fetch(row);
  for (; row < a.rows; row += stride) {
    const bool now = live;  // a masked row is zero whatever the weights hold
    u32x4 h[S];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      float p[V], q[V];
      const int e0 = (at + i * kStep) * V;
      unpack16<DT>(settle<DT, kShort>(x[i], e0, a.d), p);
      unpack16<DT>(settle<DT, kShort>(r[i], e0, a.d), q);
#pragma unroll
      for (int e = 0; e < V; ++e) p[e] += q[e];
      h[i] = pack16<DT>(p);
      unpack16<DT>(h[i], p);
#pragma unroll
      for (int e = 0; e < V; ++e) sum += p[e] * p[e];
    }
    fetch(row + stride);
    sum = over_row<NW>(sum, parts, slot, add_f);
    const float rstd = 1.f / __builtin_sqrtf(sum / (float)a.d + a.eps);
    char* total = a.total ? a.total + row * a.d * ES : nullptr;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int e0 = (at + i * kStep) * V;
      if (total) store_run<DT, kStream>(total, e0, a.d, h[i]);
      float p[V], f[V];
      unpack16<DT>(h[i], p);
      w.get(i, f);
#pragma unroll
      for (int e = 0; e < V; ++e) p[e] = now ? p[e] * f[e] * rstd : 0.f;
      if constexpr (kOut == kPlain) {
        store_run<DT, kStream>(a.out + row * a.d * ES, e0, a.d, pack16<DT>(p));
      } else {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) top = fmaxf(top, fabsf(p[e]));
        if constexpr (kOut == kRowScale) {
          most = fmaxf(most, top);
        } else {
          constexpr int kLanes = kRun8 / V;  // lanes of a run: consecutive runs of 16 bytes
          top = lanes_max<kLanes>(top);
          const float scale = top < kLeast8 ? 1.f : top / kMost8;
          const Quotient of(scale);
#pragma unroll
          for (int e = 0; e < V; ++e) p[e] = of(p[e]);
          store_run8<V>(a.out + row * a.d, e0, a.d, p);
          if (at % kLanes == 0 && e0 < a.d) a.scales[row * a.runs + e0 / kRun8] = scale;
        }
      }
    }
    if constexpr (kOut == kRowScale) {
      most = over_row<NW>(most, parts, slot, max_f);
      const float scale = most < kLeast8 ? 1.f : most / kMost8;
      const Quotient of(scale);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        float p[V], f[V];
        unpack16<DT>(h[i], p);
        w.get(i, f);
#pragma unroll
        for (int e = 0; e < V; ++e) p[e] = now ? of(p[e] * f[e] * rstd) : 0.f;
        store_run8<V>(a.out + row * a.d, (at + i * kStep) * V, a.d, p);
      }
      if (at == 0) a.scales[row] = scale;
    }
  }
}

// ---------------------------------------------------------------------------
// Backward.  Workgroup (sample, chunk): its tokens' dx, and their sum of g t.
// ---------------------------------------------------------------------------
template <int DT, bool kWide, int NW, int S, bool kStream, bool kShort>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * kWave, S <= 2 ? 2 : 1) void add_norm_backward(AddNormArgs a) {
  constexpr int ES = Elem<DT>::kBytes, V = Elem<DT>::kVec, kStep = NW * kWave;
  constexpr int kRows = NW == 1 ? 4 : 1;
  __shared__ float2 parts[2][NW];
  __shared__ float sums[NW == 1 ? 3 * S * V * kWave : 1];
  const int at = NW == 1 ? threadIdx.x % kWave : threadIdx.x, wave = threadIdx.x / kWave;
  int slot = 0;
  const int64_t b = blockIdx.x / a.chunks, c = blockIdx.x - b * a.chunks;
  const int64_t t1 = min((c + 1) * a.chunk, a.tokens);
  int64_t t = c * a.chunk + (NW == 1 ? wave : 0);
  Weights<DT, kWide, S, kShort> w;
  w.load(a.weight, at, kStep, a.d);
  const uint8_t* mask = a.mask ? a.mask + b * a.mask_b : nullptr;
  const char* g0 = a.x + b * a.x_b * ES;
  const char* gt0 = a.residual ? a.residual + b * a.r_b * ES : nullptr;
  const char* h0 = a.total_in + b * a.h_b * ES;
  u32x4 g[S], gt[S], h[S];
  bool live = false;
  auto fetch = [&](int64_t to) {
    live = to < t1 && (!mask || mask[to * a.mask_t]);
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int e0 = (at + i * kStep) * V;
      g[i] = gt[i] = h[i] = u32x4{0, 0, 0, 0};
      if (live) {
        h[i] = load_run<DT, kStream, kShort>(h0 + to * a.h_t * ES, e0, a.d);
        g[i] = load_run<DT, kStream, kShort>(g0 + to * a.x_t * ES, e0, a.d);
        if (gt0) gt[i] = load_run<DT, kStream, kShort>(gt0 + to * a.r_t * ES, e0, a.d);
      }
    }
  };
  float dw[S][V];
#pragma unroll
  for (int i = 0; i < S; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = 0.f;
  fetch(t);
  for (; t < t1; t += kRows) {
    const bool now = live;
    float sq = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int e0 = (at + i * kStep) * V;
      h[i] = settle<DT, kShort>(h[i], e0, a.d);
      g[i] = settle<DT, kShort>(g[i], e0, a.d);
      gt[i] = settle<DT, kShort>(gt[i], e0, a.d);
      float hf[V], gf[V], wf[V];
      unpack16<DT>(h[i], hf);
      unpack16<DT>(g[i], gf);
      w.get(i, wf);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        sq += hf[e] * hf[e];
        dot += gf[e] * wf[e] * hf[e];
      }
    }
    sums_over_row<NW>(sq, dot, parts, slot);
    const float rstd = now ? 1.f / __builtin_sqrtf(sq / (float)a.d + a.eps) : 0.f;
    const float mean = dot * rstd / (float)a.d * rstd;  // mean(h t) r
    char* out = a.out + (b * a.tokens + t) * a.d * ES;
    u32x4 dx[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      float hf[V], gf[V], wf[V], tf[V];
      unpack16<DT>(h[i], hf);
      unpack16<DT>(g[i], gf);
      unpack16<DT>(gt[i], tf);
      w.get(i, wf);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x_hat = hf[e] * rstd;
        dw[i][e] += gf[e] * x_hat;
        tf[e] = now ? tf[e] + rstd * (gf[e] * wf[e]) - x_hat * mean : 0.f;
      }
      dx[i] = pack16<DT>(tf);
    }
    fetch(t + kRows);
#pragma unroll
    for (int i = 0; i < S; ++i) store_run<DT, kStream>(out, (at + i * kStep) * V, a.d, dx[i]);
  }
  if (!a.partial) return;
  if constexpr (NW == 1) {  // the four waves, in order
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (wave) sums[((wave - 1) * S * V + i * V + e) * kWave + at] = dw[i][e];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e)
#pragma unroll
        for (int v = 0; v < 3; ++v) dw[i][e] += sums[(v * S * V + i * V + e) * kWave + at];
  }
  float* to = a.partial + (int64_t)blockIdx.x * a.d;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int e0 = (at + i * kStep) * V;
#pragma unroll
    for (int k = 0; k < V; k += 4)
      store_run<DA_F32>((char*)to, e0 + k, a.d, pack16<DA_F32>(&dw[i][k]));
  }
}

// dw[b, e]: a sample's chunks in order.  16 groups of threads stride over them, then the groups.
constexpr int kJoinGroups = 16, kJoinWidth = 64;
__global__ __launch_bounds__(kJoinGroups * kJoinWidth) void add_norm_join(const float* partial, float* out,
                                                                          int64_t chunks, int d) {
  __shared__ float parts[kJoinGroups][kJoinWidth];
  const int x = threadIdx.x % kJoinWidth, group = threadIdx.x / kJoinWidth;
  const int e = blockIdx.x * kJoinWidth + x;
  const int64_t b = blockIdx.y;
  float v = 0.f;
  if (e < d)
#pragma unroll 4
    for (int64_t c = group; c < chunks; c += kJoinGroups) v += partial[(b * chunks + c) * d + e];
  parts[group][x] = v;
  __syncthreads();
  if (group || e >= d) return;
#pragma unroll
  for (int k = 1; k < kJoinGroups; ++k) v += parts[k][x];
  out[b * d + e] = v;
}

// ---------------------------------------------------------------------------
// Launches.
// ---------------------------------------------------------------------------
struct Plan {
  int waves, runs;  // waves of a row, runs of 16 bytes a lane
  bool small;       // rows of less than a run
};

// Four tensors that together take half the last-level cache (256 MB) and more are read and
// written past it (8 x 2048 rows of 4096: 94 us forward and 116 backward, through it 101 and
// 122; smaller ones are left to it, for whoever reads them next).
constexpr int64_t kStreamBytes = 128 << 20;

// As many waves as leave a lane two runs where the rows are wide enough; one run in the
// backward pass, whose sums and three operands fill the registers (rows of 4096 bf16: 105 us
// with eight waves, 109 with four).
Plan plan(int64_t d, int dtype, bool backward) {
  const int64_t vec = dtype == DA_F32 ? 4 : 8, n = (d + vec - 1) / vec;
  if (d < vec) return {1, 1, true};
  if (n <= 64) return {1, 1};
  if (n <= 128) return {1, 2};
  if (n <= 256) return {4, 1};
  if (n <= 512) return backward ? Plan{8, 1} : Plan{4, 2};
  if (n <= 1024) return {4, 4};
  if (n <= 2048) return {8, 4};
  return {16, 4};
}

// Chunks of a sample's tokens: four workgroups of four waves a CU, or two larger ones (twice
// as many: 105 us in place of 101 for 8 x 2048 rows of 4096), no chunk under 8 tokens.
int chunks_of(int64_t batch, int64_t tokens, int64_t d, int dtype, int64_t* chunk, int64_t* chunks) {
  int64_t cus;
  const int rc = device_cu_count(&cus);
  if (rc) return rc;
  const int waves = plan(d, dtype, true).waves;
  const int64_t least = waves == 1 ? 32 : 8;
  const int64_t want = std::max<int64_t>(1, (waves < 8 ? 4 : 2) * cus / std::max<int64_t>(batch, 1));
  *chunk = std::max(least, (tokens + want - 1) / want);
  *chunks = std::max<int64_t>(1, (tokens + *chunk - 1) / *chunk);
  return DA_OK;
}

int check_rows(const char* what, int dtype, int weight_dtype, int64_t batch, int64_t tokens, int64_t d) {
  if (!valid_dtype(dtype)) return set_error(DA_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  if (weight_dtype != dtype && weight_dtype != DA_F32)
    return set_error(DA_ERR_UNSUPPORTED, "%s: weights are in the rows' dtype or fp32, got %d", what, weight_dtype);
  if (batch < 0 || tokens < 0) return set_error(DA_ERR_INVALID, "%s: negative size", what);
  const int most = kMaxRuns * 16 / (int)elem_bytes(dtype);
  if (d < 1 || d > most)
    return set_error(DA_ERR_UNSUPPORTED, "%s: rows of 1 to %d entries, got %lld", what, most, (long long)d);
  if (tokens && batch > INT64_MAX / (64 * (int64_t)most) / tokens)
    return set_error(DA_ERR_UNSUPPORTED, "%s: too many rows", what);
  return DA_OK;
}

// f(waves, runs, small) with all as constants.
template <class F>
int by_plan(const Plan& p, F g) {
  const auto f = [&](auto waves, auto runs) { return g(waves, runs, std::false_type{}); };
  if (p.small) return g(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{}, std::true_type{});
  if (p.waves == 1) return p.runs == 1 ? f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{})
                                       : f(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
  if (p.waves == 16) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
  if (p.waves == 8)
    return p.runs == 1 ? f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{})
                       : f(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
  if (p.runs == 1) return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
  if (p.runs == 2) return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
}

// f(dtype, fp32 weights) with both as constants.
template <class F>
int by_types(int dtype, int weight_dtype, F f) {
  const bool wide = weight_dtype == DA_F32;
#define DA_TYPES(DT) f(std::integral_constant<int, DT>{}, std::true_type{})
  if (dtype == DA_F32) return DA_TYPES(DA_F32);
  if (dtype == DA_BF16)
    return wide ? DA_TYPES(DA_BF16) : f(std::integral_constant<int, DA_BF16>{}, std::false_type{});
  return wide ? DA_TYPES(DA_F16) : f(std::integral_constant<int, DA_F16>{}, std::false_type{});
#undef DA_TYPES
}

}  // namespace
}  // namespace da

extern "C" {

int da_add_rms_norm(const void* x, const void* residual, const void* weight, int dtype, int weight_dtype,
                    int64_t batch, int64_t tokens, int64_t d, int64_t x_bstride, int64_t x_tstride,
                    int64_t r_bstride, int64_t r_tstride, const uint8_t* mask, int64_t mask_bstride,
                    int64_t mask_tstride, float eps, int quantize, void* out, void* total, float* scales,
                    void* stream) {
  using namespace da;
  const int rc = check_rows("da_add_rms_norm", dtype, weight_dtype, batch, tokens, d);
  if (rc) return rc;
  if (quantize < kPlain || quantize > kRunScale)
    return set_error(DA_ERR_INVALID, "da_add_rms_norm: quantize is 0, 1 (a scale a row) or 2 (each 128 entries)");
  if (batch == 0 || tokens == 0) return DA_OK;
  if (!x || !weight || !out || (quantize && !scales)) return set_error(DA_ERR_INVALID, "da_add_rms_norm: NULL pointer");
  int64_t cus;
  if (const int err = device_cu_count(&cus)) return err;
  AddNormArgs a = {};
  a.x = (const char*)x;
  a.residual = (const char*)residual;
  a.weight = (const char*)weight;
  a.mask = mask;
  a.out = (char*)out;
  a.total = (char*)total;
  a.scales = scales;
  a.tokens = tokens;
  a.rows = batch * tokens;
  a.x_b = x_bstride, a.x_t = x_tstride, a.r_b = r_bstride, a.r_t = r_tstride;
  a.mask_b = mask_bstride, a.mask_t = mask_tstride;
  a.d = (int)d;
  a.runs = quantize == kRunScale ? (int)((d + kRun8 - 1) / kRun8) : 1;
  a.eps = eps;
  const hipStream_t st = (hipStream_t)stream;
  const Plan p = plan(d, dtype, false);
  return by_types(dtype, weight_dtype, [&](auto dt, auto wide) {
    return by_plan(p, [&](auto nw, auto s, auto small) {
      constexpr int DT = decltype(dt)::value, NW = decltype(nw)::value, S = decltype(s)::value;
      constexpr bool kWide = decltype(wide)::value, kShort = decltype(small)::value;
      const int64_t groups = NW == 1 ? (a.rows + 3) / 4 : a.rows;
      const unsigned grid = (unsigned)std::min<int64_t>(groups, cus * (NW > 4 ? 2 : 8));
      const int64_t step = (int64_t)grid * (NW == 1 ? 4 : 1);
      a.step_b = step / tokens, a.step_t = step % tokens;
      constexpr int kN = NW == 1 ? 256 : NW * kWave;
      const auto launch = [&](auto stream) {
        constexpr bool kStream = decltype(stream)::value;
        if (quantize == kPlain) add_norm_forward<DT, kWide, NW, S, kPlain, kStream, kShort><<<grid, kN, 0, st>>>(a);
        else if (quantize == kRowScale) add_norm_forward<DT, kWide, NW, S, kRowScale, kStream, kShort><<<grid, kN, 0, st>>>(a);
        else add_norm_forward<DT, kWide, NW, S, kRunScale, kStream, kShort><<<grid, kN, 0, st>>>(a);
      };
      if (!kShort && a.rows * d * (int64_t)elem_bytes(dtype) > kStreamBytes / 4) launch(std::bool_constant<!kShort>{});
      else launch(std::false_type{});
      return check_launch("da_add_rms_norm");
    });
  });
}

int da_add_rms_norm_grad_workspace(int dtype, int64_t batch, int64_t tokens, int64_t d, size_t* bytes) {
  using namespace da;
  if (!bytes) return set_error(DA_ERR_INVALID, "da_add_rms_norm_grad_workspace: NULL pointer");
  *bytes = 0;
  int rc = check_rows("da_add_rms_norm_grad_workspace", dtype, dtype, batch, tokens, d);
  if (rc || batch == 0 || tokens == 0) return rc;
  int64_t chunk, chunks;
  rc = chunks_of(batch, tokens, d, dtype, &chunk, &chunks);
  if (rc == DA_OK && chunks > 1) *bytes = (size_t)(batch * chunks * d) * sizeof(float);
  return rc;
}

int da_add_rms_norm_grad(const void* g, const void* g_total, const void* total, const void* weight, int dtype,
                         int weight_dtype, int64_t batch, int64_t tokens, int64_t d, int64_t g_bstride,
                         int64_t g_tstride, int64_t gt_bstride, int64_t gt_tstride, int64_t total_bstride,
                         int64_t total_tstride, const uint8_t* mask, int64_t mask_bstride, int64_t mask_tstride,
                         float eps, void* dx, float* weight_grad, void* workspace, size_t workspace_bytes,
                         void* stream) {
  using namespace da;
  int rc = check_rows("da_add_rms_norm_grad", dtype, weight_dtype, batch, tokens, d);
  if (rc) return rc;
  if (batch == 0) return DA_OK;
  const hipStream_t st = (hipStream_t)stream;
  if (tokens == 0) return weight_grad ? zero_f32_2d(weight_grad, batch, d, d, st) : DA_OK;
  if (!g || !total || !weight || !dx) return set_error(DA_ERR_INVALID, "da_add_rms_norm_grad: NULL pointer");
  AddNormArgs a = {};
  rc = chunks_of(batch, tokens, d, dtype, &a.chunk, &a.chunks);
  if (rc) return rc;
  if (batch > kMaxBlocks / 4 / a.chunks) return set_error(DA_ERR_UNSUPPORTED, "da_add_rms_norm_grad: too many samples");
  const size_t need = weight_grad && a.chunks > 1 ? (size_t)(batch * a.chunks * d) * sizeof(float) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "da_add_rms_norm_grad: workspace of %zu bytes needed", need);
  a.x = (const char*)g;
  a.residual = (const char*)g_total;
  a.total_in = (const char*)total;
  a.weight = (const char*)weight;
  a.mask = mask;
  a.out = (char*)dx;
  a.partial = need ? (float*)workspace : weight_grad;
  a.tokens = tokens;
  a.x_b = g_bstride, a.x_t = g_tstride, a.r_b = gt_bstride, a.r_t = gt_tstride;
  a.h_b = total_bstride, a.h_t = total_tstride, a.mask_b = mask_bstride, a.mask_t = mask_tstride;
  a.d = (int)d;
  a.eps = eps;
  rc = by_types(dtype, weight_dtype, [&](auto dt, auto wide) {
    return by_plan(plan(d, dtype, true), [&](auto nw, auto s, auto small) {
      constexpr int NW = decltype(nw)::value;
      constexpr bool kShort = decltype(small)::value;
      const auto launch = [&](auto stream) {
        add_norm_backward<decltype(dt)::value, decltype(wide)::value, NW, decltype(s)::value, decltype(stream)::value,
                          kShort><<<(unsigned)(batch * a.chunks), NW == 1 ? 256 : NW * kWave, 0, st>>>(a);
      };
      if (!kShort && batch * tokens * d * (int64_t)elem_bytes(dtype) > kStreamBytes / 4) launch(std::bool_constant<!kShort>{});
      else launch(std::false_type{});
      return check_launch("da_add_rms_norm_grad");
    });
  });
  if (rc || !need) return rc;
  // grid.y holds 65535 samples at most
  for (int64_t b = 0; b < batch; b += 65535) {
    const dim3 grid((unsigned)((d + kJoinWidth - 1) / kJoinWidth), (unsigned)std::min<int64_t>(65535, batch - b));
    add_norm_join<<<grid, kJoinGroups * kJoinWidth, 0, st>>>(a.partial + b * a.chunks * d, weight_grad + b * d,
                                                            a.chunks, (int)d);
  }
  return check_launch("da_add_rms_norm_grad");
}

}  // extern "C"
