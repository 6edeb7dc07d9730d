// Log probabilities of given tokens with the entropy and the most likely
// alternatives, and the logits' gradient.
//
// Per live token, z = logits / temperature, m its largest, d_v = z_v - m:
//
//   lse = m + log sum e^d,   logprob = z_target - lse,
//   entropy = log sum e^d - (sum d e^d) / (sum e^d)
//   dlogits_v = (up [v = target] + p_v (up_lse - up - up_h (log p_v + entropy))) / temperature
//
// (a masked token: zeros; a target outside the vocabulary: none, logprob 0.)  One pass
// over the row: each thread keeps the running maximum, sum and weighted sum of its runs of
// 16 bytes, with one rescaling a batch of runs.  A row is one workgroup's,
// or with few rows cut into parts that a second launch joins.
//
// The alternatives need no second pass over the row.  Every thread knows its largest
// value and the batch of runs that has it first, so the k-th largest of 64 groups' maxima is
// a bound that at least k entries reach; the runs of the threads whose maximum may reach
// it, few of them, are read again by all threads, and what reaches it goes to LDS.  Entries
// are ordered by (value, lower index first), as one 64-bit key each, so that no two are
// alike and their ranks are their places.
//
// Logits are read in their type and everything from there on is fp32, differences from the row's
// maximum; only the gradient is rounded, once.  It takes the row's lse as the forward call returned
// it, and sums a row again whose lse is large (kFar).
//
// 2 x 1024 rows of 128256 in bf16 with five alternatives take 92 us (525 MB, 5.7 TB/s; an exponential
// and some eight instructions an entry nearly fill the vector unit), 16 rows with twenty 9 and 6 us;
// 4 x 1024 rows forward and backward 540 us (3.15 GB, 5.8 TB/s).
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace da {
namespace {

constexpr int kMaxTop = 32;
constexpr int kGroups = 64;       // groups whose maxima bound the alternatives: kMaxTop and more
constexpr int kCandidates = 2048; // entries that reach the bound, at most: past it the row is searched
constexpr int kBatch = 4;         // runs of 16 bytes a thread has under way
constexpr int64_t kLastLevel = 256 << 20;  // bytes of the last-level cache
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kFloor = -3.4028234663852886e38f;  // the maximum where there is none or -inf: the lowest value

struct LpArgs {
  const char* logits;
  const int64_t* targets;
  const uint8_t* mask;
  int64_t tokens, rows, vocab;
  int64_t l_b, l_t, t_b, t_t, m_b, m_t;  // elements
  float inv_temperature;
  int top;
  int64_t part, parts;  // entries of a part (whole runs), parts of a row
  float* logprob;
  float* entropy;
  float* lse;
  float* top_logprob;
  int64_t* top_index;
  float4* stats;    // (rows, parts): maximum, sum, weighted sum
  uint64_t* keys;   // (rows, parts, top)
  // backward
  const float* up;
  const float* up_h;
  const float* up_lse;
  const float* entropy_in;
  const float* lse_in;
  int64_t u_b, u_t, h_b, h_t, ul_b, ul_t;
  bool alone;  // whether one workgroup takes the whole of a row with a large lse
  char* grad;
};

// a b, 0 where either is 0 whatever the other one is.
extern "C" __device__ float da_mul_or_zero(float a, float b) __asm("llvm.amdgcn.fmul.legacy");

template <int DT>
__device__ __forceinline__ uint32_t none() {  // -inf in every place of a word
  return DT == DA_F32 ? 0xff800000u : DT == DA_BF16 ? 0xff80ff80u : 0xfc00fc00u;
}

// The run at v0 of a row where all of it lies before `end`, else -inf and nothing is read.
// (No other case: a row's last entries that are no whole run are read one a thread, so that
// no load has a branch behind it that would have to wait for the others.)
template <int DT>
__device__ __forceinline__ u32x4 load_run(const char* row, int64_t v0, int64_t end) {
  u32x4 w = {none<DT>(), none<DT>(), none<DT>(), none<DT>()};
  if (v0 + Elem<DT>::kVec <= end) w = ld16_any<Elem<DT>::kBytes>(row + v0 * Elem<DT>::kBytes);
  return w;
}

// The order of two entries as whole numbers: by value, then by the lower index.  -0 is +0.
__device__ __forceinline__ uint64_t key_of(float x, int64_t v) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t up = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)up << 32 | (0xffffffffu - (uint32_t)v);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t up = (uint32_t)(key >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
__device__ __forceinline__ int64_t key_index(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// Sums of 2^d and of d 2^d, d = (logit - m) c, relative to the largest logit m.  The
// difference comes first: logits of a type's lowest value do not overflow.  Their distance from
// others does, times c: what a new maximum leaves nothing of is 0, not 0 times it.
__device__ __forceinline__ float moved(float e, float s, float by, float scale) {
  return da_mul_or_zero(scale, e + da_mul_or_zero(s, by));
}
struct Stats {
  float m, s, e;
  __device__ void join(float m2, float s2, float e2, float c) {
    const float top = fmaxf(m, m2), d1 = (m - top) * c, d2 = (m2 - top) * c;
    const float f1 = __builtin_amdgcn_exp2f(d1), f2 = __builtin_amdgcn_exp2f(d2);
    // s = 0 where nothing was seen: its distance does not count.
    e = moved(e, s, d1, f1) + moved(e2, s2, d2, f2);
    s = s * f1 + s2 * f2;
    m = top;
  }
};

// A row's outputs from its sums and its target's logit.
__device__ void finish(const LpArgs& a, int64_t row, bool named, float logit, float c, const Stats& x) {
  const float bits = log2f(x.s);
  a.logprob[row] = named ? ((logit - x.m) * c - bits) * kLn2 : 0.f;
  a.entropy[row] = (bits - x.e / x.s) * kLn2;
  a.lse[row] = fmaf(x.m, a.inv_temperature, bits * kLn2);
}

// The largest of a wave's keys.
__device__ __forceinline__ uint64_t wave_max_key(uint64_t k) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)k, off, kWave);
    k = o > k ? o : k;
  }
  return k;
}

// The top-th largest of 64 keys, one a lane (0: none).
__device__ __forceinline__ uint64_t bound_of(uint64_t k, int top) {
  const int hi = (int)(k >> 32), lo = (int)(uint32_t)k;
  const auto of = [&](int l) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, l) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, l);
  };
  int above = 0;
#pragma unroll 8
  for (int l = 0; l < kWave; ++l) above += of(l) > k;
  const uint64_t at = __ballot(k != 0 && above == top - 1);
  return at ? of(__ffsll((unsigned long long)at) - 1) : 0;
}

// The top largest of n different keys in LDS, in order, to f(place, key).
template <int NT, class F>
__device__ __forceinline__ void place(const uint64_t* keys, int n, int top, F f) {
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t k = keys[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += keys[j] > k;
    if (above < top) f(above, k);
  }
}

// ---------------------------------------------------------------------------
// Forward: workgroup (row, part).
// ---------------------------------------------------------------------------
template <int DT, int NT, bool kTop>
__global__ __launch_bounds__(NT) void logprobs_forward(LpArgs a) {
  constexpr int ES = Elem<DT>::kBytes, V = Elem<DT>::kVec, kWaves = NT / kWave;
  __shared__ float stat[3][kWaves];
  __shared__ uint64_t maxima[kTop ? kGroups : 1];
  __shared__ uint64_t found[kTop ? kCandidates : 1];
  __shared__ uint16_t winner[kTop ? NT : 1];
  __shared__ uint64_t bound_at;
  __shared__ int count, winners;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  const int64_t b = row / a.tokens, t = row - b * a.tokens;
  if (a.mask && !a.mask[b * a.m_b + t * a.m_t]) {
    if (part) return;
    if (tid == 0) a.logprob[row] = a.entropy[row] = a.lse[row] = 0.f;
    if (kTop && tid < a.top) {
      a.top_logprob[row * a.top + tid] = 0.f;
      a.top_index[row * a.top + tid] = -1;
    }
    return;
  }
  const char* logits = a.logits + (b * a.l_b + t * a.l_t) * ES;
  const int64_t v0 = part * a.part, end = min(v0 + a.part, a.vocab);
  const float c = a.inv_temperature * kLog2e;
  // The target's logit comes with the first runs.
  const int64_t target = a.targets[b * a.t_b + t * a.t_t];
  const bool named = target >= 0 && target < a.vocab;
  const float logit = named && a.parts == 1 ? Elem<DT>::load(logits, target) : 0.f;
  constexpr int64_t kStride = (int64_t)NT * V * kBatch;
  const int64_t whole = end - (end - v0) % V;  // where the whole runs end
  Stats x = {kFloor, 0.f, 0.f};
  float most = -__builtin_inff();  // the thread's largest logit, and the batch that has it first
  int64_t most_at = v0 + (int64_t)tid * V;
  const auto add = [&](const u32x4 (&raw)[kBatch], int64_t v) __attribute__((always_inline)) {
    float f[kBatch][V], top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      unpack16<DT>(raw[i], f[i]);
#pragma unroll
      for (int e = 0; e < V; ++e) top = fmaxf(top, f[i][e]);
    }
    if (kTop && top > most) most = top, most_at = v;
    if (__any(top > x.m)) {
      const float m = fmaxf(x.m, top), by = (x.m - m) * c, scale = __builtin_amdgcn_exp2f(by);
      x.e = moved(x.e, x.s, by, scale);
      x.s *= scale;
      x.m = m;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = (f[i][e] - x.m) * c, p = __builtin_amdgcn_exp2f(d);
        x.s += p;
        x.e += da_mul_or_zero(p, d);  // 0 where p is: a logit of -inf
      }
  };
  // Batches that are whole for every thread, the next one on its way (the last again in its
  // place: no load has a condition); then one that is not.
  const int64_t full = (whole - v0) / kStride;
  int64_t v = v0 + (int64_t)tid * V;
  u32x4 raw[kBatch];
  if (full) {
    const char* at = logits + v * ES;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) raw[i] = ld16_any<ES>(at + i * (NT * 16));
    for (int64_t n = full; n > 0; --n, v += kStride) {
      u32x4 now[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) now[i] = raw[i];
      at += n > 1 ? kStride * ES : 0;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) raw[i] = ld16_any<ES>(at + i * (NT * 16));
      add(now, v);
    }
  }
  const bool left = v0 + full * kStride < end;
  float rest = -__builtin_inff();  // one of the last entries, no whole run
  const bool has_rest = tid < end - whole;
  if (left) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) raw[i] = load_run<DT>(logits, v + (int64_t)i * NT * V, whole);
    if (has_rest) rest = Elem<DT>::load(logits, whole + tid);
    add(raw, v);
    const float m = fmaxf(x.m, rest), by = (x.m - m) * c, scale = __builtin_amdgcn_exp2f(by);
    const float d = (rest - m) * c, p = __builtin_amdgcn_exp2f(d);
    x.e = moved(x.e, x.s, by, scale) + da_mul_or_zero(p, d);
    x.s = x.s * scale + p;
    x.m = m;
  }
  {  // the wave's, relative to its maximum
    const float m = lanes_max<kWave>(x.m), by = (x.m - m) * c, scale = __builtin_amdgcn_exp2f(by);
    const float s = lanes_sum<kWave>(x.s * scale);
    const float e = lanes_sum<kWave>(moved(x.e, x.s, by, scale));
    if (lane == 0) stat[0][wave] = m, stat[1][wave] = s, stat[2][wave] = e;
  }
  const bool mine = kTop && v0 + (int64_t)tid * V < whole;
  if constexpr (kTop) {
    // At least as good as this is one entry of the thread: the last place of that batch.
    uint64_t k = mine ? key_of(most, most_at + (kBatch - 1) * (int64_t)NT * V + V - 1) : 0;
    if (has_rest) {
      const uint64_t o = key_of(rest, whole + tid);
      k = o > k ? o : k;
    }
    constexpr int kEach = NT / kGroups;  // threads of a group
#pragma unroll
    for (int off = 1; off < kEach; off <<= 1) {
      const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)k, off, kWave);
      k = o > k ? o : k;
    }
    if (tid % kEach == 0) maxima[tid / kEach] = k;
    if (tid == 0) count = winners = 0;
  }
  __syncthreads();
  if (wave == 0) {
    Stats all = {stat[0][0], stat[1][0], stat[2][0]};
    for (int w = 1; w < kWaves; ++w) all.join(stat[0][w], stat[1][w], stat[2][w], c);
    if (a.parts == 1) {
      stat[0][0] = all.m, stat[1][0] = all.s;
      if (lane == 0) finish(a, row, named, logit, c, all);
    } else if (lane == 0) {
      a.stats[blockIdx.x] = float4{all.m, all.s, all.e, 0.f};
    }
    if constexpr (kTop) {
      const uint64_t bound = bound_of(maxima[lane], a.top);
      if (lane == 0) bound_at = bound;
    }
  }
  if constexpr (!kTop) return;
  __syncthreads();
  const uint64_t bound = bound_at;
  // At best the thread's largest is the first place of its batch.
  if (mine && key_of(most, most_at) >= bound) winner[atomicAdd(&winners, 1)] = (uint16_t)tid;
  __syncthreads();
  const auto keep = [&](float f, int64_t at) __attribute__((always_inline)) {
    const uint64_t k = key_of(f, at);
    if (k < bound) return;
    const int place = atomicAdd(&count, 1);  // places do not matter: keys are ranked
    if (place < kCandidates) found[place] = k;
  };
  if (has_rest) keep(rest, whole + tid);
  // Runs of a thread, the same for all (those past the end hold nothing).
  const int each = (int)((whole - v0 + (int64_t)NT * V - 1) / ((int64_t)NT * V)), again = winners * each;
#pragma unroll 2
  for (int i = tid; i < again; i += NT) {
    const int w = i / each;
    const int64_t v = v0 + ((int64_t)winner[w] + (int64_t)(i - w * each) * NT) * V;
    if (v + V > whole) continue;
    float f[V];
    unpack16<DT>(load_run<DT>(logits, v, whole), f);
#pragma unroll
    for (int e = 0; e < V; ++e) keep(f[e], v + e);
  }
  __syncthreads();
  int n = count;
  const float m = stat[0][0], bits = a.parts == 1 ? log2f(stat[1][0]) : 0.f;
  auto put = [&](int at, uint64_t key) {
    if (a.parts > 1) {
      a.keys[(int64_t)blockIdx.x * a.top + at] = key;
    } else {
      a.top_logprob[row * a.top + at] = ((key_value(key) - m) * c - bits) * kLn2;
      a.top_index[row * a.top + at] = key_index(key);
    }
  };
  if (n <= kCandidates) {
    place<NT>(found, n, a.top, put);
    if (tid >= n && tid < a.top) {  // a part of fewer entries; a row with NaN
      if (a.parts > 1) {
        a.keys[(int64_t)blockIdx.x * a.top + tid] = 0;
      } else {
        a.top_logprob[row * a.top + tid] = __builtin_nanf("");
        a.top_index[row * a.top + tid] = -1;
      }
    }
    return;
  }
  // More entries reach the bound than LDS holds (sorted logits, say): the largest one below
  // the last, `top` times over.
  uint64_t last = ~0ull;
  for (int at = 0; at < a.top; ++at) {
    uint64_t k = 0;
    const auto larger = [&](float f, int64_t v) __attribute__((always_inline)) {
      const uint64_t o = key_of(f, v);
      if (o < last && o > k) k = o;
    };
    if (has_rest) larger(rest, whole + tid);
    for (int64_t v = v0 + (int64_t)tid * V; v < whole; v += (int64_t)NT * V) {
      float f[V];
      unpack16<DT>(load_run<DT>(logits, v, whole), f);
#pragma unroll
      for (int e = 0; e < V; ++e) larger(f[e], v + e);
    }
    k = wave_max_key(k);
    __syncthreads();
    if (lane == 0) found[wave] = k;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) k = found[w] > k ? found[w] : k;
    if (tid == 0) put(at, k);
    last = k;
  }
}

// The parts of a row: their sums in order, and the largest of their alternatives.
constexpr int kJoin = 256, kMaxParts = 64;
template <bool kTop>
__global__ __launch_bounds__(kJoin) void logprobs_join(LpArgs a, int dt) {
  __shared__ uint64_t keys[kTop ? kMaxParts * kMaxTop : 1];
  __shared__ uint64_t kept[kTop ? kMaxParts * kMaxTop : 1];
  __shared__ float stat[2];
  __shared__ uint64_t bound_at;
  __shared__ int count;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x, b = row / a.tokens, t = row - b * a.tokens;
  if (a.mask && !a.mask[b * a.m_b + t * a.m_t]) return;  // written by the first launch
  const float c = a.inv_temperature * kLog2e;
  const int parts = (int)a.parts, n = kTop ? parts * a.top : 0;
  const int64_t target = a.targets[b * a.t_b + t * a.t_t];
  const bool named = target >= 0 && target < a.vocab;
  const char* logits = a.logits + (b * a.l_b + t * a.l_t) * (dt == DA_F32 ? 4 : 2);
  const float logit = !named ? 0.f : dt == DA_F32 ? Elem<DA_F32>::load(logits, target)
                      : dt == DA_BF16 ? Elem<DA_BF16>::load(logits, target) : Elem<DA_F16>::load(logits, target);
  if (tid < kWave) {
    Stats x = {kFloor, 0.f, 0.f};
    if (tid < parts) {
      const float4 v = a.stats[row * parts + tid];
      x = Stats{v.x, v.y, v.z};
    }
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1)
      x.join(__shfl_xor(x.m, off, kWave), __shfl_xor(x.s, off, kWave), __shfl_xor(x.e, off, kWave), c);
    if (tid == 0) {
      finish(a, row, named, logit, c, x);
      stat[0] = x.m, stat[1] = x.s;
      count = 0;
    }
  }
  if constexpr (!kTop) return;
  for (int i = tid; i < n; i += kJoin) keys[i] = a.keys[row * n + i];
  __syncthreads();
  if (tid < kWave) {
    uint64_t k = 0;
    for (int i = tid; i < n; i += kWave) k = keys[i] > k ? keys[i] : k;
    const uint64_t bound = bound_of(k, a.top);
    if (tid == 0) bound_at = bound;
  }
  __syncthreads();
  const uint64_t bound = bound_at;
  for (int i = tid; i < n; i += kJoin)
    if (keys[i] && keys[i] >= bound) kept[atomicAdd(&count, 1)] = keys[i];
  __syncthreads();
  const float m = stat[0], bits = log2f(stat[1]);
  if (tid >= count && tid < a.top) {
    a.top_logprob[row * a.top + tid] = __builtin_nanf("");
    a.top_index[row * a.top + tid] = -1;
  }
  place<kJoin>(kept, count, a.top, [&](int at, uint64_t key) {
    a.top_logprob[row * a.top + at] = ((key_value(key) - m) * c - bits) * kLn2;
    a.top_index[row * a.top + at] = key_index(key);
  });
}

// Over the workgroup's row: its largest logit m, and log sum e^((z - m) / temperature).
template <int DT, int NT>
__device__ float2 row_sums(const char* logits, int64_t vocab, float c, float (*stat)[NT / kWave]) {
  constexpr int V = Elem<DT>::kVec, kWaves = NT / kWave;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t whole = vocab - vocab % V;
  float m = kFloor, s = 0.f;
  for (int64_t v = (int64_t)threadIdx.x * V; v < whole; v += (int64_t)NT * V * kBatch) {
    float f[kBatch][V], top = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      unpack16<DT>(load_run<DT>(logits, v + (int64_t)i * NT * V, whole), f[i]);
#pragma unroll
      for (int e = 0; e < V; ++e) top = fmaxf(top, f[i][e]);
    }
    s *= __builtin_amdgcn_exp2f((m - top) * c);
    m = top;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) s += __builtin_amdgcn_exp2f((f[i][e] - m) * c);
  }
  if ((int)threadIdx.x < vocab - whole) {
    const float f = Elem<DT>::load(logits, whole + threadIdx.x), top = fmaxf(m, f);
    s = s * __builtin_amdgcn_exp2f((m - top) * c) + __builtin_amdgcn_exp2f((f - top) * c);
    m = top;
  }
  float most = lanes_max<kWave>(m);
  s = lanes_sum<kWave>(s * __builtin_amdgcn_exp2f((m - most) * c));
  if (lane == 0) stat[0][wave] = most, stat[1][wave] = s;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) most = fmaxf(most, stat[0][w]);
  s = 0.f;
  for (int w = 0; w < kWaves; ++w) s += stat[1][w] * __builtin_amdgcn_exp2f((stat[0][w] - most) * c);
  return float2{most, log2f(s) * kLn2};
}

// How far from 0 a row's lse may lie for the gradient to take probabilities from it: as an fp32
// number it is off by 2^-25 of its size and more, and so are all of the row's probabilities,
// relatively.  2^-20 in fp32; in 16 bits a sixteenth of the gradient's own half step.
template <int DT>
constexpr float kFar = DT == DA_F32 ? 32.f : DT == DA_F16 ? 512.f : 4096.f;

// ---------------------------------------------------------------------------
// Backward: workgroup (row, part), the last rows first: a forward call just before left them
// in the last-level cache.  Rows whose lse is large (a common offset, a small temperature) are
// read twice, for their maximum and sum apart: by one part's workgroup, which then writes the
// whole row, or with few rows by each.  kStream: gradients that do not fit there are written past it, and
// leave it to the logits (3 x 509 rows of 50257 in fp32, forward and backward: 195 us without,
// 163 with both).
// ---------------------------------------------------------------------------
template <int DT, int NT, bool kStream>
__global__ __launch_bounds__(NT) void logprobs_backward(LpArgs a) {
  constexpr int ES = Elem<DT>::kBytes, V = Elem<DT>::kVec;
  const int64_t id = gridDim.x - 1 - blockIdx.x, row = id / a.parts, part = id - row * a.parts;
  const int64_t b = row / a.tokens, t = row - b * a.tokens;
  const bool live = !a.mask || a.mask[b * a.m_b + t * a.m_t];
  const char* logits = a.logits + (b * a.l_b + t * a.l_t) * ES;
  char* grad = a.grad + row * a.vocab * ES;
  int64_t v0 = part * a.part, end = min(v0 + a.part, a.vocab);
  int64_t target = a.targets[b * a.t_b + t * a.t_t];
  const bool named = live && target >= 0 && target < a.vocab;
  target = named ? target : -1;
  const float up = named && a.up ? a.up[b * a.u_b + t * a.u_t] * a.inv_temperature : 0.f;
  const float up_h = live && a.up_h ? a.up_h[b * a.h_b + t * a.h_t] * a.inv_temperature : 0.f;
  const float up_lse = live && a.up_lse ? a.up_lse[b * a.ul_b + t * a.ul_t] * a.inv_temperature : 0.f;
  float m = 0.f, lse = live ? a.lse_in[row] : 0.f;
  if (live && !(fabsf(lse) <= kFar<DT>)) {  // the same in all threads
    __shared__ float stat[2][NT / kWave];
    if (a.alone) {  // any one part, so that those that stay lie on all dies
      if (part != ((uint32_t)row * 0x9e3779b1u >> 8) % a.parts) return;
      v0 = 0, end = a.vocab;
    }
    const float2 x = row_sums<DT, NT>(logits, a.vocab, a.inv_temperature * kLog2e, stat);
    m = x.x, lse = x.y;
  }
  const float whole = up_lse - up - (a.up_h && live ? up_h * a.entropy_in[row] : 0.f), slope = -up_h;
  const auto of = [&](float f) __attribute__((always_inline)) {
    const float d = fmaf(f - m, a.inv_temperature, -lse), p = __builtin_amdgcn_exp2f(d * kLog2e);
    return live ? da_mul_or_zero(p, fmaf(d, slope, whole)) : 0.f;
  };
  const int64_t runs = end - (end - v0) % V;  // where the whole runs end
  const int last = (int)(end - runs);
  if ((int)threadIdx.x < last) {
    const int64_t at = runs + threadIdx.x;
    Elem<DT>::store(grad, at, of(live ? Elem<DT>::load(logits, at) : 0.f) + (at == target ? up : 0.f));
  }
  for (int64_t v = v0 + (int64_t)threadIdx.x * V; v < runs; v += (int64_t)NT * V * kBatch) {
    u32x4 raw[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) raw[i] = load_run<DT>(logits, v + (int64_t)i * NT * V, live ? runs : 0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t at = v + (int64_t)i * NT * V;
      if (at >= runs) continue;
      float f[V];
      unpack16<DT>(raw[i], f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = of(f[e]);
      if (target >= at && target < at + V) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] += at + e == target ? up : 0.f;
      }
      u32x4 w;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (DT == DA_F32) w[k] = __float_as_uint(f[k]);
        else w[k] = pack2<DT>(f[2 * k], f[2 * k + 1]);
      }
      if constexpr (kStream) st16_any_nt<ES>(grad + at * ES, w);
      else st16_any<ES>(grad + at * ES, w);
    }
  }
}

// ---------------------------------------------------------------------------
// Launches.
// ---------------------------------------------------------------------------
int check_rows(const char* what, int dtype, int64_t batch, int64_t tokens, int64_t vocab, float temperature) {
  if (!valid_dtype(dtype)) return set_error(DA_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || tokens < 0) return set_error(DA_ERR_INVALID, "%s: negative size", what);
  if (vocab < 1 || vocab > INT32_MAX) return set_error(DA_ERR_UNSUPPORTED, "%s: vocabularies of 1 to 2^31 - 1 tokens", what);
  // Both 1 / temperature and -inf times it have to be what they say.
  if (!(temperature > 0.f) || !(1.f / temperature < 1e30f) || !(1.f / temperature >= 0x1p-126f))
    return set_error(DA_ERR_INVALID, "%s: the temperature must lie between 1e-30 and 8e37", what);
  if (tokens && batch > kMaxBlocks / 4 / tokens) return set_error(DA_ERR_UNSUPPORTED, "%s: too many rows", what);
  return DA_OK;
}

// Threads of a row's workgroup: one wave where rows are short and many (bf16 with five
// alternatives, 4096 rows of 1000: 18 us, with eight waves 45; of 8000: 30 and 47; 32000: 69 and
// 63; 16 rows of 4000: 15 and 10).
int threads_of(int64_t rows, int64_t vocab, int dtype, int64_t cus) {
  return rows >= 4 * cus && vocab * (int64_t)elem_bytes(dtype) <= 32768 ? 64 : 512;
}

// Parts of a row: enough workgroups for every CU, no part under two runs a thread.
int parts_of(int64_t rows, int64_t vocab, int dtype, int* threads, int64_t* part, int64_t* parts) {
  int64_t cus;
  const int rc = device_cu_count(&cus);
  if (rc) return rc;
  *threads = threads_of(rows, vocab, dtype, cus);
  const int64_t vec = dtype == DA_F32 ? 4 : 8, least = 2 * *threads * vec;
  int64_t n = rows >= cus ? 1 : std::min<int64_t>(kMaxParts, 2 * cus / std::max<int64_t>(rows, 1));
  n = std::max<int64_t>(1, std::min(n, vocab / least));
  *part = ((vocab + n - 1) / n + vec - 1) / vec * vec;
  *parts = (vocab + *part - 1) / *part;
  return DA_OK;
}

size_t workspace_of(int64_t rows, int64_t parts, int top) {
  return parts > 1 ? (size_t)(rows * parts) * (sizeof(float4) + (size_t)top * sizeof(uint64_t)) : 0;
}

template <class F>
int by_type(int dtype, int threads, F f) {
#define DA_LP(DT)                                                                                 \
  return threads == 64 ? f(std::integral_constant<int, DT>{}, std::integral_constant<int, 64>{}) \
                       : f(std::integral_constant<int, DT>{}, std::integral_constant<int, 512>{});
  if (dtype == DA_F32) DA_LP(DA_F32)
  if (dtype == DA_BF16) DA_LP(DA_BF16)
  DA_LP(DA_F16)
#undef DA_LP
}

}  // namespace
}  // namespace da

extern "C" {

int da_token_logprobs_workspace(int dtype, int64_t batch, int64_t tokens, int64_t vocab, int top, size_t* bytes) {
  using namespace da;
  if (!bytes) return set_error(DA_ERR_INVALID, "da_token_logprobs_workspace: NULL pointer");
  *bytes = 0;
  int rc = check_rows("da_token_logprobs_workspace", dtype, batch, tokens, vocab, 1.f);
  if (rc) return rc;
  if (top < 0 || top > kMaxTop || top > vocab)
    return set_error(DA_ERR_UNSUPPORTED, "da_token_logprobs_workspace: 0 to %d alternatives, no more than tokens", kMaxTop);
  int threads;
  int64_t part, parts;
  rc = parts_of(batch * tokens, vocab, dtype, &threads, &part, &parts);
  if (rc == DA_OK) *bytes = workspace_of(batch * tokens, parts, top);
  return rc;
}

int da_token_logprobs(const void* logits, int dtype, int64_t batch, int64_t tokens, int64_t vocab, int64_t l_bstride,
                      int64_t l_tstride, const int64_t* targets, int64_t t_bstride, int64_t t_tstride,
                      const uint8_t* mask, int64_t mask_bstride, int64_t mask_tstride, float temperature, int top,
                      float* logprob, float* entropy, float* lse, float* top_logprob, int64_t* top_index,
                      void* workspace, size_t workspace_bytes, void* stream) {
  using namespace da;
  int rc = check_rows("da_token_logprobs", dtype, batch, tokens, vocab, temperature);
  if (rc) return rc;
  if (top < 0 || top > kMaxTop || top > vocab)
    return set_error(DA_ERR_UNSUPPORTED, "da_token_logprobs: 0 to %d alternatives, no more than tokens", kMaxTop);
  if (batch == 0 || tokens == 0) return DA_OK;
  if (!logits || !targets || !logprob || !entropy || !lse || (top && (!top_logprob || !top_index)))
    return set_error(DA_ERR_INVALID, "da_token_logprobs: NULL pointer");
  LpArgs a = {};
  int threads;
  rc = parts_of(batch * tokens, vocab, dtype, &threads, &a.part, &a.parts);
  if (rc) return rc;
  a.rows = batch * tokens;
  const size_t need = workspace_of(a.rows, a.parts, top);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "da_token_logprobs: workspace of %zu bytes needed", need);
  if ((uintptr_t)workspace % 16) return set_error(DA_ERR_INVALID, "da_token_logprobs: workspace must be 16-byte aligned");
  a.logits = (const char*)logits;
  a.targets = targets;
  a.mask = mask;
  a.tokens = tokens, a.vocab = vocab;
  a.l_b = l_bstride, a.l_t = l_tstride, a.t_b = t_bstride, a.t_t = t_tstride, a.m_b = mask_bstride, a.m_t = mask_tstride;
  a.inv_temperature = 1.f / temperature;
  a.top = top;
  a.logprob = logprob, a.entropy = entropy, a.lse = lse, a.top_logprob = top_logprob, a.top_index = top_index;
  a.stats = (float4*)workspace;
  a.keys = need ? (uint64_t*)((float4*)workspace + a.rows * a.parts) : nullptr;
  const hipStream_t st = (hipStream_t)stream;
  rc = by_type(dtype, threads, [&](auto dt, auto nt) {
    constexpr int DT = decltype(dt)::value, NT = decltype(nt)::value;
    const unsigned grid = (unsigned)(a.rows * a.parts);
    if (top) logprobs_forward<DT, NT, true><<<grid, NT, 0, st>>>(a);
    else logprobs_forward<DT, NT, false><<<grid, NT, 0, st>>>(a);
    return check_launch("da_token_logprobs");
  });
  if (rc || a.parts == 1) return rc;
  if (top) logprobs_join<true><<<(unsigned)a.rows, kJoin, 0, st>>>(a, dtype);
  else logprobs_join<false><<<(unsigned)a.rows, kJoin, 0, st>>>(a, dtype);
  return check_launch("da_token_logprobs");
}

int da_token_logprobs_grad(const float* up, int64_t up_bstride, int64_t up_tstride, const float* up_entropy,
                           int64_t uh_bstride, int64_t uh_tstride, const float* up_lse, int64_t ul_bstride,
                           int64_t ul_tstride, const void* logits, int dtype, int64_t batch, int64_t tokens,
                           int64_t vocab, int64_t l_bstride, int64_t l_tstride, const int64_t* targets,
                           int64_t t_bstride, int64_t t_tstride, const float* lse, const float* entropy,
                           const uint8_t* mask, int64_t mask_bstride, int64_t mask_tstride, float temperature,
                           void* grad, void* stream) {
  using namespace da;
  const int rc = check_rows("da_token_logprobs_grad", dtype, batch, tokens, vocab, temperature);
  if (rc) return rc;
  if (batch == 0 || tokens == 0) return DA_OK;
  if (!logits || !targets || !lse || !grad || (up_entropy && !entropy))
    return set_error(DA_ERR_INVALID, "da_token_logprobs_grad: NULL pointer");
  LpArgs a = {};
  a.rows = batch * tokens;
  const int64_t vec = dtype == DA_F32 ? 4 : 8;
  int64_t cus;
  if (const int err = device_cu_count(&cus)) return err;
  const int nt = threads_of(a.rows, vocab, dtype, cus);
  // Parts of two batches a thread: nothing is joined.
  a.part = 2 * (int64_t)kBatch * nt * vec;
  a.parts = (vocab + a.part - 1) / a.part;
  if (a.rows > kMaxBlocks / 4 / a.parts) return set_error(DA_ERR_UNSUPPORTED, "da_token_logprobs_grad: too many rows");
  a.alone = a.rows * a.parts > 4 * cus;
  a.up = up, a.u_b = up_bstride, a.u_t = up_tstride;
  a.up_h = up_entropy, a.h_b = uh_bstride, a.h_t = uh_tstride;
  a.up_lse = up_lse, a.ul_b = ul_bstride, a.ul_t = ul_tstride;
  a.logits = (const char*)logits;
  a.targets = targets;
  a.mask = mask;
  a.tokens = tokens, a.vocab = vocab;
  a.l_b = l_bstride, a.l_t = l_tstride, a.t_b = t_bstride, a.t_t = t_tstride, a.m_b = mask_bstride, a.m_t = mask_tstride;
  a.inv_temperature = 1.f / temperature;
  a.lse_in = lse, a.entropy_in = entropy;
  a.grad = (char*)grad;
  const hipStream_t st = (hipStream_t)stream;
  return by_type(dtype, nt, [&](auto dt, auto n) {
    constexpr int NT = decltype(n)::value;
    constexpr int DT = decltype(dt)::value;
    const unsigned grid = (unsigned)(a.rows * a.parts);
    if (a.rows * vocab * (int64_t)elem_bytes(dtype) > kLastLevel / 2) logprobs_backward<DT, NT, true><<<grid, NT, 0, st>>>(a);
    else logprobs_backward<DT, NT, false><<<grid, NT, 0, st>>>(a);
    return check_launch("da_token_logprobs_grad");
  });
}

}  // extern "C"
