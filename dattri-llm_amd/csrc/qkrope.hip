// RMS norms of the queries and keys of each head with the position rotation,
// and their gradients (the norm weights' per sample).
//
// One row is a head's D entries at one token, x; w the side's weight, p the
// token's position, f_i the rotation's inverse frequencies (i < R/2, R <= D):
//
//   r = (mean(x^2) + eps)^(-1/2),  y = x r w
//   z_a = s (y_a cos(p f_i) - y_b sin(p f_i)),  z_b = s (y_b cos(p f_i) + y_a sin(p f_i))
//   z = y past R
//
// for the pairs (a, b) = (i, i + R/2), or (2i, 2i+1) interleaved.  Backward,
// with dz given: dy = the pairs turned back (times s), g = dy w,
//
//   dx = r (g - x r^2 mean(g x)),  dw[b] = sum over tokens and heads of dy x r.
//
// The angle is position times frequency in fp64, reduced to its fraction of a
// turn there (a position of 10^6 leaves 10^-10 of a turn), and only then fp32:
// fp32 products would lose the angles of far positions.
//
// A row's pairs lie in slots of V; a group of kL lanes owns a head, lane l its
// slots l, l + kL, ..., and a wave 64 / kL heads of one token at a time, so that
// one token's angles serve all the heads its wave visits.  Both members of a
// pair are in one lane: the rotation needs no exchange, and a row's two sums
// (x^2; and g x in the backward pass) are one butterfly over the kL lanes.  The
// slots are 16 bytes where the widths and every row's alignment allow it; else 4
// entries, else 1 (any width, any stride).
//
// Bound by HBM: each row is read once and written once, and the angles are fp64
// work for one lane a pair and token.  8 x 2048 tokens, 32 + 8 heads of 128, bf16:
// forward 57 us for 335 MB (5.9 TB/s; one wave a head 150 us, 16-byte slots 93,
// angles once a token 88, weights in LDS and waves over many tokens 70, streamed
// loads 57), backward 99 us for 503 MB (5.1 TB/s; 361 with one wave a head) and 4 us
// to join its chunks.  A new token of 16 sequences: 4 us, a launch.
#include <algorithm>

#include "common.h"

namespace da {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int64_t kMaxD = 1024;
// Forward: a token's heads are spread over waves while there are fewer than
// kWantWaves (a new token of 16 sequences: 10.3 us on a wave each, 4.1 spread); at
// most kMostBlocks workgroups, whose waves stride over the tokens (1024 to 16384
// differ by 1%, and each loads the weights).
constexpr int64_t kWantWaves = 4096;
constexpr int64_t kMostBlocks = 2048;
// Rows of this many bytes in all are read past the caches.  Fewer may lie in the
// last-level cache (256 MB) from the kernel that wrote them: at 84 MB of rows
// (4 x 2048 tokens, 32 + 8 heads of 128, bf16) both take 34 us forward, at 168 MB
// 70 us with cached loads, 58 us with streamed ones; 21 MB: 10.9 and 12.7 us.
constexpr int64_t kStreamBytes = 128 << 20;
constexpr int64_t kRows = 1024;
constexpr int64_t kWantBlocks = 512;

struct Rows {  // one side's rows; strides in bytes
  const char* x;
  const char* gz;
  char* out;
  const void* w;
  float* wgrad;    // (batch, D), NULL: not wanted
  float* partial;  // (batch, chunks, D)
  int64_t heads;
  int64_t chunk, chunks;  // backward: tokens of a workgroup, workgroups of a sample
  int64_t x_b, x_t, x_h, g_b, g_t, g_h, o_b, o_t, o_h;
};

struct QkArgs {
  Rows side[2];
  int64_t batch, tokens;
  int d, rot, w_dtype;
  const float* inv_freq;
  const void* pos;  // NULL: the token's index
  int pos_bytes;
  int64_t pos_b, pos_t;  // elements
  const uint8_t* mask;   // NULL: every token lives
  int64_t mask_b, mask_t;
  float scaling, eps;
  int parts;  // forward: waves that share a token's heads
};

__device__ __forceinline__ float load_any(const void* p, int dt, int64_t i) {
  if (dt == DA_F32) return ((const float*)p)[i];
  const uint32_t h = ((const uint16_t*)p)[i];
  return dt == DA_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}

// LDS written by a wave's lanes is read by its other lanes: the hardware keeps a
// wave's LDS accesses in order, this keeps the compiler to it.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Where a slot's two runs of V entries start, and what of them exists.
template <int V, bool kInter>
struct Slot {
  int a, b;       // first entry of each run; interleaved: the runs follow one another
  bool in, turn;  // the slot holds entries; they rotate
  bool has_b;     // V == 1 only: the second entry exists (odd remainders)
  __device__ void at(int s, int d, int rot) {
    if constexpr (kInter) {
      a = 2 * s * V;
      b = a + V;
      turn = a < rot;
    } else {
      const int half = rot / 2, p = s * V;
      turn = p < half;
      const int rest = (d - rot + 1) / 2, q = p - half;
      a = turn ? p : (q < rest ? rot + q : d);
      b = turn ? half + p : rot + rest + q;
    }
    in = a < d;
    has_b = b < d;
  }
};

template <int DT, int V>
struct Run {  // V entries as they lie in memory, in one access
  static constexpr int kBytes = V * Elem<DT>::kBytes, kWords = kBytes < 4 ? 1 : kBytes / 4;
  typedef uint32_t Words __attribute__((ext_vector_type(kWords)));
  Words w;
  template <bool kStream>
  __device__ void load(const char* p, bool in) {
    w = Words(0);
    if (!in) return;
    if constexpr (kBytes == 2) w[0] = *(const uint16_t*)p;
    else if constexpr (kStream) w = __builtin_nontemporal_load((const Words*)p);
    else w = *(const Words*)p;
  }
  __device__ float get(int i) const {
    if constexpr (DT == DA_F32) return __uint_as_float(w[i]);
    else return Elem<DT>::from_bits(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu);
  }
  template <class Vec>
  __device__ void pack(const Vec& v) {
    if constexpr (DT == DA_F32) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(v[i]);
    } else if constexpr (V == 1) {
      w[0] = DT == DA_BF16 ? f32_to_bf16_bits(v[0]) : f32_to_f16_bits(v[0]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) w[i] = pack2<DT>(v[2 * i], v[2 * i + 1]);
    }
  }
  __device__ void store(char* p, bool in) const {
    if (!in) return;
    if constexpr (kBytes == 2) *(uint16_t*)p = (uint16_t)w[0];
    else *(Words*)p = w;
  }
};

// The lane's runs of one row as they lie in memory.
template <int DT, int V, int S, bool kInter>
struct RawRow {
  Run<DT, V> u[S], v[S];
  template <bool kStream>
  __device__ void load(const char* p, const Slot<V, kInter>* slots, bool live) {
    constexpr int ES = Elem<DT>::kBytes;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      u[i].template load<kStream>(p + (int64_t)slots[i].a * ES, live && slots[i].in);
      v[i].template load<kStream>(p + (int64_t)slots[i].b * ES, live && slots[i].in && slots[i].has_b);
    }
  }
};

// Its pairs: fp32 values, first and second members.  Interleaved runs hold both
// members alternately.
template <int DT, int V, int S, bool kInter>
struct Row {
  typedef float Vec __attribute__((ext_vector_type(V)));
  Vec a[S], b[S];
  __device__ void unpack(const RawRow<DT, V, S, kInter>& raw) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (kInter && V > 1) {
          if constexpr (DT == DA_F32) {
            a[i][e] = __uint_as_float(e < V / 2 ? raw.u[i].w[2 * e % V] : raw.v[i].w[2 * e % V]);
            b[i][e] = __uint_as_float(e < V / 2 ? raw.u[i].w[2 * e % V + 1] : raw.v[i].w[2 * e % V + 1]);
          } else {  // a pair is a word
            const uint32_t pair = e < V / 2 ? raw.u[i].w[e % (V / 2)] : raw.v[i].w[e % (V / 2)];
            a[i][e] = Elem<DT>::from_bits(pair & 0xffffu);
            b[i][e] = Elem<DT>::from_bits(pair >> 16);
          }
        } else {
          a[i][e] = raw.u[i].get(e);
          b[i][e] = raw.v[i].get(e);
        }
      }
    }
  }
  __device__ void store(char* p, const Slot<V, kInter>* slots, bool live) const {
    constexpr int ES = Elem<DT>::kBytes;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      if constexpr (kInter && V > 1) {
        Run<DT, V> u, v;
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          if constexpr (DT == DA_F32) {
            u.w[2 * e] = __float_as_uint(a[i][e]);
            u.w[2 * e + 1] = __float_as_uint(b[i][e]);
            v.w[2 * e] = __float_as_uint(a[i][V / 2 + e]);
            v.w[2 * e + 1] = __float_as_uint(b[i][V / 2 + e]);
          } else {
            u.w[e] = pack2<DT>(a[i][e], b[i][e]);
            v.w[e] = pack2<DT>(a[i][V / 2 + e], b[i][V / 2 + e]);
          }
        }
        u.store(p + (int64_t)slots[i].a * ES, live && slots[i].in);
        v.store(p + (int64_t)slots[i].b * ES, live && slots[i].in);
        continue;
      }
      Run<DT, V> u, v;
      u.pack(a[i]);
      v.pack(b[i]);
      u.store(p + (int64_t)slots[i].a * ES, live && slots[i].in);
      v.store(p + (int64_t)slots[i].b * ES, live && slots[i].in && slots[i].has_b);
    }
  }
};

// Cosine and sine of a token's pairs, one pair a lane: a wave's heads share them
// through its own part of the LDS (`table`: kL S V pairs).  Pairs past the
// rotated ones get (1, 0) and are not turned by it: 0 times a partner that is not
// finite is no zero.  (A selection a value: no difference in time.)
template <int V, int kL, int S>
__device__ __forceinline__ void angles(const QkArgs& a, int64_t b, int64_t t, float2* table, int lane, int l,
                                       float (&c)[S][V], float (&s)[S][V]) {
  double pos = (double)t;
  if (a.pos) {
    const int64_t at = b * a.pos_b + t * a.pos_t;
    pos = a.pos_bytes == 8 ? (double)((const int64_t*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
  }
  wave_sync();  // the last token's are read
  for (int pair = lane; pair < kL * S * V; pair += kWave) {
    float sn = 0.f, cs = 1.f;
    if (pair < a.rot / 2) {
      const double turns = pos * ((double)a.inv_freq[pair] * 0.15915494309189535);  // 1 / (2 pi)
      sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);                    // half turns, [-1, 1]
      sn *= a.scaling;
      cs *= a.scaling;
    }
    table[pair] = make_float2(cs, sn);
  }
  wave_sync();
#pragma unroll
  for (int i = 0; i < S; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float2 cs = table[(l + i * kL) * V + e];
      c[i][e] = cs.x;
      s[i][e] = cs.y;
    }
}

// The weight in the order of the pairs, in LDS: first members, then second.
template <bool kInter>
__device__ __forceinline__ void weights(const QkArgs& a, const void* w, float* to, int pairs) {
  const int half = a.rot / 2, rest = (a.d - a.rot + 1) / 2;
  for (int n = threadIdx.x; n < 2 * pairs; n += kThreads) {
    const int p = n < pairs ? n : n - pairs, second = n >= pairs;
    int at = kInter ? 2 * p + second : p < half ? p + second * half : a.rot + p - half + second * rest;
    if (!kInter && p >= half + rest) at = a.d;
    to[n] = at < a.d ? load_any(w, a.w_dtype, at) : 0.f;
  }
}
template <int V, int kL, int S>
__device__ __forceinline__ void lane_weights(const float* from, int l, float (&wa)[S][V], float (&wb)[S][V]) {
#pragma unroll
  for (int i = 0; i < S; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      wa[i][e] = from[(l + i * kL) * V + e];
      wb[i][e] = from[(kL * S + l + i * kL) * V + e];
    }
}

// A wave takes units in turn: a token's heads, or every `parts`-th group of them
// where the tokens are few.
template <int DT, int V, int kL, int S, bool kInter, bool kStream>
__global__ __launch_bounds__(kThreads) void qk_rope_forward(QkArgs a) {
  constexpr int kHeads = kWave / kL, kPairs = kL * S * V;  // heads of a wave's step, pairs of a head
  __shared__ float2 tables[kWaves][kPairs];
  __shared__ float w[2][2 * kPairs];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane % kL, sub = lane / kL;
  Slot<V, kInter> slots[S];
#pragma unroll
  for (int i = 0; i < S; ++i) slots[i].at(l + i * kL, a.d, a.rot);
#pragma unroll
  for (int side = 0; side < 2; ++side)
    if (a.side[side].heads) weights<kInter>(a, a.side[side].w, w[side], kPairs);
  __syncthreads();
  const float inv_d = 1.f / (float)a.d;
  const uint32_t units = (uint32_t)(a.batch * a.tokens) * (uint32_t)a.parts;
  for (uint32_t unit = blockIdx.x * kWaves + wave; unit < units; unit += gridDim.x * kWaves) {
    const uint32_t token = unit / (uint32_t)a.parts, part = unit - token * (uint32_t)a.parts;
    const int64_t b = token / (uint32_t)a.tokens, t = token - (uint32_t)b * (uint32_t)a.tokens;
    const bool live = !a.mask || a.mask[b * a.mask_b + t * a.mask_t];
    float c[S][V], s[S][V];
    bool turned = false;
    int g = part, base = 0;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const Rows& r = a.side[side];
      const int heads = (int)r.heads, groups = (heads + kHeads - 1) / kHeads, end = base + groups;
      if (g < end) {
        int head = (g - base) * kHeads + sub;
        const char* x_row = r.x + b * r.x_b + t * r.x_t + head * r.x_h;
        char* out_row = r.out + b * r.o_b + t * r.o_t + head * r.o_h;
        const int64_t x_step = r.x_h * kHeads * a.parts, out_step = r.o_h * kHeads * a.parts;
        RawRow<DT, V, S, kInter> raw;
        raw.template load<kStream>(x_row, slots, head < heads && live);
        if (!turned) angles<V, kL, S>(a, b, t, tables[wave], lane, l, c, s);
        turned = true;
        float wa[S][V], wb[S][V];
        lane_weights<V, kL, S>(w[side], l, wa, wb);
        for (; g < end; g += a.parts) {
          Row<DT, V, S, kInter> x;
          x.unpack(raw);
          const bool in = head < heads;
          head += kHeads * a.parts;
          x_row += x_step;
          if (g + a.parts < end) raw.template load<kStream>(x_row, slots, head < heads && live);
          if (live) {  // a dead token's rows hold zeros, and stay so whatever weights and angles are
            float sq = 0.f;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
              for (int e = 0; e < V; ++e) sq += x.a[i][e] * x.a[i][e] + x.b[i][e] * x.b[i][e];
            const float rms = rsqrtf(lanes_sum<kL>(sq) * inv_d + a.eps);
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float ya = x.a[i][e] * rms * wa[i][e], yb = x.b[i][e] * rms * wb[i][e];
                x.a[i][e] = slots[i].turn ? ya * c[i][e] - yb * s[i][e] : ya;
                x.b[i][e] = slots[i].turn ? yb * c[i][e] + ya * s[i][e] : yb;
              }
          }
          x.store(out_row, slots, in);
          out_row += out_step;
        }
      }
      base = end;
    }
  }
}

// A workgroup owns one side's rows of `chunk` tokens of a sample; its waves
// take (token, group of heads) steps in turn and add their lanes' dw up, the
// waves' sums meet in LDS and go to the chunk's place of the partials in fp32.
// Three waves a SIMD fit its registers (130 for 8 lanes of bf16 runs, half-split); held
// to four at 139, it spilled (241 us).
template <int DT, int V, int kL, int S, bool kInter, bool kStream>
__global__ __launch_bounds__(kThreads) void qk_rope_backward(QkArgs a, int64_t q_blocks) {
  constexpr int kHeads = kWave / kL;
  constexpr int kPairs = kL * S * V;
  __shared__ float2 tables[kWaves][kPairs];
  __shared__ float w[2 * kPairs];
  __shared__ float sums[kWaves][2 * kPairs];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane % kL, sub = lane / kL;
  const int which = (int64_t)blockIdx.x >= q_blocks;
  const Rows& r = a.side[which];
  const int64_t block = (int64_t)blockIdx.x - (which ? q_blocks : 0);
  const int64_t b = block / r.chunks, chunk = block - b * r.chunks;
  Slot<V, kInter> slots[S];
#pragma unroll
  for (int i = 0; i < S; ++i) slots[i].at(l + i * kL, a.d, a.rot);
  const float inv_d = 1.f / (float)a.d;
  float wa[S][V], wb[S][V], da_[S][V], db_[S][V];
  const int groups = ((int)r.heads + kHeads - 1) / kHeads;
  if (groups) weights<kInter>(a, r.w, w, kPairs);  // an absent side has no weight to read
  __syncthreads();
#pragma unroll
  for (int i = 0; i < S; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) da_[i][e] = db_[i][e] = 0.f;
  const int64_t t0 = chunk * r.chunk, t1 = min(t0 + r.chunk, a.tokens);
  // Steps of (token, group of heads), the waves in turn; the next step's rows are loaded ahead.
  int64_t t = groups ? t0 + wave / groups : t1, last = -1;
  int g = groups ? wave % groups : 0;
  RawRow<DT, V, S, kInter> raw_x, raw_z;
  bool live = true;
  auto load = [&]() {
    live = !a.mask || a.mask[b * a.mask_b + t * a.mask_t];
    const int64_t head = g * kHeads + sub;
    raw_x.template load<kStream>(r.x + b * r.x_b + t * r.x_t + head * r.x_h, slots, head < r.heads && live);
    raw_z.template load<kStream>(r.gz + b * r.g_b + t * r.g_t + head * r.g_h, slots, head < r.heads && live);
  };
  if (t < t1) load();
  float c[S][V], s[S][V];
  while (t < t1) {
    if (t != last) {
      angles<V, kL, S>(a, b, t, tables[wave], lane, l, c, s);
      last = t;
    }
    const int64_t head = g * kHeads + sub;
    const bool in = head < r.heads, lives = live;
    char* out = r.out + b * r.o_b + t * r.o_t + head * r.o_h;
    Row<DT, V, S, kInter> x, z;
    x.unpack(raw_x);
    z.unpack(raw_z);
    for (g += kWaves; g >= groups; g -= groups) ++t;
    if (t < t1) load();
    asm volatile("" ::: "memory");  // the weights stay in LDS: registers bound the waves of a SIMD
    lane_weights<V, kL, S>(w, l, wa, wb);
    if (lives) {  // as in the forward pass: nothing into dw, dx as loaded, zero
      float sq = 0.f, along = 0.f;
#pragma unroll
      for (int i = 0; i < S; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float ya = slots[i].turn ? z.a[i][e] * c[i][e] + z.b[i][e] * s[i][e] : z.a[i][e];
          const float yb = slots[i].turn ? z.b[i][e] * c[i][e] - z.a[i][e] * s[i][e] : z.b[i][e];
          z.a[i][e] = ya;
          z.b[i][e] = yb;
          sq += x.a[i][e] * x.a[i][e] + x.b[i][e] * x.b[i][e];
          along += ya * wa[i][e] * x.a[i][e] + yb * wb[i][e] * x.b[i][e];
        }
      // Rows that are not there are zero, and stay zero without an eps.
      const float rms = in ? rsqrtf(lanes_sum<kL>(sq) * inv_d + a.eps) : 0.f;
      const float back = lanes_sum<kL>(along) * inv_d * rms * rms;
#pragma unroll
      for (int i = 0; i < S; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          da_[i][e] += z.a[i][e] * (x.a[i][e] * rms);
          db_[i][e] += z.b[i][e] * (x.b[i][e] * rms);
          z.a[i][e] = rms * (z.a[i][e] * wa[i][e] - x.a[i][e] * back);
          z.b[i][e] = rms * (z.b[i][e] * wb[i][e] - x.b[i][e] * back);
        }
    }
    z.store(out, slots, in);
  }
  if (!r.partial) return;
#pragma unroll
  for (int i = 0; i < S; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float u = da_[i][e], v = db_[i][e];
#pragma unroll
      for (int off = kL; off < kWave; off <<= 1) {
        u += __shfl_xor(u, off, kWave);
        v += __shfl_xor(v, off, kWave);
      }
      if (sub == 0) {
        sums[wave][((2 * i) * V + e) * kL + l] = u;
        sums[wave][((2 * i + 1) * V + e) * kL + l] = v;
      }
    }
  __syncthreads();
  if (wave == 0 && sub == 0) {
    float* out = r.partial + (b * r.chunks + chunk) * a.d;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float u = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          u += sums[w][((2 * i) * V + e) * kL + l];
          v += sums[w][((2 * i + 1) * V + e) * kL + l];
        }
        const int ia = kInter ? slots[i].a + 2 * e : slots[i].a + e;
        const int ib = kInter ? slots[i].a + 2 * e + 1 : slots[i].b + e;
        if (slots[i].in) out[ia] = u;
        if (slots[i].in && slots[i].has_b) out[ib] = v;
      }
  }
}

// dw of a sample: eight threads an entry take its chunks in turn and are added in
// order.
__global__ __launch_bounds__(kThreads) void qk_rope_join(QkArgs a) {
  __shared__ float sums[8][32];
  const Rows& r = a.side[blockIdx.z];
  if (!r.wgrad) return;
  const int64_t b = blockIdx.y;
  const int x = threadIdx.x % 32, y = threadIdx.x / 32, i = blockIdx.x * 32 + x;
  float v = 0.f;
  if (i < a.d) {
    const float* p = r.partial + b * r.chunks * a.d + i;
#pragma unroll 4
    for (int64_t c = y; c < r.chunks; c += 8) v += p[c * a.d];
  }
  sums[y][x] = v;
  __syncthreads();
  if (y == 0 && i < a.d) {
#pragma unroll
    for (int k = 1; k < 8; ++k) v += sums[k][x];
    r.wgrad[b * a.d + i] = v;
  }
}

int check_args(const char* what, const da_qk_side* sides, int dtype, int weight_dtype, int64_t batch, int64_t tokens,
               int64_t d, int64_t rot, const float* inv_freq, const void* positions, int position_bytes) {
  if (!valid_dtype(dtype) || !valid_dtype(weight_dtype))
    return set_error(DA_ERR_INVALID, "%s: bad dtype %d / %d", what, dtype, weight_dtype);
  if (!sides) return set_error(DA_ERR_INVALID, "%s: NULL sides", what);
  if (batch < 0 || tokens < 0 || sides[0].heads < 0 || sides[1].heads < 0)
    return set_error(DA_ERR_INVALID, "%s: negative size", what);
  if (d < 1 || d > kMaxD) return set_error(DA_ERR_UNSUPPORTED, "%s: head width %lld outside 1..1024", what, (long long)d);
  if (rot < 0 || rot % 2 || rot > d)
    return set_error(DA_ERR_INVALID, "%s: rotated width %lld must be even and at most the head width %lld", what,
                     (long long)rot, (long long)d);
  if (rot && !inv_freq) return set_error(DA_ERR_INVALID, "%s: NULL inv_freq", what);
  if (positions && position_bytes != 4 && position_bytes != 8)
    return set_error(DA_ERR_INVALID, "%s: positions must have 4 or 8 bytes", what);
  return DA_OK;
}

void fill_side(Rows& r, const da_qk_side& s, int es) {
  r = Rows{};
  r.x = (const char*)s.x;
  r.gz = (const char*)s.gz;
  r.out = (char*)s.out;
  r.w = s.weight;
  r.wgrad = s.weight_grad;
  r.heads = s.heads;
  r.x_b = s.x_bstride * es, r.x_t = s.x_tstride * es, r.x_h = s.x_hstride * es;
  r.g_b = s.gz_bstride * es, r.g_t = s.gz_tstride * es, r.g_h = s.gz_hstride * es;
  r.o_b = s.out_bstride * es, r.o_t = s.out_tstride * es, r.o_h = s.out_hstride * es;
}

// Backward: tokens of a workgroup of one side, about kRows rows, fewer where that
// leaves less than kWantBlocks workgroups.  (32 + 8 heads of 128, 8 x 2048 tokens:
// 256 rows 108 us, 1024 101, 2048 123.)
int64_t chunk_tokens(int64_t batch, int64_t tokens, int64_t heads) {
  const int64_t most = std::max<int64_t>(1, kRows / std::max<int64_t>(heads, 1));
  return std::max<int64_t>(1, std::min(most, batch * tokens / kWantBlocks));
}

}  // namespace
}  // namespace da

using namespace da;

// Entries of a lane's run: what every slot and every row's alignment allow, up to
// 16 bytes; then the lanes of a head, or its slots a lane.
namespace {
int run_entries(const QkArgs& a, int es, bool grad) {
  const int64_t d = a.d, rot = a.rot;
  for (int v = 16 / es; v > 1; v = v == 8 ? 4 : 1) {
    bool fits = rot / 2 % v == 0 && (d - rot) % (2 * v) == 0;
    for (int i = 0; i < 2 && fits; ++i) {
      const Rows& s = a.side[i];
      if (!s.heads) continue;
      int64_t all = (int64_t)s.x | (int64_t)s.out;
      if (grad) all |= (int64_t)s.gz;
      // the stride of an axis of one entry says nothing
      if (a.batch > 1) all |= s.x_b | s.o_b | (grad ? s.g_b : 0);
      if (a.tokens > 1) all |= s.x_t | s.o_t | (grad ? s.g_t : 0);
      if (s.heads > 1) all |= s.x_h | s.o_h | (grad ? s.g_h : 0);
      fits = (uint64_t)all % (uint64_t)(v * es) == 0;
    }
    if (fits) return v;
  }
  return 1;
}
}  // namespace

namespace {

// Launches the forward or the backward kernel for the operands' type, the entries
// of a run, the lanes of a head (one slot each, or several slots of 64 lanes) and
// the order of the pairs.
struct Launch {
  const QkArgs& a;
  bool grad;
  int64_t blocks, q_blocks;
  hipStream_t stream;

  template <int DT, int V, int kL, int S, bool kInter, bool kStream>
  void kernel() const {
    if (grad) qk_rope_backward<DT, V, kL, S, kInter, kStream><<<(unsigned)blocks, kThreads, 0, stream>>>(a, q_blocks);
    else qk_rope_forward<DT, V, kL, S, kInter, kStream><<<(unsigned)blocks, kThreads, 0, stream>>>(a);
  }
  template <int DT, int V, bool kInter, bool kStream>
  void lanes(int64_t slots) const {
    if (slots <= 4) kernel<DT, V, 4, 1, kInter, kStream>();
    else if (slots <= 8) kernel<DT, V, 8, 1, kInter, kStream>();
    else if (slots <= 16) kernel<DT, V, 16, 1, kInter, kStream>();
    else if (slots <= 32) kernel<DT, V, 32, 1, kInter, kStream>();
    else if (V == 8 || slots <= 64) kernel<DT, V, 64, 1, kInter, kStream>();
    else if constexpr (V == 4) kernel<DT, V, 64, 2, kInter, kStream>();
  }
  template <int DT, bool kInter>
  void runs(int v, int64_t pairs, bool streamed) const {
    constexpr int kFull = 16 / Elem<DT>::kBytes;
    if (v == kFull && streamed) lanes<DT, kFull, kInter, true>(pairs / v);
    else if (v == kFull) lanes<DT, kFull, kInter, false>(pairs / v);
    else if (v == 4) lanes<DT, 4, kInter, false>(pairs / v);
    else if (pairs <= 64) kernel<DT, 1, 64, 1, kInter, false>();
    else if (pairs <= 128) kernel<DT, 1, 64, 2, kInter, false>();
    else if (pairs <= 256) kernel<DT, 1, 64, 4, kInter, false>();
    else kernel<DT, 1, 64, 8, kInter, false>();
  }
  void operator()(int dtype, bool interleaved, int v, int64_t pairs) const {
    const bool streamed = rows_bytes() >= kStreamBytes;
    if (dtype == DA_BF16) interleaved ? runs<DA_BF16, true>(v, pairs, streamed) : runs<DA_BF16, false>(v, pairs, streamed);
    else if (dtype == DA_F16) interleaved ? runs<DA_F16, true>(v, pairs, streamed) : runs<DA_F16, false>(v, pairs, streamed);
    else interleaved ? runs<DA_F32, true>(v, pairs, streamed) : runs<DA_F32, false>(v, pairs, streamed);
  }
  int64_t rows_bytes() const {
    return a.batch * a.tokens * (a.side[0].heads + a.side[1].heads) * a.d * bytes * (grad ? 2 : 1);
  }
  int bytes;  // of an entry
};

}  // namespace

extern "C" {

int da_qk_norm_rope(const da_qk_side* sides, int dtype, int weight_dtype, int64_t batch, int64_t tokens, int64_t d,
                    int64_t rot, const float* inv_freq, const void* positions, int position_bytes,
                    int64_t pos_bstride, int64_t pos_tstride, const uint8_t* mask, int64_t mask_bstride,
                    int64_t mask_tstride, int interleaved, float scaling, float eps, void* stream) {
  if (int rc = check_args("da_qk_norm_rope", sides, dtype, weight_dtype, batch, tokens, d, rot, inv_freq, positions,
                          position_bytes))
    return rc;
  QkArgs a{};
  const int es = (int)elem_bytes(dtype);
  for (int i = 0; i < 2; ++i) {
    if (batch && tokens && sides[i].heads && (!sides[i].x || !sides[i].out || !sides[i].weight))
      return set_error(DA_ERR_INVALID, "da_qk_norm_rope: NULL pointer of side %d", i);
    fill_side(a.side[i], sides[i], es);
  }
  if (!batch || !tokens || !(sides[0].heads + sides[1].heads)) return DA_OK;
  a.batch = batch, a.tokens = tokens, a.d = (int)d, a.rot = (int)rot, a.w_dtype = weight_dtype;
  a.inv_freq = inv_freq, a.pos = positions, a.pos_bytes = position_bytes, a.pos_b = pos_bstride, a.pos_t = pos_tstride;
  a.mask = mask, a.mask_b = mask_bstride, a.mask_t = mask_tstride, a.scaling = scaling, a.eps = eps;
  hipStream_t st = (hipStream_t)stream;
  const int64_t pairs = rot / 2 + (d - rot + 1) / 2;
  const int v = run_entries(a, es, false);
  const int64_t slots = pairs / v;
  int lanes = 4;
  while (lanes < 64 && lanes < slots) lanes *= 2;
  const int64_t per_step = kWave / lanes;  // heads
  const int64_t groups = (sides[0].heads + per_step - 1) / per_step + (sides[1].heads + per_step - 1) / per_step;
  a.parts = (int)std::min<int64_t>(groups, std::max<int64_t>(1, kWantWaves / (batch * tokens)));
  if (batch * tokens * a.parts > 0x7fffffff || sides[0].heads > 65535 || sides[1].heads > 65535)
    return set_error(DA_ERR_UNSUPPORTED, "da_qk_norm_rope: up to 2^31 tokens and 65535 heads");
  const int64_t blocks = std::min<int64_t>((batch * tokens * a.parts + kWaves - 1) / kWaves, kMostBlocks);
  Launch{a, false, blocks, 0, st, es}(dtype, interleaved, v, pairs);
  return check_launch("da_qk_norm_rope");
}

int da_qk_norm_rope_grad_workspace(int64_t batch, int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t d,
                                   size_t* bytes) {
  if (!bytes || batch < 0 || tokens < 0 || q_heads < 0 || k_heads < 0 || d < 0)
    return set_error(DA_ERR_INVALID, "da_qk_norm_rope_grad_workspace: bad argument");
  *bytes = 0;
  for (int64_t heads : {q_heads, k_heads}) {
    const int64_t chunk = chunk_tokens(batch, tokens, heads);
    *bytes += (size_t)(batch * ((tokens + chunk - 1) / chunk) * d) * sizeof(float);
  }
  return DA_OK;
}

int da_qk_norm_rope_grad(const da_qk_side* sides, int dtype, int weight_dtype, int64_t batch, int64_t tokens,
                         int64_t d, int64_t rot, const float* inv_freq, const void* positions, int position_bytes,
                         int64_t pos_bstride, int64_t pos_tstride, const uint8_t* mask, int64_t mask_bstride,
                         int64_t mask_tstride, int interleaved, float scaling, float eps, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (int rc = check_args("da_qk_norm_rope_grad", sides, dtype, weight_dtype, batch, tokens, d, rot, inv_freq,
                          positions, position_bytes))
    return rc;
  QkArgs a{};
  const int es = (int)elem_bytes(dtype);
  bool wanted = false;
  for (int i = 0; i < 2; ++i) {
    if (batch && tokens && sides[i].heads && (!sides[i].x || !sides[i].gz || !sides[i].out || !sides[i].weight))
      return set_error(DA_ERR_INVALID, "da_qk_norm_rope_grad: NULL pointer of side %d", i);
    fill_side(a.side[i], sides[i], es);
    wanted |= sides[i].weight_grad != nullptr;
  }
  if (!batch) return DA_OK;
  hipStream_t st = (hipStream_t)stream;
  size_t need = 0;
  for (int i = 0; i < 2; ++i) {
    Rows& r = a.side[i];
    r.chunk = chunk_tokens(batch, tokens, r.heads);
    r.chunks = (tokens + r.chunk - 1) / r.chunk;
    if (!r.wgrad) continue;
    r.partial = (float*)((char*)workspace + need);
    need += (size_t)(batch * r.chunks * d) * sizeof(float);
  }
  if (need && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "da_qk_norm_rope_grad: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  a.batch = batch, a.tokens = tokens, a.d = (int)d, a.rot = (int)rot, a.w_dtype = weight_dtype;
  a.inv_freq = inv_freq, a.pos = positions, a.pos_bytes = position_bytes, a.pos_b = pos_bstride, a.pos_t = pos_tstride;
  a.mask = mask, a.mask_b = mask_bstride, a.mask_t = mask_tstride, a.scaling = scaling, a.eps = eps;
  const int64_t pairs = rot / 2 + (d - rot + 1) / 2;
  const int v = run_entries(a, es, true);
  const int64_t q_blocks = batch * a.side[0].chunks, blocks = q_blocks + batch * a.side[1].chunks;
  if (blocks > kMaxBlocks || batch > 65535 || sides[0].heads > 65535 || sides[1].heads > 65535)
    return set_error(DA_ERR_UNSUPPORTED, "da_qk_norm_rope_grad: too many tokens; up to 65535 samples and heads");
  if (blocks) {
    Launch{a, true, blocks, q_blocks, st, es}(dtype, interleaved, v, pairs);
    if (int rc = check_launch("da_qk_norm_rope_grad")) return rc;
  }
  if (wanted) {
    qk_rope_join<<<dim3((unsigned)((d + 31) / 32), (unsigned)batch, 2), kThreads, 0, st>>>(a);
    return check_launch("da_qk_norm_rope_grad (join)");
  }
  return DA_OK;
}

}  // extern "C"
