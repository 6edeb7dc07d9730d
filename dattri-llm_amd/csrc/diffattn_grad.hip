// Attention by the difference of two softmax maps, backward.
//
// With p_m the maps (from the scores, and the forward call's largest ones and sums), g the
// gradient of out:
//
//   dp = g v^T,   delta_m = g . o_m
//   ds_1 = p_1 (dp - delta_1),   ds_2 = -lam p_2 (dp - delta_2)
//   dq_m = scale ds_m k_m,   dk_m = scale ds_m^T q_m,   dv = (p_1 - lam p_2)^T g
//   dlam[sample] = -sum of delta_2
//
// No atomic sums, so that results do not change from run to run, and five launches: delta; dq, a
// wave holding 32 rows and going over their keys; the records of rows and dlam's parts; these
// joined; dk and dv, a wave holding 32 keys and going over all rows of their heads.  Either large
// pass has a join more where it is split, and fp16 two launches for the sizes of g and v.  The
// scores are formed twice, the price of sums that are nobody else's.  Where keys are columns, the
// scores' registers are rows and stand as the operand that is contracted over rows; where rows are
// columns, they are keys: neither pass moves a score between lanes.
//
// What is rounded to 16 bits: ds and the maps' mixture where they are operands, by half a step
// of each entry, no more than the outputs' own rounding; and out and o_2, from which delta
// comes, off by as much for a whole row.  dq therefore takes ds as the sum of two 16-bit
// values (with one, its error was 1.6 times that of its rounding; it costs 79 of 800 us at the
// size below), and its pass sums ds in fp32: the sum of ds_m is how far delta_m was off, as the
// maps sum to one.  The pass of dk and dv and dlam have delta from there, and so has dq where a
// row sees few keys (kFewKeys).
//
// fp16 would lose small values of ds: there ds is scaled by the power of two that brings the
// bound of the largest to 2^14, and the maps' mixture by one that its factors allow; their products
// are scaled back.  Each sample's key heads have a bound of their own: what a sample gets does not
// depend on the others in its batch.
//
// 4 x 2048 tokens, 32 heads on 8, two 64-wide maps, 128-wide values, causal, bf16: delta 36 us,
// dq 355 us and dk, dv 437 us of 275 GFLOP each (770 and 630 TFLOP/s), records 11 us.  Both large
// passes are bound by the vector unit (two exponentials and some twenty instructions an entry of
// the maps) and the matrix unit nearly in sum: with the registers of two waves a SIMD there is
// little to put under the other one's work.  dk and dv wait for the first keys' workgroups besides,
// which have the most rows.
#include <algorithm>
#include <type_traits>

#include "diffattn.h"

namespace da {
namespace diff {
namespace {

// ---------------------------------------------------------------------------
// delta, its records, parts of dlam, largest |g|: workgroups (b, h, chunk of tokens), 16 lanes
// a token.
//
// Where keys are columns, a row's lse and delta are needed in every lane, by register.  In
// 16 bits they come with the products instead: one more step of contraction over their parts
// (three bf16 values hold 24 bits) against ones makes the scores' accumulators z - top - lse / c
// and g v^T - delta, from two reads of LDS in place of sixteen.  A record then is the parts of
// [-top_1, -lse_1 / c | -delta_1 | -top_2, -lse_2' / c | delta_1 - delta_2], eight entries each;
// else it is the six values in fp32.  lse_2' = lse_2 - log2 |lam|: the factor comes with the
// exponential.  A tile with large scores takes top and lse in two steps: the sum of both would
// be rounded to top's last place.  A row without keys has an exponential of nothing, by a finite
// number: no product is NaN.
// ---------------------------------------------------------------------------
constexpr int kLanes = 16;
constexpr float kNothing = -1e30f;
// In 16 bits lse + top c as one number is off by half a unit of its last place, 2^-15 up to here:
// no more than a tenth of the half step that the maps are rounded by.
constexpr float kNear = 1024.f;
__device__ __forceinline__ bool near(float top0, float top1, float c) {
  return fabsf(top0 * c) < kNear && fabsf(top1 * c) < kNear;
}

template <int DT>
struct Record {
  static constexpr bool kParts = DT != DA_F32;
  static constexpr int kBytes = kParts ? 64 : 32;
};

__device__ __forceinline__ u32x4 three_parts(float x) {
  const uint32_t hi = f32_to_bf16_bits(x);
  const float r1 = x - bf16_bits_to_f32(hi);
  const uint32_t mid = f32_to_bf16_bits(r1);
  const uint32_t lo = f32_to_bf16_bits(r1 - bf16_bits_to_f32(mid));
  return u32x4{hi | mid << 16, lo, 0, 0};
}
__device__ __forceinline__ u32x4 six_parts(float x, float y) {
  const u32x4 u = three_parts(x), v = three_parts(y);
  return u32x4{u[0], u[1] | v[0] << 16, v[0] >> 16 | v[1] << 16, 0};
}

template <int DT>
__device__ __forceinline__ void put_record(char* to, float c, float top0, float top1, float lse0, float lse1, float de0,
                                           float de1) {
  if constexpr (Record<DT>::kParts) {
    const bool some0 = lse0 != __builtin_inff(), some1 = lse1 != __builtin_inff();
    st16(to, six_parts(some0 ? -top0 : kNothing, some0 ? -lse0 / c : 0.f));
    st16(to + 16, three_parts(-de0));
    st16(to + 32, six_parts(some1 ? -top1 : kNothing, some1 ? -lse1 / c : 0.f));
    st16(to + 48, three_parts(de0 - de1));
  } else {
    *(f32x4*)to = f32x4{top0, top1, lse0, lse1};
    *(f32x4*)(to + 16) = f32x4{de0, de1, 0.f, 0.f};
  }
}

// Rows that are not finite have no say in a scale.
__device__ __forceinline__ float finite(float norm) { return norm < __builtin_inff() ? norm : 0.f; }

template <int DT>
__global__ __launch_bounds__(256) void diff_delta(Args a) {
  constexpr int ES = Type<DT>::ES, V = Type<DT>::V, kRows = 256 / kLanes;
  const int heads = a.Hk * a.G, l = threadIdx.x % kLanes, sub = threadIdx.x / kLanes;
  const int chunk = blockIdx.x % a.chunks;
  const int h = blockIdx.x / a.chunks % heads, b = blockIdx.x / a.chunks / heads;
  const int hk = h / a.G, rows = a.T * a.G;
  const float lam = lam_of(a, h);
  const int t1 = min((chunk + 1) * a.chunk, a.T);
  float most = 0.f;
  for (int t = chunk * a.chunk + sub; t < t1; t += kRows) {
    const int64_t of = (int64_t)b * a.Hk + hk;
    const int r = t * a.G + (h - hk * a.G);
    // Of a row that sees no key nothing is read: its gradient may be anything.
    const bool live = a.lse[of * 2 * rows + r] != __builtin_inff();
    float d0 = 0.f, d1 = 0.f, norm = 0.f;
    if (live) {
      const char* g = a.g + (b * a.g_b + t * a.g_t + h * a.g_h) * ES;
      const int64_t at = (((int64_t)b * a.T + t) * heads + h) * a.Dv * ES;
      for (int e0 = l * V; e0 < a.Dv; e0 += kLanes * V) {
        float x[V], y[V], z[V];
        unpack16<DT>(load_run<DT>(g, e0, a.Dv), x);
        unpack16<DT>(load_run<DT>(a.out + at, e0, a.Dv), y);
        unpack16<DT>(load_run<DT>(a.second + at, e0, a.Dv), z);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          d0 += x[e] * y[e];
          d1 += x[e] * z[e];
          if constexpr (DT == DA_F16) norm += x[e] * x[e];
        }
      }
    }
    d0 = lanes_sum<kLanes>(d0);
    d1 = lanes_sum<kLanes>(d1);
    if constexpr (DT == DA_F16) most = fmaxf(most, finite(lanes_sum<kLanes>(norm)));
    if (l == 0) {
      float* to = a.delta + of * 2 * rows + r;
      to[0] = d0 + lam * d1;  // o_1 = out + lam o_2
      to[rows] = d1;
    }
  }
  if constexpr (DT == DA_F16) {  // a maximum: the order does not matter
    most = lanes_max<64>(most) * fmaxf(1.f, lam * lam);
    if (threadIdx.x % 64 == 0 && most > 0.f)
      atomicMax((unsigned*)a.most + 2 * ((int64_t)b * a.Hk + hk), __float_as_uint(most));
  }
}

// The largest norm of the values' rows that a query may see, squared: 16 lanes a row.  Workgroup
// (b, key head, one of `parts`).
__global__ __launch_bounds__(256) void diff_values_norm(Args a, int parts) {
  constexpr int V = Type<DA_F16>::V, kRows = 256 / kLanes;
  const int l = threadIdx.x % kLanes, part = blockIdx.x % parts;
  const int64_t of = blockIdx.x / parts;
  const int hk = (int)(of % a.Hk), b = (int)(of / a.Hk);
  float most = 0.f;
  for (int64_t at = (int64_t)part * kRows + threadIdx.x / kLanes; at < a.S; at += (int64_t)parts * kRows) {
    const int key = (int)at;
    float norm = 0.f;
    if (!(a.causal && key >= a.T + a.q_start) && (!a.mask || a.mask[b * a.m_b + key * a.m_k])) {
      const char* v = a.v + (b * a.v_b + key * a.v_t + hk * a.v_h) * 2;
      for (int e0 = l * V; e0 < a.Dv; e0 += kLanes * V) {
        float x[V];
        unpack16<DA_F16>(load_run<DA_F16>(v, e0, a.Dv), x);
#pragma unroll
        for (int e = 0; e < V; ++e) norm += x[e] * x[e];
      }
    }
    most = fmaxf(most, finite(lanes_sum<kLanes>(norm)));
  }
  most = lanes_max<64>(most);
  if (threadIdx.x % 64 == 0 && most > 0.f) atomicMax((unsigned*)a.most + 2 * of + 1, __float_as_uint(most));
}

// After dq: delta as the maps in fp32 have it, the records, and dlam's parts.
template <int DT>
__global__ __launch_bounds__(256) void diff_records(Args a) {
  __shared__ float parts[256 / kWave];
  const int heads = a.Hk * a.G, chunk = blockIdx.x % a.chunks;
  const int h = blockIdx.x / a.chunks % heads, b = blockIdx.x / a.chunks / heads;
  const int hk = h / a.G, rows = a.T * a.G;
  const float lam = lam_of(a, h), c = a.scale * kLog2e, bits = log2f(fabsf(lam));
  const int t1 = min((chunk + 1) * a.chunk, a.T);
  const int64_t of = (int64_t)b * a.Hk + hk, all = (int64_t)a.batch * a.Hk * 2 * rows;
  float sum = 0.f;
  for (int t = chunk * a.chunk + threadIdx.x; t < t1; t += 256) {
    const int r = t * a.G + (h - hk * a.G);
    const int64_t at = of * 2 * rows + r;
    float d0 = a.delta[at], d1 = a.delta[at + rows];
    if constexpr (DT != DA_F32)
      for (int p = 0; p < a.row_splits; ++p) d0 += a.off[p * all + at], d1 += a.off[p * all + at + rows];
    const float* tops = a.lse + tops_at(a) + at;
    const float lse0 = a.lse[at];
    put_record<DT>(a.records + (of * rows + r) * Record<DT>::kBytes, c, tops[0], tops[rows], lse0, a.lse[at + rows] - bits,
                   d0, d1);
    a.takes_part[of * rows + r] = lse0 == __builtin_inff() ? 0 : near(tops[0], tops[rows], c) ? 1 : 3;
    sum += d1;
  }
  sum = lanes_sum<kWave>(sum);
  if (threadIdx.x % kWave == 0) parts[threadIdx.x / kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.lam_part[blockIdx.x] = -(parts[0] + parts[1] + parts[2] + parts[3]);
}

__global__ __launch_bounds__(256) void diff_lam_join(const float* parts, float* out, int64_t n, int chunks) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float v = 0.f;
  for (int c = 0; c < chunks; ++c) v += parts[i * chunks + c];
  out[i] = v;
}

// fp16: a power of two under which no |ds| <= 2 max(1, |lam|) |g| |v| passes 2^14, and the
// largest are near it: the maps' small entries keep their bits.  1 where there is none.
template <int DT>
__device__ __forceinline__ float small_scale(const Args& a, int b, int hk) {
  if constexpr (DT != DA_F16) return 1.f;
  const float* most = a.most + 2 * ((int64_t)b * a.Hk + hk);
  const float bound = __builtin_sqrtf(most[0]) * __builtin_sqrtf(most[1]);
  const uint32_t e = __float_as_uint(bound) >> 23;  // bound < 2^(e - 126); of a float from zero on
  return e < 40 || e > 220 ? 1.f : __uint_as_float((266u - e) << 23);  // 2^(139 - e)
}

// ---------------------------------------------------------------------------
// dk and dv: four waves of 32 keys over the rows r = t G + g of their key head.
// ---------------------------------------------------------------------------
constexpr int kWaves = 4, kThreads = kWaves * kWave;

// In 16 bits the values of a wave's keys lie in LDS, read again for every tile of rows: with
// them in registers there is room for one wave a SIMD only.
template <int DT, int DP, int DVP>
struct KeySmem {
  static constexpr int kQ = Tile<DT, DP, kThreads>::kBytes, kG = Tile<DT, DVP, kThreads>::kBytes;
  static constexpr int kR = Record<DT>::kParts ? kTile * 64 : 1024;  // one load a wave writes 1 KB
  static constexpr int kStage = 2 * kQ + kG + kR;
  static constexpr bool kValues = DT != DA_F32;
  static constexpr int kOf = kValues ? kG : 0;  // a wave's values
  // A thread's offsets of rows.  They lie in LDS too: kept in registers they would be spilled,
  // and a load of a spilled one waits for the tiles under way.
  static constexpr int kOffsets = (Tile<DT, DP, kThreads>::N + Tile<DT, DVP, kThreads>::N + 3) / 4;
  static constexpr int kOffsetsAt = 2 * kStage + kWaves * kOf;
  static constexpr int kBytes = kOffsetsAt + kOffsets * kThreads * 16;
};

template <int DT, int DP, int DVP>
__global__ __launch_bounds__(kThreads, DT != DA_F32 && DP == 64 ? 2 : 1) void diff_grad_keys(Args a) {
  using L = KeySmem<DT, DP, DVP>;
  using Rec = Record<DT>;
  constexpr int ES = Type<DT>::ES, V = Type<DT>::V;
  constexpr int KD = DP / Type<DT>::kStep, KV = DVP / Type<DT>::kStep, KC = Type<DT>::kChunks;
  constexpr int ND = DP / 32, NV = DVP / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int at, block;
  deal(a.batch * a.Hk * a.splits, a.blocks, &at, &block);  // the first keys have the most rows
  const int split = at % a.splits;
  at /= a.splits;
  const int hk = at % a.Hk, b = at / a.Hk;
  const int key0 = (block * kWaves + wave) * kTile, key = key0 + (lane & 31);
  const int rows = a.T * a.G, end = min(rows, (split + 1) * a.each);
  // The rows that see a key are those from this one on.
  const auto first_row = [&](int to) {
    const int64_t t = to - a.q_start;
    return !a.causal || t <= 0 ? 0 : t >= a.T ? rows : (int)t * a.G;
  };
  const bool alive = key < a.S && first_row(key) < rows && (!a.mask || a.mask[b * a.m_b + key * a.m_k]);
  u32x4 k[2][KD], v[L::kValues ? 1 : KV];
#pragma unroll
  for (int kk = 0; kk < KD; ++kk)
#pragma unroll
    for (int m = 0; m < 2; ++m)
      k[m][kk] = alive ? load_run<DT>(a.k + (b * a.k_b + key * a.k_t + (2 * hk + m) * a.k_h) * ES,
                                      (2 * kk + half) * V, a.D) : u32x4{0, 0, 0, 0};
  char* lv = lds + 2 * L::kStage + wave * L::kOf;
#pragma unroll
  for (int kk = 0; kk < KV; ++kk) {
    const u32x4 x = alive ? load_run<DT>(a.v + (b * a.v_b + key * a.v_t + hk * a.v_h) * ES, (2 * kk + half) * V, a.Dv)
                          : u32x4{0, 0, 0, 0};
    if constexpr (L::kValues) {
      constexpr int kRow = DVP * ES;
      const int row = lane & 31;
      st16(lv + row * kRow + (((2 * kk + half) ^ swizzle<kRow>(row)) << 4), x);
    } else {
      v[kk] = x;
    }
  }
  const bool work = __any(alive);
  f32x16 dk[2][ND], dv[NV];
#pragma unroll
  for (int n = 0; n < ND; ++n) dk[0][n] = zeros(), dk[1][n] = zeros();
#pragma unroll
  for (int n = 0; n < NV; ++n) dv[n] = zeros();
  const float c = a.scale * kLog2e, small = small_scale<DT>(a, b, hk);
  // Ones against the parts of one half's records.
  constexpr uint32_t kOnes = 0x3f803f80u, kOne = 0x3f80u;
  const uint32_t in_low = half ? 0u : ~0u;

  // Of the wave's keys, some and all.
  const int from_some = first_row(key0), from_all = first_row(key0 + kTile - 1);
  const int first = max(split * a.each, first_row(block * kWaves * kTile) / kTile * kTile);
  const uint32_t q_token = (uint32_t)(a.q_t * ES), q_head = (uint32_t)(2 * a.q_h * ES);
  const uint32_t g_token = (uint32_t)(a.g_t * ES), g_head = (uint32_t)(a.g_h * ES);
  const char* qp = a.q + (b * a.q_b + (int64_t)2 * hk * a.G * a.q_h) * ES;
  const char* gp = a.g + (b * a.g_b + (int64_t)hk * a.G * a.g_h) * ES;
  const char* records = a.records + ((int64_t)b * a.Hk + hk) * rows * Rec::kBytes;
  const bool steady = kTile % a.G == 0;
  using Q = Rows<DT, DP, kThreads>;
  using G = Rows<DT, DVP, kThreads>;
  const auto place = [&](int r0, uint32_t* at) __attribute__((always_inline)) {
    Q::place(a, r0, q_token, q_head, a.D, at);
    G::place(a, r0, g_token, g_head, a.Dv, at + Q::N);
  };
  {
    uint32_t at[4 * L::kOffsets] = {};
    place(first, at);
#pragma unroll
    for (int i = 0; i < L::kOffsets; ++i)
      st16(lds + L::kOffsetsAt + (i * kThreads + threadIdx.x) * 16,
           u32x4{at[4 * i], at[4 * i + 1], at[4 * i + 2], at[4 * i + 3]});
  }
  // Negative factors: their sign is not in the exponential.  fp16: the maps' mixture, at most
  // 1 + |lam|, times the power of two that brings that bound to 2^15.
  bool any_minus = false;
  float most_lam = 0.f;
  for (int i = lane; i < a.G; i += kWave) {
    const float lam = lam_of(a, hk * a.G + i);
    any_minus |= lam < 0.f;
    most_lam = fmaxf(most_lam, fabsf(lam));
  }
  any_minus = __any(any_minus);
  float mixture = 1.f;
  if constexpr (DT == DA_F16)  // 1 + |lam| < 2^(e - 126)
    mixture = __uint_as_float((268u - (__float_as_uint(1.f + lanes_max<kWave>(most_lam)) >> 23)) << 23);
  const uint8_t* takes_part = a.takes_part + ((int64_t)b * a.Hk + hk) * rows;
  auto row_byte = [&](int r0) {
    const int r = r0 + (lane & 31);
    return r < end ? takes_part[r] : 0;
  };
  auto fetch = [&](int r0, int stage, uint32_t live) {
    const int64_t t0 = token_of(a, r0);
    const uint32_t l = lds_address(lds) + stage * L::kStage;
    int thread = threadIdx.x;
    asm("" : "+v"(thread) : "s"(r0));  // what follows from it is formed anew in each tile
    uint32_t at[4 * L::kOffsets];
    if (steady) {
#pragma unroll
      for (int i = 0; i < L::kOffsets; ++i) {
        const u32x4 x = lds16(lds_address(lds) + L::kOffsetsAt + (i * kThreads + thread) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) at[4 * i + e] = x[e];
      }
    } else {
      place(r0, at);
    }
    Q::fetch(qp + t0 * a.q_t * ES, l, at, live, thread);
    Q::fetch(qp + (t0 * a.q_t + a.q_h) * ES, l + L::kQ, at, live, thread);
    G::fetch(gp + t0 * a.g_t * ES, l + 2 * L::kQ, at + Q::N, live, thread);
    if (wave * 1024 < kTile * Rec::kBytes) {  // rows past the end have records of zeros
      const int row = thread / (Rec::kBytes / 16);
      int column = thread % (Rec::kBytes / 16);
      if constexpr (Rec::kParts) column ^= swizzle<64>(row);
      dma16(uniform4(make_rsrc(records + (int64_t)r0 * Rec::kBytes, kOutside - 1)), l + 2 * L::kQ + L::kG + wave * 1024,
            row < kTile && r0 + row < end ? row * Rec::kBytes + column * 16 : kOutside);
    }
  };
  int byte = 0;
  bool far_next = false;  // whether the tile under way has large scores
  if (first < end) {
    byte = row_byte(first);
    far_next = __any(byte & 2);
    fetch(first, 0, key_word(byte));
    byte = row_byte(first + kTile);
  }
  const Reader<DT, DP> q_reader(lds, lane);
  const Reader<DT, DVP> g_reader(lds + 2 * L::kQ, lane);
  const int to_values = 2 * L::kStage + wave * L::kOf - 2 * L::kQ;  // of the wave's keys, from g's tile
  const Reader<DT, 32> record_reader(lds + 2 * L::kQ + L::kG, lane);
  const auto step = [&](int r0, auto of) __attribute__((always_inline)) {
    constexpr int stage = decltype(of)::value;
    constexpr int skip = stage * L::kStage;
    tiles_barrier();
    const bool far = far_next;
    if (r0 + kTile < end) {
      far_next = __any(byte & 2);
      fetch(r0 + kTile, stage ^ 1, key_word(byte));
      byte = row_byte(r0 + 2 * kTile);
    }
    if (!work || r0 + kTile <= from_some) return;
    const auto lq = q_reader.fresh(r0);
    const auto lg = g_reader.fresh(r0);
    f32x16 s0 = zeros(), s1 = zeros(), dp = zeros(), dp1;
#pragma unroll
    for (int kk = 0; kk < KD; ++kk) {
      Mfma32<DT>::mma(s0, lq.rows(skip, kk), k[0][kk]);
      Mfma32<DT>::mma(s1, lq.rows(skip + L::kQ, kk), k[1][kk]);
    }
#pragma unroll
    for (int kk = 0; kk < KV; ++kk) {
      if constexpr (L::kValues) Mfma32<DT>::mma(dp, lg.rows(skip, kk), lg.rows(to_values, kk));
      else Mfma32<DT>::mma(dp, lg.rows(skip, kk), v[kk]);
    }
    if constexpr (Rec::kParts) {
      const auto lr = record_reader.fresh(r0);
      const u32x4 r1 = lr.rows(skip, 0), r2 = lr.rows(skip, 1);
      uint32_t low = in_low;
      asm("" : "+v"(low) : "s"(r0));  // two instructions a tile instead of eight registers
      u32x4 of_low = {kOnes & low, kOnes & low, kOnes & low, 0};
      const u32x4 of_high = {kOnes & ~low, kOne & ~low, 0, 0};
      if (far) {
        const u32x4 of_top = {kOnes & low, kOne & low, 0, 0};
        Mfma32<DA_BF16>::mma(s0, r1, of_top);
        Mfma32<DA_BF16>::mma(s1, r2, of_top);
        of_low[0] = 0, of_low[1] = kOne << 16 & low;
      }
      Mfma32<DA_BF16>::mma(s0, r1, of_low);
      Mfma32<DA_BF16>::mma(s1, r2, of_low);
      Mfma32<DA_BF16>::mma(dp, r1, of_high);
      dp1 = dp;
      Mfma32<DA_BF16>::mma(dp1, r2, of_high);
    } else {
      dp1 = dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const f32x4* record = (const f32x4*)(lds + skip + 2 * L::kQ + L::kG + acc_at(i, half) * Rec::kBytes);
        const f32x4 x = record[0], y = record[1];
        s0[i] = fmaf(s0[i] - x[0], c, -x[2]);
        s1[i] = fmaf(s1[i] - x[1], c, -x[3]);
        dp[i] -= y[0];
        dp1[i] -= y[1];
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s0[i] = __builtin_amdgcn_exp2f(Rec::kParts ? s0[i] * c : s0[i]);
      s1[i] = __builtin_amdgcn_exp2f(Rec::kParts ? s1[i] * c : s1[i]);
    }
    if (any_minus) {
      const int r = r0 + (lane & 31);
      const uint32_t minus =
          (uint32_t)__ballot(r < rows && lam_of(a, hk * a.G + r - token_of(a, r) * a.G) < 0.f) >> (4 * half);
#pragma unroll
      for (int i = 0; i < 16; ++i) s1[i] = minus & 1u << acc_at(i, 0) ? -s1[i] : s1[i];
    }
    if (r0 < from_all) {
      const int n = first_row(key0 + (lane & 31)) - r0;
      const uint32_t seen = (n <= 0 ? ~0u : n >= kTile ? 0u : ~0u << n) >> (4 * half);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s0[i] = seen & 1u << acc_at(i, 0) ? s0[i] : 0.f;
        s1[i] = seen & 1u << acc_at(i, 0) ? s1[i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p0 = s0[i], p1 = s1[i];
      s0[i] = (DT == DA_F16 ? p0 * small : p0) * dp[i];
      s1[i] = (DT == DA_F16 ? p1 * small : p1) * -dp1[i];
      dp[i] = DT == DA_F16 ? (p0 - p1) * mixture : p0 - p1;
    }
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      const u32x4 x = from_acc<DT>(dp, j), y0 = from_acc<DT>(s0, j), y1 = from_acc<DT>(s1, j);
#pragma unroll
      for (int n = 0; n < NV; ++n) Mfma32<DT>::mma(dv[n], lg.columns(skip, n, j), x);
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        Mfma32<DT>::mma(dk[0][n], lq.columns(skip, n, j), y0);
        Mfma32<DT>::mma(dk[1][n], lq.columns(skip + L::kQ, n, j), y1);
      }
    }
  };
  for (int r0 = first; r0 < end; r0 += 2 * kTile) {
    step(r0, std::integral_constant<int, 0>{});
    if (r0 + kTile < end) step(r0 + kTile, std::integral_constant<int, 1>{});
  }
  if (key >= a.S) return;
  const float by = a.scale / small, by_v = 1.f / mixture;
  const int64_t n_keys = (int64_t)a.batch * a.S * a.Hk;
  const int64_t to = ((int64_t)b * a.S + key) * a.Hk + hk;
  // A key that takes no part was a column of its own: whatever it holds is dropped here.
  auto put = [&](char* whole, int64_t skip, int64_t row, int d, int e, f32x4 x) {
    if (!alive) x = f32x4{0, 0, 0, 0};
    if (a.splits > 1) {
      if (e < d) *(f32x4*)(a.part + split * n_keys * (2 * a.D + a.Dv) + skip + row * d + e) = x;
    } else {
      store4<DT>(whole + row * d * ES, e, d, x[0], x[1], x[2], x[3]);
    }
  };
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        put(a.dk, 0, 2 * to + m, a.D, 32 * n + acc_at(i, half),
            f32x4{dk[m][n][i], dk[m][n][i + 1], dk[m][n][i + 2], dk[m][n][i + 3]} * by);
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      put(a.dv, n_keys * 2 * a.D, to, a.Dv, 32 * n + acc_at(i, half),
          f32x4{dv[n][i], dv[n][i + 1], dv[n][i + 2], dv[n][i + 3]} * by_v);
}

// ---------------------------------------------------------------------------
// dq: four waves of 32 rows over their keys.  In 16 bits, where a workgroup's rows see few of them,
// twice: a first time for the sums that delta comes from.  Of few keys each counts for much: dq's
// error was twice its rounding, and of a row's only key, whose score has no gradient, all there
// was.  Of many it is hidden behind theirs.  (64 x 200 tokens of 16 heads on 4: both passes 181 us
// with one, 240 with two.)  The whole sum is known where all the keys lie in one split.
constexpr int kFewKeys = 256;
// ---------------------------------------------------------------------------
template <int DT, int DP, int DVP>
struct RowSmem {
  static constexpr int kK = Tile<DT, DP, kThreads>::kBytes, kV = Tile<DT, DVP, kThreads>::kBytes;
  static constexpr int kStage = 2 * kK + kV;
  // A lane's largest scores and logarithms apart: few tiles want them, and a spilled register's
  // load waits for the tiles under way.
  static constexpr int kFarAt = 2 * kStage;
  static constexpr int kBytes = kFarAt + kThreads * 16;
};

// Two waves a SIMD where the operands of 64-wide maps leave room for them (128-wide ones spill:
// 2 x 2048 tokens of 16 heads, 128 and 128 wide, both passes 670 us with two, 431 with one).
template <int DT, int DP, int DVP>
__global__ __launch_bounds__(kThreads, DT != DA_F32 && DP == 64 ? 2 : 1) void diff_grad_rows(Args a) {
  using L = RowSmem<DT, DP, DVP>;
  constexpr int ES = Type<DT>::ES, V = Type<DT>::V;
  constexpr int KD = DP / Type<DT>::kStep, KV = DVP / Type<DT>::kStep, KC = Type<DT>::kChunks, ND = DP / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int at = (int)xcd_remap(blockIdx.x, gridDim.x);
  const int block = a.blocks - 1 - at % a.blocks;  // the rows with the most keys first
  at /= a.blocks;
  const int split = at % a.splits;
  at /= a.splits;
  const int hk = at % a.Hk, b = at / a.Hk;
  const int rows = a.T * a.G;
  const int r = (block * kWaves + wave) * kTile + (lane & 31);
  const int t = token_of(a, r), h = hk * a.G + (r - t * a.G);
  const int64_t base = ((int64_t)b * a.Hk + hk) * 2 * rows + r;
  int last = r < rows ? last_key(a, b, t) : -1;
  const float lse0 = last >= 0 ? a.lse[base] : __builtin_inff();
  if (lse0 == __builtin_inff()) last = -1;  // no key that it could see is live
  int most = last, least = last;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    most = max(most, __shfl_xor(most, off, kWave));
    least = min(least, __shfl_xor(least, off, kWave));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);
  int end = a.S;
  if (a.causal) {
    const int64_t t_last = token_of(a, min((block + 1) * kWaves * kTile, rows) - 1);
    end = (int)max((int64_t)0, min((int64_t)a.S, t_last + a.q_start + 1));
  }
  int key = split * a.each;
  // Whether the keys up to `end` are few, and all of them in this split: the same in all waves.
  bool few = false;
  if constexpr (DT != DA_F32) {
    if (a.mask) {
      int live = 0, here = 0;
      for (int k = 0; k < end && live <= kFewKeys; k += 4 * kWave) {
        int byte[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = k + i * kWave + lane;
          byte[i] = at < end ? a.mask[b * a.m_b + at * a.m_k] : 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = k + i * kWave + lane - key;
          live += __popcll(__ballot(byte[i] != 0));
          here += __popcll(__ballot(byte[i] != 0 && at >= 0 && at < a.each));
        }
      }
      few = live <= kFewKeys && here == live;
    } else {
      few = end <= kFewKeys && key == 0 && end <= a.each;
    }
  }
  end = min(end, key + a.each);
  const bool in = last >= 0;
  u32x4 q[2][KD], g[KV];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int kk = 0; kk < KD; ++kk)
      q[m][kk] = in ? load_run<DT>(a.q + (b * a.q_b + t * a.q_t + (2 * h + m) * a.q_h) * ES, (2 * kk + half) * V, a.D)
                    : u32x4{0, 0, 0, 0};
#pragma unroll
  for (int kk = 0; kk < KV; ++kk)
    g[kk] = in ? load_run<DT>(a.g + (b * a.g_b + t * a.g_t + h * a.g_h) * ES, (2 * kk + half) * V, a.Dv)
               : u32x4{0, 0, 0, 0};
  // The size of the second map's factor comes with its exponential, the sign at the end.
  const float lam = in ? lam_of(a, h) : 0.f;
  const float lse1 = in ? a.lse[base + rows] - log2f(fabsf(lam)) : __builtin_inff();
  const int64_t tops = tops_at(a) + base;
  const float top0 = in ? a.lse[tops] : 0.f, top1 = in ? a.lse[tops + rows] : 0.f;
  float de0 = in ? a.delta[base] : 0.f, de1 = in ? a.delta[base + rows] : 0.f;
  const float c = a.scale * kLog2e, small = small_scale<DT>(a, b, hk);
  // Large scores: the difference from the largest first.
  const bool far = DT == DA_F32 || __any(!near(top0, top1, c));
  const float whole0 = fmaf(top0, c, lse0), whole1 = fmaf(top1, c, lse1);
  *(f32x4*)(lds + L::kFarAt + threadIdx.x * 16) = f32x4{top0, top1, lse0, lse1};

  const Keys<DT, DP, kThreads> keys(a.k_t, a.D);
  const Keys<DT, DVP, kThreads> values(a.v_t, a.Dv);
  const char* kp = a.k + (b * a.k_b + 2 * hk * a.k_h) * ES;
  const char* vp = a.v + (b * a.v_b + hk * a.v_h) * ES;
  auto fetch = [&](int to, int stage, uint32_t live) {
    const uint32_t l = lds_address(lds) + stage * L::kStage;
    keys.fetch(kp + to * a.k_t * ES, l, live);
    keys.fetch(kp + (to * a.k_t + a.k_h) * ES, l + L::kK, live);
    values.fetch(vp + to * a.v_t * ES, l + 2 * L::kK, live);
  };
  float off0 = 0.f, off1 = 0.f;
  f32x16 dq[2][ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) dq[0][n] = zeros(), dq[1][n] = zeros();
  const int start = key;
  Live live(a, b, key, end, lane);
  if (live.word) fetch(live.key, 0, live.word);
  bool sums_only = few;
  const Reader<DT, DP> key_reader(lds, lane);
  const Reader<DT, DVP> value_reader(lds + 2 * L::kK, lane);
  const auto step = [&](auto of) __attribute__((always_inline)) {
    constexpr int stage = decltype(of)::value;
    key = live.key;
    const uint32_t word = live.word;
    live.next(a, b, end, lane);
    tiles_barrier();
    if (live.word) fetch(live.key, stage ^ 1, live.word);
    if (key > most) return;
    constexpr int skip = stage * L::kStage;
    const auto lk = key_reader.fresh(key);
    const auto lv = value_reader.fresh(key);
    f32x16 s0 = zeros(), s1 = zeros(), dp = zeros();
#pragma unroll
    for (int kk = 0; kk < KD; ++kk) {
      Mfma32<DT>::mma(s0, lk.rows(skip, kk), q[0][kk]);
      Mfma32<DT>::mma(s1, lk.rows(skip + L::kK, kk), q[1][kk]);
    }
#pragma unroll
    for (int kk = 0; kk < KV; ++kk) Mfma32<DT>::mma(dp, lv.rows(skip, kk), g[kk]);
    const bool some = word != ~0u || key + kTile - 1 > least;
    const uint32_t seen = some ? seen_of(word, key, last, half) : ~0u;
    if (far) {
      const f32x4 x = __builtin_bit_cast(f32x4, lds16(lds_address(lds) + L::kFarAt + threadIdx.x * 16));
#pragma unroll
      for (int i = 0; i < 16; ++i) s0[i] = fmaf(s0[i] - x[0], c, -x[2]), s1[i] = fmaf(s1[i] - x[1], c, -x[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) s0[i] = fmaf(s0[i], c, -whole0), s1[i] = fmaf(s1[i], c, -whole1);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float p0 = __builtin_amdgcn_exp2f(s0[i]);
      float p1 = __builtin_amdgcn_exp2f(s1[i]);
      if constexpr (DT == DA_F16) p0 *= small, p1 *= small;
      if (some) {
        p0 = seen & 1u << acc_at(i, 0) ? p0 : 0.f;
        p1 = seen & 1u << acc_at(i, 0) ? p1 : 0.f;
      }
      s0[i] = p0 * (dp[i] - de0);
      s1[i] = p1 * (de1 - dp[i]);
      if constexpr (DT != DA_F32) off0 += s0[i], off1 += s1[i];
    }
    if (DT != DA_F32 && sums_only) return;
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      // A map after the other: both at once would spill.
      const auto add = [&](const f32x16& x, int at, f32x16 (&to)[ND]) __attribute__((always_inline)) {
        const u32x4 y = from_acc<DT>(x, j);
        u32x4 rest;
        if constexpr (DT != DA_F32) rest = rest_of<DT>(x, j, y);
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const u32x4 k = lk.columns(at, n, j);
          Mfma32<DT>::mma(to[n], k, y);
          if constexpr (DT != DA_F32) Mfma32<DT>::mma(to[n], k, rest);
        }
      };
      add(s0, skip, dq[0]);
      add(s1, skip + L::kK, dq[1]);
    }
  };
  // A factor so small that its map's entries vanish tells nothing of delta.
  const float size = fabsf(lam), to_off0 = 1.f / small, to_off1 = size > 0x1p-60f ? -1.f / (size * small) : 0.f;
  for (;;) {
    while (live.word) {
      step(std::integral_constant<int, 0>{});
      if (live.word) step(std::integral_constant<int, 1>{});
    }
    if constexpr (DT == DA_F32) break;
    off0 = (off0 + other_half(off0)) * to_off0;
    off1 = (off1 + other_half(off1)) * to_off1;
    if (!sums_only) break;
    sums_only = false;
    de0 += off0, de1 += off1;
    off0 = off1 = 0.f;
    __syncthreads();  // the tiles have been read
    live = Live(a, b, start, end, lane);
    if (live.word) fetch(live.key, 0, live.word);
  }
  if (r >= rows) return;
  if (DT != DA_F32 && half == 0) {
    float* to = a.off + (int64_t)split * a.batch * a.Hk * 2 * rows + base;
    if (few && in) off0 += de0 - a.delta[base], off1 += de1 - a.delta[base + rows];
    to[0] = off0;
    to[rows] = off1;
  }
  const float by = a.scale / small, by_map[2] = {by, lam < 0.f ? -by : by};
  const int64_t to = ((int64_t)b * a.T + t) * (a.Hk * a.G) + h;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int e = 32 * n + acc_at(i, half);
        const f32x4 x = f32x4{dq[m][n][i], dq[m][n][i + 1], dq[m][n][i + 2], dq[m][n][i + 3]} * by_map[m];
        if (a.splits == 1)
          store4<DT>(a.dq + (2 * to + m) * a.D * ES, e, a.D, x[0], x[1], x[2], x[3]);
        else if (e < a.D)
          *(f32x4*)(a.part + (split * (int64_t)a.batch * rows * a.Hk + to) * 2 * a.D + m * a.D + e) = x;
      }
}

// Sums of splits, in order, four entries a thread: to `first` up to n_first, then to `second`.
template <int DT>
__global__ __launch_bounds__(256) void diff_grad_join(const float* part, int splits, int64_t n, char* first,
                                                      int64_t n_first, char* second) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  f32x4 v = *(const f32x4*)(part + at);
  for (int p = 1; p < splits; ++p) v += *(const f32x4*)(part + p * n + at);
  char* to = at < n_first ? first + at * Type<DT>::ES : second + (at - n_first) * Type<DT>::ES;
  store4<DT>(to, 0, 4, v[0], v[1], v[2], v[3]);
}

// Tokens of a chunk of delta: about four workgroups a CU, no fewer than 16 tokens.
void chunks_of(int64_t groups, int64_t T, int64_t cus, int* chunk, int* chunks) {
  const int64_t want = std::max<int64_t>(1, 4 * cus / std::max<int64_t>(groups, 1));
  const int64_t each = std::max<int64_t>(16, (T + want - 1) / want);
  *chunk = (int)each;
  *chunks = (int)std::max<int64_t>(1, (T + each - 1) / each);
}

// Blocks of one side's entries, and splits of the other's: so many that every CU has two
// workgroups, none under kLeastSplit entries (18 heads of 509 keys in fp32, both passes: 269 us
// from 256 on, which leaves it whole, 136 from 128, 152 from 64).
constexpr int kLeastSplit = 128;
void share(int64_t mine, int64_t others, int64_t groups, int64_t cus, int* blocks, int* splits, int* each) {
  const int64_t n = std::max<int64_t>(1, (mine + kWaves * kTile - 1) / (kWaves * kTile));
  int64_t want = std::max<int64_t>(1, 2 * cus / std::max<int64_t>(1, groups * n));
  want = std::max<int64_t>(1, std::min(want, others / kLeastSplit));
  const int64_t e = std::max<int64_t>(kTile, ((others + want - 1) / want + kTile - 1) / kTile * kTile);
  *blocks = (int)n, *each = (int)e;
  *splits = (int)std::max<int64_t>(1, (others + e - 1) / e);
}

// How the two passes are shared out, and the workspace: delta, the parts of dlam, the largest
// |g| and |v|, the records, whether a row takes part, and the sums of the splits (of one pass after the other).
struct Plan {
  Args keys, rows;  // blocks, splits, each
  int64_t records_at, parts_at, most_at, off_at, takes_part_at, sums_at;  // in floats
  size_t bytes;
};

int plan(int dtype, int64_t batch, int64_t heads, int64_t k_heads, int64_t T, int64_t S, int64_t D, int64_t Dv, Args* a, Plan* p) {
  int64_t cus;
  const int rc = device_cu_count(&cus);
  if (rc) return rc;
  const int64_t rows = T * (heads / k_heads);
  chunks_of(batch * heads, T, cus, &a->chunk, &a->chunks);
  share(S, rows, batch * k_heads, cus, &p->keys.blocks, &p->keys.splits, &p->keys.each);
  share(rows, S, batch * k_heads, cus, &p->rows.blocks, &p->rows.splits, &p->rows.each);
  p->records_at = (batch * heads * T * 2 + 3) / 4 * 4;
  p->parts_at = p->records_at + batch * heads * T * (dtype == DA_F32 ? Record<DA_F32>::kBytes : Record<DA_BF16>::kBytes) / 4;
  p->most_at = p->parts_at + batch * heads * a->chunks;
  p->off_at = p->most_at + (dtype == DA_F16 ? 2 * batch * k_heads : 0);
  p->takes_part_at = p->off_at + (dtype == DA_F32 ? 0 : p->rows.splits * batch * heads * T * 2);
  p->sums_at = (p->takes_part_at + (batch * heads * T + 3) / 4 + 3) / 4 * 4;
  const int64_t of_keys = p->keys.splits > 1 ? p->keys.splits * batch * S * k_heads * (2 * D + Dv) : 0;
  const int64_t of_rows = p->rows.splits > 1 ? p->rows.splits * batch * T * heads * 2 * D : 0;
  p->bytes = (size_t)(p->sums_at + std::max(of_keys, of_rows)) * sizeof(float);
  return DA_OK;
}

template <int DT>
int join(const float* part, int splits, int64_t n, void* first, int64_t n_first, void* second, hipStream_t st) {
  const int64_t blocks = (n / 4 + 255) / 256;
  if (blocks > kMaxBlocks) return set_error(DA_ERR_UNSUPPORTED, "da_diff_attention_grad: too many rows");
  diff_grad_join<DT><<<(unsigned)blocks, 256, 0, st>>>(part, splits, n, (char*)first, n_first, (char*)second);
  return DA_OK;
}

}  // namespace
}  // namespace diff
}  // namespace da

extern "C" {

int da_diff_attention_grad_workspace(int dtype, int64_t batch, int64_t q_len, int64_t k_len, int64_t heads,
                                     int64_t k_heads, int64_t d, int64_t dv, size_t* bytes) {
  using namespace da;
  using namespace da::diff;
  if (!bytes) return set_error(DA_ERR_INVALID, "da_diff_attention_grad_workspace: NULL pointer");
  *bytes = 0;
  int rc = check_sizes("da_diff_attention_grad_workspace", dtype, batch, q_len, k_len, heads, k_heads, d, dv, 0);
  if (rc || batch == 0) return rc;
  Args a;
  Plan p;
  rc = plan(dtype, batch, heads, k_heads, q_len, k_len, d, dv, &a, &p);
  if (rc == DA_OK) *bytes = p.bytes;
  return rc;
}

int da_diff_attention_grad(const da_diff_inputs* in, const void* g, int64_t g_bstride, int64_t g_tstride,
                           int64_t g_hstride, const void* out, const void* second, const float* lse, int dtype,
                           int64_t batch, int64_t q_len, int64_t k_len, int64_t heads, int64_t k_heads, int64_t d,
                           int64_t dv, float scale, int causal, int64_t q_start, void* dq, void* dk, void* dvalue,
                           float* dlam, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace da;
  using namespace da::diff;
  const char* what = "da_diff_attention_grad";
  int rc = check_sizes(what, dtype, batch, q_len, k_len, heads, k_heads, d, dv, q_start);
  if (rc) return rc;
  if (batch == 0) return DA_OK;
  if (!in || !in->lam || !dlam || (q_len && (!in->q || !g || !out || !second || !lse || !dq)) ||
      (k_len && (!in->k || !in->v || !dk || !dvalue)))
    return set_error(DA_ERR_INVALID, "%s: NULL pointer", what);
  Args a = {};
  rc = fill_args(a, what, dtype, in, batch, q_len, k_len, heads, k_heads, d, dv, scale, causal, q_start);
  if (rc == DA_OK)
    rc = check_side(what, "g", g, (int)elem_bytes(dtype), dv, q_len, a.G, g_bstride, g_tstride, g_hstride);
  if (rc) return rc;
  Plan p;
  rc = plan(dtype, batch, heads, k_heads, q_len, k_len, d, dv, &a, &p);
  if (rc) return rc;
  if (!workspace || workspace_bytes < p.bytes)
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", what, p.bytes);
  if ((uintptr_t)workspace % 16) return set_error(DA_ERR_INVALID, "%s: workspace must be 16-byte aligned", what);
  const int64_t rows = q_len * a.G, pairs = batch * k_heads;
  if (batch * heads > kMaxBlocks / a.chunks || pairs > kMaxBlocks / p.rows.blocks / p.rows.splits ||
      pairs > kMaxBlocks / p.keys.blocks / p.keys.splits)
    return set_error(DA_ERR_UNSUPPORTED, "%s: too many rows", what);
  a.g = (const char*)g, a.g_b = g_bstride, a.g_t = g_tstride, a.g_h = g_hstride;
  a.out = (char*)const_cast<void*>(out), a.second = (char*)const_cast<void*>(second);
  a.lse = const_cast<float*>(lse);
  a.delta = (float*)workspace;
  a.records = (char*)(a.delta + p.records_at);
  a.lam_part = a.delta + p.parts_at;
  a.most = a.delta + p.most_at;
  a.off = a.delta + p.off_at;
  a.row_splits = p.rows.splits;
  a.takes_part = (uint8_t*)(a.delta + p.takes_part_at);
  a.part = a.delta + p.sums_at;
  a.dq = (char*)dq, a.dk = (char*)dk, a.dv = (char*)dvalue;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == DA_F16 && (rc = zero_f32_2d(a.most, 1, 2 * pairs, 2 * pairs, st))) return rc;
  const unsigned delta_grid = (unsigned)(batch * heads * a.chunks);
  if (dtype == DA_BF16) diff_delta<DA_BF16><<<delta_grid, 256, 0, st>>>(a);
  else if (dtype == DA_F16) diff_delta<DA_F16><<<delta_grid, 256, 0, st>>>(a);
  else diff_delta<DA_F32><<<delta_grid, 256, 0, st>>>(a);
  if (dtype == DA_F16 && k_len) {  // about 1024 workgroups
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(1024 / pairs, (k_len + 15) / 16));
    diff_values_norm<<<(unsigned)(pairs * parts), 256, 0, st>>>(a, (int)parts);
  }
  rc = by_widths(dtype, widths(d, dv), [&](auto dt, auto dp, auto dvp) {
    constexpr int DT = decltype(dt)::value, DP = decltype(dp)::value, DVP = decltype(dvp)::value;
    if (rows) {
      constexpr int kBytes = RowSmem<DT, DP, DVP>::kBytes;
      const auto kernel = diff_grad_rows<DT, DP, DVP>;
      if (const int err = allow_lds((const void*)kernel, kBytes)) return err;
      a.blocks = p.rows.blocks, a.splits = p.rows.splits, a.each = p.rows.each;
      kernel<<<(unsigned)(pairs * a.blocks * a.splits), kThreads, kBytes, st>>>(a);
      const int64_t n = batch * q_len * heads * 2 * d;
      if (a.splits > 1)
        if (const int err = join<DT>(a.part, a.splits, n, dq, n, nullptr, st)) return err;
    }
    diff_records<DT><<<delta_grid, 256, 0, st>>>(a);
    diff_lam_join<<<(unsigned)((batch * heads + 255) / 256), 256, 0, st>>>(a.lam_part, dlam, batch * heads, a.chunks);
    if (k_len) {
      constexpr int kBytes = KeySmem<DT, DP, DVP>::kBytes;
      if (const int err = allow_lds((const void*)diff_grad_keys<DT, DP, DVP>, kBytes)) return err;
      a.blocks = p.keys.blocks, a.splits = p.keys.splits, a.each = p.keys.each;
      diff_grad_keys<DT, DP, DVP><<<(unsigned)(pairs * a.blocks * a.splits), kThreads, kBytes, st>>>(a);
      const int64_t n_first = pairs * k_len * 2 * d, n = n_first + pairs * k_len * dv;
      if (a.splits > 1)
        if (const int err = join<DT>(a.part, a.splits, n, dk, n_first, dvalue, st)) return err;
    }
    return check_launch("da_diff_attention_grad");
  });
  return rc;
}

}  // extern "C"
