// Attention by the difference of two softmax maps, backward.
//
// With p_m the maps (from the scores and the forward call's lse), g the gradient of out:
//
//   dp = g v^T,   delta_m = g . o_m
//   ds_1 = p_1 (dp - delta_1),   ds_2 = -lam p_2 (dp - delta_2)
//   dq_m = scale ds_m k_m,   dk_m = scale ds_m^T q_m,   dv = (p_1 - lam p_2)^T g
//   dlam[sample] = -sum of delta_2
//
// Three launches and no atomic sums, so that results do not change from run to run: delta
// and dlam's parts; dk and dv, a wave holding 32 keys and going over all rows of their
// heads; dq, a wave holding 32 rows and going over their keys.  The scores are formed
// twice, the price of sums that are nobody else's.  Where keys are columns, the scores'
// registers are rows and stand as the operand that is contracted over rows; where rows are
// columns, they are keys: neither pass moves a score between lanes.
//
// 16-bit floats of five exponent bits lose small values of ds: there ds is scaled by the
// power of two that brings the largest |g| near one, and its products back.
#include <algorithm>

#include "diffattn.h"

namespace da {
namespace diff {
namespace {

// ---------------------------------------------------------------------------
// delta, parts of dlam, largest |g|.  Workgroup (b, h, chunk of tokens), 16 lanes a token.
// ---------------------------------------------------------------------------
constexpr int kLanes = 16;

template <int DT>
__global__ __launch_bounds__(256) void diff_delta(Args a) {
  constexpr int ES = Type<DT>::ES, V = Type<DT>::V, kRows = 256 / kLanes;
  __shared__ float parts[kRows];
  const int heads = a.Hk * a.G, l = threadIdx.x % kLanes, sub = threadIdx.x / kLanes;
  const int chunk = blockIdx.x % a.chunks;
  const int h = blockIdx.x / a.chunks % heads, b = blockIdx.x / a.chunks / heads;
  const int hk = h / a.G, rows = a.T * a.G;
  const float lam = lam_of(a, h);
  const int t1 = min((chunk + 1) * a.chunk, a.T);
  float all = 0.f, most = 0.f;
  for (int t = chunk * a.chunk + sub; t < t1; t += kRows) {
    const bool live = !a.q_mask || a.q_mask[b * a.qm_b + t * a.qm_t];
    float d0 = 0.f, d1 = 0.f;
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
          if constexpr (DT == DA_F16) most = fmaxf(most, fabsf(x[e]));
        }
      }
    }
    d0 = lanes_sum<kLanes>(d0);
    d1 = lanes_sum<kLanes>(d1);
    if (l == 0) {
      float* to = a.delta + ((int64_t)b * a.Hk + hk) * 2 * rows + t * a.G + (h - hk * a.G);
      to[0] = d0 + lam * d1;  // o_1 = out + lam o_2
      to[rows] = d1;
    }
    all += d1;
  }
  if constexpr (DT == DA_F16) {  // a maximum: the order does not matter
    most = lanes_max<64>(most);
    if (threadIdx.x % 64 == 0 && most > 0.f) atomicMax((unsigned*)a.most, __float_as_uint(most));
  }
  if (l == 0) parts[sub] = all;
  __syncthreads();
  if (threadIdx.x) return;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) v += parts[i];
  a.lam_part[blockIdx.x] = -v;
}

__global__ __launch_bounds__(256) void diff_lam_join(const float* parts, float* out, int64_t n, int chunks) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float v = 0.f;
  for (int c = 0; c < chunks; ++c) v += parts[i * chunks + c];
  out[i] = v;
}

// The power of two that brings the largest |g| to [1, 2): 1 where there is no such.
template <int DT>
__device__ __forceinline__ float small_scale(const Args& a) {
  if constexpr (DT != DA_F16) return 1.f;
  const uint32_t e = __float_as_uint(*a.most) >> 23;  // of a float above zero
  return e == 0 || e == 255 ? 1.f : __uint_as_float((254 - e) << 23);
}

// ---------------------------------------------------------------------------
// dk and dv: four waves of 32 keys over all rows r = t G + g of their key head.
// ---------------------------------------------------------------------------
constexpr int kKeyWaves = 4;

template <int DT, int DP, int DVP>
struct KeySmem {
  static constexpr int NT = kKeyWaves * kWave;
  static constexpr int kQ = Tile<DT, DP, NT>::kBytes, kG = Tile<DT, DVP, NT>::kBytes;
  static constexpr int kRow = 6 * kTile * 4;  // of each row: lse, delta of both maps, lam, the last key
  static constexpr int kStage = 2 * kQ + kG + kRow;
  static constexpr int kBytes = 2 * kStage;
};

template <int DT, int DP, int DVP>
__global__ __launch_bounds__(kKeyWaves * kWave) void diff_grad_keys(Args a) {
  using L = KeySmem<DT, DP, DVP>;
  constexpr int NT = L::NT, ES = Type<DT>::ES, V = Type<DT>::V;
  constexpr int KD = DP / Type<DT>::kStep, KV = DVP / Type<DT>::kStep, KC = Type<DT>::kChunks;
  constexpr int ND = DP / 32, NV = DVP / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int blocks = (a.S + kKeyWaves * kTile - 1) / (kKeyWaves * kTile);
  const int block = blockIdx.x % blocks, hk = blockIdx.x / blocks % a.Hk, b = blockIdx.x / blocks / a.Hk;
  const int key0 = (block * kKeyWaves + wave) * kTile, key = key0 + (lane & 31);
  const bool alive = key < a.S && (!a.mask || a.mask[b * a.m_b + key * a.m_k]);
  const int rows = a.T * a.G;
  u32x4 k[2][KD], v[KV];
#pragma unroll
  for (int kk = 0; kk < KD; ++kk)
#pragma unroll
    for (int m = 0; m < 2; ++m)
      k[m][kk] = alive ? load_run<DT>(a.k + (b * a.k_b + key * a.k_t + (2 * hk + m) * a.k_h) * ES,
                                      (2 * kk + half) * V, a.D) : u32x4{0, 0, 0, 0};
#pragma unroll
  for (int kk = 0; kk < KV; ++kk)
    v[kk] = alive ? load_run<DT>(a.v + (b * a.v_b + key * a.v_t + hk * a.v_h) * ES, (2 * kk + half) * V, a.Dv)
                  : u32x4{0, 0, 0, 0};
  const bool work = __any(alive);
  const bool whole = __all(alive);
  f32x16 dk[2][ND], dv[NV];
#pragma unroll
  for (int n = 0; n < ND; ++n) dk[0][n] = zeros(), dk[1][n] = zeros();
#pragma unroll
  for (int n = 0; n < NV; ++n) dv[n] = zeros();
  const float c = a.scale * kLog2e, small = small_scale<DT>(a);

  Tile<DT, DP, NT> q0, q1;
  Tile<DT, DVP, NT> g;
  float row_value = 0.f;
  // One value of a row a thread: 32 rows of lse and delta of both maps, lam, the last key.
  const int what = threadIdx.x / kTile, which = threadIdx.x % kTile;
  auto fetch = [&](int r0) {
    auto place = [&](int i, int64_t st, int64_t sh, int maps) -> int64_t {
      const int r = r0 + i, t = r / a.G;
      if (r >= rows || (a.q_mask && !a.q_mask[b * a.qm_b + t * a.qm_t])) return -1;
      return b * (maps == 2 ? a.q_b : a.g_b) + t * st + (int64_t)(hk * a.G + r - t * a.G) * maps * sh;
    };
    q0.fetch([&](int i) { const int64_t at = place(i, a.q_t, a.q_h, 2); return at < 0 ? nullptr : a.q + at * ES; }, a.D);
    q1.fetch([&](int i) { const int64_t at = place(i, a.q_t, a.q_h, 2); return at < 0 ? nullptr : a.q + (at + a.q_h) * ES; },
             a.D);
    g.fetch([&](int i) { const int64_t at = place(i, a.g_t, a.g_h, 1); return at < 0 ? nullptr : a.g + at * ES; }, a.Dv);
    const int r = r0 + which;
    const int64_t base = ((int64_t)b * a.Hk + hk) * 2 * rows;
    if (what < 2) row_value = r < rows ? a.lse[base + what * rows + r] : __builtin_inff();
    else if (what < 4) row_value = r < rows ? a.delta[base + (what - 2) * rows + r] : 0.f;
    else if (what == 4) row_value = r < rows ? lam_of(a, hk * a.G + r % a.G) : 0.f;
    else if (what == 5) row_value = __int_as_float(r < rows ? last_key(a, b, r / a.G) : -1);
  };
  // The first row that sees the workgroup's first key.
  int first = 0;
  if (a.causal) {
    const int64_t t = (int64_t)block * kKeyWaves * kTile - a.q_start;
    first = t <= 0 ? 0 : t >= a.T ? rows : (int)t * a.G / kTile * kTile;
  }
  if (first < rows) fetch(first);
  int stage = 0;
  for (int r0 = first; r0 < rows; r0 += kTile, stage ^= 1) {
    char* l = lds + stage * L::kStage;
    q0.put(l, ~0u);
    q1.put(l + L::kQ, ~0u);
    g.put(l + 2 * L::kQ, ~0u);
    float* of_rows = (float*)(l + 2 * L::kQ + L::kG);
    if (what < 6) of_rows[what * kTile + which] = row_value;
    if (r0 + kTile < rows) fetch(r0 + kTile);
    __syncthreads();
    if (!work) continue;
    const int last_row = min(r0 + kTile, rows) - 1;
    if (a.causal && last_row / a.G + a.q_start < key0) continue;
    const char* lg = l + 2 * L::kQ;
    f32x16 s0 = zeros(), s1 = zeros(), dp = zeros();
#pragma unroll
    for (int kk = 0; kk < KD; ++kk) {
      Mfma32<DT>::mma(s0, by_rows<DT, DP>(l, kk, lane), k[0][kk]);
      Mfma32<DT>::mma(s1, by_rows<DT, DP>(l + L::kQ, kk, lane), k[1][kk]);
    }
#pragma unroll
    for (int kk = 0; kk < KV; ++kk) Mfma32<DT>::mma(dp, by_rows<DT, DVP>(lg, kk, lane), v[kk]);
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int x = acc_at(i, half);
      const f32x4 lse0 = *(const f32x4*)(of_rows + x), lse1 = *(const f32x4*)(of_rows + kTile + x);
      const f32x4 de0 = *(const f32x4*)(of_rows + 2 * kTile + x), de1 = *(const f32x4*)(of_rows + 3 * kTile + x);
      const f32x4 lam = *(const f32x4*)(of_rows + 4 * kTile + x), last = *(const f32x4*)(of_rows + 5 * kTile + x);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float p0 = __builtin_amdgcn_exp2f(fmaf(s0[i + e], c, -lse0[e]));
        float p1 = __builtin_amdgcn_exp2f(fmaf(s1[i + e], c, -lse1[e]));
        const bool seen = alive && key <= __float_as_int(last[e]);
        p0 = seen ? p0 : 0.f;
        p1 = seen ? p1 * lam[e] : 0.f;
        const float x0 = p0 * small, x1 = p1 * small;
        s0[i + e] = x0 * (dp[i + e] - de0[e]);
        s1[i + e] = x1 * (de1[e] - dp[i + e]);
        dp[i + e] = p0 - p1;
      }
    }
    (void)whole;
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      const u32x4 x = from_acc<DT>(dp, j), y0 = from_acc<DT>(s0, j), y1 = from_acc<DT>(s1, j);
#pragma unroll
      for (int n = 0; n < NV; ++n) Mfma32<DT>::mma(dv[n], by_columns<DT, DVP>(lg, n, j, lane), x);
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        Mfma32<DT>::mma(dk[0][n], by_columns<DT, DP>(l, n, j, lane), y0);
        Mfma32<DT>::mma(dk[1][n], by_columns<DT, DP>(l + L::kQ, n, j, lane), y1);
      }
    }
  }
  if (key >= a.S) return;
  const float by = a.scale / small;
  const int64_t at = ((int64_t)b * a.S + key) * a.Hk + hk;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        store4<DT>(a.dk + (2 * at + m) * a.D * ES, 32 * n + acc_at(i, half), a.D, dk[m][n][i] * by, dk[m][n][i + 1] * by,
                   dk[m][n][i + 2] * by, dk[m][n][i + 3] * by);
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      store4<DT>(a.dv + at * a.Dv * ES, 32 * n + acc_at(i, half), a.Dv, dv[n][i], dv[n][i + 1], dv[n][i + 2], dv[n][i + 3]);
}

// ---------------------------------------------------------------------------
// dq: four waves of 32 rows over their keys.
// ---------------------------------------------------------------------------
constexpr int kRowWaves = 4;

template <int DT, int DP, int DVP>
struct RowSmem {
  static constexpr int NT = kRowWaves * kWave;
  static constexpr int kK = Tile<DT, DP, NT>::kBytes, kV = Tile<DT, DVP, NT>::kBytes;
  static constexpr int kStage = 2 * kK + kV;
  static constexpr int kBytes = 2 * kStage;
};

template <int DT, int DP, int DVP>
__global__ __launch_bounds__(kRowWaves * kWave) void diff_grad_rows(Args a) {
  using L = RowSmem<DT, DP, DVP>;
  constexpr int NT = L::NT, ES = Type<DT>::ES, V = Type<DT>::V;
  constexpr int KD = DP / Type<DT>::kStep, KV = DVP / Type<DT>::kStep, KC = Type<DT>::kChunks, ND = DP / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int block = a.row_blocks - 1 - blockIdx.x % a.row_blocks;  // the rows with the most keys first
  const int hk = blockIdx.x / a.row_blocks % a.Hk, b = blockIdx.x / a.row_blocks / a.Hk;
  const int rows = a.T * a.G;
  const int r = (block * kRowWaves + wave) * kTile + (lane & 31);
  const int t = r / a.G, h = hk * a.G + (r - t * a.G);
  const int last = r < rows ? last_key(a, b, t) : -1;
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
    const int64_t t_last = min((block + 1) * kRowWaves * kTile, rows) - 1;
    end = (int)max((int64_t)0, min((int64_t)a.S, t_last / a.G + a.q_start + 1));
  }
  u32x4 q[2][KD], g[KV];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int kk = 0; kk < KD; ++kk)
      q[m][kk] = last >= 0 ? load_run<DT>(a.q + (b * a.q_b + t * a.q_t + (2 * h + m) * a.q_h) * ES, (2 * kk + half) * V, a.D)
                           : u32x4{0, 0, 0, 0};
#pragma unroll
  for (int kk = 0; kk < KV; ++kk)
    g[kk] = last >= 0 ? load_run<DT>(a.g + (b * a.g_b + t * a.g_t + h * a.g_h) * ES, (2 * kk + half) * V, a.Dv)
                      : u32x4{0, 0, 0, 0};
  const int64_t base = ((int64_t)b * a.Hk + hk) * 2 * rows + r;
  const bool in = last >= 0;
  const float lse0 = in ? a.lse[base] : __builtin_inff(), lse1 = in ? a.lse[base + rows] : __builtin_inff();
  const float de0 = in ? a.delta[base] : 0.f, de1 = in ? a.delta[base + rows] : 0.f;
  const float c = a.scale * kLog2e, small = small_scale<DT>(a);
  const float lam = in ? lam_of(a, h) * small : 0.f;

  Tile<DT, DP, NT> k0, k1;
  Tile<DT, DVP, NT> v;
  const char* kp = a.k + (b * a.k_b + 2 * hk * a.k_h) * ES;
  const char* vp = a.v + (b * a.v_b + hk * a.v_h) * ES;
  auto fetch = [&](int key) {
    k0.fetch([&](int i) { return key + i < end ? kp + (key + i) * a.k_t * ES : nullptr; }, a.D);
    k1.fetch([&](int i) { return key + i < end ? kp + ((key + i) * a.k_t + a.k_h) * ES : nullptr; }, a.D);
    v.fetch([&](int i) { return key + i < end ? vp + (key + i) * a.v_t * ES : nullptr; }, a.Dv);
  };
  f32x16 dq[2][ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) dq[0][n] = zeros(), dq[1][n] = zeros();
  uint32_t word = end > 0 ? key_word(key_byte(a, b, 0, end, lane)) : 0;
  int byte = key_byte(a, b, kTile, end, lane);
  if (word) fetch(0);
  int stage = 0;
  for (int key = 0; key < end; key += kTile) {
    char* l = lds + stage * L::kStage;
    const uint32_t live = word;
    if (live) {
      k0.put(l, live);
      k1.put(l + L::kK, live);
      v.put(l + 2 * L::kK, live);
    }
    word = key_word(byte);
    if (word) fetch(key + kTile);
    byte = key_byte(a, b, key + 2 * kTile, end, lane);
    if (!live) continue;
    __syncthreads();
    stage ^= 1;
    if (key > most) continue;
    f32x16 s0 = zeros(), s1 = zeros(), dp = zeros();
#pragma unroll
    for (int kk = 0; kk < KD; ++kk) {
      Mfma32<DT>::mma(s0, by_rows<DT, DP>(l, kk, lane), q[0][kk]);
      Mfma32<DT>::mma(s1, by_rows<DT, DP>(l + L::kK, kk, lane), q[1][kk]);
    }
#pragma unroll
    for (int kk = 0; kk < KV; ++kk) Mfma32<DT>::mma(dp, by_rows<DT, DVP>(l + 2 * L::kK, kk, lane), g[kk]);
    const bool some = live != ~0u || key + kTile - 1 > least;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float p0 = __builtin_amdgcn_exp2f(fmaf(s0[i], c, -lse0)) * small;
      float p1 = __builtin_amdgcn_exp2f(fmaf(s1[i], c, -lse1)) * lam;
      if (some) {
        const int x = acc_at(i, half);
        const bool seen = key + x <= last && (live >> x & 1);
        p0 = seen ? p0 : 0.f;
        p1 = seen ? p1 : 0.f;
      }
      s0[i] = p0 * (dp[i] - de0);
      s1[i] = p1 * (de1 - dp[i]);
    }
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      const u32x4 y0 = from_acc<DT>(s0, j), y1 = from_acc<DT>(s1, j);
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        Mfma32<DT>::mma(dq[0][n], by_columns<DT, DP>(l, n, j, lane), y0);
        Mfma32<DT>::mma(dq[1][n], by_columns<DT, DP>(l + L::kK, n, j, lane), y1);
      }
    }
  }
  if (r >= rows) return;
  const float by = a.scale / small;
  const int64_t at = ((int64_t)b * a.T + t) * (a.Hk * a.G) + h;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        store4<DT>(a.dq + (2 * at + m) * a.D * ES, 32 * n + acc_at(i, half), a.D, dq[m][n][i] * by, dq[m][n][i + 1] * by,
                   dq[m][n][i + 2] * by, dq[m][n][i + 3] * by);
}

// Tokens of a chunk of delta: about four workgroups a CU, no fewer than 16 tokens.
void chunks_of(int64_t groups, int64_t T, int64_t cus, int* chunk, int* chunks) {
  const int64_t want = std::max<int64_t>(1, 4 * cus / std::max<int64_t>(groups, 1));
  const int64_t each = std::max<int64_t>(16, (T + want - 1) / want);
  *chunk = (int)each;
  *chunks = (int)std::max<int64_t>(1, (T + each - 1) / each);
}

// The workspace: delta, the parts of dlam, the largest |g|.
size_t workspace_of(int64_t batch, int64_t heads, int64_t T, int chunks, int64_t* parts_at, int64_t* most_at) {
  *parts_at = batch * heads * T * 2;
  *most_at = *parts_at + batch * heads * chunks;
  return (size_t)(*most_at + 1) * sizeof(float);
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
  int64_t cus, parts, most;
  rc = device_cu_count(&cus);
  if (rc) return rc;
  int chunk, chunks;
  chunks_of(batch * heads, q_len, cus, &chunk, &chunks);
  *bytes = workspace_of(batch, heads, q_len, chunks, &parts, &most);
  return DA_OK;
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
  rc = fill_args(a, what, in, batch, q_len, k_len, heads, k_heads, d, dv, scale, causal, q_start);
  if (rc) return rc;
  int64_t cus, parts_at, most_at;
  rc = device_cu_count(&cus);
  if (rc) return rc;
  chunks_of(batch * heads, q_len, cus, &a.chunk, &a.chunks);
  const size_t need = workspace_of(batch, heads, q_len, a.chunks, &parts_at, &most_at);
  if (!workspace || workspace_bytes < need)
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", what, need);
  if ((uintptr_t)workspace % 16) return set_error(DA_ERR_INVALID, "%s: workspace must be 16-byte aligned", what);
  const int64_t rows = q_len * a.G;
  const int64_t row_blocks = (rows + kRowWaves * kTile - 1) / (kRowWaves * kTile);
  const int64_t key_blocks = (k_len + kKeyWaves * kTile - 1) / (kKeyWaves * kTile);
  if (batch * heads > kMaxBlocks / a.chunks || batch * k_heads > kMaxBlocks / std::max<int64_t>(1, row_blocks) ||
      batch * k_heads > kMaxBlocks / std::max<int64_t>(1, key_blocks))
    return set_error(DA_ERR_UNSUPPORTED, "%s: too many rows", what);
  a.g = (const char*)g, a.g_b = g_bstride, a.g_t = g_tstride, a.g_h = g_hstride;
  a.out = (char*)const_cast<void*>(out), a.second = (char*)const_cast<void*>(second);
  a.lse = const_cast<float*>(lse);
  a.delta = (float*)workspace;
  a.lam_part = a.delta + parts_at;
  a.most = a.delta + most_at;
  a.dq = (char*)dq, a.dk = (char*)dk, a.dv = (char*)dvalue;
  a.row_blocks = (int)row_blocks;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == DA_F16 && (rc = zero_f32_2d(a.most, 1, 1, 1, st))) return rc;
  const unsigned delta_grid = (unsigned)(batch * heads * a.chunks);
  if (dtype == DA_BF16) diff_delta<DA_BF16><<<delta_grid, 256, 0, st>>>(a);
  else if (dtype == DA_F16) diff_delta<DA_F16><<<delta_grid, 256, 0, st>>>(a);
  else diff_delta<DA_F32><<<delta_grid, 256, 0, st>>>(a);
  diff_lam_join<<<(unsigned)((batch * heads + 255) / 256), 256, 0, st>>>(a.lam_part, dlam, batch * heads, a.chunks);
  rc = by_widths(dtype, widths(d, dv), [&](auto dt, auto dp, auto dvp) {
    constexpr int DT = decltype(dt)::value, DP = decltype(dp)::value, DVP = decltype(dvp)::value;
    if (k_len) {
      constexpr int kBytes = KeySmem<DT, DP, DVP>::kBytes;
      if (const int err = allow_lds((const void*)diff_grad_keys<DT, DP, DVP>, kBytes)) return err;
      diff_grad_keys<DT, DP, DVP>
          <<<(unsigned)(batch * k_heads * key_blocks), kKeyWaves * kWave, kBytes, st>>>(a);
    }
    if (rows) {
      constexpr int kBytes = RowSmem<DT, DP, DVP>::kBytes;
      if (const int err = allow_lds((const void*)diff_grad_rows<DT, DP, DVP>, kBytes)) return err;
      diff_grad_rows<DT, DP, DVP>
          <<<(unsigned)(batch * k_heads * row_blocks), kRowWaves * kWave, kBytes, st>>>(a);
    }
    return check_launch("da_diff_attention_grad");
  });
  return rc;
}

}  // extern "C"
