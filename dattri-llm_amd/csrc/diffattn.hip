// Attention by the difference of two softmax maps, forward.
//
// Head h has two query maps and its key head two key maps:
//
//   out = o_1 - lam_h o_2,   o_m = softmax(scale q_m k_m^T) v     (zero for a row without keys)
//
// One pass over the keys: a wave holds 32 rows, with each map's running maximum and sum.
// It forms the transposed scores, k q^T, so that a row is a lane's (two lanes', 16 keys
// each) and its maximum and sum stay within them; the accumulator's registers then are,
// rounded, the second operand of o^T = v^T p^T as they stand, where v is read transposed
// out of LDS and once for both maps.  The accumulators are rescaled only when a maximum
// grows by more than 2^8: what is summed meanwhile is at most that much larger.
#include <algorithm>
#include <type_traits>

#include "diffattn.h"

namespace da {
namespace diff {
namespace {

constexpr float kSlack = 8.f;  // log2 of how far exponentials may pass 1 before a rescaling

template <int DT, int DP, int DVP, int NW>
struct Smem {
  static constexpr int kK = Tile<DT, DP, NW * kWave>::kBytes, kV = Tile<DT, DVP, NW * kWave>::kBytes;
  static constexpr int kStage = 2 * kK + kV;
  static constexpr int kBytes = 2 * kStage;
};

template <int DT, int DP, int DVP, int NW>
__global__ __launch_bounds__(NW * kWave) void diff_forward(Args a) {
  using L = Smem<DT, DP, DVP, NW>;
  constexpr int NT = NW * kWave, ES = Type<DT>::ES, V = Type<DT>::V;
  constexpr int KD = DP / Type<DT>::kStep, NB = DVP / 32, KC = Type<DT>::kChunks;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  // Workgroups of one key head are neighbours; the rows with the most keys go first.
  int at = blockIdx.x;
  const int block = a.row_blocks - 1 - at % a.row_blocks;
  at /= a.row_blocks;
  const int split = at % a.splits;
  at /= a.splits;
  const int hk = at % a.Hk, b = at / a.Hk;
  const int rows = a.T * a.G;
  const int r = (block * NW + wave) * kTile + (lane & 31);
  const int t = r / a.G, h = hk * a.G + (r - t * a.G);
  const int last = r < rows ? last_key(a, b, t) : -1;
  // The wave's and the workgroup's ranges of keys: rows come in order, so the last one sees most.
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
    const int64_t t_last = min((block + 1) * NW * kTile, rows) - 1;
    end = (int)max((int64_t)0, min((int64_t)a.S, t_last / a.G + a.q_start + 1));
  }
  const int first = split * a.split_keys;
  end = min(end, first + a.split_keys);

  u32x4 q[2][KD];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int kk = 0; kk < KD; ++kk) {
      q[m][kk] = u32x4{0, 0, 0, 0};
      if (last >= 0)
        q[m][kk] = load_run<DT>(a.q + (b * a.q_b + t * a.q_t + (2 * h + m) * a.q_h) * ES, (2 * kk + half) * V, a.D);
    }

  Tile<DT, DP, NT> k0, k1;
  Tile<DT, DVP, NT> v;
  const char* kp = a.k + (b * a.k_b + 2 * hk * a.k_h) * ES;
  const char* vp = a.v + (b * a.v_b + hk * a.v_h) * ES;
  auto fetch = [&](int key) {
    k0.fetch([&](int i) { return key + i < end ? kp + (key + i) * a.k_t * ES : nullptr; }, a.D);
    k1.fetch([&](int i) { return key + i < end ? kp + ((key + i) * a.k_t + a.k_h) * ES : nullptr; }, a.D);
    v.fetch([&](int i) { return key + i < end ? vp + (key + i) * a.v_t * ES : nullptr; }, a.Dv);
  };

  const float c = a.scale * kLog2e;
  f32x16 o[2][NB];
  float top[2] = {kLowest, kLowest}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n) o[m][n] = zeros();

  // Two tiles are under way: the words of live keys one ahead of their tiles, so that a
  // tile without any is not read.
  uint32_t word = first < end ? key_word(key_byte(a, b, first, end, lane)) : 0;
  int byte = key_byte(a, b, first + kTile, end, lane);
  if (word) fetch(first);
  int stage = 0;
  for (int key = first; key < end; key += kTile) {
    char* lk = lds + stage * L::kStage;
    const uint32_t live = word;
    if (live) {
      k0.put(lk, live);
      k1.put(lk + L::kK, live);
      v.put(lk + 2 * L::kK, live);
    }
    word = key_word(byte);
    if (word) fetch(key + kTile);
    byte = key_byte(a, b, key + 2 * kTile, end, lane);
    if (!live) continue;
    __syncthreads();
    stage ^= 1;
    if (key > most) continue;
    const char* lv = lk + 2 * L::kK;
    f32x16 s[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      s[m] = zeros();
#pragma unroll
      for (int kk = 0; kk < KD; ++kk) Mfma32<DT>::mma(s[m], by_rows<DT, DP>(lk + m * L::kK, kk, lane), q[m][kk]);
    }
    if (live != ~0u || key + kTile - 1 > least) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int x = acc_at(i, half);
        const bool seen = key + x <= last && (live >> x & 1);
        s[0][i] = seen ? s[0][i] : -__builtin_inff();
        s[1][i] = seen ? s[1][i] : -__builtin_inff();
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float x = s[m][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) x = fmaxf(x, s[m][i]);
      x = fmaxf(x, __shfl_xor(x, 32, kWave)) * c;
      if (__any(x > top[m] + kSlack)) {  // kLowest + 8 is kLowest
        const float now = fmaxf(top[m], x), by = __builtin_amdgcn_exp2f(top[m] - now);
        top[m] = now;
        sum[m] *= by;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[m][n][i] *= by;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[m][i] = __builtin_amdgcn_exp2f(fmaf(s[m][i], c, -top[m]));
        sum[m] += s[m][i];
      }
    }
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      const u32x4 p0 = from_acc<DT>(s[0], j), p1 = from_acc<DT>(s[1], j);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const u32x4 x = by_columns<DT, DVP>(lv, n, j, lane);
        Mfma32<DT>::mma(o[0][n], x, p0);
        Mfma32<DT>::mma(o[1][n], x, p1);
      }
    }
  }

  if (a.splits > 1) {  // this part's sums: joined by a second launch
    if (r >= rows) return;
    sum[0] += __shfl_xor(sum[0], 32, kWave);
    sum[1] += __shfl_xor(sum[1], 32, kWave);
    float* to = a.part + ((((int64_t)split * a.batch + b) * a.Hk + hk) * rows + r) * 2 * (DVP + 2);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *(f32x4*)(to + m * DVP + 32 * n + acc_at(i, half)) =
              f32x4{o[m][n][i], o[m][n][i + 1], o[m][n][i + 2], o[m][n][i + 3]};
      if (half == 0) to[2 * DVP + 2 * m] = top[m], to[2 * DVP + 2 * m + 1] = sum[m];
    }
    return;
  }
  sum[0] += __shfl_xor(sum[0], 32, kWave);
  sum[1] += __shfl_xor(sum[1], 32, kWave);
  if (r >= rows) return;
  const float by0 = sum[0] > 0.f ? 1.f / sum[0] : 0.f, by1 = sum[1] > 0.f ? 1.f / sum[1] : 0.f;
  const float by2 = by1 != 0.f ? lam_of(a, h) * by1 : 0.f;
  const int64_t to = ((int64_t)b * a.T + t) * (a.Hk * a.G) + h;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int e = 32 * n + acc_at(i, half);
      float f[4], g[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        f[x] = o[0][n][i + x] * by0 - o[1][n][i + x] * by2;
        g[x] = o[1][n][i + x] * by1;
      }
      store4<DT>(a.out + to * a.Dv * ES, e, a.Dv, f[0], f[1], f[2], f[3]);
      if (a.second) store4<DT>(a.second + to * a.Dv * ES, e, a.Dv, g[0], g[1], g[2], g[3]);
    }
  if (a.lse && half == 0) {
    float* lse = a.lse + ((int64_t)b * a.Hk + hk) * 2 * rows + r;
    lse[0] = sum[0] > 0.f ? top[0] + log2f(sum[0]) : __builtin_inff();
    lse[rows] = sum[1] > 0.f ? top[1] + log2f(sum[1]) : __builtin_inff();
  }
}

// The parts of a row, in order.  A thread has four entries.
template <int DT, int DVP>
__global__ __launch_bounds__(256) void diff_join(Args a) {
  constexpr int kLanes = DVP / 4, kRows = 256 / kLanes, ES = Type<DT>::ES;
  const int rows = a.T * a.G, l = threadIdx.x % kLanes;
  const int64_t all = (int64_t)a.batch * a.Hk * rows;
  const int64_t at = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes;  // (b, hk, r)
  if (at >= all) return;
  f32x4 o[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
  float top[2] = {kLowest, kLowest}, sum[2] = {0.f, 0.f};
  for (int p = 0; p < a.splits; ++p) {
    const float* from = a.part + (p * all + at) * 2 * (DVP + 2);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float top2 = from[2 * DVP + 2 * m], sum2 = from[2 * DVP + 2 * m + 1];
      const f32x4 x = *(const f32x4*)(from + m * DVP + 4 * l);
      const float now = fmaxf(top[m], top2);
      const float f1 = __builtin_amdgcn_exp2f(top[m] - now), f2 = __builtin_amdgcn_exp2f(top2 - now);
      top[m] = now;
      sum[m] = sum[m] * f1 + sum2 * f2;
      o[m] = o[m] * f1 + x * f2;
    }
  }
  const int r = (int)(at % rows), hk = (int)(at / rows % a.Hk), b = (int)(at / rows / a.Hk);
  const int t = r / a.G, h = hk * a.G + (r - t * a.G);
  const float by0 = sum[0] > 0.f ? 1.f / sum[0] : 0.f, by1 = sum[1] > 0.f ? 1.f / sum[1] : 0.f;
  const float by2 = by1 != 0.f ? lam_of(a, h) * by1 : 0.f;
  const int64_t to = ((int64_t)b * a.T + t) * (a.Hk * a.G) + h;
  const f32x4 f = o[0] * by0 - o[1] * by2, g = o[1] * by1;
  store4<DT>(a.out + to * a.Dv * ES, 4 * l, a.Dv, f[0], f[1], f[2], f[3]);
  if (a.second) store4<DT>(a.second + to * a.Dv * ES, 4 * l, a.Dv, g[0], g[1], g[2], g[3]);
  if (a.lse && l == 0) {
    float* lse = a.lse + ((int64_t)b * a.Hk + hk) * 2 * rows + r;
    lse[0] = sum[0] > 0.f ? top[0] + log2f(sum[0]) : __builtin_inff();
    lse[rows] = sum[1] > 0.f ? top[1] + log2f(sum[1]) : __builtin_inff();
  }
}

}  // namespace

int widths(int64_t D, int64_t Dv) { return D <= 64 && Dv <= 128 ? (Dv <= 64 ? 0 : 1) : Dv <= 128 ? 2 : 3; }

int check_sizes(const char* what, int dtype, int64_t batch, int64_t T, int64_t S, int64_t heads, int64_t k_heads,
                int64_t D, int64_t Dv, int64_t q_start) {
  if (!valid_dtype(dtype)) return set_error(DA_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || T < 0 || S < 0) return set_error(DA_ERR_INVALID, "%s: negative size", what);
  if (k_heads < 1 || heads < 1 || heads % k_heads)
    return set_error(DA_ERR_INVALID, "%s: %lld heads do not share %lld key heads", what, (long long)heads,
                     (long long)k_heads);
  if (D < 1 || D > 128 || Dv < 1 || Dv > 256)
    return set_error(DA_ERR_UNSUPPORTED, "%s: maps of 1 to 128 entries and values of 1 to 256, got %lld and %lld", what,
                     (long long)D, (long long)Dv);
  const int64_t most = int64_t{1} << 30;
  if (batch >= most || T >= most || S >= most || heads >= most || T * (heads / k_heads) >= most ||
      q_start >= most || q_start <= -most)
    return set_error(DA_ERR_UNSUPPORTED, "%s: lengths, heads and positions below 2^30", what);
  return DA_OK;
}

int fill_args(Args& a, const char* what, const da_diff_inputs* in, int64_t batch, int64_t T, int64_t S, int64_t heads,
              int64_t k_heads, int64_t D, int64_t Dv, float scale, int causal, int64_t q_start) {
  if (!valid_dtype((int)in->lam_dtype)) return set_error(DA_ERR_INVALID, "%s: bad dtype %d", what, (int)in->lam_dtype);
  if (!(scale > 0.f) || !(scale < 1e30f)) return set_error(DA_ERR_INVALID, "%s: the scale must be positive", what);
  a.q = (const char*)in->q, a.k = (const char*)in->k, a.v = (const char*)in->v;
  a.lam = in->lam, a.lam_dtype = (int)in->lam_dtype, a.lam_stride = in->lam_stride;
  a.mask = in->mask, a.q_mask = in->q_mask;
  a.q_b = in->q_bstride, a.q_t = in->q_tstride, a.q_h = in->q_hstride;
  a.k_b = in->k_bstride, a.k_t = in->k_tstride, a.k_h = in->k_hstride;
  a.v_b = in->v_bstride, a.v_t = in->v_tstride, a.v_h = in->v_hstride;
  a.m_b = in->mask_bstride, a.m_k = in->mask_kstride, a.qm_b = in->q_mask_bstride, a.qm_t = in->q_mask_tstride;
  a.batch = (int)batch, a.T = (int)T, a.S = (int)S, a.Hk = (int)k_heads, a.G = (int)(heads / k_heads);
  a.D = (int)D, a.Dv = (int)Dv, a.causal = causal, a.q_start = q_start, a.scale = scale;
  return DA_OK;
}

int allow_lds(const void* kernel, int bytes) {
  if (bytes > 65536 && hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return set_error(DA_ERR_HIP, "da_diff_attention: hipFuncSetAttribute failed");
  return DA_OK;
}

namespace {

// One wave a workgroup where there are no more rows than it takes, and a tile of keys and
// values fits its registers on the way (16 KB: 64 a lane).
int waves_of(int64_t rows, int dtype, int w) { return rows <= kTile && dtype != DA_F32 && w < 2 ? 1 : 4; }

// Keys are split where the rows alone leave CUs without work: about eight waves' worth of
// workgroups a CU, no part under 256 keys.
int split_of(int dtype, int w, int64_t batch, int64_t T, int64_t S, int64_t k_heads, int64_t G, int* blocks, int* splits, int* keys) {
  int64_t cus;
  const int rc = device_cu_count(&cus);
  if (rc) return rc;
  const int64_t rows = T * G, nw = waves_of(rows, dtype, w);
  const int64_t n = (rows + nw * kTile - 1) / (nw * kTile), groups = batch * k_heads * n;
  int64_t want = groups >= cus ? 1 : (nw == 1 ? 8 : 2) * cus / std::max<int64_t>(groups, 1);
  if (nw == 1 && groups >= cus) want = 8 * cus / groups;
  want = std::max<int64_t>(1, std::min<int64_t>(want, S / 256));
  const int64_t each = ((S + want - 1) / want + kTile - 1) / kTile * kTile;
  *blocks = (int)n;
  *keys = (int)std::max<int64_t>(each, kTile);
  *splits = (int)std::max<int64_t>(1, (S + *keys - 1) / *keys);
  return DA_OK;
}

const int kValueWidths[] = {64, 128, 128, 256};

size_t workspace_of(int64_t batch, int64_t rows, int64_t k_heads, int splits, int w) {
  return splits > 1 ? (size_t)splits * batch * k_heads * rows * 2 * (kValueWidths[w] + 2) * sizeof(float) : 0;
}

}  // namespace
}  // namespace diff
}  // namespace da

extern "C" {

int da_diff_attention_workspace(int dtype, int64_t batch, int64_t q_len, int64_t k_len, int64_t heads,
                                int64_t k_heads, int64_t d, int64_t dv, size_t* bytes) {
  using namespace da;
  using namespace da::diff;
  if (!bytes) return set_error(DA_ERR_INVALID, "da_diff_attention_workspace: NULL pointer");
  *bytes = 0;
  int rc = check_sizes("da_diff_attention_workspace", dtype, batch, q_len, k_len, heads, k_heads, d, dv, 0);
  if (rc || batch == 0 || q_len == 0) return rc;
  int blocks, splits, keys;
  rc = split_of(dtype, widths(d, dv), batch, q_len, k_len, k_heads, heads / k_heads, &blocks, &splits, &keys);
  if (rc == DA_OK) *bytes = workspace_of(batch, q_len * (heads / k_heads), k_heads, splits, widths(d, dv));
  return rc;
}

int da_diff_attention(const da_diff_inputs* in, int dtype, int64_t batch, int64_t q_len, int64_t k_len, int64_t heads,
                      int64_t k_heads, int64_t d, int64_t dv, float scale, int causal, int64_t q_start, void* out,
                      void* second, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace da;
  using namespace da::diff;
  int rc = check_sizes("da_diff_attention", dtype, batch, q_len, k_len, heads, k_heads, d, dv, q_start);
  if (rc) return rc;
  if (batch == 0 || q_len == 0) return DA_OK;
  if (!in || !in->q || !in->lam || !out || (k_len && (!in->k || !in->v)) || !second != !lse)
    return set_error(DA_ERR_INVALID, "da_diff_attention: NULL pointer");
  Args a = {};
  rc = fill_args(a, "da_diff_attention", in, batch, q_len, k_len, heads, k_heads, d, dv, scale, causal, q_start);
  if (rc) return rc;
  a.out = (char*)out, a.second = (char*)second, a.lse = lse;
  const int w = widths(d, dv);
  rc = split_of(dtype, w, batch, q_len, k_len, k_heads, a.G, &a.row_blocks, &a.splits, &a.split_keys);
  if (rc) return rc;
  const int64_t rows = q_len * a.G;
  const size_t need = workspace_of(batch, rows, k_heads, a.splits, w);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "da_diff_attention: workspace of %zu bytes needed", need);
  if ((uintptr_t)workspace % 16) return set_error(DA_ERR_INVALID, "da_diff_attention: workspace must be 16-byte aligned");
  a.part = (float*)workspace;
  if (batch * k_heads > kMaxBlocks / a.splits / a.row_blocks)
    return set_error(DA_ERR_UNSUPPORTED, "da_diff_attention: too many rows");
  const unsigned grid = (unsigned)(batch * k_heads * a.splits * a.row_blocks);
  const hipStream_t st = (hipStream_t)stream;
  const bool one = waves_of(rows, dtype, w) == 1;
  return by_widths(dtype, w, [&](auto dt, auto dp, auto dvp) {
    constexpr int DT = decltype(dt)::value, DP = decltype(dp)::value, DVP = decltype(dvp)::value;
    if constexpr (DT != DA_F32 && DP == 64) {
      if (one) diff_forward<DT, DP, DVP, 1><<<grid, 64, Smem<DT, DP, DVP, 1>::kBytes, st>>>(a);
    }
    if (!one) {
      constexpr int kBytes = Smem<DT, DP, DVP, 4>::kBytes;
      if (const int err = allow_lds((const void*)diff_forward<DT, DP, DVP, 4>, kBytes)) return err;
      diff_forward<DT, DP, DVP, 4><<<grid, 256, kBytes, st>>>(a);
    }
    if (a.splits > 1) {
      constexpr int kRows = 256 / (DVP / 4);
      const int64_t all = batch * k_heads * rows;
      diff_join<DT, DVP><<<(unsigned)((all + kRows - 1) / kRows), 256, 0, st>>>(a);
    }
    return check_launch("da_diff_attention");
  });
}

}  // extern "C"
