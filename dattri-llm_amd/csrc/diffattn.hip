// Attention by the difference of two softmax maps, forward.
//
// Head h has two query maps and its key head two key maps:
//
//   out = o_1 - lam_h o_2,   o_m = softmax(scale q_m k_m^T) v     (zero for a row without keys,
//                                                               NaN for one with NaN or infinite scores)
//
// One pass over the keys, a wave to a map and to 32 rows, with their running maxima and
// sums.  It forms the transposed scores, k q^T, so that a row is a lane's (two lanes', 16
// keys each) and its maximum and sum stay within them; the accumulator's registers then are,
// rounded, the second operand of o^T = v^T p^T as they stand, where v is read transposed out
// of LDS.  A difference of scores is formed before it is scaled where they are large (kNear), so
// that any finite scores have finite exponentials.  These are relative to a maximum that is looked
// for again only when the sum of a lane's sixteen passes 2^10 (fp16: 2^15, the largest being 2^10):
// until then they are at most that much larger than with the last one (the first tile has none, and
// passes; with a new one in every tile that has a larger score a twelfth more time at the first size
// below).  At the end the second map's waves hand their values, divided and weighted, to the first's
// through LDS.
//
// 4 x 2048 causal tokens in bf16: 32 heads on 8, two 64-wide maps and 128-wide values 260 us
// (206 GFLOP, 790 TFLOP/s), 16 heads of 128 and 256 267 us (770 TFLOP/s): vector and matrix unit
// nearly in sum.  16 new tokens of 32 heads on 8 against 8192 positions 94 + 12 us, HBM at 4.8 TB/s.
#include <algorithm>
#include <type_traits>

#include "diffattn.h"

namespace da {
namespace diff {
namespace {

// Keys of a split (18 heads of 509 keys in fp32: 65 us with 64, 59 with 128).
constexpr int kLeastSplit = 128;
constexpr int kFewKeys = 512;

// The largest exponential is 2^kUp when it is found, and a lane's sixteen sum to kMostSum before a
// new maximum is looked for.  As fp16 operands they are lifted so that keys far below the largest
// keep bits, down to 2^-24: of 2^17 keys 17 below it, which have a tenth of a percent of the row,
// nothing was left without.
template <int DT>
struct Range {
  static constexpr float kUp = DT == DA_F16 ? 10.f : 0.f;
  static constexpr float kMostSum = DT == DA_F16 ? 32768.f : 1024.f;
};

// A row that sees keys has a sum of about 1 and more (its maximum's exponential), one that sees
// none 0.  A split whose live scores are all -inf sums to kOnlyInf: that counts for nothing beside
// another split's sum, and where it is all there is the row is NaN, as the softmax is.
constexpr float kOnlyInf = 0x1p-100f;
__device__ __forceinline__ float settled(float sum) { return sum > 0.f && sum < 0.5f ? __builtin_nanf("") : sum; }
// Of a settled sum, NaN of NaN.
__device__ __forceinline__ float inverse(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }

// The exponentials are 2^((s - top) c + shift).  shift is kUp and what rounding top c - kUp leaves of
// it, so that one fma, s c - base, gives them; where that could be large (it is half a unit of top
// c's last place), kUp, and the difference is formed first.
constexpr float kNear = 0x1p20f;
__device__ __forceinline__ bool near(float top, float c) { return fabsf(top * c) < kNear; }
template <int DT>
__device__ __forceinline__ float base_of(float top, float c) {
  return fmaf(top, c, -Range<DT>::kUp);
}
template <int DT>
__device__ __forceinline__ float shift_of(float top, float c) {
  return near(top, c) ? fmaf(top, c, -base_of<DT>(top, c)) : Range<DT>::kUp;
}

// What the backward pass needs of a row: the settled sum of 2^((s - top) c), +inf where it sees no
// key, and top.
__device__ __forceinline__ void put_lse(const Args& a, int64_t at, float top, float shift, float sum) {
  a.lse[at] = sum == 0.f ? __builtin_inff() : log2f(sum) - shift;
  a.lse[tops_at(a) + at] = sum == 0.f ? 0.f : top;
}

// NG tiles of rows, each with a wave for either map.
template <int DT, int DP, int DVP, int NG>
struct Smem {
  static constexpr int NT = 2 * NG * kWave;
  static constexpr int kK = Tile<DT, DP, NT>::kBytes, kV = Tile<DT, DVP, NT>::kBytes;
  static constexpr int kStage = 2 * kK + kV, kHanded = NG * DVP / 32 * 4096;
  static constexpr int kBytes = 2 * kStage > kHanded ? 2 * kStage : kHanded;
};

// kFine: probabilities as the sum of two 16-bit values, so that values are rounded once, at the
// end (bf16 error 1.7e-3).  Where a token's few rows leave the matrix units idle that costs
// nothing; else the products with v double.  With up to kFewKeys keys, where each counts for more, that
// is at most a fifth of the time (32 heads on 8 of 64 and 128: 16 x 256 tokens 49 us and 43 without,
// 16 x 512 120 and 99), past it more (8 x 768 118 and 93, 8 x 1024 186 and 140, 4 x 2048 332 and 242):
// there they are rounded where they are multiplied, by half a step each, no more than the output's
// own rounding (2.4e-3 together).  Sums stay in fp32.
// Two waves a SIMD but for the widest maps in fp32, which would spill (8 heads of 2 x 512 tokens
// 203 us in place of 141) and whose tiles leave LDS for one workgroup anyway.
template <int DT, int DP, int DVP, int NG, bool kFine>
__global__ __launch_bounds__(2 * NG * kWave, DT == DA_F32 && DVP == 256 ? 1 : 2) void diff_forward(Args a) {
  using L = Smem<DT, DP, DVP, NG>;
  constexpr int NT = L::NT, ES = Type<DT>::ES, V = Type<DT>::V;
  constexpr int KD = DP / Type<DT>::kStep, NB = DVP / 32, KC = Type<DT>::kChunks;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), map = wave & 1, group = wave >> 1;
  // Workgroups of one key head are neighbours on one die; the rows with the most keys go first.
  int at = (int)xcd_remap(blockIdx.x, gridDim.x);
  const int block = a.blocks - 1 - at % a.blocks;
  at /= a.blocks;
  const int split = at % a.splits;
  at /= a.splits;
  const int hk = at % a.Hk, b = at / a.Hk;
  const int rows = a.T * a.G;
  const int r = (block * NG + group) * kTile + (lane & 31), t = token_of(a, r), h = hk * a.G + (r - t * a.G);
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
  if (a.causal) {  // rows come in order: the workgroup's last one sees most
    const int64_t t_last = token_of(a, min((block + 1) * NG * kTile, rows) - 1);
    end = (int)max((int64_t)0, min((int64_t)a.S, t_last + a.q_start + 1));
  }
  int key = split * a.each;
  end = min(end, key + a.each);

  u32x4 q[KD];
#pragma unroll
  for (int kk = 0; kk < KD; ++kk)
    q[kk] = last >= 0 ? load_run<DT>(a.q + (b * a.q_b + t * a.q_t + (2 * h + map) * a.q_h) * ES, (2 * kk + half) * V, a.D)
                      : u32x4{0, 0, 0, 0};

  const Keys<DT, DP, NT> keys(a.k_t, a.D);
  const Keys<DT, DVP, NT> values(a.v_t, a.Dv);
  const char* kp = a.k + (b * a.k_b + 2 * hk * a.k_h) * ES;
  const char* vp = a.v + (b * a.v_b + hk * a.v_h) * ES;
  const auto fetch = [&](int to, int stage, uint32_t live) __attribute__((always_inline)) {
    const uint32_t l = lds_address(lds) + stage * L::kStage;
    keys.fetch(kp + to * a.k_t * ES, l, live);
    keys.fetch(kp + (to * a.k_t + a.k_h) * ES, l + L::kK, live);
    values.fetch(vp + to * a.v_t * ES, l + 2 * L::kK, live);
  };

  const float c = a.scale * kLog2e;
  f32x16 o[NB];
  // A lane without a row sees nothing, and does not make the others' scores large.
  float top = last >= 0 ? kLowest : 0.f, shift = Range<DT>::kUp, sum = 0.f;
  bool far = true;  // whether a score of the wave is large
  uint32_t saw = 0;  // whether the row has seen a key
#pragma unroll
  for (int x = 0; x < NB; ++x) o[x] = zeros();
  const Reader<DT, DP> key_reader(lds + map * L::kK, lane);
  const Reader<DT, DVP> value_reader(lds + 2 * L::kK, lane);
  // The next tile with a live key is on its way while one is multiplied.
  Live live(a, b, key, end, lane);
  if (live.word) fetch(live.key, 0, live.word);
  const auto step = [&](auto of) __attribute__((always_inline)) {
    constexpr int stage = decltype(of)::value;
    key = live.key;
    const uint32_t word = live.word;
    live.next(a, b, end, lane);
    tiles_barrier();
    if (live.word) fetch(live.key, stage ^ 1, live.word);
    if (key > most) return;
    f32x16 s = zeros();
#pragma unroll
    for (int kk = 0; kk < KD; ++kk) Mfma32<DT>::mma(s, key_reader.rows(stage * L::kStage, kk), q[kk]);
    if (word != ~0u || key + kTile - 1 > least) {
      const uint32_t seen = seen_of(word, key, last, half);
      saw |= seen;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = seen & 1u << acc_at(i, 0) ? s[i] : -__builtin_inff();
    } else {
      saw = 1;
    }
    f32x16 e;
    const auto exponentials = [&]() __attribute__((always_inline)) {
      if (far) {  // the same in all lanes
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(s[i] - top, c, shift));
      } else {
        const float base = base_of<DT>(top, c);
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -base));
      }
      return over_acc(e, [](float u, float v) { return u + v; });
    };
    float part = exponentials();
    if (__any(part > Range<DT>::kMostSum)) {
      float x = over_acc(s, [](float u, float v) { return fmaxf(u, v); });
      x = fmaxf(x, other_half(x));
      const float now = fmaxf(top, x), shift_now = shift_of<DT>(now, c);
      const float by = __builtin_amdgcn_exp2f(fmaf(top - now, c, shift_now - shift));
      top = now, shift = shift_now;
      far = __any(!near(top, c));
      sum *= by;
#pragma unroll
      for (int y = 0; y < NB; ++y)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[y][i] *= by;
      part = exponentials();
    }
    sum += part;
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      const u32x4 p = from_acc<DT>(e, j);
      u32x4 rest;
      if constexpr (kFine) rest = rest_of<DT>(e, j, p);
#pragma unroll
      for (int y = 0; y < NB; ++y) {
        const u32x4 x = value_reader.columns(stage * L::kStage, y, j);
        Mfma32<DT>::mma(o[y], x, p);
        if constexpr (kFine) Mfma32<DT>::mma(o[y], x, rest);
      }
    }
  };
  while (live.word) {
    step(std::integral_constant<int, 0>{});
    if (live.word) step(std::integral_constant<int, 1>{});
  }

  sum += other_half(sum);
  saw |= __float_as_uint(other_half(__uint_as_float(saw)));
  if (sum == 0.f && saw) sum = kOnlyInf;
  if (a.splits > 1) {  // this split's sums
    if (r >= rows) return;
    float* to = a.part + ((((int64_t)split * a.batch + b) * a.Hk + hk) * rows + r) * 2 * (DVP + 2);
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *(f32x4*)(to + map * DVP + 32 * y + acc_at(i, half)) = f32x4{o[y][i], o[y][i + 1], o[y][i + 2], o[y][i + 3]};
    if (half == 0) to[2 * DVP + 2 * map] = top, to[2 * DVP + 2 * map + 1] = sum;
    return;
  }
  f32x4* handed = (f32x4*)(lds + group * (L::kHanded / NG));
  const bool in = r < rows;
  sum = settled(sum);
  const float by = inverse(sum);
  const int64_t to = (((int64_t)b * a.T + t) * (a.Hk * a.G) + h) * a.Dv * ES;
  if (a.lse && half == 0 && in) put_lse(a, (((int64_t)b * a.Hk + hk) * 2 + map) * rows + r, top, shift, sum);
  __syncthreads();  // the tiles have been read
  if (map) {
    const float lam = in && by != 0.f ? lam_of(a, h) : 0.f;
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 v = f32x4{o[y][i], o[y][i + 1], o[y][i + 2], o[y][i + 3]} * by;
        if (a.second && in) store4<DT>(a.second + to, 32 * y + acc_at(i, half), a.Dv, v[0], v[1], v[2], v[3]);
        handed[(y * 4 + i / 4) * kWave + lane] = v * lam;
      }
  }
  __syncthreads();
  if (!map && in) {
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 v = handed[(y * 4 + i / 4) * kWave + lane];
        store4<DT>(a.out + to, 32 * y + acc_at(i, half), a.Dv, o[y][i] * by - v[0], o[y][i + 1] * by - v[1],
                   o[y][i + 2] * by - v[2], o[y][i + 3] * by - v[3]);
      }
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
  const float c = a.scale * kLog2e;
#pragma unroll 4
  for (int p = 0; p < a.splits; ++p) {
    const float* from = a.part + (p * all + at) * 2 * (DVP + 2);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const float top2 = from[2 * DVP + 2 * m], sum2 = from[2 * DVP + 2 * m + 1];
      const f32x4 x = *(const f32x4*)(from + m * DVP + 4 * l);
      const float now = fmaxf(top[m], top2);
      const float f1 = __builtin_amdgcn_exp2f((top[m] - now) * c);
      const float f2 = __builtin_amdgcn_exp2f(fmaf(top2 - now, c, -shift_of<DT>(top2, c)));
      top[m] = now;
      sum[m] = sum[m] * f1 + sum2 * f2;
      o[m] = o[m] * f1 + x * f2;
    }
  }
  const int r = (int)(at % rows), hk = (int)(at / rows % a.Hk), b = (int)(at / rows / a.Hk);
  const int t = r / a.G, h = hk * a.G + (r - t * a.G);
  sum[0] = settled(sum[0]), sum[1] = settled(sum[1]);
  const float by0 = inverse(sum[0]), by1 = inverse(sum[1]);
  const float by2 = by1 != 0.f ? lam_of(a, h) * by1 : 0.f;
  const int64_t to = ((int64_t)b * a.T + t) * (a.Hk * a.G) + h;
  const f32x4 f = o[0] * by0 - o[1] * by2, g = o[1] * by1;
  store4<DT>(a.out + to * a.Dv * ES, 4 * l, a.Dv, f[0], f[1], f[2], f[3]);
  if (a.second) store4<DT>(a.second + to * a.Dv * ES, 4 * l, a.Dv, g[0], g[1], g[2], g[3]);
  if (a.lse && l == 0) {
    const int64_t to = ((int64_t)b * a.Hk + hk) * 2 * rows + r;
    put_lse(a, to, top[0], 0.f, sum[0]);
    put_lse(a, to + rows, top[1], 0.f, sum[1]);
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

// Rows are read in runs of 16 bytes, and a tile's by 31-bit offsets from its first row.
int check_side(const char* what, const char* name, const void* x, int es, int64_t width, int64_t tokens,
                      int64_t heads, int64_t bs, int64_t ts, int64_t hs) {
  if (!x) return DA_OK;
  const int64_t most = int64_t{1} << 31;
  if (((uintptr_t)x | (uint64_t)(bs * es) | (uint64_t)(ts * es) | (uint64_t)(hs * es) | (uint64_t)(width * es)) & 15)
    return set_error(DA_ERR_INVALID, "%s: rows of %s must be whole 16-byte runs at 16-byte aligned addresses", what, name);
  if (bs < 0 || ts < 0 || hs < 0) return set_error(DA_ERR_INVALID, "%s: negative stride of %s", what, name);
  if (ts >= most || hs >= most || (std::min<int64_t>(tokens, kTile + 1) * ts + heads * hs + width) * es >= most)
    return set_error(DA_ERR_UNSUPPORTED, "%s: tokens of %s lie too far apart", what, name);
  return DA_OK;
}

int fill_args(Args& a, const char* what, int dtype, const da_diff_inputs* in, int64_t batch, int64_t T, int64_t S, int64_t heads,
              int64_t k_heads, int64_t D, int64_t Dv, float scale, int causal, int64_t q_start) {
  if (!valid_dtype((int)in->lam_dtype)) return set_error(DA_ERR_INVALID, "%s: bad dtype %d", what, (int)in->lam_dtype);
  if (!(scale >= 1e-20f) || !(scale <= 1e20f))  // a logarithm over it stays in range, and 1e30 times it is large
    return set_error(DA_ERR_INVALID, "%s: the scale must lie between 1e-20 and 1e20", what);
  const int es = (int)elem_bytes(dtype);
  const int64_t group = heads / k_heads;
  int rc = check_side(what, "q", in->q, es, D, T, 2 * group, in->q_bstride, in->q_tstride, in->q_hstride);
  if (rc == DA_OK) rc = check_side(what, "k", in->k, es, D, S, 2, in->k_bstride, in->k_tstride, in->k_hstride);
  if (rc == DA_OK) rc = check_side(what, "v", in->v, es, Dv, S, 1, in->v_bstride, in->v_tstride, in->v_hstride);
  if (rc) return rc;
  a.q = (const char*)in->q, a.k = (const char*)in->k, a.v = (const char*)in->v;
  a.lam = in->lam, a.lam_dtype = (int)in->lam_dtype, a.lam_stride = in->lam_stride;
  a.mask = in->mask, a.q_mask = in->q_mask;
  a.q_b = in->q_bstride, a.q_t = in->q_tstride, a.q_h = in->q_hstride;
  a.k_b = in->k_bstride, a.k_t = in->k_tstride, a.k_h = in->k_hstride;
  a.v_b = in->v_bstride, a.v_t = in->v_tstride, a.v_h = in->v_hstride;
  a.m_b = in->mask_bstride, a.m_k = in->mask_kstride, a.qm_b = in->q_mask_bstride, a.qm_t = in->q_mask_tstride;
  a.batch = (int)batch, a.T = (int)T, a.S = (int)S, a.Hk = (int)k_heads, a.G = (int)(heads / k_heads);
  int bits = 0;
  while ((1 << bits) < a.G) ++bits;
  a.g_factor = (uint32_t)(((uint64_t{1} << (31 + bits)) + a.G - 1) / a.G);
  a.g_shift = 31 + bits;
  a.D = (int)D, a.Dv = (int)Dv, a.causal = causal, a.q_start = q_start, a.scale = scale;
  return DA_OK;
}

int allow_lds(const void* kernel, int bytes) {
  if (bytes > 65536 && hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return set_error(DA_ERR_HIP, "da_diff_attention: hipFuncSetAttribute failed");
  return DA_OK;
}

namespace {

// How rows are shared out: *ng tiles a workgroup.  Two share the keys they read (18 heads of
// 509 rows in fp32: 59 us, with one 88; 16 on 4 of 1024, 128 and 256 wide in bf16: 74 and 100).
int plan(int64_t batch, int64_t T, int64_t S, int64_t k_heads, int64_t G, int* ng, Args* a) {
  int64_t cus;
  const int rc = device_cu_count(&cus);
  if (rc) return rc;
  const int64_t rows = T * G, heads = batch * k_heads;
  const auto blocks_of = [&](int64_t n) { return (rows + n * kTile - 1) / (n * kTile); };
  *ng = rows > kTile ? 2 : 1;
  const int64_t blocks = blocks_of(*ng), groups = std::max<int64_t>(1, heads * blocks);
  // Keys are split where the rows leave CUs without work: up to sixteen waves a CU, no split
  // under kLeastSplit keys.
  int64_t want = std::max<int64_t>(1, (*ng == 1 ? 8 : 4) * cus / groups);
  want = std::max<int64_t>(1, std::min(want, S / kLeastSplit));
  const int64_t each = std::max<int64_t>(kTile, ((S + want - 1) / want + kTile - 1) / kTile * kTile);
  a->blocks = (int)blocks;
  a->each = (int)each;
  a->splits = (int)std::max<int64_t>(1, (S + each - 1) / each);
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
  int ng;
  Args a;
  rc = plan(batch, q_len, k_len, k_heads, heads / k_heads, &ng, &a);
  if (rc == DA_OK) *bytes = workspace_of(batch, q_len * (heads / k_heads), k_heads, a.splits, widths(d, dv));
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
  rc = fill_args(a, "da_diff_attention", dtype, in, batch, q_len, k_len, heads, k_heads, d, dv, scale, causal, q_start);
  if (rc) return rc;
  a.out = (char*)out, a.second = (char*)second, a.lse = lse;
  const int w = widths(d, dv);
  int ng;
  rc = plan(batch, q_len, k_len, k_heads, a.G, &ng, &a);
  if (rc) return rc;
  const int64_t rows = q_len * a.G;
  const size_t need = workspace_of(batch, rows, k_heads, a.splits, w);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "da_diff_attention: workspace of %zu bytes needed", need);
  if ((uintptr_t)workspace % 16) return set_error(DA_ERR_INVALID, "da_diff_attention: workspace must be 16-byte aligned");
  a.part = (float*)workspace;
  if (batch * k_heads > kMaxBlocks / a.splits / a.blocks)
    return set_error(DA_ERR_UNSUPPORTED, "da_diff_attention: too many rows");
  const unsigned grid = (unsigned)(batch * k_heads * a.splits * a.blocks);
  const hipStream_t st = (hipStream_t)stream;
  return by_widths(dtype, w, [&](auto dt, auto dp, auto dvp) {
    constexpr int DT = decltype(dt)::value, DP = decltype(dp)::value, DVP = decltype(dvp)::value;
    const auto launch = [&](auto groups, auto fine) {
      constexpr int NG = decltype(groups)::value;
      constexpr bool kFine = DT != DA_F32 && decltype(fine)::value;
      constexpr int kBytes = Smem<DT, DP, DVP, NG>::kBytes;
      const auto kernel = diff_forward<DT, DP, DVP, NG, kFine>;
      if (const int err = allow_lds((const void*)kernel, kBytes)) return err;
      kernel<<<grid, 2 * NG * kWave, kBytes, st>>>(a);
      return (int)DA_OK;
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    const int err = ng == 1 ? launch(One{}, std::true_type{})
                    : k_len <= kFewKeys ? launch(Two{}, std::true_type{}) : launch(Two{}, std::false_type{});
    if (err) return err;
    if (a.splits > 1) {
      constexpr int kRows = 256 / (DVP / 4);
      const int64_t all = batch * k_heads * rows;
      diff_join<DT, DVP><<<(unsigned)((all + kRows - 1) / kRows), 256, 0, st>>>(a);
    }
    return check_launch("da_diff_attention");
  });
}

}  // extern "C"
