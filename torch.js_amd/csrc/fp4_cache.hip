// Values into four bits and back: weights (tjh_fp4_quantize, _dequantize) and
// the positions of a key / value cache (tjh_fp4_cache_append, _read).
#include "fp4.h"

namespace tjh {
namespace {

using namespace fp4;

constexpr int64_t kGrid = 1 << 21;  // workgroups of a launch: a grid has less than 2^32 threads

// Largest of 4, 8 or 16 neighbouring lanes.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  const uint32_t w = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
  return v > w ? v : w;
}
template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = dpp_max<kDppXor2>(dpp_max<kDppXor1>(v));
  if (LANES > 4) v = dpp_max<0x141>(v);  // row_half_mirror: the other four of eight
  if (LANES > 8) v = dpp_max<kDppRor8>(v);
  return v;
}

// ------------------------------------------------------------------ weights

// 16 lanes a row's 128 columns, 8 columns a lane (one word of codes), 4, 8 or
// 16 lanes a scale.  Runs once for a layer: 50257 x 768 (154 MB) 75 us.
__global__ __launch_bounds__(256) void k_fp4_quantize(const float* __restrict__ w, int64_t ld,
                                                      int64_t K, uint32_t nb, uint32_t items,
                                                      int lanes, uint32_t* __restrict__ codes,
                                                      float* __restrict__ scales) {
  const uint32_t at = blockIdx.x * 256 + threadIdx.x;
  const bool on = at < items;
  const uint32_t block = (on ? at : items - 1) >> 4;  // n nb + b
  const int i = threadIdx.x & 15;
  const int64_t n = block / nb, k = (int64_t)(block % nb) * 128 + 8 * i;
  float x[8];
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = k + e < K ? w[n * ld + k + e] : 0.f;
    top = max(top, magnitude(x[e]));
  }
  const uint32_t most = lanes == 4 ? row_max<4>(top) : lanes == 8 ? row_max<8>(top) : row_max<16>(top);
  const float scale = scale_of(most);
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) word |= code_of(x[e], scale) << (4 * e);
  if (!on) return;
  codes[block * 16 + 4 * (i & 3) + (i >> 2)] = word;
  if (i % lanes == 0) scales[(block * 16 + i) / (uint32_t)lanes] = scale;
}

// One word a thread.
__global__ __launch_bounds__(256) void k_fp4_dequantize(const uint32_t* __restrict__ codes,
                                                        const float* __restrict__ scales,
                                                        int64_t K, uint32_t nb, uint32_t items,
                                                        int lanes, float* __restrict__ out,
                                                        int64_t ldo) {
  const uint32_t at = blockIdx.x * 256 + threadIdx.x;
  if (at >= items) return;
  const uint32_t block = at >> 4;
  const int i = at & 15;
  const int64_t n = block / nb, k = (int64_t)(block % nb) * 128 + 8 * i;
  const float scale = scales[at / (uint32_t)lanes];
  float v[8];
  unpack(codes[block * 16 + 4 * (i & 3) + (i >> 2)], v);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (k + e < K) out[n * ldo + k + e] = v[e] * scale;
}

// -------------------------------------------------------------------- cache

struct AppendArgs {
  const float* x[2];
  uint8_t* codes[2];
  float* scales[2];
  int64_t st[2][4];
  int64_t L, pos;
  uint32_t H, T, rows;
  const int32_t* positions;
  int D, P;
};

// LR lanes a position, 8 columns and a word of codes a lane (VEC: as 16-byte
// loads), the rows of K (grid y 0) and of V.  8 x 12 heads of 1024 positions by 64,
// K and V (50 MB read, 7 written): 13.5 us, 4.2 TB/s.
template <int LR, bool VEC>
__global__ __launch_bounds__(256) void k_fp4_append(AppendArgs a) {
  const int which = blockIdx.y;
  const uint32_t at = (blockIdx.x * 256 + threadIdx.x) / LR;
  const bool on = at < a.rows;
  const uint32_t row = on ? at : a.rows - 1;  // (b H + h) T + t
  const int d = 8 * (threadIdx.x % LR);
  const uint32_t bhu = row / a.T;
  const int64_t bh = bhu, t = row - bhu * a.T, b = bhu / a.H, h = bhu % a.H;
  const int64_t* st = a.st[which];
  const float* p = a.x[which] + b * st[0] + h * st[1] + t * st[2] + d * st[3];
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  if (VEC) {
#pragma unroll
    for (int q = 0; q < 8; q += 4) {
      if (d + q >= a.D) continue;
      const floatx4 v = *reinterpret_cast<const floatx4*>(p + q);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[q + e] = v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (d + e < a.D) x[e] = p[e * st[3]];
  }
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, magnitude(x[e]));
  const float scale = scale_of(row_max<LR>(top));
  const int64_t to = (a.positions ? (int64_t)a.positions[b] : a.pos) + t;
  if (!on || to < 0 || to >= a.L) return;
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) word |= code_of(x[e], scale) << (4 * e);
  const int64_t place = bh * a.L + to;
  if (d < 2 * a.P)
    *reinterpret_cast<uint32_t*>(a.codes[which] + place * a.P + d / 2) = word;
  if (d == 0) a.scales[which][place] = scale;
}

struct ReadArgs {
  const uint8_t* codes[2];
  const float* scales[2];
  float* out[2];
  int64_t L, start;
  uint32_t n, items;
  int D, P;
};

// 8 columns a thread, keys (grid y 0) and values.  8 x 12 heads of 1024 positions
// by 64, 50 MB written: 11.6 us, 4.9 TB/s.
__global__ __launch_bounds__(256) void k_fp4_read(ReadArgs a) {
  const uint32_t at = blockIdx.x * 256 + threadIdx.x;
  if (at >= a.items) return;
  const uint32_t per = (a.D + 7) / 8, rw = at / per, bh = rw / a.n;
  const int64_t row = rw, from = bh * a.L + a.start + (rw - bh * a.n);
  const int d = 8 * (int)(at - rw * per), D = a.D;
  const float scale = a.scales[blockIdx.y][from];
  float v[8];
  unpack(*reinterpret_cast<const uint32_t*>(a.codes[blockIdx.y] + from * a.P + d / 2), v);
  float* o = a.out[blockIdx.y] + row * D + d;
  if (D % 4 == 0) {
    *reinterpret_cast<floatx4*>(o) = floatx4{v[0], v[1], v[2], v[3]} * scale;
    if (d + 4 < D) *reinterpret_cast<floatx4*>(o + 4) = floatx4{v[4], v[5], v[6], v[7]} * scale;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (d + e < D) o[e] = v[e] * scale;
  }
}

int check_weights(const char* who, int64_t N, int64_t K, int64_t group) {
  TJH_ARG(N >= 0 && K >= 0 && N < (int64_t(1) << 31) && K < (int64_t(1) << 30), "%s: bad sizes",
          who);
  TJH_ARG(group == 32 || group == 64 || group == 128, "%s: groups of %lld columns (32, 64 or 128)",
          who, (long long)group);
  return TJH_OK;
}

}  // namespace
}  // namespace tjh

using namespace tjh;

extern "C" {

int tjh_fp4_quantize(const float* w, int64_t ld, int64_t N, int64_t K, int64_t group,
                     uint8_t* codes, float* scales) {
  TJH_REQUIRE_INIT();
  const int rc = check_weights("tjh_fp4_quantize", N, K, group);
  if (rc != TJH_OK) return rc;
  TJH_ARG(ld >= K, "tjh_fp4_quantize: bad sizes");
  if (N == 0 || K == 0) return TJH_OK;
  TJH_ARG(w && codes && scales && aligned16(codes), "tjh_fp4_quantize: NULL or unaligned pointer");
  const int64_t nb = cdiv(K, 128), step = kGrid * 256;
  TJH_ARG(nb * 16 <= step, "tjh_fp4_quantize: rows too long");
  const int64_t rows = step / (nb * 16);  // of one launch
  KernelScope ks("fp4_quantize");
  for (int64_t n = 0; n < N; n += rows) {
    const int64_t m = N - n < rows ? N - n : rows;
    tjh_launch(k_fp4_quantize, dim3((unsigned)cdiv(m * nb * 16, 256)), dim3(256), 0, stream(),
               w + n * ld, ld, K, (uint32_t)nb, (uint32_t)(m * nb * 16),
               (int)group / 8,
               reinterpret_cast<uint32_t*>(codes) + n * nb * 16, scales + n * nb * 128 / group);
  }
  return check_launch("fp4_quantize");
}

int tjh_fp4_dequantize(const uint8_t* codes, const float* scales, int64_t N, int64_t K,
                       int64_t group, float* out, int64_t ldo) {
  TJH_REQUIRE_INIT();
  const int rc = check_weights("tjh_fp4_dequantize", N, K, group);
  if (rc != TJH_OK) return rc;
  TJH_ARG(ldo >= K, "tjh_fp4_dequantize: bad sizes");
  if (N == 0 || K == 0) return TJH_OK;
  TJH_ARG(out && codes && scales && aligned16(codes),
          "tjh_fp4_dequantize: NULL or unaligned pointer");
  const int64_t nb = cdiv(K, 128), step = kGrid * 256;
  TJH_ARG(nb * 16 <= step, "tjh_fp4_dequantize: rows too long");
  const int64_t rows = step / (nb * 16);
  KernelScope ks("fp4_dequantize");
  for (int64_t n = 0; n < N; n += rows) {
    const int64_t m = N - n < rows ? N - n : rows;
    tjh_launch(k_fp4_dequantize, dim3((unsigned)cdiv(m * nb * 16, 256)), dim3(256), 0, stream(),
               reinterpret_cast<const uint32_t*>(codes) + n * nb * 16,
               scales + n * nb * 128 / group, K, (uint32_t)nb, (uint32_t)(m * nb * 16),
               (int)group / 8, out + n * ldo,
               ldo);
  }
  return check_launch("fp4_dequantize");
}

int tjh_fp4_cache_append(const float* k, const float* v, const int64_t* k_strides,
                         const int64_t* v_strides, uint8_t* k_codes, float* k_scales,
                         uint8_t* v_codes, float* v_scales, int64_t B, int64_t H, int64_t T,
                         int64_t D, int64_t L, int64_t pos, const int32_t* positions) {
  TJH_REQUIRE_INIT();
  TJH_ARG(B >= 0 && H >= 0 && T >= 0 && D > 0 && L >= 0, "tjh_fp4_cache_append: bad sizes");
  if (D > 128 || L >= (int64_t(1) << 24))
    return set_error(TJH_ERR_UNSUPPORTED,
                     "tjh_fp4_cache_append: head dim %lld, length %lld (128, 2^24 - 1 at most)",
                     (long long)D, (long long)L);
  TJH_ARG(positions || (pos >= 0 && pos + T <= L), "tjh_fp4_cache_append: positions [%lld, %lld) of %lld",
          (long long)pos, (long long)(pos + T), (long long)L);
  if (B == 0 || H == 0 || T == 0 || L == 0) return TJH_OK;
  TJH_ARG(k && v && k_strides && v_strides && k_codes && k_scales && v_codes && v_scales &&
              aligned16(k_codes) && aligned16(v_codes),
          "tjh_fp4_cache_append: NULL or unaligned pointer");
  const int64_t rows = B * H * T;
  const int lanes = D <= 32 ? 4 : D <= 64 ? 8 : 16;
  TJH_ARG(B < (1 << 29) && H < (1 << 29) && T < (1 << 29) && B * H < (1 << 29) &&
              rows < (1 << 29) && cdiv(rows * lanes, 256) <= kGrid,
          "tjh_fp4_cache_append: too many rows");
  AppendArgs a{{k, v}, {k_codes, v_codes}, {k_scales, v_scales}, {}, L, pos, (uint32_t)H,
               (uint32_t)T, (uint32_t)rows, positions, (int)D, fp4::row_bytes((int)D)};
  bool vec = D % 4 == 0 && aligned16(k) && aligned16(v);
  for (int i = 0; i < 4; ++i) {
    a.st[0][i] = k_strides[i];
    a.st[1][i] = v_strides[i];
    vec = vec && (i == 3 ? k_strides[i] == 1 && v_strides[i] == 1
                         : k_strides[i] % 4 == 0 && v_strides[i] % 4 == 0);
  }
  const dim3 grid((unsigned)cdiv(rows * lanes, 256), 2), block(256);
  KernelScope ks("fp4_append");
  if (lanes == 4 && vec) tjh_launch(k_fp4_append<4, true>, grid, block, 0, stream(), a);
  else if (lanes == 4) tjh_launch(k_fp4_append<4, false>, grid, block, 0, stream(), a);
  else if (lanes == 8 && vec) tjh_launch(k_fp4_append<8, true>, grid, block, 0, stream(), a);
  else if (lanes == 8) tjh_launch(k_fp4_append<8, false>, grid, block, 0, stream(), a);
  else if (vec) tjh_launch(k_fp4_append<16, true>, grid, block, 0, stream(), a);
  else tjh_launch(k_fp4_append<16, false>, grid, block, 0, stream(), a);
  return check_launch("fp4_append");
}

int tjh_fp4_cache_read(const uint8_t* codes, const float* scales, const uint8_t* codes2,
                       const float* scales2, int64_t B, int64_t H, int64_t L, int64_t D,
                       int64_t start, int64_t n, float* out, float* out2) {
  TJH_REQUIRE_INIT();
  TJH_ARG(B >= 0 && H >= 0 && D > 0 && start >= 0 && n >= 0 && start + n <= L,
          "tjh_fp4_cache_read: bad sizes");
  if (D > 128 || L >= (int64_t(1) << 24))
    return set_error(TJH_ERR_UNSUPPORTED,
                     "tjh_fp4_cache_read: head dim %lld, length %lld (128, 2^24 - 1 at most)",
                     (long long)D, (long long)L);
  if (B == 0 || H == 0 || n == 0) return TJH_OK;
  TJH_ARG(codes && scales && out && aligned16(codes) && aligned16(out) &&
              (!codes2 || (scales2 && out2 && aligned16(codes2) && aligned16(out2))),
          "tjh_fp4_cache_read: NULL or unaligned pointer");
  const int64_t items = B * H * n * cdiv(D, 8);
  TJH_ARG(B < (1 << 29) && H < (1 << 29) && B * H < (1 << 29) && cdiv(items, 256) <= kGrid,
          "tjh_fp4_cache_read: too many rows");
  const ReadArgs a{{codes, codes2}, {scales, scales2}, {out, out2}, L, start, (uint32_t)n,
                   (uint32_t)items, (int)D, fp4::row_bytes((int)D)};
  KernelScope ks("fp4_read");
  tjh_launch(k_fp4_read, dim3((unsigned)cdiv(items, 256), codes2 ? 2 : 1), dim3(256), 0, stream(),
             a);
  return check_launch("fp4_read");
}

}  // extern "C"
