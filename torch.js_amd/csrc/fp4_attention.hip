// Attention over a key / value cache held in 4 bits (beside
// F.scaled_dot_product_attention, src/nn/functional.ts:866-890):
//
//   o_i = sum over j <= p_i of softmax_j(scale ks_j (q_i . kc_j)) vs_j vc_j
//
// with the codes' steps kc, vc and one scale a position, ks, vs; query i of Tq
// stands at position p_i = length - Tq + i.
#include "fp4.h"

#include <math.h>

namespace tjh {
namespace {

using namespace fp4;

constexpr float kLog2e = 1.4426950408889634f;

struct AttArgs {
  const float* q;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  float* o;
  float *pm, *pl, *po;  // partial results of slices
  const int32_t* lengths;
  int64_t qb, qh, qt, ob, oh, ot;
  int64_t L, length;
  int B, H, Hkv, Tq, D, group;
  int row_tiles, slices;
  float scale;
};

__device__ __forceinline__ int length_of(const AttArgs& a, int b) {
  if (!a.lengths) return (int)a.length;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n > a.L ? (int)a.L : n;
}

// A row is one query of one of the heads that share a key head; a wave takes 16
// rows of one key head and walks tiles of 32 keys.  No operand changes lanes:
//
//   S^T[key, row] = K q^T: lane (j, n) feeds key n of each half tile and row n,
//     columns 8 NB j + 8 t + e in product t (any order serves that is the same in
//     both), q as three bfloat16 parts, and gets the scores of row n with the keys
//     4 j + r of both halves;
//   O[row, column] = P V: those eight keys are what lane (j, n) feeds of row n, in
//     three parts, so it feeds the same keys of V: eight words, one of each key,
//     whose 8 x 8 codes are transposed in registers.
//
// A matrix instruction cuts off what does not reach a sum's last bit.  Over thousands
// of keys a row's sum would outgrow what the third parts of P add to it, always to
// the same side where V's columns have a mean: 7e-6 of the result at 32768 keys of a
// wave.  So O (and the sum of the weights) goes on for kFold tiles only, and is then
// rounded to the float sum of those before, which waits in LDS: 1e-7, for up to 3% of
// the time over thousands of keys and none where a wave has fewer tiles.
//
// Running maxima are raised only when a score is kSlack above them, the same in the
// four lanes of a row; then the sums are rescaled.  So a weight is up to 2^kSlack, and
// a row's sum finite for 2^24 keys with values under 2^94.  A key takes 2 (D / 2 + 4)
// bytes and three products for 2 D / 512 of a matrix instruction each, so up to 16
// rows (a group's heads, or some queries) cost as much as one.
//
// Bound for one query by reading the cache: 32 sequences of 4096 to 8192 positions,
// 32 heads over 8 of 128, 217 MB: 51 us, 4.3 TB/s (with float multiply-adds in
// place of the matrix cores 131); for many by issuing some 260 vector instructions
// a tile beside its 42 to 48 products: the last 1999 of 4095 positions, 16 heads
// over 4 of 80: 178 us, 178 TFLOP/s, more than the float matrix cores' 154 (by
// float multiply-adds 1600).  Few short sequences by latency: 48 heads of 64, 1000
// positions 10.7 us.
constexpr float kSlack = 10.f;
constexpr int kWaves = 4, kTile = 32;
constexpr int kFold = 16;  // tiles; 8: 1% slower, 32: 1% faster at twice the error

// NB: words of a key that a lane feeds, a quarter of its codes.
template <int NB>
struct Dims {
  static constexpr int CH = NB == 1 ? 4 : NB == 2 ? 8 : 16;  // words of V's rows, over the lanes
  static constexpr int NT = CH / 2;                          // column tiles
  static constexpr int DP = 8 * CH;
  // column of lane n in tile d
  __device__ __forceinline__ static int column(int n, int d) {
    return 8 * (n % CH) + n / CH + 16 / CH * d;
  }
};

// w[d] = the d-th of the lane's columns: the codes of the eight keys whose words
// are a[0..8).
template <int NB>
__device__ __forceinline__ void transpose(const uint32_t (&a)[8], int n,
                                          uint32_t (&w)[Dims<NB>::NT]) {
  uint32_t u[8], v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // columns 0 to 3 and 4 to 7
    u[i] = __builtin_amdgcn_perm(a[i + 4], a[i], 0x05040100);
    u[i + 4] = __builtin_amdgcn_perm(a[i + 4], a[i], 0x07060302);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // pairs of columns
    if (i & 2) continue;
    v[i] = __builtin_amdgcn_perm(u[i + 2], u[i], 0x06020400);
    v[i + 2] = __builtin_amdgcn_perm(u[i + 2], u[i], 0x07030501);
  }
  constexpr uint32_t kLow = 0x0f0f0f0fu;
  const auto even = [&](uint32_t x, uint32_t y) { return (x & kLow) | ((y << 4) & ~kLow); };
  const auto odd = [&](uint32_t x, uint32_t y) { return ((x >> 4) & kLow) | (y & ~kLow); };
  if constexpr (Dims<NB>::CH == 16) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      w[i] = even(v[i], v[i + 1]);
      w[i + 1] = odd(v[i], v[i + 1]);
    }
  } else if constexpr (Dims<NB>::CH == 8) {  // columns n / 8 + 2 d
    const int s = n < 8 ? 0 : 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = ((v[2 * i] >> s) & kLow) | ((v[2 * i + 1] << (4 - s)) & ~kLow);
  } else {  // columns n / 4 + 4 d
    const int s = n & 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t x = n < 8 ? v[4 * i] : v[4 * i + 2], y = n < 8 ? v[4 * i + 1] : v[4 * i + 3];
      w[i] = ((x >> s) & kLow) | ((y << (4 - s)) & ~kLow);
    }
  }
}

template <int NB>
__device__ __forceinline__ void load_words(uint32_t (&w)[NB], const uint8_t* p) {
  typedef uint32_t uintx3 __attribute__((ext_vector_type(3), aligned(4)));
  if constexpr (NB == 4) {
    const uintx4 x = *reinterpret_cast<const uintx4*>(p);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else if constexpr (NB == 3) {
    const uintx3 x = *reinterpret_cast<const uintx3*>(p);
    w[0] = x.x; w[1] = x.y; w[2] = x.z;
  } else if constexpr (NB == 2) {
    const uintx2 x = *reinterpret_cast<const uintx2*>(p);
    w[0] = x.x; w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// SPLIT: the waves of a workgroup share 16 rows' keys, tile by tile; otherwise
// each has rows of its own.
template <int NB, bool SPLIT>
__global__ __launch_bounds__(64 * kWaves, NB < 4 ? 3 : 2) void k_fp4_attend(AttArgs a) {
  typedef Dims<NB> Z;
  constexpr int NT = Z::NT, P = 16 * NB;
  const int lane = threadIdx.x & 63, n = lane & 15, j = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = blockIdx.x;
  const int groups = SPLIT ? a.row_tiles : (a.row_tiles + kWaves - 1) / kWaves;
  const int g = groups - 1 - id % groups;  // the last queries have the most keys: first
  id /= groups;
  const int slice = id % a.slices, bh = id / a.slices;
  const int tile = SPLIT ? g : g * kWaves + w;
  if (!SPLIT && tile >= a.row_tiles) return;
  const int b = bh / a.Hkv, kh = bh - b * a.Hkv, len = length_of(a, b);
  const int rows = a.group * a.Tq, r0 = 16 * tile;
  // keys that this lane's row sees; that any and that all of the rows see
  const int row = min(r0 + n, rows - 1), h = row / a.Tq, i = row - h * a.Tq;
  const int seen = max(0, len - a.Tq + i + 1);
  const int last = min(r0 + 15, rows - 1), h0 = r0 / a.Tq, h1 = last / a.Tq;
  const int most = max(0, h0 == h1 ? len - a.Tq + last - h1 * a.Tq + 1 : len);
  const int least = max(0, len - a.Tq + (h0 == h1 ? r0 - h0 * a.Tq : 0) + 1);
  const int per = ((most + a.slices - 1) / a.slices + kTile - 1) / kTile * kTile;
  const int from = min(most, slice * per), to = min(most, from + per);
  const int64_t base = (int64_t)bh * a.L;
  const uint8_t* __restrict__ kc = a.kc + base * P;
  const uint8_t* __restrict__ vc = a.vc + base * P;
  const float* __restrict__ ks = a.ks + base;
  const float* __restrict__ vs = a.vs + base;
  const uint32_t kat = n * P + 4 * NB * j, vat = 4 * j * P + 4 * min(n % Z::CH, 4 * NB - 1);
  // one of keys or values of a tile; a key past the cache's end is its last one,
  // a key past `to` or not seen is whatever the cache holds: weights of 0 below
  const int end = (int)a.L;
  uint32_t kw[2][NB], vw[8];
  floatx4 kscale[2], vscale[2];
  const auto load_scales = [&](const float* p, int t0, floatx4 (&x)[2]) {
    if (t0 + kTile <= end) {
      const float* at = p + (uint32_t)(t0 + 4 * j);
#pragma unroll
      for (int y = 0; y < 2; ++y) x[y] = *reinterpret_cast<const floatx4u*>(at + 16 * y);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e >> 2][e & 3] = p[min(t0 + 16 * (e >> 2) + 4 * j + (e & 3), end - 1)];
    }
  };
  const auto load_k = [&](int t0) {
    if (t0 + kTile <= end) {
      const uint8_t* at = kc + ((uint32_t)t0 * P + kat);
      load_words(kw[0], at);
      load_words(kw[1], at + 16 * P);
    } else {
#pragma unroll
      for (int y = 0; y < 2; ++y)
        load_words(kw[y], kc + ((uint32_t)min(t0 + 16 * y + n, end - 1) * P + 4 * NB * j));
    }
    load_scales(ks, t0, kscale);
  };
  const auto load_v = [&](int t0) {
    if (t0 + kTile <= end) {
      const uint8_t* at = vc + ((uint32_t)t0 * P + vat);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        vw[e] = *reinterpret_cast<const uint32_t*>(at + (16 * (e >> 2) + (e & 3)) * P);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        vw[e] = *reinterpret_cast<const uint32_t*>(
            vc + ((uint32_t)min(t0 + 16 * (e >> 2) + 4 * j + (e & 3), end - 1) * P +
                  4 * min(n % Z::CH, 4 * NB - 1)));
    }
    load_scales(vs, t0, vscale);
  };
  const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
  floatx4 o[NT];
#pragma unroll
  for (int d = 0; d < NT; ++d) o[d] = zero;
  float m = -INFINITY, l = 0.f;
  // O and l of the tiles before the last fold, and by what maxima raised since scale
  // them; SPLIT: then what the waves add up, a wave's in its own place
  __shared__ floatx4 lds[kWaves][SPLIT ? 4 * (Z::DP + 4) : NT * 64];
  __shared__ float lds_l[kWaves][64];
  floatx4* const before = lds[w] + lane;
  float raised = 1.f;
  bool folded = false;
  const auto add_before = [&] {
    floatx4 f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = __shfl(raised, 4 * j + r, 64);
#pragma unroll
    for (int d = 0; d < NT; ++d) o[d] += before[64 * d] * f;
    l += lds_l[w][lane] * raised;
  };
  const int step = SPLIT ? kTile * kWaves : kTile;
  int t0 = from + (SPLIT ? w * kTile : 0);
  if (t0 < to) {
    load_k(t0);
    load_v(t0);
  }
  bf16x8 q[NB][3];
  {
    const float* p = a.q + b * a.qb + (int64_t)(kh * a.group + h) * a.qh + i * a.qt;
    const float f = a.scale * kLog2e;
#pragma unroll
    for (int t = 0; t < NB; ++t) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = 8 * (NB * j + t) + e;
        const float y = p[min(d, a.D - 1)];
        x[e] = d < a.D ? y * f : 0.f;
      }
      split8(x, q[t]);
    }
  }
  while (t0 < to) {
    const int stop = min(to, t0 + kFold * step);
    for (; t0 < stop; t0 += step) {
      const int tn = t0 + step < to ? t0 + step : t0;  // the last tile is loaded twice
      floatx4 s[2] = {zero, zero};
      {
        bf16x8 kf[2][NB];
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int t = 0; t < NB; ++t) kf[y][t] = steps(kw[y][t]);
#pragma unroll
        for (int part = 2; part >= 0; --part)
#pragma unroll
          for (int t = 0; t < NB; ++t)
#pragma unroll
            for (int y = 0; y < 2; ++y)
              s[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[y][t], q[t][part], s[y], 0, 0, 0);
      }
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = s[e >> 2][e & 3] * kscale[e >> 2][e & 3];
      load_k(tn);
      const bool masked = t0 + kTile > min(to, least);
      if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = t0 + 16 * (e >> 2) + 4 * j + (e & 3);
          if (t >= min(to, seen)) {
            p[e] = -INFINITY;
            vscale[e >> 2][e & 3] = 0.f;  // may be NaN
          }
        }
      }
      float top = p[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, p[e]);
      if (__any(top > m + kSlack)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float up = fmaxf(m, top);
        const float f = up == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - up);
        m = up;
        l *= f;
        raised *= f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float fr = __shfl(f, 4 * j + r, 64);
#pragma unroll
          for (int d = 0; d < NT; ++d) o[d][r] *= fr;
        }
      }
      const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __builtin_amdgcn_exp2f(p[e] - ms);
        l += y;
        p[e] = y * vscale[e >> 2][e & 3];
      }
      bf16x8 pp[3];
      split8_finite(p, pp);
      uint32_t v[NT];
      transpose<NB>(vw, n, v);
      load_v(tn);
#pragma unroll
      for (int d = 0; d < NT; d += 2) {  // two chains at a time
        const bf16x8 vb[2] = {steps(v[d]), steps(v[d + 1])};
#pragma unroll
        for (int part = 2; part >= 0; --part)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            o[d + y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pp[part], vb[y], o[d + y], 0, 0, 0);
      }
    }
    if (folded) add_before();
    if (t0 < to) {
#pragma unroll
      for (int d = 0; d < NT; ++d) {
        before[64 * d] = o[d];
        o[d] = zero;
      }
      lds_l[w][lane] = l;
      l = 0.f;
      raised = 1.f;
      folded = true;
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  // lane (j, n) has the columns of lane n of rows 4 j + r
  const auto put = [&](int r, int d, float num, float den, float top) {
    const int at = r0 + r;
    if (at >= rows || d >= a.D) return;
    if (a.slices == 1) {
      const int hh = at / a.Tq, t = at - hh * a.Tq;
      // zeros where no key is seen, NaN where all scores are -infinity
      a.o[b * a.ob + (int64_t)(kh * a.group + hh) * a.oh + t * a.ot + d] =
          len - a.Tq + t < 0 ? 0.f : num / den;
    } else {
      const int64_t p = ((int64_t)bh * rows + at) * a.slices + slice;
      a.po[p * a.D + d] = num;
      if (d == 0) {
        a.pm[p] = top;
        a.pl[p] = den;
      }
    }
  };
  if constexpr (SPLIT) {
    __shared__ float sm[kWaves][16], sl[kWaves][16];
    float(*const so)[16][Z::DP + 4] = reinterpret_cast<float(*)[16][Z::DP + 4]>(lds);
    if (lane < 16) {
      sm[w][n] = m;
      sl[w][n] = l;
    }
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) so[w][4 * j + r][Z::column(n, d)] = o[d][r];
    __syncthreads();
    const int live = min(16, rows - r0);
    for (int e = threadIdx.x; e < live * Z::DP; e += 64 * kWaves) {
      const int r = e / Z::DP, d = e % Z::DP;
      float top = sm[0][r];
#pragma unroll
      for (int y = 1; y < kWaves; ++y) top = fmaxf(top, sm[y][r]);
      const float ts = top == -INFINITY ? 0.f : top;
      float num = 0.f, den = 0.f;
#pragma unroll
      for (int y = 0; y < kWaves; ++y) {
        const float f = __builtin_amdgcn_exp2f(sm[y][r] - ts);
        num = __builtin_fmaf(so[y][r][d], f, num);
        den = __builtin_fmaf(sl[y][r], f, den);
      }
      put(r, d, num, den, top);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float den = __shfl(l, 4 * j + r, 64), top = __shfl(m, 4 * j + r, 64);
#pragma unroll
      for (int d = 0; d < NT; ++d) put(4 * j + r, Z::column(n, d), o[d][r], den, top);
    }
  }
}

// The slices' results of a row together, one thread a column; 4 us, a launch and
// two rounds of loads.
__global__ __launch_bounds__(128) void k_fp4_join(AttArgs a) {
  const int64_t row = blockIdx.x;  // (b Hkv + kh) group Tq + h Tq + t
  const int d = threadIdx.x;
  if (d >= a.D) return;
  const int64_t p = row * a.slices;
  float top = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < a.slices; ++s) top = fmaxf(top, a.pm[p + s]);
  const float ts = top == -INFINITY ? 0.f : top;
  float num = 0.f, den = 0.f;
#pragma unroll 8
  for (int s = 0; s < a.slices; ++s) {
    const float f = __builtin_amdgcn_exp2f(a.pm[p + s] - ts);
    den = __builtin_fmaf(a.pl[p + s], f, den);
    num = __builtin_fmaf(a.po[(p + s) * a.D + d], f, num);
  }
  const int64_t bh = row / a.Tq;
  const int t = (int)(row - bh * a.Tq);
  const int64_t b = bh / a.H, h = bh - b * a.H;
  const bool none = length_of(a, (int)b) - a.Tq + t < 0;
  a.o[b * a.ob + h * a.oh + t * a.ot + d] = none ? 0.f : num / den;
}

template <int NB>
void launch_attend(const AttArgs& a, bool split) {
  const dim3 block(64 * kWaves);
  const int groups = split ? a.row_tiles : (int)cdiv(a.row_tiles, kWaves);
  const dim3 grid((unsigned)(a.B * a.Hkv * a.slices * groups));
  if (split) tjh_launch((k_fp4_attend<NB, true>), grid, block, 0, stream(), a);
  else tjh_launch((k_fp4_attend<NB, false>), grid, block, 0, stream(), a);
}

}  // namespace
}  // namespace tjh

using namespace tjh;

extern "C" int tjh_fp4_attention(const float* q, const uint8_t* k_codes, const float* k_scales,
                                 const uint8_t* v_codes, const float* v_scales, float* o, int64_t B,
                                 int64_t H, int64_t Hkv, int64_t Tq, int64_t L, int64_t D,
                                 const int64_t* q_strides, const int64_t* o_strides,
                                 int64_t length, const int32_t* lengths, float scale) {
  TJH_REQUIRE_INIT();
  TJH_ARG(B >= 0 && H >= 0 && Hkv >= 0 && Tq >= 0 && L >= 0 && D > 0 && (H == 0) == (Hkv == 0) &&
              (Hkv == 0 || H % Hkv == 0),
          "tjh_fp4_attention: bad sizes");
  TJH_ARG(lengths || (length >= 0 && length <= L), "tjh_fp4_attention: length %lld of %lld",
          (long long)length, (long long)L);
  if (D > 128 || L >= (int64_t(1) << 24))
    return set_error(TJH_ERR_UNSUPPORTED,
                     "tjh_fp4_attention: head dim %lld, length %lld (128, 2^24 - 1 at most)",
                     (long long)D, (long long)L);
  if (B == 0 || H == 0 || Tq == 0) return TJH_OK;
  TJH_ARG(Tq < (int64_t(1) << 24) && B * H * Tq < (int64_t(1) << 30),
          "tjh_fp4_attention: too many queries");
  TJH_ARG(q && o && q_strides && o_strides &&
              (L == 0 || (k_codes && k_scales && v_codes && v_scales && aligned16(k_codes) &&
                          aligned16(v_codes))),
          "tjh_fp4_attention: NULL or unaligned pointer");
  AttArgs a{};
  a.q = q; a.kc = k_codes; a.vc = v_codes; a.ks = k_scales; a.vs = v_scales; a.o = o;
  a.lengths = lengths;
  a.qb = q_strides[0]; a.qh = q_strides[1]; a.qt = q_strides[2];
  a.ob = o_strides[0]; a.oh = o_strides[1]; a.ot = o_strides[2];
  a.L = L; a.length = length;
  a.B = (int)B; a.H = (int)H; a.Hkv = (int)Hkv; a.Tq = (int)Tq; a.D = (int)D;
  a.group = (int)(H / Hkv);
  a.scale = scale;
  const int64_t rows = a.group * Tq;
  a.row_tiles = (int)cdiv(rows, 16);
  // The waves of a workgroup share a row tile's keys where there are too few
  // tiles for a wave on every SIMD.  Then slices of the keys until the CUs have
  // two workgroups each, if there are more than 1024: joining them is a launch of
  // its own (12 heads of 64, 1000 keys: 10 us, in eight slices 11.6, in two 12).
  const int64_t keys = lengths ? L : length, tiles = B * Hkv * a.row_tiles;
  const bool split = tiles < 4 * num_cus();
  const int64_t wgs = split ? tiles : B * Hkv * cdiv(a.row_tiles, kWaves);
  const int64_t want = 2 * wgs >= 3 * num_cus() ? 1 : cdiv(2 * num_cus(), wgs);
  const int64_t can = keys > 1024 ? cdiv(keys, 512) : 1;
  a.slices = (int)(want < can ? want : can);
  if (a.slices < 1) a.slices = 1;
  KernelScope ks("fp4_attention");
  Scratch s(a.slices > 1 ? (size_t)(B * H * Tq * a.slices) * (D + 2) * sizeof(float) : 0);
  if (a.slices > 1) {
    if (!s.ok()) return set_error(TJH_ERR_OOM, "tjh_fp4_attention: no scratch");
    const int64_t n = B * H * Tq * a.slices;
    a.pm = s.as<float>();
    a.pl = a.pm + n;
    a.po = a.pl + n;
  }
  TJH_ARG(wgs * a.slices < (int64_t(1) << 23), "tjh_fp4_attention: too many queries");
  if (D <= 32) launch_attend<1>(a, split);
  else if (D <= 64) launch_attend<2>(a, split);
  else if (D <= 96) launch_attend<3>(a, split);
  else launch_attend<4>(a, split);
  int rc = check_launch("fp4_attend");
  if (rc != TJH_OK || a.slices == 1) return rc;
  tjh_launch(k_fp4_join, dim3((unsigned)(B * H * Tq)), dim3(128), 0, stream(), a);
  return check_launch("fp4_join");
}
