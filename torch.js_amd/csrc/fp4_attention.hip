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
  int B, H, Hkv, Tq, D, P, group;
  int row_groups, slices;
  float scale;
};

__device__ __forceinline__ int length_of(const AttArgs& a, int b) {
  if (!a.lengths) return (int)a.length;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n > a.L ? (int)a.L : n;
}

// Few queries.  A row is one query of one of the heads that share a key head;
// a workgroup takes R rows of one key head and a slice of the keys.  LPK lanes
// have a key, 16 columns each; each lane group walks its own keys, U of them at
// a time, with sums of its own; the maxima are raised only when a score is
// 2^kSlack above them, so that sums are rescaled once or twice in a walk.
constexpr float kSlack = 10.f;
constexpr int kWaves = 4;

template <int LPK, int R, int U>
__global__ __launch_bounds__(64 * kWaves) void k_fp4_attend(AttArgs a) {
  constexpr int SPW = 64 / LPK, kSlots = SPW * kWaves, DP = 16 * LPK, PR = 4 * kWaves;
  __shared__ float sm[PR][R], sl[PR][R];
  __shared__ float so[PR][R][DP];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int part = lane % LPK, slot = w * SPW + lane / LPK;
  int id = blockIdx.x;
  const int rg = id % a.row_groups;
  id /= a.row_groups;
  const int slice = id % a.slices;
  const int bh = id / a.slices, b = bh / a.Hkv, kh = bh - b * a.Hkv;
  const int len = length_of(a, b);
  const int rows = a.group * a.Tq, r0 = rg * R;
  // keys that each row sees, and all of them together
  int seen[R], most = 0;
  float q[R][16];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = r0 + r < rows ? r0 + r : rows - 1;
    const int h = row / a.Tq, i = row - h * a.Tq;
    seen[r] = max(0, len - a.Tq + i + 1);
    most = max(most, seen[r]);
    const float* p = a.q + b * a.qb + (int64_t)(kh * a.group + h) * a.qh + i * a.qt + 16 * part;
#pragma unroll
    for (int d = 0; d < 16; ++d)
      q[r][d] = 16 * part + d < a.D ? p[d] * (a.scale * kLog2e) : 0.f;
  }
  // this slice's keys: equal runs of the sequence's own
  const int per = (most + a.slices - 1) / a.slices;
  const int from = min(most, slice * per), to = min(most, from + per);
  const int64_t base = (int64_t)bh * a.L;
  const uint8_t* __restrict__ kc = a.kc + base * a.P + 8 * part;
  const uint8_t* __restrict__ vc = a.vc + base * a.P + 8 * part;
  const float* __restrict__ ks = a.ks + base;
  const float* __restrict__ vs = a.vs + base;
  const bool held = 8 * part < a.P;
  float m[R], l[R], o[R][16];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int d = 0; d < 16; ++d) o[r][d] = 0.f;
  }
  for (int t0 = from + slot; __any(t0 < to); t0 += kSlots * U) {
    uintx2 kw[U], vw[U];
    float kscale[U], vscale[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = min(t0 + u * kSlots, to - 1);  // past the slice: its last key, not used
      kw[u] = held ? *reinterpret_cast<const uintx2*>(kc + (int64_t)t * a.P) : uintx2{0, 0};
      vw[u] = held ? *reinterpret_cast<const uintx2*>(vc + (int64_t)t * a.P) : uintx2{0, 0};
      kscale[u] = ks[t];
      vscale[u] = vs[t];
    }
    float s[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float k[16];
      unpack(kw[u].x, reinterpret_cast<float(&)[8]>(k[0]));
      unpack(kw[u].y, reinterpret_cast<float(&)[8]>(k[8]));
      const int t = t0 + u * kSlots;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float x = 0.f;
#pragma unroll
        for (int d = 0; d < 16; ++d) x = __builtin_fmaf(q[r][d], k[d], x);
        if (LPK > 1) x += dpp_f<kDppXor1>(x);
        if (LPK > 2) x += dpp_f<kDppXor2>(x);
        if (LPK > 4) x += dpp_f<0x141>(x);  // row_half_mirror: the other four of eight
        s[u][r] = t < to && t < seen[r] ? x * kscale[u] : -INFINITY;
      }
    }
    float ms[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = s[0][r];
#pragma unroll
      for (int u = 1; u < U; ++u) top = fmaxf(top, s[u][r]);
      if (__any(top > m[r] + kSlack)) {
        const float up = fmaxf(m[r], top);
        const float f = up == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - up);
        m[r] = up;
        l[r] *= f;
#pragma unroll
        for (int d = 0; d < 16; ++d) o[r][d] *= f;
      }
      ms[r] = m[r] == -INFINITY ? 0.f : m[r];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[16];
      unpack(vw[u].x, reinterpret_cast<float(&)[8]>(v[0]));
      unpack(vw[u].y, reinterpret_cast<float(&)[8]>(v[8]));
      const int t = t0 + u * kSlots;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool sees = t < to && t < seen[r];
        const float p = sees ? __builtin_amdgcn_exp2f(s[u][r] - ms[r]) : 0.f;
        const float pv = sees ? p * vscale[u] : 0.f;  // what is not seen may hold NaN
        l[r] += p;
#pragma unroll
        for (int d = 0; d < 16; ++d) o[r][d] = __builtin_fmaf(pv, v[d], o[r][d]);
      }
    }
  }
  // one sum of each 16 lanes, then of all of them
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float top = m[r];
    if (LPK <= 2) top = fmaxf(top, dpp_f<kDppXor2>(top));
    if (LPK <= 4) top = fmaxf(top, dpp_f<kDppRor4>(top));
    top = fmaxf(top, dpp_f<kDppRor8>(top));
    const float f = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - top);
    const auto join = [&](float x) {
      if (LPK <= 2) x += dpp_f<kDppXor2>(x);
      if (LPK <= 4) x += dpp_f<kDppRor4>(x);
      return x + dpp_f<kDppRor8>(x);
    };
    const float sum = join(l[r] * f);
    const int at = w * 4 + (lane >> 4);
    if ((lane & 15) == 0) {
      sm[at][r] = top;
      sl[at][r] = sum;
    }
#pragma unroll
    for (int d = 0; d < 16; ++d) {
      const float x = join(o[r][d] * f);
      if ((lane & 15) < LPK) so[at][r][16 * part + d] = x;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * DP; i += 64 * kWaves) {
    const int r = i / DP, d = i - r * DP;
    if (r0 + r >= rows || d >= a.D) continue;
    float top = -INFINITY;
    for (int s = 0; s < PR; ++s) top = fmaxf(top, sm[s][r]);
    const float ts = top == -INFINITY ? 0.f : top;
    float num = 0.f, den = 0.f;
    for (int s = 0; s < PR; ++s) {
      const float f = __builtin_amdgcn_exp2f(sm[s][r] - ts);
      den = __builtin_fmaf(sl[s][r], f, den);
      num = __builtin_fmaf(so[s][r][d], f, num);
    }
    const int h = (r0 + r) / a.Tq, t = r0 + r - h * a.Tq;
    if (a.slices == 1) {
      // no key seen: zeros
      a.o[b * a.ob + (int64_t)(kh * a.group + h) * a.oh + t * a.ot + d] = den == 0.f ? 0.f : num / den;
    } else {
      const int64_t to = ((int64_t)bh * rows + r0 + r) * a.slices + slice;
      a.po[to * a.D + d] = num;
      if (d == 0) {
        a.pm[to] = top;
        a.pl[to] = den;
      }
    }
  }
}

// The slices' results of a row together, one thread a column.
__global__ __launch_bounds__(128) void k_fp4_join(AttArgs a) {
  const int64_t row = blockIdx.x;  // (b Hkv + kh) group Tq + h Tq + t
  const int d = threadIdx.x;
  if (d >= a.D) return;
  const int64_t p = row * a.slices;
  float top = -INFINITY;
  for (int s = 0; s < a.slices; ++s) top = fmaxf(top, a.pm[p + s]);
  const float ts = top == -INFINITY ? 0.f : top;
  float num = 0.f, den = 0.f;
  for (int s = 0; s < a.slices; ++s) {
    const float f = __builtin_amdgcn_exp2f(a.pm[p + s] - ts);
    den = __builtin_fmaf(a.pl[p + s], f, den);
    num = __builtin_fmaf(a.po[(p + s) * a.D + d], f, num);
  }
  const int64_t bh = row / a.Tq;
  const int t = (int)(row - bh * a.Tq);
  const int64_t b = bh / a.H, h = bh - b * a.H;
  a.o[b * a.ob + h * a.oh + t * a.ot + d] = den == 0.f ? 0.f : num / den;
}

template <int LPK>
void launch_few(AttArgs& a, int R) {
  const dim3 grid((unsigned)(a.B * a.Hkv * a.slices * a.row_groups)), block(64 * kWaves);
  if (R == 1) tjh_launch((k_fp4_attend<LPK, 1, 4>), grid, block, 0, stream(), a);
  else if (R == 2) tjh_launch((k_fp4_attend<LPK, 2, 4>), grid, block, 0, stream(), a);
  else tjh_launch((k_fp4_attend<LPK, 4, 2>), grid, block, 0, stream(), a);
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
  a.P = fp4::row_bytes((int)D);
  a.group = (int)(H / Hkv);
  a.scale = scale;
  const int64_t rows = a.group * Tq;
  const int R = rows == 1 ? 1 : rows == 2 ? 2 : 4;
  a.row_groups = (int)cdiv(rows, R);
  // slices of the keys until the CUs have two workgroups each, none under 128 keys
  const int64_t keys = lengths ? L : length, wgs = B * Hkv * a.row_groups;
  const int64_t want = cdiv(2 * num_cus(), wgs), can = cdiv(keys, 128);
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
  if (D <= 32) launch_few<2>(a, R);
  else if (D <= 64) launch_few<4>(a, R);
  else launch_few<8>(a, R);
  int rc = check_launch("fp4_attend");
  if (rc != TJH_OK || a.slices == 1) return rc;
  tjh_launch(k_fp4_join, dim3((unsigned)(B * H * Tq)), dim3(128), 0, stream(), a);
  return check_launch("fp4_join");
}
