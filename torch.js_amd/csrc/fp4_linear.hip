// y = x W^T + bias for weights in 4 bits with a float scale for each 32, 64 or
// 128 columns (beside nn.Linear, src/nn/linear.ts:43-66).
//
//   y[m, n] = bias[n] + sum over groups g of scale[n, g] sum over k in g of
//             x[m, k] step[n, k]
//
// Products.  A step of 4 bits is a bfloat16 exactly, and a float x is the sum
// of three bfloat16 parts (its significand's bits by eights), so three products
// on the bf16 matrix cores form the float product of each group; the groups'
// sums are scaled and added up in floats.
#include "fp4.h"

namespace tjh {
namespace {

using namespace fp4;

struct LinArgs {
  const float* x;
  const uintx4* parts;  // x in fragments (k_split_rows), or NULL
  const uint8_t* codes;
  const float* scales;
  const float* bias;
  float* y;
  int64_t ldx, ldy, M, N, K;
  int nb;    // blocks of 128 columns
  int rows;  // of x a workgroup takes (grid y)
};

// Part `part` of eight floats.
__device__ __forceinline__ bf16x8 parts_of(const float (&x)[8], int part) {
  uintx4 v;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float r = rest(x[2 * q + i]);
      y[i] = part == 0 ? x[2 * q + i] : part == 1 ? r : r - cut(r);
    }
    v[q] = pack_high(y[0], y[1]);
  }
  return __builtin_bit_cast(bf16x8, v);
}

// x[k0, k0 + 8) of a row, 0 past K.
__device__ __forceinline__ void load8(const float* __restrict__ row, int64_t k0, int64_t K,
                                      float (&x)[8]) {
  if (k0 + 8 <= K) {
    const floatx4 a = *reinterpret_cast<const floatx4u*>(row + k0);
    const floatx4 b = *reinterpret_cast<const floatx4u*>(row + k0 + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = k0 + e < K ? row[k0 + e] : 0.f;
  }
}

// The parts of x's rows in the order in which the matrix cores take them: for
// each chunk of R rows, each 32 columns and each 16 of its 3 R (row, part)
// pairs, part by part, 64 lanes of 8 columns.
__global__ __launch_bounds__(256) void k_split_rows(const float* __restrict__ x, int64_t ldx,
                                                    int64_t M, int64_t K, int R, int MT,
                                                    int kb, int64_t items,
                                                    uintx4* __restrict__ parts) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= items) return;
  const int lane = at & 63;
  const int64_t f = at >> 6, chunk = f / ((int64_t)kb * MT);
  const int rest = (int)(f - chunk * kb * MT), k32 = rest / MT, tile = rest - k32 * MT;
  const int r = tile * 16 + (lane & 15), part = r / R;
  int64_t m = chunk * R + r - part * R;
  m = m < M ? m : M - 1;
  float v[8];
  load8(x + m * ldx, 32 * (int64_t)k32 + 8 * (lane >> 4), K, v);
  parts[at] = __builtin_bit_cast(uintx4, parts_of(v, part));
}

// The scales of a row's 128 columns, one for each 32.
template <int G>
__device__ __forceinline__ floatx4 scales_of(const float* __restrict__ s) {
  if (G == 32) return *reinterpret_cast<const floatx4u*>(s);
  if (G == 64) {
    const floatx2 v = *reinterpret_cast<const floatx2u*>(s);
    return floatx4{v.x, v.x, v.y, v.y};
  }
  return floatx4{*s, *s, *s, *s};
}

// Few rows of x.  A workgroup has 16 NT columns of y, its waves share the
// columns of x by blocks of 128 and add up through LDS.  A matrix tile's 16
// rows are (row, part) pairs: one tile holds five rows, MT of them 16 MT / 3.
template <int G, int MT, int NT, int WAVES, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES) void k_fp4_rows(LinArgs a) {
  __shared__ float red[WAVES][MT][16][16];
  const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * 16 * NT, m0 = (int64_t)blockIdx.y * a.rows;
  const int R = (int)(a.M - m0 < a.rows ? a.M - m0 : a.rows);
  const uint8_t* __restrict__ cp[NT];
  const float* __restrict__ sp[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = n0 + 16 * t + c < a.N ? n0 + 16 * t + c : a.N - 1;
    cp[t] = a.codes + n * a.nb * 64 + 16 * j;
    sp[t] = a.scales + n * a.nb * (128 / G);
  }
  // this lane's row of x and part of it
  const int part = SPLIT ? c / a.rows : 0;
  const float* __restrict__ xr = a.x;
  if (SPLIT) xr += (m0 + min(c - part * a.rows, R - 1)) * a.ldx;
  const uintx4* __restrict__ frag = a.parts + (int64_t)blockIdx.y * a.nb * 4 * MT * 64 + lane;
  floatx4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = floatx4{0.f, 0.f, 0.f, 0.f};
  for (int b = w; b < a.nb; b += WAVES) {
    uintx4 code[NT];
    floatx4 s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      code[t] = *reinterpret_cast<const uintx4*>(cp[t] + (int64_t)b * 64);
      s[t] = scales_of<G>(sp[t] + b * (128 / G));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      bf16x8 xa[MT];
      if (SPLIT) {
        float v[8];
        load8(xr, 128 * (int64_t)b + 32 * u + 8 * j, a.K, v);
        xa[0] = parts_of(v, part);
      } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
          xa[i] = __builtin_bit_cast(bf16x8, frag[((b * 4 + u) * MT + i) * 64]);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const bf16x8 wb = steps(code[t][u]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const floatx4 p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              xa[i], wb, floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][t][r] = __builtin_fmaf(s[t][u], p[r], acc[i][t][r]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t) __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[w][i][4 * j + r][c] = acc[i][t][r];
    __syncthreads();
    for (int o = threadIdx.x; o < R * 16; o += 64 * WAVES) {
      const int m = o >> 4, col = o & 15;
      const int64_t n = n0 + 16 * t + col;
      float v = 0.f;
#pragma unroll
      for (int p = 2; p >= 0; --p) {
        const int row = p * a.rows + m;
#pragma unroll
        for (int q = 0; q < WAVES; ++q) v += red[q][row >> 4][row & 15][col];
      }
      if (n < a.N) a.y[(m0 + m) * a.ldy + n] = a.bias ? v + a.bias[n] : v;
    }
  }
}

template <int G, int MT, int NT, bool SPLIT>
void launch_waves(const LinArgs& a, int chunks) {
  const dim3 grid((unsigned)cdiv(a.N, 16 * NT), (unsigned)chunks);
  if (a.nb <= 4)
    tjh_launch((k_fp4_rows<G, MT, NT, 4, SPLIT>), grid, dim3(256), 0, stream(), a);
  else
    tjh_launch((k_fp4_rows<G, MT, NT, 8, SPLIT>), grid, dim3(512), 0, stream(), a);
}

template <int G, int MT, bool SPLIT>
void launch_cols(const LinArgs& a, int chunks) {
  if (a.N * chunks >= 64LL * 2 * num_cus()) launch_waves<G, MT, 4, SPLIT>(a, chunks);
  else launch_waves<G, MT, 1, SPLIT>(a, chunks);
}

template <int G>
int launch_rows(LinArgs a) {
  if (a.M <= 5) {
    a.rows = 5;
    launch_cols<G, 1, true>(a, 1);
    return check_launch("fp4_rows");
  }
  const int chunks = (int)cdiv(a.M, 32);
  a.rows = (int)cdiv(a.M, chunks);
  const int MT = (int)cdiv(3 * a.rows, 16);
  const int64_t items = (int64_t)chunks * a.nb * 4 * MT * 64;
  TJH_ARG(chunks < 65536 && cdiv(items, 256) < (1 << 23), "tjh_fp4_linear: too many rows");
  Scratch s((size_t)(items ? items : 1) * 16);
  if (!s.ok()) return set_error(TJH_ERR_OOM, "tjh_fp4_linear: no scratch");
  // a last chunk of fewer rows has its parts as far apart as the others
  if (items)
    tjh_launch(k_split_rows, dim3((unsigned)cdiv(items, 256)), dim3(256), 0, stream(), a.x, a.ldx,
               a.M, a.K, a.rows, MT, a.nb * 4, items, s.as<uintx4>());
  a.parts = s.as<uintx4>();
  switch (MT) {
    case 2: launch_cols<G, 2, false>(a, chunks); break;
    case 3: launch_cols<G, 3, false>(a, chunks); break;
    case 4: launch_cols<G, 4, false>(a, chunks); break;
    case 5: launch_cols<G, 5, false>(a, chunks); break;
    default: launch_cols<G, 6, false>(a, chunks); break;
  }
  return check_launch("fp4_rows");
}

}  // namespace
}  // namespace tjh

using namespace tjh;

extern "C" int tjh_fp4_linear(const float* x, int64_t ldx, int64_t M, int64_t N, int64_t K,
                              const uint8_t* codes, const float* scales, int64_t group,
                              const float* bias, float* y, int64_t ldy) {
  TJH_REQUIRE_INIT();
  TJH_ARG(M >= 0 && N >= 0 && K >= 0 && M < (int64_t(1) << 31) && N < (int64_t(1) << 31) &&
              K < (int64_t(1) << 30) && ldx >= K && ldy >= N,
          "tjh_fp4_linear: bad sizes");
  TJH_ARG(group == 32 || group == 64 || group == 128,
          "tjh_fp4_linear: groups of %lld columns (32, 64 or 128)", (long long)group);
  if (M == 0 || N == 0) return TJH_OK;
  TJH_ARG(y && (K == 0 || (x && codes && scales && aligned16(codes))),
          "tjh_fp4_linear: NULL or unaligned pointer");
  LinArgs a{x, nullptr, codes, scales, bias, y, ldx, ldy, M, N, K, (int)cdiv(K, 128), 0};
  KernelScope ks("fp4_linear");
  if (group == 32) return launch_rows<32>(a);
  if (group == 64) return launch_rows<64>(a);
  return launch_rows<128>(a);
}
