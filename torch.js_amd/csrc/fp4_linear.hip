// y = x W^T + bias for weights in 4 bits with a float scale for each 32, 64 or
// 128 columns (beside nn.Linear, src/nn/linear.ts:43-66).
//
//   y[m, n] = bias[n] + sum over groups g of scale[n, g] sum over k in g of
//             x[m, k] step[n, k]
//
// Products.  A step of 4 bits is a bfloat16 exactly, and a float x is the sum
// of three bfloat16 parts (its significand's bits by eights), so three products
// on the bf16 matrix cores form the float product of each group; the groups'
// sums are scaled and added up in floats.  An error of 7e-8 to 1.4e-7 against 64
// bits (2-norm), a fifth of a float matrix product's with the same weights.
//
// Three kernels, by the rows of x (product() below):
//   up to 5    k_fp4_rows    bound by reading the weights and by latency
//   some       k_fp4_some    by latency of a chain of steps, by forming x's parts
//   many       k_fp4_gemm    by the bf16 matrix cores
#include "fp4.h"
#include "ops_math.h"

namespace tjh {
namespace {

using namespace fp4;

struct LinArgs {
  const float* x;
  const uintx4* parts;  // x's parts in fragments, or NULL
  const uint8_t* codes;
  const float* scales;
  const float* bias;
  const float* residual;
  float* y;
  int64_t ldx, ldy, ldr, M, N, K;
  int nb;       // blocks of 128 columns
  int m_tiles;  // 16 rows each, of `parts`
  int act;      // 1: GELU, 3: plus residual
  float* sums;  // [slices, M, N] of k_fp4_some, or NULL
  int per;      // blocks of a slice
};

// The end of an element of y.
__device__ __forceinline__ void finish(const LinArgs& a, int64_t m, int64_t n, float v) {
  if (a.bias) v += a.bias[n];
  if (a.act == 1) v = gelu_f(v);
  else if (a.act == 3) v = a.residual[m * a.ldr + n] + v;
  a.y[m * a.ldy + n] = v;
}

constexpr int kWaves = 8;

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

// ----------------------------------------------------------------- few rows

// Up to five rows of x: a matrix operand's 16 rows are (part, row) pairs.  A
// workgroup's eight waves have 8 / KS tiles of 16 columns of y; KS of them share
// a tile's columns of x by blocks of 128 and add up through LDS.  x's parts for KB
// = KS U blocks at a time are split into LDS; the codes of the next U blocks of a
// wave are loaded before.  One launch: the parts of five rows cost a workgroup a
// few hundred instructions, a kernel for them 3 us.
//
// Bound by reading the weights once, and by a chain of loads, split, barrier and
// products for each KB blocks.  One row, 2304 x 768: 4.0 us (0.2 at the rate of a
// copy).  Four rows: 50257 x 768 in groups of 32, 24.9 MB: 9.4 us, 2.6 TB/s;
// 65536 x 1024: 12.5 us, 3.4 TB/s; 16384 x 4096: 17.3 us, 2.1 TB/s.  Loading the
// next blocks' x ahead too gained 10% at 65536 x 1024 and lost 20% at 11000 x
// 4000 (a quarter fewer waves fit).
template <int G, int KS, int U>
__global__ __launch_bounds__(64 * kWaves) void k_fp4_rows(LinArgs a) {
  constexpr int KB = KS * U, kParts = KB * 4 * 64;
  constexpr int kRed = kWaves * 64;  // 16-byte items of the sums
  __shared__ uintx4 lds[kParts > kRed ? kParts : kRed];
  const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ks = w % KS;
  const int R = (int)a.M;
  const int64_t n0 = ((int64_t)blockIdx.x * (kWaves / KS) + w / KS) * 16;
  const int64_t n = n0 + c < a.N ? n0 + c : a.N - 1;
  const uint8_t* __restrict__ cp = a.codes + n * a.nb * 64 + 16 * j;
  const float* __restrict__ sp = a.scales + n * a.nb * (128 / G);
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  uintx4 code[U], next[U];
  floatx4 s[U], snext[U];
  const auto load = [&](int b0, uintx4 (&cd)[U], floatx4 (&sc)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b0 + u * KS + ks;
      if (b < a.nb) {
        cd[u] = *reinterpret_cast<const uintx4*>(cp + (int64_t)b * 64);
        sc[u] = scales_of<G>(sp + b * (128 / G));
      }
    }
  };
  load(0, next, snext);
  for (int b0 = 0; b0 < a.nb; b0 += KB) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      code[u] = next[u];
      s[u] = snext[u];
    }
    if (b0 + KB < a.nb) load(b0 + KB, next, snext);
    if (b0) __syncthreads();
    const int k32s = 4 * (KB < a.nb - b0 ? KB : a.nb - b0);
    // 16 octets of columns of a row a time, which lie in one line
    for (int i = threadIdx.x; i < k32s * 4 * R; i += 64 * kWaves) {
      const int o = i & 15, r = (i >> 4) % R, k = ((i >> 4) / R) * 16 + o;  // octet
      float v[8];
      load8(a.x + r * a.ldx, 128 * (int64_t)b0 + 8 * k, a.K, v);
      bf16x8 p[3];
      split8(v, p);
#pragma unroll
      for (int q = 0; q < 3; ++q)
        lds[(k >> 2) * 64 + 16 * (k & 3) + q * R + r] = __builtin_bit_cast(uintx4, p[q]);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = u * KS + ks;
      if (b0 + at >= a.nb) break;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const floatx4 p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, lds[(at * 4 + t) * 64 + lane]), steps(code[u][t]),
            floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(s[u][t], p[r], acc[r]);
      }
    }
  }
  __syncthreads();
  float* red = reinterpret_cast<float*>(lds);  // [wave][pair][column]
#pragma unroll
  for (int r = 0; r < 4; ++r) red[(w * 16 + 4 * j + r) * 16 + c] = acc[r];
  __syncthreads();
  for (int o = threadIdx.x; o < R * (kWaves / KS) * 16; o += 64 * kWaves) {
    const int col = o & 15, tile = (o >> 4) % (kWaves / KS), m = (o >> 4) / (kWaves / KS);
    const int64_t at = ((int64_t)blockIdx.x * (kWaves / KS) + tile) * 16 + col;
    if (at >= a.N) continue;
    float v = 0.f;
#pragma unroll
    for (int p = 2; p >= 0; --p)
#pragma unroll
      for (int q = 0; q < KS; ++q) v += red[((tile * KS + q) * 16 + p * R + m) * 16 + col];
    finish(a, m, at, v);
  }
}

template <int G, int KS>
void launch_rows(const LinArgs& a) {
  constexpr int U = 16 / KS > 4 ? 4 : 16 / KS;  // 64 KB of parts at most
  tjh_launch((k_fp4_rows<G, KS, U>), dim3((unsigned)cdiv(a.N, 16 * (kWaves / KS))),
             dim3(64 * kWaves), 0, stream(), a);
}

template <int G>
int few_rows(const LinArgs& a) {
  // waves share a tile's columns of x until the CUs have a workgroup each
  const int64_t tiles = cdiv(a.N, 16);
  if (a.nb >= 8 && tiles < 2 * num_cus()) launch_rows<G, 8>(a);
  else if (a.nb >= 4 && tiles < 4 * num_cus()) launch_rows<G, 4>(a);
  else if (a.nb >= 2 && tiles < 8 * num_cus()) launch_rows<G, 2>(a);
  else launch_rows<G, 1>(a);
  return check_launch("fp4_rows");
}

// ---------------------------------------------------------------- some rows

// Parts of x for k_fp4_some and k_fp4_gemm: for each 32 columns, each 16 rows and
// each part a matrix operand.
__global__ __launch_bounds__(256) void k_fp4_split(const float* __restrict__ x, int64_t ldx,
                                                   int64_t M, int64_t K, uint32_t m_tiles,
                                                   uint32_t items, uintx4* __restrict__ parts) {
  const uint32_t at = blockIdx.x * 256 + threadIdx.x;
  if (at >= items) return;
  const int lane = at & 63;
  const uint32_t fu = at >> 6;
  const int64_t f = fu, k32 = fu / m_tiles, m = (fu % m_tiles) * 16 + (lane & 15);
  float v[8];
  load8(x + (m < M ? m : M - 1) * ldx, 32 * k32 + 8 * (lane >> 4), K, v);
  bf16x8 p[3];
  split8(v, p);
#pragma unroll
  for (int i = 0; i < 3; ++i) parts[(f * 3 + i) * 64 + lane] = __builtin_bit_cast(uintx4, p[i]);
}

// A wave has RT times 16 rows and NT times 16 columns of y; the eight waves of a
// workgroup share the columns of x (a slice's of them, grid z) by blocks of 128 and
// add up through LDS.  x comes from memory as lanes feed it, a step of 32 columns
// ahead, codes a block ahead; PARTS: cut into its parts by a launch before, else by
// every wave for itself, which takes 60 instructions for each 16 rows of a step.
//
// Bound by the latency of a wave's steps while the workgroups fit the CUs, and by
// those instructions; by loading the parts (3 KB for 3 NT products) where there are
// more.  8, 32 and 64 rows: 2304 x 768 4.0, 4.8 and 6.3 us, 4096 x 4096 10.6, 14.7
// and 19, 16384 x 4096 18, 23 and 33, 50257 x 768 14, 24 and 39 us.
template <int G, int RT, int NT, bool PARTS>
__global__ __launch_bounds__(64 * kWaves, 2) void k_fp4_some(LinArgs a) {
  constexpr int CT = RT * NT <= 8 ? NT : 8 / RT;  // column tiles that are added up at a time
  __shared__ float red[kWaves][RT * 16][CT * 16 + 4];
  const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m0 = (int64_t)blockIdx.y * (16 * RT), n0 = (int64_t)blockIdx.x * 16 * NT;
  const int R = (int)(a.M - m0 < 16 * RT ? a.M - m0 : 16 * RT);
  const uint8_t* __restrict__ cp[NT];
  const float* __restrict__ sp[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = n0 + 16 * t + c < a.N ? n0 + 16 * t + c : a.N - 1;
    cp[t] = a.codes + n * a.nb * 64 + 16 * j;
    sp[t] = a.scales + n * a.nb * (128 / G);
  }
  const float* __restrict__ xp[RT];
  const uintx4* __restrict__ pp[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int64_t m = m0 + 16 * i + c, tile = m0 / 16 + i;
    xp[i] = a.x + (m < a.M ? m : a.M - 1) * a.ldx + 8 * j;
    pp[i] = a.parts + (tile < a.m_tiles ? tile : a.m_tiles - 1) * 192 + lane;
  }
  floatx4 acc[RT][NT], s[NT], snext[NT];
  uintx4 code[NT], cnext[NT], pn[RT][3];
  float xn[RT][8];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = floatx4{0.f, 0.f, 0.f, 0.f};
  const auto load_w = [&](int b) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      cnext[t] = *reinterpret_cast<const uintx4*>(cp[t] + (int64_t)b * 64);
      snext[t] = scales_of<G>(sp[t] + b * (128 / G));
    }
  };
  const auto load_x = [&](int k32) {
    const int64_t k0 = 32 * (int64_t)k32;
    if (PARTS) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int q = 0; q < 3; ++q) pn[i][q] = pp[i][(int64_t)k32 * a.m_tiles * 192 + q * 64];
    } else if (k0 + 32 <= a.K) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const floatx4 p = *reinterpret_cast<const floatx4u*>(xp[i] + k0);
        const floatx4 q = *reinterpret_cast<const floatx4u*>(xp[i] + k0 + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          xn[i][e] = p[e];
          xn[i][4 + e] = q[e];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) xn[i][e] = k0 + 8 * j + e < a.K ? xp[i][k0 + e] : 0.f;
    }
  };
  const int first = blockIdx.z * a.per, end = min(first + a.per, a.nb);
  if (first + w < end) {
    load_w(first + w);
    load_x(4 * (first + w));
  }
  for (int b = first + w; b < end; b += kWaves) {
    const int bn = b + kWaves < end ? b + kWaves : b;  // the last block is loaded twice
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      code[t] = cnext[t];
      s[t] = snext[t];
    }
    load_w(bn);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      bf16x8 x[RT][3];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        if (PARTS) {
#pragma unroll
          for (int q = 0; q < 3; ++q) x[i][q] = __builtin_bit_cast(bf16x8, pn[i][q]);
        } else {
          split8(xn[i], x[i]);
        }
      }
      load_x(u < 3 ? 4 * b + u + 1 : 4 * bn);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const bf16x8 wb = steps(code[t][u]);
        floatx4 p[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) p[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 2; q >= 0; --q)
#pragma unroll
          for (int i = 0; i < RT; ++i)
            p[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i][q], wb, p[i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[i][t][r] = __builtin_fmaf(s[t][u], p[i][r], acc[i][t][r]);
      }
    }
  }
#pragma unroll
  for (int t0 = 0; t0 < NT; t0 += CT) {
    if (t0) __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[w][16 * i + 4 * j + r][16 * t + c] = acc[i][t0 + t][r];
    __syncthreads();
    for (int o = threadIdx.x; o < R * CT * 16; o += 64 * kWaves) {
      const int m = o / (CT * 16), col = o % (CT * 16);
      const int64_t n = n0 + 16 * t0 + col;
      if (n >= a.N) continue;
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < kWaves; ++q) v += red[q][m][col];
      if (a.sums) a.sums[(blockIdx.z * a.M + m0 + m) * a.N + n] = v;
      else finish(a, m0 + m, n, v);
    }
  }
}

// The slices' sums together, always in one order.
__global__ __launch_bounds__(256) void k_fp4_sums(LinArgs a, int slices) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;
  if (n >= a.N) return;
  float v = 0.f;
#pragma unroll 4
  for (int i = 0; i < slices; ++i) v += a.sums[(i * a.M + m) * a.N + n];
  finish(a, m, n, v);
}

// How k_fp4_some takes some rows, and what that costs: 20 for a round of
// workgroups of 16 x 16 of y and eight blocks of columns (1.7 us).  Wider tiles
// cost less than their products, but fewer workgroups leave CUs idle:
// 4096 x 4096, 8 rows by 16 columns 10.6 us, by 32 12.1; 6400 x 1600 8.7 and 6.6.
struct Some {
  int rt, nt;
  int64_t slices, cost;
  bool parts;
};
Some plan_some(const LinArgs& a) {
  const struct {
    int rt, nt, cost;
  } tiles[] = {{1, 1, 20}, {1, 2, 25}, {1, 4, 40}, {2, 4, 54}, {4, 4, 84}};
  const int64_t cus = num_cus(), blocks = cdiv(a.nb, kWaves);
  Some best{4, 4, 1, INT64_MAX, true};
  for (const auto& t : tiles) {
    const int64_t wgs = cdiv(a.M, 16 * t.rt) * cdiv(a.N, 16 * t.nt);
    if (t.nt < 4 && wgs > cus) continue;
    // cut by a launch before (4 us) where that is done often: 4096 x 4096, 96 rows
    // 22.4 us (28 without); 2304 x 768, 8 rows 7 (4.0)
    const bool parts = t.rt > 1 || wgs > cus;
    for (int64_t n = 1; n <= 4 && n <= blocks && (n == 1 || wgs * n <= cus); n *= 2) {
      // adding slices up is a launch: 1000 x 8000, 8 rows 10.5 us by four and 14 by
      // one; 4096 x 4096 12.7 and 10.6
      const int64_t cost = cdiv(wgs * n, cus) * cdiv(blocks, n) * t.cost + (n > 1 ? 60 : 0) +
                           (parts ? 50 : 0);
      if (cost < best.cost) best = {t.rt, t.nt, n, cost, parts};
    }
  }
  return best;
}

template <int G>
int some_rows(LinArgs a, const Some& plan) {
  a.m_tiles = (int)cdiv(a.M, 16);
  a.per = (int)(cdiv(cdiv(a.nb, kWaves), plan.slices) * kWaves);
  const int slices = a.nb ? (int)cdiv(a.nb, a.per) : 1;
  const dim3 grid((unsigned)cdiv(a.N, 16 * plan.nt), (unsigned)cdiv(a.M, 16 * plan.rt),
                  (unsigned)slices);
  const dim3 block(64 * kWaves);
  const int64_t items = plan.parts ? (int64_t)a.m_tiles * a.nb * 4 * 64 : 0;
  const int64_t sums = slices > 1 ? slices * a.M * a.N : 0;
  TJH_ARG(cdiv(a.M, 16 * plan.rt) < 65536 && cdiv(items, 256) < (1 << 23) &&
              (int64_t)grid.x * grid.y < (1 << 23),
          "tjh_fp4_linear: too many rows");
  Scratch s((size_t)items * 48 + (size_t)sums * 4);
  if (items || sums) {
    if (!s.ok()) return set_error(TJH_ERR_OOM, "tjh_fp4_linear: no scratch");
    a.parts = s.as<uintx4>();
    if (sums) a.sums = s.as<float>() + items * 12;
  }
  if (items)
    tjh_launch(k_fp4_split, dim3((unsigned)cdiv(items, 256)), dim3(256), 0, stream(), a.x, a.ldx,
               a.M, a.K, (uint32_t)a.m_tiles, (uint32_t)items, s.as<uintx4>());
  if (plan.rt == 4) tjh_launch((k_fp4_some<G, 4, 4, true>), grid, block, 0, stream(), a);
  else if (plan.rt == 2) tjh_launch((k_fp4_some<G, 2, 4, true>), grid, block, 0, stream(), a);
  else if (plan.parts) tjh_launch((k_fp4_some<G, 1, 4, true>), grid, block, 0, stream(), a);
  else if (plan.nt == 4) tjh_launch((k_fp4_some<G, 1, 4, false>), grid, block, 0, stream(), a);
  else if (plan.nt == 2) tjh_launch((k_fp4_some<G, 1, 2, false>), grid, block, 0, stream(), a);
  else tjh_launch((k_fp4_some<G, 1, 1, false>), grid, block, 0, stream(), a);
  if (sums)
    tjh_launch(k_fp4_sums, dim3((unsigned)cdiv(a.N, 256), (unsigned)a.M), dim3(256), 0, stream(), a,
               slices);
  return check_launch("fp4_some");
}

// ---------------------------------------------------------------- many rows

// 128 x 16 C of y a workgroup, 32 rows of it a wave.  A wave's parts of x come straight
// from memory as its lanes feed them, one step of 32 columns ahead; codes and
// scales, which all four waves feed, go through one of two LDS buffers, 128
// columns at a time and loaded as many ahead.
//
// Bound by the matrix cores' power: 2047 x 1600 x 6400 takes 112 us, 1.17 PFLOP/s
// of bfloat16 products or 375 TFLOP/s of float ones, at 1.9 to 2 GHz with the
// matrix cores of a working CU busy 62% of the time; a plain bfloat16 product of
// 8192^3 by the library reaches 1.13 PFLOP/s.  Without its loads, its conversions,
// or half of its sums the kernel takes as long.  13 us of it are the writing of y
// by all workgroups at the end of their one round.  64 x 64 a wave with x through
// LDS: 156 us; products and sums of one column tile one after the other: 138.
constexpr int kGemmWaves = 4, kRowTiles = 2;

// ACT: with an epilogue (104 GELUs in line cost every call 14 us of 111).
template <int G, int C, bool ACT>
__global__ __launch_bounds__(64 * kGemmWaves, 2) void k_fp4_gemm(LinArgs a) {
  constexpr int T = 64 * kGemmWaves, kBM = 16 * kRowTiles * kGemmWaves, kBN = 16 * C;
  constexpr int kItems = (C + kGemmWaves - 1) / kGemmWaves;  // column tiles a wave loads
  __shared__ uint32_t lw[2][4][C * 64];
  __shared__ float ls[2][4][kBN];
  const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // each XCD has a run of tiles: row blocks, in each all column blocks
  const int nt = (int)((a.N + kBN - 1) / kBN), total = nt * (a.m_tiles * 16 / kBM);
  const int per = (total + 7) / 8, t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (t >= total) return;
  const int mb = t / nt, cb = t - mb * nt;
  const int64_t n0 = (int64_t)cb * kBN;
  const uint8_t* __restrict__ cp[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    // (the last one again where there are fewer)
    const int64_t n = n0 + 16 * min(w + kGemmWaves * i, C - 1) + c;
    cp[i] = a.codes + (n < a.N ? n : a.N - 1) * a.nb * 64 + 16 * j;
  }
  const int64_t ns = n0 + threadIdx.x % kBN;
  const float* __restrict__ sp = a.scales + (ns < a.N ? ns : a.N - 1) * a.nb * (128 / G);
  const int64_t hop = (int64_t)a.m_tiles * 3 * 64;  // to the next 32 columns
  const uintx4* __restrict__ from =
      a.parts + (int64_t)(mb * (kBM / 16) + w * kRowTiles) * 3 * 64 + lane;
  floatx4 acc[kRowTiles][C];
#pragma unroll
  for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
    for (int n = 0; n < C; ++n) acc[i][n] = floatx4{0.f, 0.f, 0.f, 0.f};
  uintx4 code[kItems], xr[kRowTiles][3];
  floatx4 sc;
  const auto load_w = [&](int b) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) code[i] = *reinterpret_cast<const uintx4*>(cp[i] + (int64_t)b * 64);
    sc = scales_of<G>(sp + b * (128 / G));
  };
  // no branches in the loop: the last step and block are loaded twice (with
  // branches the compiler moves products past them and spills)
  int left = 4 * a.nb;
  const auto load_x = [&] {
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
      for (int p = 0; p < 3; ++p) xr[i][p] = from[(i * 3 + p) * 64];
    --left;
    from += left > 0 ? hop : 0;
  };
  load_w(0);
  load_x();
  for (int b = 0; b < a.nb; ++b) {
    const int to = b & 1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int i = 0; i < kItems; ++i)
        lw[to][u][min(w + kGemmWaves * i, C - 1) * 64 + lane] = code[i][u];
      ls[to][u][threadIdx.x % kBN] = sc[u];
    }
    load_w(b + 1 < a.nb ? b + 1 : b);
    __syncthreads();
    // The products of a column tile are issued between the sums of the one
    // before and the conversions of the one after: a wave alone keeps its
    // matrix cores busy.
    bf16x8 xa[kRowTiles][3], wb = steps(lw[to][0][lane]);
    float f = ls[to][0][c], fnext = ls[to][0][16 + c], fy = 0.f;
    uint32_t word = lw[to][0][64 + lane];
    floatx4 y[kRowTiles];
#pragma unroll
    for (int q = 0; q < 4 * C; ++q) {
      const int u = q / C, n = q % C;
      if (n == 0) {
#pragma unroll
        for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
          for (int p = 0; p < 3; ++p) xa[i][p] = __builtin_bit_cast(bf16x8, xr[i][p]);
        load_x();
      }
      floatx4 z[kRowTiles];
#pragma unroll
      for (int i = 0; i < kRowTiles; ++i) z[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < kRowTiles; ++i)
          z[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xa[i][p], wb, z[i], 0, 0, 0);
      const float fz = f;
      if (q + 1 < 4 * C) {
        wb = steps(word);
        f = fnext;
        if (q + 2 < 4 * C) {
          word = lw[to][(q + 2) / C][(q + 2) % C * 64 + lane];
          fnext = ls[to][(q + 2) / C][(q + 2) % C * 16 + c];
        }
      }
      if (q > 0) {
        const int before = (n + C - 1) % C;
#pragma unroll
        for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[i][before][r] = __builtin_fmaf(fy, y[i][r], acc[i][before][r]);
      }
      fy = fz;
#pragma unroll
      for (int i = 0; i < kRowTiles; ++i) y[i] = z[i];
#pragma unroll
      for (int i = 0; i < 3 * kRowTiles; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product,
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);  // two of the other operations
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[i][C - 1][r] = __builtin_fmaf(fy, y[i][r], acc[i][C - 1][r]);
  }
#pragma unroll
  for (int n = 0; n < C; ++n) {
    const int64_t at = n0 + n * 16 + c;
    if (at >= a.N) continue;
    const float bias = a.bias ? a.bias[at] : 0.f;
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t m = (int64_t)mb * kBM + (w * kRowTiles + i) * 16 + 4 * j + r;
        if (m >= a.M) continue;
        if (ACT) finish(a, m, at, acc[i][n][r]);
        else a.y[m * a.ldy + at] = acc[i][n][r] + bias;
      }
  }
}

template <int G, int C>
void launch_gemm(const LinArgs& a) {
  const int64_t tiles = cdiv(a.N, 16 * C) * (a.m_tiles / 8);
  const dim3 grid((unsigned)(cdiv(tiles, 8) * 8)), block(64 * kGemmWaves);
  if (a.act) tjh_launch((k_fp4_gemm<G, C, true>), grid, block, 0, stream(), a);
  else tjh_launch((k_fp4_gemm<G, C, false>), grid, block, 0, stream(), a);
}

// Column tiles of a workgroup of k_fp4_gemm, and what that costs, as for
// k_fp4_some: by the column tiles of the CU that has most.  2047 x 1600 x 6400 139 us
// by 4 or 8, 121 by 13; 2600 x 1600 x 4800 138 and 121; 2600 x 6400 x 1600 231 and 218;
// but 2047 x 768 x 2304 40 by 4 and 47 by 13, which is taken.  Over 70 sizes of 300 to
// 4096 rows 13 saves 0.1% beside 4 and 8 alone; the best of 4, 8 and 10 to 13 for each
// size would save 3.6%.
struct Gemm {
  int C;
  int64_t cost;
};
Gemm plan_gemm(const LinArgs& a) {
  const int64_t rows = cdiv(a.M, 128);
  const auto load = [&](int C) { return cdiv(cdiv(a.N, 16 * C) * rows, num_cus()) * C; };
  const int64_t l4 = load(4) * 5 / 4, l8 = load(8), l13 = load(13);
  const auto plan = [&](int C, int64_t l) { return Gemm{C, l * a.nb * 7 / 2 + 150}; };
  if (l13 <= l8 && l13 <= l4) return plan(13, l13);
  return l8 <= l4 ? plan(8, l8) : plan(4, load(4) * 3 / 2);
}

template <int G>
int many_rows(LinArgs a) {
  // a GB of parts at a time: long prompts in pieces of rows
  const int64_t piece = ((int64_t(1) << 30) / (a.nb * 128 * 6) / 128 + 1) * 128;
  if (a.M > piece) {
    LinArgs b = a;
    for (int64_t m = 0; m < a.M; m += piece) {
      b.M = a.M - m < piece ? a.M - m : piece;
      b.x = a.x + m * a.ldx;
      b.y = a.y + m * a.ldy;
      if (a.residual) b.residual = a.residual + m * a.ldr;
      const int rc = many_rows<G>(b);
      if (rc != TJH_OK) return rc;
    }
    return TJH_OK;
  }
  a.m_tiles = (int)cdiv(a.M, 128) * 8;
  const int64_t items = (int64_t)a.m_tiles * a.nb * 4 * 64, rows = a.m_tiles / 8;
  TJH_ARG(cdiv(items, 256) < (1 << 23) && cdiv(a.N, 64) * rows < (1 << 23),
          "tjh_fp4_linear: too many rows");
  Scratch s((size_t)items * 3 * 16);
  if (!s.ok()) return set_error(TJH_ERR_OOM, "tjh_fp4_linear: no scratch");
  tjh_launch(k_fp4_split, dim3((unsigned)cdiv(items, 256)), dim3(256), 0, stream(), a.x, a.ldx, a.M,
             a.K, (uint32_t)a.m_tiles, (uint32_t)items, s.as<uintx4>());
  a.parts = s.as<uintx4>();
  const int C = plan_gemm(a).C;
  if (C == 13) launch_gemm<G, 13>(a);
  else if (C == 8) launch_gemm<G, 8>(a);
  else launch_gemm<G, 4>(a);
  return check_launch("fp4_gemm");
}

template <int G>
int product(const LinArgs& a) {
  const Some plan = plan_some(a);
  // few rows of many columns take k_fp4_rows a barrier and a split for each 16
  // blocks: 1000 x 8000, 2 rows 10.7 us (11.1 by slices), 4 rows 13.5 (10.9); 1000 x
  // 16000, one row 15.5 (13.7)
  if (a.M <= 5 && (plan.slices == 1 || (a.M + 1) * a.nb < 250)) return few_rows<G>(a);
  // 50257 x 768, 64 rows 38 us by k_fp4_some and 41 by k_fp4_gemm, 96 rows 51 and 42;
  // 4096 x 4096, 512 rows 62 and 66, 1024 117 and 95.  Over 210 sizes what is taken
  // is 12% slower than the other at most.
  const int64_t parts = plan.parts ? a.M * a.nb * 128 * 6 : 0;  // bytes
  if (a.nb && (parts > (int64_t(1) << 30) || plan_gemm(a).cost < plan.cost)) return many_rows<G>(a);
  return some_rows<G>(a, plan);
}

}  // namespace

int fp4_linear(const float* x, int64_t ldx, int64_t M, int64_t N, int64_t K, const uint8_t* codes,
               const float* scales, int64_t group, const float* bias, float* y, int64_t ldy,
               const float* residual, int64_t ldr, int act) {
  TJH_ARG(M >= 0 && N >= 0 && K >= 0 && M < (int64_t(1) << 31) && N < (int64_t(1) << 26) &&
              K < (int64_t(1) << 26) && ldx >= K && ldy >= N,
          "tjh_fp4_linear: bad sizes");
  TJH_ARG(group == 32 || group == 64 || group == 128,
          "tjh_fp4_linear: groups of %lld columns (32, 64 or 128)", (long long)group);
  if (M == 0 || N == 0) return TJH_OK;
  TJH_ARG(y && (K == 0 || (x && codes && scales && aligned16(codes))),
          "tjh_fp4_linear: NULL or unaligned pointer");
  LinArgs a{x,   nullptr, codes, scales, bias, residual, y, ldx, ldy, ldr, M, N, K,
            (int)cdiv(K, 128), 0, act, nullptr, 0};
  KernelScope ks("fp4_linear");
  if (group == 32) return product<32>(a);
  if (group == 64) return product<64>(a);
  return product<128>(a);
}

}  // namespace tjh

extern "C" int tjh_fp4_linear(const float* x, int64_t ldx, int64_t M, int64_t N, int64_t K,
                              const uint8_t* codes, const float* scales, int64_t group,
                              const float* bias, float* y, int64_t ldy) {
  TJH_REQUIRE_INIT();
  return tjh::fp4_linear(x, ldx, M, N, K, codes, scales, group, bias, y, ldy, nullptr, 0, 0);
}
