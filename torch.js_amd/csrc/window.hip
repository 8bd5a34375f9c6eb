// Causal attention over a sliding window with sinks
// (F.sliding_window_attention, beside the full attention of flash.hip behind
// src/nn/functional.ts:866-890): the query at position i = Tk - Tq + t sees
// the keys j <= i with j > i - window or j < sinks, H query heads share Hkv
// heads of keys and values, and time and memory grow with the keys seen.
//
// Layouts and products are flash.hip's (flash_tile.h).  Forward and dQ: a wave
// has 32 queries, its operands straight from memory, and walks the tiles of
// keys that those see: the ones that hold sinks, then the window's.  It masks
// only the tiles that it sees in part.  dK and dV: a key-block kernel walks
// the query heads that share its keys and their query tiles, accumulating dV
// and dK and storing each 32x32 block of dS in a band of `nsl` slots a query
// tile (sink tiles, then window tiles); the query kernel turns those into dQ,
// so S and dP are formed once.  The key blocks with sinks are seen by every
// later query: their steps are cut into slices, whose sums a last kernel adds
// in order.  Deterministic, no atomics.
//
// Keys that a query does not see may hold anything, infinities and NaN
// included: their scores are replaced, never multiplied, and where a tile
// that is seen in part holds such values of V (or of K, for dQ) they are kept
// out of the products, in which 0 times them would be NaN.
//
// Bound by the fp32 matrix cores: 4 D operations forward and 10 D backward
// for each key that a query sees, 8 floats moved a head and position.
#include "flash_tile.h"

#include <math.h>

namespace tjh {
namespace {

struct WinArgs {
  const float *q, *k, *v, *o, *dout, *lse, *dsum;
  float *out, *out2, *lse_out;
  Strides3 qs, ks, vs, os, gs, o1s, o2s;
  int H, G;            // query heads, query heads to one of keys and values
  int Tq, Tk, off;     // off = Tk - Tq: the first query's position
  int D;
  float scale;
  int win, sinks, nst; // nst: key tiles that hold sinks
  int nblk;            // row blocks of a head
  // forward in slices of `kslice` key tiles: part
  // [slice][b*H + h][Tq][D] unscaled sums, pml {maximum, sum}
  float* part;
  float2* pml;
  int kslice;
  // backward: dS blocks [bh - bh0][query tile][nsl], of the key heads from
  // bkv0 on
  float* dsblk;
  int nqt, nkt, nsl;
  int bkv0, nbkv;
  // slices of the steps of the nsb key blocks with sinks and of the others;
  // sums [slice][bkv - bkv0][keys of those blocks][D] of dK, then dV, of each
  int nsb, nslice, nsplit;
  float* sums;
};

constexpr int PROWS = 64;  // keys of a workgroup of the key-block kernel

// Workgroups go round the XCDs: neighbours in `i` are on one XCD, where they
// find the keys and values that they share in its L2.
__device__ __forceinline__ int xcd_item(int id, int n) {
  const int per = n / kXcds, rem = n % kXcds, x = id % kXcds, j = id / kXcds;
  return x * per + min(x, rem) + j;
}

// The key tiles that queries at positions [lo, hi] see: i -> tile.
struct Tiles {
  int ns, w0, n;  // sink tiles, the window's first tile, all
  __device__ __forceinline__ Tiles(const WinArgs& a, int lo, int hi) {
    w0 = max(0, lo - a.win + 1) / TILE;
    ns = min(a.nst, w0);
    n = ns + hi / TILE - w0 + 1;
  }
  __device__ __forceinline__ int operator()(int i) const { return i < ns ? i : w0 + i - ns; }
};

// Whether a query at a position in [lo, lo + 31] sees a key of tile kt, and
// whether they all see all of it.
__device__ __forceinline__ bool tile_seen(const WinArgs& a, int lo, int kt) {
  const int k0 = kt * TILE;
  return k0 <= lo + TILE - 1 && (k0 + TILE - 1 > lo - a.win || k0 < a.sinks);
}
__device__ __forceinline__ bool tile_whole(const WinArgs& a, int lo, int kt) {
  const int k1 = kt * TILE + TILE - 1;
  return k1 <= lo && (kt * TILE > lo + TILE - 1 - a.win || k1 < a.sinks);
}
__device__ __forceinline__ bool sees(const WinArgs& a, int pos, int key) {
  // key <= pos and key > pos - win as one comparison.  No short circuits here
  // or where this is used: a branch around one element of an accumulator has
  // been compiled wrongly (ROCm 7.2: the element's other value went to every
  // lane that took the branch)
  return ((unsigned)(pos - key) < (unsigned)a.win) | ((key < a.sinks) & (key <= pos));
}
// Slot of tile kt among the dS blocks of the queries at [lo, lo + 31].
__device__ __forceinline__ int ds_slot(const WinArgs& a, int lo, int kt) {
  return kt < a.nst ? kt : a.nst + kt - max(a.nst, max(0, lo - a.win + 1) / TILE);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// Sets values that are not finite to 0; whether the wave had any.
template <int NC>
__device__ __forceinline__ bool drop_nonfinite(float (&x)[NC][16]) {
  float top = 0.f;  // the maximum that NaN is larger than everything for
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int s = 0; s < 16; s += 2)
      top = __builtin_elementwise_maximum(
          __builtin_elementwise_maximum(top, fabsf(x[c][s])), fabsf(x[c][s + 1]));
  if (__ballot(!finite(top)) == 0) return false;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int s = 0; s < 16; ++s) {
      asm volatile("" : "+v"(x[c][s]));  // compared anew: else every mask is kept
      x[c][s] = finite(x[c][s]) ? x[c][s] : 0.f;
    }
  return true;
}

// Operands straight from memory, with no LDS between: the waves of a
// workgroup then need no barriers, and each walks just the tiles that its own
// 32 queries see (a 128-query block's list is a third longer at a window of
// 256).  What they share comes from the L1.

// One 32-row tile of a [T, D] matrix with row stride st, as a buffer from the
// tile's first element to the last one of its rows: loads past that give 0,
// and addresses are one register and scalars.  Row strides are below 2^23, so
// that a tile's offsets fit 32 bits.
constexpr int kBufferFlags = 0x00020000;  // 32-bit data, raw addressing (gfx9)
constexpr int64_t kMaxRowStride = int64_t(1) << 23;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_buffer(const float* tile, int64_t st,
                                                              int left, int D) {
  const int rows = min(left, TILE);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(tile), 0,
                                           4 * ((rows - 1) * (int)st + D), kBufferFlags);
}

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

// Operand of a product over the head dim, row l32 of the tile: lane (l32, h)
// has row[8 i + 4 h + e] as x[4 i + e].  GUARD: columns >= D are zero (read
// past the buffer).
template <int HD, bool GUARD, int RUN>
__device__ __forceinline__ void row_operand(__amdgpu_buffer_rsrc_t tile, int st, int D, int l32,
                                            int h, float (&x)[RUN]) {
  const int at = 4 * (l32 * st + 4 * h);
#pragma unroll
  for (int i = 0; i < RUN / 4; ++i) {
    const bool in = !GUARD || 8 * i + 4 * h < D;
    const uint4v v = __builtin_amdgcn_raw_buffer_load_b128(tile, in ? at : 0x7ffffff0, 32 * i, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * i + e] = __uint_as_float(v[e]);
  }
}

// Operand of a product over the tile's rows (lds_cols's): x[c][s] is column
// c * 32 + l32 of row kappa(s, h).  Columns past D hold anything: they go to
// columns of the result that are not written.
template <int HD>
__device__ __forceinline__ void col_operand(__amdgpu_buffer_rsrc_t tile, int st, int l32, int h,
                                            float (&x)[Hd<HD>::NC][16]) {
  const int at = 4 * (4 * h * st + l32);
#pragma unroll
  for (int s = 0; s < 16; ++s)
#pragma unroll
    for (int c = 0; c < Hd<HD>::NC; ++c)
      x[c][s] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
          tile, at + 128 * c, 4 * kappa(s, 0) * st, 0));
}

// ------------------------------------------------------------ forward

// Waves per SIMD the registers leave room for.
template <int HD> constexpr int waves_fwd() { return HD <= 64 ? 3 : HD <= 96 ? 2 : 1; }

// One wave 32 queries.  GUARD: D < HD.  PART: one slice of the key tiles,
// joined by k_win_merge.  96 heads of 1024 positions, D 64, window 256: 87 us,
// 66 TFLOP/s of the keys seen (80 of the tiles formed); 16 of 8192, D 128,
// window 1024: 718 us, 91.  A part of a prompt, 16 heads of 93 positions, D
// 80, window 300, in slices: 15 us and 4 for the join.
template <int HD, bool GUARD, bool PART, int RUN>
__global__ __launch_bounds__(256, waves_fwd<HD>()) void k_win_fwd(WinArgs a) {
  using S_ = Hd<HD>;
  __shared__ __attribute__((aligned(16))) float buf[WAVES][TILE * S_::W];  // the output's rows
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, h = lane >> 5;
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const int64_t bh = item / a.nblk;
  const int qb = item % a.nblk;
  const int64_t b = bh / a.H, hh = bh % a.H, kh = hh / a.G;
  const float* Q = a.q + b * a.qs.b + hh * a.qs.h;
  const float* K = a.k + b * a.ks.b + kh * a.ks.h;
  const float* V = a.v + b * a.vs.b + kh * a.vs.h;
  const int q0 = qb * ROWS + w * TILE;  // this wave's first query
  if (q0 >= a.Tq) return;
  const int myq = q0 + l32, lo = a.off + q0, pos = lo + l32;
  const Tiles tiles(a, lo, min(lo + TILE, a.Tk) - 1);
  const int i0 = PART ? (int)blockIdx.y * a.kslice : 0;
  const int i1 = PART ? min(tiles.n, i0 + a.kslice) : tiles.n;
  if (PART && i0 >= i1) return;

  float qf[RUN];
  row_operand<HD, GUARD>(tile_buffer(Q + q0 * a.qs.t, a.qs.t, a.Tq - q0, a.D), (int)a.qs.t, a.D,
                         l32, h, qf);
#pragma unroll
  for (int s = 0; s < RUN; ++s) qf[s] *= a.scale * kLog2e;
  const auto load_keys = [&](int kt, float (&x)[RUN]) {
    const int k0 = kt * TILE;
    row_operand<HD, GUARD>(tile_buffer(K + k0 * a.ks.t, a.ks.t, a.Tk - k0, a.D), (int)a.ks.t, a.D,
                           l32, h, x);
  };
  floatx16 acc[S_::NC];
  zero_acc(acc);
  float m = -INFINITY, lsum = 0.f;
  float ka[RUN];
  load_keys(tiles(i0), ka);
  for (int i = i0; i < i1; ++i) {
    const int kt = tiles(i), k0 = kt * TILE;
    // values on their way during the first product, the next keys during the
    // second
    float va[S_::NC][16];
    col_operand<HD>(tile_buffer(V + k0 * a.vs.t, a.vs.t, a.Tk - k0, a.D), (int)a.vs.t, l32, h, va);
    floatx16 st = chain0<HD>(ka, qf);  // S^T[key][query], base-2 units
    load_keys(tiles(min(i + 1, i1 - 1)), ka);
    bool bad = false;
    if (!tile_whole(a, lo, kt)) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const bool in = sees(a, pos, k0 + kappa(j, h));
        st[j] = in ? st[j] : -INFINITY;
      }
      bad = drop_nonfinite(va);
    }
    float bm = st[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) bm = fmaxf(bm, st[j]);
    bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
    const float mn = fmaxf(m, bm);
    const float ms = mn == -INFINITY ? 0.f : mn;  // nothing seen so far
    const float alpha = exp2_hw(m - ms);
    float rs = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      st[j] = exp2_hw(st[j] - ms);
      rs += st[j];
    }
    rs += __shfl_xor(rs, 32, 64);
    lsum = lsum * alpha + rs;
    m = mn;
#pragma unroll
    for (int c = 0; c < S_::NC; ++c) acc[c] *= alpha;
#pragma unroll
    for (int s = 0; s < 16; ++s)  // O^T += V^T P^T
#pragma unroll
      for (int c = 0; c < S_::NC; ++c) acc[c] = mfma(va[c][s], st[s], acc[c]);
    if (bad) {  // values that are not finite, for the queries that see them
#pragma unroll 1
      for (int r = 0; r < TILE; ++r) {
        if (!sees(a, pos, k0 + r) || k0 + r >= a.Tk) continue;
        const float* row = V + (int64_t)(k0 + r) * a.vs.t;
#pragma unroll
        for (int c = 0; c < S_::NC; ++c)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int d = c * 32 + kappa(j, h);
            const float x = d < a.D ? row[d] : 0.f;
            acc[c][j] += finite(x) ? 0.f : x;
          }
      }
    }
  }
  if constexpr (PART) {
    const int64_t row0 = ((int64_t)blockIdx.y * (gridDim.x / a.nblk) + bh) * a.Tq;
    write_rows<HD, false>(buf[w], acc, 1.0f, a.part + row0 * a.D, a.D, q0, a.Tq, a.D, l32, h, lane);
    if (h == 0 && myq < a.Tq) a.pml[row0 + myq] = make_float2(m, lsum);
    return;
  }
  const float inv = 1.0f / lsum;  // a query sees itself: the sum is at least 1
  write_rows<HD, false>(buf[w], acc, inv, a.out + b * a.os.b + hh * a.os.h, a.os.t, q0, a.Tq, a.D,
                        l32, h, lane);
  if (a.lse_out && h == 0 && myq < a.Tq) a.lse_out[bh * a.Tq + myq] = m + __log2f(lsum);
}

// Joins the slices of a query: o = sum 2^(m_s - m) acc_s / sum 2^(m_s - m)
// l_s, in slice order.  One float4 a lane; n: slices of each row, or 0 and
// those of its 32 queries.
__global__ __launch_bounds__(256) void k_win_merge(WinArgs a, int64_t n4, int nslices) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n4) return;
  const int d4 = a.D / 4;
  const int64_t row = i / d4, rows = n4 / d4;
  const int c = (int)(i - row * d4);
  const int64_t bh = row / a.Tq;
  const int q = (int)(row - bh * a.Tq);
  int n = nslices;
  if (n == 0) {
    const int lo = a.off + q / TILE * TILE;
    const Tiles tiles(a, lo, min(lo + TILE, a.Tk) - 1);
    n = (tiles.n + a.kslice - 1) / a.kslice;
  }
  // eight slices at a time, their loads together: they come from other XCDs
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, den = 0.f;
  for (int s0 = 0; s0 < n; s0 += 8) {
    float2 ml[8];
    floatx4 x[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const int64_t at = min(s0 + s, n - 1) * rows + row;  // past the end: not used
      ml[s] = a.pml[at];
      x[s] = *reinterpret_cast<const floatx4*>(a.part + at * a.D + 4 * c);
    }
    float m = top;
#pragma unroll
    for (int s = 0; s < 8; ++s) m = fmaxf(m, ml[s].x);
    const float ms = m == -INFINITY ? 0.f : m;
    const float alpha = exp2_hw(top - ms);
    top = m;
    den *= alpha;
    o *= alpha;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const float f = s0 + s < n ? exp2_hw(ml[s].x - ms) : 0.f;
      // a slice that this query sees nothing of has sums of 0 and a factor of
      // 0, and infinities of other slices stay what they are
      if (f != 0.f) {
        den = __builtin_fmaf(ml[s].y, f, den);
        o += f * x[s];
      }
    }
  }
  const int64_t b = bh / a.H, h = bh % a.H;
  *reinterpret_cast<floatx4*>(a.out + b * a.os.b + h * a.os.h + q * a.os.t + 4 * c) =
      o * (1.0f / den);
  if (a.lse_out && c == 0) a.lse_out[row] = top + __log2f(den);
}

// Few queries (a decoding step): one query head and position a workgroup,
// its keys over groups of 16 lanes, each with a running softmax of its own
// over every NG-th key, joined once at the end in a fixed order.  grid.y
// slices of the keys, joined by k_win_merge, where there are few rows.
// Bound by the latency of its loads where rows are few: 48 of 260 keys, D 64,
// 5.5 us; by memory where they are many: 64 sequences of 8 heads, 4096 keys, D
// 128, 355 us, 6.1 TB/s.  Query heads that share keys each fetch them, on
// different XCDs: 32 over those 8 heads take 1239 us, 1.7 TB/s of the cache.
constexpr int kFewThreads = 512, kFewGroups = kFewThreads / 16, kFewUnroll = 4;

template <int NC, bool PART>  // NC: 64-column pieces of the head dim
__global__ __launch_bounds__(kFewThreads) void k_win_few(WinArgs a) {
  __shared__ float sm[kFewGroups], sl[kFewGroups];
  __shared__ __attribute__((aligned(16))) float so[kFewGroups][NC * 64];
  const int64_t row = blockIdx.x;  // (b * H + h) * Tq + t
  const int64_t bh = row / a.Tq, b = bh / a.H, hh = bh % a.H, kh = hh / a.G;
  const int q = (int)(row - bh * a.Tq), pos = a.off + q;
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15;
  const float* __restrict__ K = a.k + b * a.ks.b + kh * a.ks.h;
  const float* __restrict__ V = a.v + b * a.vs.b + kh * a.vs.h;
  // the i-th key that it sees
  const int first = max(0, pos - a.win + 1), ns = min(a.sinks, first);
  const int seen = ns + pos - first + 1;
  const int i0 = PART ? (int)blockIdx.y * a.kslice : 0;
  const int i1 = PART ? min(seen, i0 + a.kslice) : seen;
  const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
  floatx4 qv[NC], o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int d = 64 * c + 4 * l;
    o[c] = zero;
    qv[c] = zero;
    if (d < a.D)
      qv[c] = *reinterpret_cast<const floatx4*>(a.q + b * a.qs.b + hh * a.qs.h + q * a.qs.t + d) *
              (a.scale * kLog2e);
  }
  float m = -INFINITY, sum = 0.f;
  for (int t0 = i0 + g; t0 < i1; t0 += kFewGroups * kFewUnroll) {
    floatx4 kv[kFewUnroll][NC], vv[kFewUnroll][NC];
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u) {
      // keys past the end repeat the last one with a score of -infinity
      const int i = min(t0 + u * kFewGroups, i1 - 1);
      const int64_t t = i < ns ? i : first + i - ns;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = 64 * c + 4 * l;
        kv[u][c] = d < a.D ? *reinterpret_cast<const floatx4*>(K + t * a.ks.t + d) : zero;
        vv[u][c] = d < a.D ? *reinterpret_cast<const floatx4*>(V + t * a.vs.t + d) : zero;
      }
    }
    float s[kFewUnroll], mn = m;
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u) {
      float x = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) x = __builtin_fmaf(qv[c][e], kv[u][c][e], x);
      x = row16_sum(x);
      s[u] = t0 + u * kFewGroups < i1 ? x : -INFINITY;
      mn = fmaxf(mn, s[u]);
    }
    const float ms = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2_hw(m - ms);
    m = mn;
    sum *= alpha;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[c] *= alpha;
#pragma unroll
    for (int u = 0; u < kFewUnroll; ++u) {
      const float p = exp2_hw(s[u] - ms);
      sum += p;
      if (t0 + u * kFewGroups < i1) {  // 0 times infinity of a repeated key stays out
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][e] = __builtin_fmaf(p, vv[u][c][e], o[c][e]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) *reinterpret_cast<floatx4*>(&so[g][64 * c + 4 * l]) = o[c];
  if (l == 0) {
    sm[g] = m;
    sl[g] = sum;
  }
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= NC * 64 || d >= a.D) return;
  float top = -INFINITY;
  for (int i = 0; i < kFewGroups; ++i) top = fmaxf(top, sm[i]);
  const float ts = top == -INFINITY ? 0.f : top;
  float den = 0.f, num = 0.f;
#pragma unroll 8
  for (int i = 0; i < kFewGroups; ++i) {
    const float f = exp2_hw(sm[i] - ts);
    den = __builtin_fmaf(sl[i], f, den);
    num = __builtin_fmaf(so[i][d], f, num);
  }
  if constexpr (PART) {
    const int64_t at = (int64_t)blockIdx.y * gridDim.x + row;
    a.part[at * a.D + d] = num;
    if (d == 0) a.pml[at] = make_float2(top, den);
  } else {
    a.out[b * a.os.b + hh * a.os.h + q * a.os.t + d] = num * (1.0f / den);
    if (d == 0 && a.lse_out) a.lse_out[row] = top + __log2f(den);
  }
}

// ------------------------------------------------------------ backward

// Where the sums of the key blocks without sinks begin.
__host__ __device__ inline int64_t sums_at(const WinArgs& a) {
  return a.nslice > 1 ? (int64_t)2 * a.nslice * a.nbkv * a.nsb * PROWS * a.D : 0;
}

// Key-block kernel: 64 keys a workgroup, each 32 of them a pair of waves; wave
// A forms P and accumulates dV^T += dO^T P, wave B forms dS = P (dP - D),
// stores it and accumulates dK^T += Q^T dS (flash.hip's split of the work, the
// tiles of Q and dO through LDS: straight from memory they took 2 % less at a
// head dim of 64 and a sixth more at 128).  GUARD: Tq or Tk is not a multiple
// of 32, or D < HD.  The sizes of k_win_fwd: 168 us, 68 TFLOP/s of the keys
// seen; 1239 us, 105.
template <int HD, bool GUARD, int RUN>
__global__ __launch_bounds__(256, occ_pair<HD>()) void k_win_dkv(WinArgs a) {
  using S_ = Hd<HD>;
  __shared__ __attribute__((aligned(16))) float Qs[2][TILE * S_::W];
  __shared__ __attribute__((aligned(16))) float Gs[2][TILE * S_::W];
  __shared__ __attribute__((aligned(16))) float Ps[2][16 * 64];
  __shared__ __attribute__((aligned(16))) float Rs[2][2][TILE];  // [role][tile][row]: lse, D
  // unequal wave priorities keep a CU's workgroups out of step (flash.hip)
  if (blockIdx.x % 3 == 0) __builtin_amdgcn_s_setprio(2);
  else if (blockIdx.x % 3 == 1) __builtin_amdgcn_s_setprio(1);
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int role = wv >> 1, pr = wv & 1;  // role 0: A (P, dV), 1: B (dS, dK)
  const int l32 = lane & 31, h = lane >> 5;
  // the slices of the sinks' blocks first, then the blocks by position: the
  // last ones are seen by fewer queries and fill the CUs at the end
  const int nlong = a.nbkv * a.nsb * a.nslice;
  const bool sunk = (int)blockIdx.x < nlong;
  const int slices = sunk ? a.nslice : a.nsplit;
  int id = sunk ? blockIdx.x : blockIdx.x - nlong;
  const int bkv = id % a.nbkv;
  id /= a.nbkv;
  const int slice = id % slices, kb = (sunk ? 0 : a.nsb) + id / slices;
  const int hkv = a.H / a.G;
  const int64_t b = (a.bkv0 + bkv) / hkv, kh = (a.bkv0 + bkv) % hkv;
  const float* K = a.k + b * a.ks.b + kh * a.ks.h;
  const float* V = a.v + b * a.vs.b + kh * a.vs.h;
  const int k0 = kb * PROWS + pr * TILE, kt = k0 / TILE;  // the pair's keys
  const int mykey = k0 + l32;

  float kv[RUN];
  if (role == 0)
    gl_run<HD, GUARD>(K, a.ks.t, mykey, a.Tk, a.D, h, a.scale * kLog2e, kv);
  else
    gl_run<HD, GUARD>(V, a.vs.t, mykey, a.Tk, a.D, h, 1.0f, kv);
  // complete the loads here: a wait for them inside the loop would also
  // wait for every step's prefetch
#pragma unroll
  for (int i = 0; i < RUN; ++i) asm volatile("" : "+v"(kv[i]));
  floatx16 acc[S_::NC];  // A: dV^T, B: dK^T
  zero_acc(acc);

  // the query tiles that see some of the 64 keys
  const int qt0 = max(0, kb * PROWS - a.off) / TILE;
  int last = a.Tq - 1;
  if (!sunk) last = (int)min((int64_t)last, (int64_t)kb * PROWS + PROWS - 2 + a.win - a.off);
  const int qt1 = last < 0 ? qt0 : max(qt0, last / TILE + 1), nt = qt1 - qt0;
  // this slice of the steps, the query heads' tiles one head after the other
  const int per = (nt * a.G + slices - 1) / slices;
  const int f0 = min(nt * a.G, slice * per), steps = min(nt * a.G - f0, per);
  // of the current and the next step: query head and tile
  int hh = (int)kh * a.G + (nt ? f0 / nt : 0), qt = qt0 + (nt ? f0 % nt : 0);
  const auto qrows = [&](const float* x, const Strides3& s, int head) {
    return x + b * s.b + (int64_t)head * s.h;
  };
  // lse (A) or D (B) of the tile's rows: subtracted after the products.  As
  // the products' first term, as in flash.hip, they would have every later
  // sum rounded at their own size, three times the error in P at 260 keys
  const auto row_term = [&](int head, int t) {
    const float* L = (role == 0 ? a.lse : a.dsum) + (b * a.H + head) * (int64_t)a.Tq;
    return L[min(t * TILE + l32, a.Tq - 1)];
  };
  floatx4 rq[S_::NC], rg[S_::NC];
  float term = 0.f;
  if (steps > 0) {
    load_tile<HD, GUARD>(qrows(a.q, a.qs, hh), a.qs.t, qt * TILE, a.Tq, a.D, rq);
    load_tile<HD, GUARD>(qrows(a.dout, a.gs, hh), a.gs.t, qt * TILE, a.Tq, a.D, rg);
    term = row_term(hh, qt);
    store_tile<HD>(Qs[0], rq);
    store_tile<HD>(Gs[0], rg);
    if (pr == 0 && h == 0) Rs[role][0][l32] = term;
  }
  __syncthreads();
  float* pbuf = Ps[pr];
  for (int step = 0; step < steps; ++step) {
    const int cur = step & 1;
    const bool more = step + 1 < steps;
    int hn = hh, qn = qt + 1;
    if (qn == qt1) {
      qn = qt0;
      ++hn;
    }
    if (more) {
      load_tile<HD, GUARD>(qrows(a.q, a.qs, hn), a.qs.t, qn * TILE, a.Tq, a.D, rq);
      load_tile<HD, GUARD>(qrows(a.dout, a.gs, hn), a.gs.t, qn * TILE, a.Tq, a.D, rg);
      term = row_term(hn, qn);
    }
    const int lo = a.off + qt * TILE;  // the tile's first position
    const bool seen = k0 < a.Tk && tile_seen(a, lo, kt);
    const bool edge = !tile_whole(a, lo, kt) || (GUARD && qt * TILE + TILE > a.Tq);
    const auto ok = [&](int j) {
      const int r = kappa(j, h);
      return (!GUARD | (qt * TILE + r < a.Tq)) & sees(a, lo + r, mykey);
    };
    floatx16 x = zero16();  // A: P; B: dP - D, then dS
    if (seen) {
      float xa[RUN];
      // A: S[q][key] - lse[q] from Q rows; B: dP[q][key] - D[q] from dO rows
      lds_run<HD>(role == 0 ? Qs[cur] : Gs[cur], l32, h, xa);
      x = chain0<HD>(xa, kv);
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const floatx4 r = *reinterpret_cast<const floatx4*>(&Rs[role][cur][kappa(j, h)]);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j + e] -= r[e];
      }
      if (role == 0) {
        if (edge) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float e = exp2_hw(x[j]);
            x[j] = ok(j) ? e : 0.f;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] = exp2_hw(x[j]);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) pbuf[j * 64 + lane] = x[j];
      }
    }
    __syncthreads();
    if (seen) {
      float ct[S_::NC][16];
      if (role == 0) {
        lds_cols<HD>(Gs[cur], l32, h, ct);
#pragma unroll
        for (int s = 0; s < 16; ++s)  // dV^T += dO^T P
#pragma unroll
          for (int c = 0; c < S_::NC; ++c) acc[c] = mfma(ct[c][s], x[s], acc[c]);
      } else {
        if (edge) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float ds = x[j] * pbuf[j * 64 + lane];
            x[j] = ok(j) ? ds : 0.f;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] *= pbuf[j * 64 + lane];
        }
        lds_cols<HD>(Qs[cur], l32, h, ct);
#pragma unroll
        for (int s = 0; s < 16; ++s)  // dK^T += Q^T dS
#pragma unroll
          for (int c = 0; c < S_::NC; ++c) acc[c] = mfma(ct[c][s], x[s], acc[c]);
      }
    }
    if (more) {
      store_tile<HD>(Qs[cur ^ 1], rq);
      store_tile<HD>(Gs[cur ^ 1], rg);
      if (pr == 0 && h == 0) Rs[role][cur ^ 1][l32] = term;
    }
    if (seen && role == 1) {
      const int64_t bh = (int64_t)bkv * a.G + hh - kh * a.G;
      float* blk = a.dsblk + ((bh * a.nqt + qt) * a.nsl + ds_slot(a, lo, kt)) * (TILE * TILE) +
                   ds_col(l32);
#pragma unroll
      for (int j = 0; j < 16; ++j) __builtin_nontemporal_store(x[j], blk + kappa(j, h) * TILE);
    }
    hh = hn;
    qt = qn;
    __syncthreads();
  }
  float* buf = (wv < 2 ? Qs[wv] : Gs[wv - 2]);
  const float mul = role == 0 ? 1.0f : a.scale;
  if (slices > 1) {  // rows of `sums`: the sinks' blocks, then the others
    const int64_t rows = (int64_t)(sunk ? a.nsb : a.nblk - a.nsb) * PROWS;
    float* to = a.sums + (sunk ? 0 : sums_at(a)) +
                (((int64_t)(role == 0 ? slices : 0) + slice) * a.nbkv + bkv) * rows * a.D;
    write_rows<HD>(buf, acc, mul, to - (sunk ? 0 : (int64_t)a.nsb * PROWS * a.D), a.D, k0, a.Tk,
                   a.D, l32, h, lane);
  } else {
    const Strides3& st = role == 0 ? a.o2s : a.o1s;
    write_rows<HD>(buf, acc, mul, (role == 0 ? a.out2 : a.out) + b * st.b + kh * st.h, st.t, k0,
                   a.Tk, a.D, l32, h, lane);
  }
}

// dK and dV of the key blocks whose steps were cut into slices: the slices'
// sums, in order.  Blocks [blk0, blk0 + nb) and their part of `sums`.
__global__ __launch_bounds__(256) void k_win_sums(WinArgs a, const float* __restrict__ sums,
                                                  int blk0, int nb, int slices, int64_t n4) {
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * n4) return;
  const bool v = i >= n4;
  const int64_t rows = (int64_t)nb * PROWS, all = a.nbkv * rows * a.D;
  const float* src = sums + (v ? slices * all : 0);
  if (v) i -= n4;
  const int d4 = a.D / 4;
  const int64_t row = i / d4, bkv = row / rows, key = row - bkv * rows + (int64_t)blk0 * PROWS;
  const int c = 4 * (int)(i - row * d4);
  if (key >= a.Tk) return;
  floatx4 x = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < slices; ++s)
    x += *reinterpret_cast<const floatx4*>(src + s * all + row * a.D + c);
  const int hkv = a.H / a.G;
  const int64_t b = (a.bkv0 + bkv) / hkv, kh = (a.bkv0 + bkv) % hkv;
  const Strides3& st = v ? a.o2s : a.o1s;
  *reinterpret_cast<floatx4*>((v ? a.out2 : a.out) + b * st.b + kh * st.h + key * st.t + c) = x;
}

// Query kernel: dQ^T += K^T dS^T from the stored dS blocks, one wave 32
// queries, the next tile's operands on their way during a tile's products.
// Half the products of a tile for the same loads as the forward's: the sizes
// of k_win_fwd, 58 us, 49 TFLOP/s of the keys seen; 375 us, 87.  JOIN: where
// that leaves CUs idle, a workgroup's waves have a quarter each of the tiles
// of the same 32 queries and add their sums up in order.
template <int HD, bool JOIN>
__global__ __launch_bounds__(256, HD <= 64 ? 3 : HD <= 96 ? 2 : 1) void k_win_dq(WinArgs a) {
  using S_ = Hd<HD>;
  __shared__ __attribute__((aligned(16))) float buf[WAVES][TILE * S_::W];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, h = lane >> 5;
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const int per_head = JOIN ? a.nqt : a.nblk;
  const int64_t bhl = item / per_head;  // from the launch's first head on
  const int qb = item % per_head;
  const int64_t bh = (int64_t)a.bkv0 * a.G + bhl;
  const int64_t b = bh / a.H, hh = bh % a.H;
  const float* K = a.k + b * a.ks.b + (hh / a.G) * a.ks.h;
  const int q0 = JOIN ? qb * TILE : qb * ROWS + w * TILE, lo = a.off + q0;
  if (q0 >= a.Tq) return;  // JOIN: never
  const float* dsrow = a.dsblk + (bhl * a.nqt + q0 / TILE) * a.nsl * (TILE * TILE) + l32 * TILE +
                       h * 16;
  const Tiles tiles(a, lo, min(lo + TILE, a.Tk) - 1);
  const auto load = [&](int kt, float (&k)[S_::NC][16], floatx4 (&d)[4]) {
    const int k0 = kt * TILE;
    col_operand<HD>(tile_buffer(K + k0 * a.ks.t, a.ks.t, a.Tk - k0, a.D), (int)a.ks.t, l32, h, k);
    const floatx4* src =
        reinterpret_cast<const floatx4*>(dsrow + (int64_t)ds_slot(a, lo, kt) * (TILE * TILE));
#pragma unroll
    for (int u = 0; u < 4; ++u) d[u] = src[u];
  };
  floatx16 dq[S_::NC];
  zero_acc(dq);
  const auto products = [&](int kt, float (&k)[S_::NC][16], const floatx4 (&d)[4]) {
    // a query that sees a key that is not finite has NaN in dS already
    if (!tile_whole(a, lo, kt)) drop_nonfinite(k);
#pragma unroll
    for (int s = 0; s < 16; ++s)
#pragma unroll
      for (int c = 0; c < S_::NC; ++c) dq[c] = mfma(k[c][s], d[s >> 2][s & 3], dq[c]);
  };
  const int per = JOIN ? (tiles.n + WAVES - 1) / WAVES : tiles.n;
  const int i0 = JOIN ? min(w * per, tiles.n) : 0, i1 = min(i0 + per, tiles.n);
  if (!JOIN || i0 < i1) {
    float k0[S_::NC][16], k1[S_::NC][16];
    floatx4 d0[4], d1[4];
    load(tiles(i0), k0, d0);
    for (int i = i0; i < i1; i += 2) {
      load(tiles(min(i + 1, i1 - 1)), k1, d1);
      products(tiles(i), k0, d0);
      load(tiles(min(i + 2, i1 - 1)), k0, d0);
      if (i + 1 < i1) products(tiles(i + 1), k1, d1);
    }
  }
  float* out = a.out + b * a.o1s.b + hh * a.o1s.h;
  if constexpr (!JOIN) {
    write_rows<HD, false>(buf[w], dq, a.scale, out, a.o1s.t, q0, a.Tq, a.D, l32, h, lane);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int c = 0; c < S_::NC; ++c) buf[w][l32 * S_::W + c * 32 + kappa(j, h)] = dq[c][j];
    __syncthreads();
    for (int f = threadIdx.x; f < TILE * S_::F4; f += 256) {
      const int row = f / S_::F4, c4 = f % S_::F4, at = row * S_::W + 4 * c4;
      if (q0 + row >= a.Tq || 4 * c4 >= a.D) continue;
      floatx4 sum = *reinterpret_cast<const floatx4*>(&buf[0][at]);
#pragma unroll
      for (int i = 1; i < WAVES; ++i) sum += *reinterpret_cast<const floatx4*>(&buf[i][at]);
      *reinterpret_cast<floatx4*>(out + (int64_t)(q0 + row) * a.o1s.t + 4 * c4) = sum * a.scale;
    }
  }
}

// ------------------------------------------------------------ host

Strides3 s3(const int64_t* s) { return Strides3{s[0], s[1], s[2]}; }

// 16 or more of the padded columns empty: shorter products over the head dim
template <int HD>
bool short_run(const WinArgs& a) { return a.D <= HD - 16; }

template <int HD, bool PART>
void launch_fwd(const WinArgs& a, dim3 grid) {
  if (short_run<HD>(a))
    tjh_launch(k_win_fwd<HD, true, PART, HD / 2 - 8>, grid, dim3(256), 0, stream(), a);
  else if (a.D != HD)
    tjh_launch(k_win_fwd<HD, true, PART, HD / 2>, grid, dim3(256), 0, stream(), a);
  else
    tjh_launch(k_win_fwd<HD, false, PART, HD / 2>, grid, dim3(256), 0, stream(), a);
}

template <int HD>
void launch_fwd(const WinArgs& a, dim3 grid, bool part) {
  if (part) launch_fwd<HD, true>(a, grid);
  else launch_fwd<HD, false>(a, grid);
}

template <int HD>
int launch_bwd(WinArgs a, unsigned keys, float* dq, const int64_t* dq_st) {
  if (short_run<HD>(a))
    tjh_launch(k_win_dkv<HD, true, HD / 2 - 8>, dim3(keys), dim3(256), 0, stream(), a);
  else if (a.Tq % TILE || a.Tk % TILE || a.D != HD)
    tjh_launch(k_win_dkv<HD, true, HD / 2>, dim3(keys), dim3(256), 0, stream(), a);
  else
    tjh_launch(k_win_dkv<HD, false, HD / 2>, dim3(keys), dim3(256), 0, stream(), a);
  int rc = check_launch("window_dkv");
  if (rc != TJH_OK) return rc;
  for (int sunk = 0; sunk < 2; ++sunk) {
    const int nb = sunk ? a.nsb : a.nblk - a.nsb, slices = sunk ? a.nslice : a.nsplit;
    if (slices < 2 || nb == 0) continue;
    const int64_t n4 = (int64_t)a.nbkv * nb * PROWS * a.D / 4;
    tjh_launch(k_win_sums, dim3((unsigned)cdiv(2 * n4, 256)), dim3(256), 0, stream(), a,
               (const float*)(a.sums + (sunk ? 0 : sums_at(a))), sunk ? 0 : a.nsb, nb, slices, n4);
    if ((rc = check_launch("window_sums")) != TJH_OK) return rc;
  }
  a.nblk = (int)cdiv(a.Tq, ROWS);
  a.out = dq;
  a.o1s = s3(dq_st);
  const unsigned heads = (unsigned)(a.nbkv * a.G), grid = heads * a.nblk;
  // the whole backward of one head of 4096, window 2000 (32 workgroups): 171
  // us, joined 115; 12 of 1024, all seen (96): 116, 102; 8 x 4 of 700, window
  // 64 (192): 81, 83
  if (3 * (int64_t)grid <= 2 * (num_cus() > 0 ? num_cus() : 256))
    tjh_launch(k_win_dq<HD, true>, dim3(heads * a.nqt), dim3(256), 0, stream(), a);
  else
    tjh_launch(k_win_dq<HD, false>, dim3(grid), dim3(256), 0, stream(), a);
  return check_launch("window_dq");
}

// Over how many workgroups the steps of a key block are split.  The
// workgroups are about equally long, so the last round that they fill the CUs
// in stands half empty on average; each split costs a prologue of some 3
// steps, and its sums' way through memory about 2.  4 key heads of 8192, 4
// query heads each (508 workgroups of 140 steps on 512 places): 1424 us, as
// two splits 1315, as four 1292; one head of 4096, D 64, window 2000, the
// whole backward: 300 us, split 171.
int key_splits(const WinArgs& a, int64_t nbkv, int64_t tiles) {
  const int64_t cus = num_cus() > 0 ? num_cus() : 256, places = cus * (a.D <= 64 ? 3 : 2);
  int best = 1;
  int64_t cost = 0;
  for (int n = 1; n <= 8 && n <= tiles * a.G; ++n) {
    const int64_t each = cdiv(tiles * a.G, n) + 3;
    const int64_t c = 2 * nbkv * a.nblk * n * each / places + each + (n > 1 ? 4 * n : 0);
    if (n == 1 || c < cost) {
      cost = c;
      best = n;
    }
  }
  return best;
}

int check_window(const char* who, int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk,
                 int64_t D, int64_t window, int64_t sinks, const void* const* ptrs,
                 const int64_t* const* strides, int n) {
  TJH_ARG(B >= 0 && H >= 0 && Hkv >= 0 && Tq >= 0 && D > 0, "%s: bad sizes", who);
  TJH_ARG(Tk >= Tq, "%s: %lld queries over %lld keys", who, (long long)Tq, (long long)Tk);
  TJH_ARG(window >= 1 && sinks >= 0, "%s: window %lld, sinks %lld", who, (long long)window,
          (long long)sinks);
  TJH_ARG(H == 0 || (Hkv > 0 && H % Hkv == 0), "%s: %lld heads over %lld", who, (long long)H,
          (long long)Hkv);
  TJH_ARG(Tk < (int64_t(1) << 30) && B < (int64_t(1) << 30) && H < (int64_t(1) << 30),
          "%s: too large", who);
  // a grid has less than 2^32 threads: up to 4 queries take kFewThreads each in
  // the forward, a tile of 32 at most 256
  const int64_t groups = Tq <= 4 ? Tq * (kFewThreads / 256) : cdiv(Tq, TILE);
  TJH_ARG(groups == 0 || B * H <= ((int64_t(1) << 24) - 1) / groups, "%s: too large", who);
  for (int i = 0; i < n; ++i) TJH_ARG(strides[i], "%s: NULL strides", who);
  bool wide = false;
  for (int i = 0; i < n; ++i) wide |= strides[i][2] >= kMaxRowStride || strides[i][2] < 0;
  if (B == 0 || H == 0 || Tq == 0) return TJH_OK;
  for (int i = 0; i < n; ++i) TJH_ARG(ptrs[i], "%s: NULL pointer", who);
  if (wide || !flash_supported(D, ptrs, strides, n))
    return set_error(TJH_ERR_UNSUPPORTED,
                     "%s: head dims up to 128 that are multiples of 4, in 16-byte aligned rows "
                     "less than 2^23 apart (head dim %lld)", who, (long long)D);
  return TJH_OK;
}

WinArgs win_args(int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t D, float scale,
                 int64_t window, int64_t sinks) {
  WinArgs a{};
  a.H = (int)H; a.G = (int)(H / Hkv);
  a.Tq = (int)Tq; a.Tk = (int)Tk; a.off = (int)(Tk - Tq); a.D = (int)D;
  a.scale = scale;
  a.win = (int)(window < Tk ? window : Tk);
  a.sinks = (int)(sinks < Tk ? sinks : Tk);
  // sinks that every query's window holds are none
  if (a.win >= a.Tk) a.sinks = 0;
  a.nst = (int)cdiv(a.sinks, TILE);
  return a;
}

}  // namespace
}  // namespace tjh

using namespace tjh;

extern "C" {

int tjh_window_forward(const float* q, const float* k, const float* v, float* o, float* lse,
                       int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t D,
                       const int64_t* q_strides, const int64_t* k_strides,
                       const int64_t* v_strides, const int64_t* o_strides, float scale,
                       int64_t window, int64_t sinks) {
  TJH_REQUIRE_INIT();
  const void* ptrs[4] = {q, k, v, o};
  const int64_t* sts[4] = {q_strides, k_strides, v_strides, o_strides};
  int rc = check_window("tjh_window_forward", B, H, Hkv, Tq, Tk, D, window, sinks, ptrs, sts, 4);
  if (rc != TJH_OK || B == 0 || H == 0 || Tq == 0) return rc;
  WinArgs a = win_args(H, Hkv, Tq, Tk, D, scale, window, sinks);
  a.q = q; a.k = k; a.v = v; a.out = o; a.lse_out = lse;
  a.qs = s3(q_strides); a.ks = s3(k_strides); a.vs = s3(v_strides); a.os = s3(o_strides);
  KernelScope ks("window_fwd");
  const int64_t cus = num_cus() > 0 ? num_cus() : 256, rows = B * H * Tq;
  // keys that a query sees at most
  const int64_t most = a.win + a.sinks < a.Tk ? a.win + a.sinks : a.Tk;
  const auto room = [&](Scratch& s, int64_t n) {
    if (!s.ok()) return false;
    a.part = s.as<float>();
    a.pml = reinterpret_cast<float2*>(a.part + n * rows * D);
    return true;
  };
  if (Tq <= 4) {
    int64_t n = 1;
    if (rows < cus && most > 512)
      n = cdiv(most, 256) < cus / rows ? cdiv(most, 256) : cus / rows;
    a.kslice = (int)cdiv(most, n);
    n = cdiv(most, a.kslice);
    Scratch s(n > 1 ? (size_t)(n * rows * (D + 2)) * sizeof(float) : 0);
    const bool split = n > 1 && room(s, n);
    const dim3 grid((unsigned)rows, split ? (unsigned)n : 1), block(kFewThreads);
    if (split && D <= 64) tjh_launch(k_win_few<1, true>, grid, block, 0, stream(), a);
    else if (split) tjh_launch(k_win_few<2, true>, grid, block, 0, stream(), a);
    else if (D <= 64) tjh_launch(k_win_few<1, false>, grid, block, 0, stream(), a);
    else tjh_launch(k_win_few<2, false>, grid, block, 0, stream(), a);
    if ((rc = check_launch("window_few")) != TJH_OK || !split) return rc;
    const int64_t n4 = rows * D / 4;
    tjh_launch(k_win_merge, dim3((unsigned)cdiv(n4, 256)), dim3(256), 0, stream(), a, n4, (int)n);
    return check_launch("window_merge");
  }
  a.nblk = (int)cdiv(Tq, ROWS);
  const int64_t blocks = B * H * a.nblk;
  // slices of the key tiles where the blocks of queries leave CUs idle and
  // a wave is spared four tiles or more, some 3 us each, for the join.  2 heads
  // of 3000, D 128, window 1000: 173 us, in slices 54; 3 of 300, D 64, window
  // 100 (4 spared): 22, 16; 16 of 1500, D 64, window 300 (3 spared): 39, 46
  const int64_t wt = cdiv((int64_t)a.win + TILE - 2, TILE) + 1 + a.nst, all = cdiv(Tk, TILE);
  const int64_t nt = wt < all ? wt : all;  // tiles of 32 queries at most
  int64_t n = 1;
  a.kslice = (int)(cdiv(nt * blocks, cus) < 2 ? 2 : cdiv(nt * blocks, cus));
  if (blocks < cus && nt - a.kslice >= 4) n = cdiv(nt, a.kslice);
  Scratch s(n > 1 ? (size_t)(n * rows * (D + 2)) * sizeof(float) : 0);
  const bool split = n > 1 && room(s, n);
  const dim3 grid((unsigned)blocks, split ? (unsigned)n : 1);
  switch (cdiv(D, 32)) {
    case 1: launch_fwd<32>(a, grid, split); break;
    case 2: launch_fwd<64>(a, grid, split); break;
    case 3: launch_fwd<96>(a, grid, split); break;
    default: launch_fwd<128>(a, grid, split); break;
  }
  if ((rc = check_launch("window_fwd")) != TJH_OK || !split) return rc;
  const int64_t n4 = rows * D / 4;
  tjh_launch(k_win_merge, dim3((unsigned)cdiv(n4, 256)), dim3(256), 0, stream(), a, n4, 0);
  return check_launch("window_merge");
}

int tjh_window_backward(const float* q, const float* k, const float* v, const float* o,
                        const float* do_, const float* lse, float* dq, float* dk, float* dv,
                        int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t D,
                        const int64_t* const* strides, float scale, int64_t window,
                        int64_t sinks) {
  TJH_REQUIRE_INIT();
  TJH_ARG(strides, "tjh_window_backward: NULL strides");
  const void* ptrs[8] = {q, k, v, o, do_, dq, dk, dv};
  int rc = check_window("tjh_window_backward", B, H, Hkv, Tq, Tk, D, window, sinks, ptrs, strides, 8);
  if (rc != TJH_OK || B == 0 || H == 0 || Tq == 0) return rc;
  TJH_ARG(lse, "tjh_window_backward: NULL pointer");
  WinArgs a = win_args(H, Hkv, Tq, Tk, D, scale, window, sinks);
  a.q = q; a.k = k; a.v = v; a.o = o; a.dout = do_; a.lse = lse; a.out = dk; a.out2 = dv;
  a.qs = s3(strides[0]); a.ks = s3(strides[1]); a.vs = s3(strides[2]); a.os = s3(strides[3]);
  a.gs = s3(strides[4]); a.o1s = s3(strides[6]); a.o2s = s3(strides[7]);
  Scratch ds((size_t)(B * H * Tq) * sizeof(float));
  if (!ds.ok()) return set_error(TJH_ERR_OOM, "tjh_window_backward: no scratch");
  a.dsum = ds.as<float>();
  KernelScope ks("window_bwd");
  if ((rc = attn_dsum(do_, o, strides[4], strides[3], B, H, Tq, D, ds.as<float>())) != TJH_OK)
    return rc;
  a.nqt = (int)cdiv(Tq, TILE);
  a.nkt = (int)cdiv(Tk, TILE);
  // the window tiles of 32 queries: window + 31 keys from anywhere in a tile
  const int64_t wt = cdiv((int64_t)a.win + 30, TILE) + 1;
  a.nsl = (int)(a.nst + (wt < a.nkt ? wt : a.nkt));
  a.nblk = (int)cdiv(Tk, PROWS);
  a.nsb = (int)cdiv(a.sinks, PROWS);
  // steps (32 queries of a head) of a key block without sinks, at most
  const int64_t tiles = cdiv((int64_t)a.win + PROWS, TILE) + 1;
  const int64_t tq = tiles < a.nqt ? tiles : a.nqt;
  // key heads at once: the dS blocks of all of them up to 4 GiB
  const int64_t nbkv = B * Hkv;
  const size_t per = (size_t)a.G * a.nqt * a.nsl * (TILE * TILE) * sizeof(float);
  int64_t chunk = (int64_t)((size_t(4) << 30) / per);
  chunk = chunk < 1 ? 1 : chunk > nbkv ? nbkv : chunk;
  for (;;) {
    a.nsplit = key_splits(a, chunk, tq);
    // slices of the sinks' blocks about as long as the others' steps
    const int64_t each = cdiv(tq * a.G, a.nsplit);
    a.nslice = a.nsb ? (int)cdiv((int64_t)a.nqt * a.G, each < 8 ? 8 : each) : 1;
    a.nbkv = (int)chunk;
    const int64_t rest = a.nsplit > 1
                             ? (int64_t)2 * a.nsplit * chunk * (a.nblk - a.nsb) * PROWS * D : 0;
    const size_t room = (size_t)(sums_at(a) + rest) * sizeof(float);
    Scratch blocks(per * chunk);
    Scratch sums(room);
    if (!blocks.ok() || (room && !sums.ok())) {
      if (chunk == 1) return set_error(TJH_ERR_OOM, "tjh_window_backward: no scratch");
      chunk = cdiv(chunk, 2);
      continue;
    }
    a.dsblk = blocks.as<float>();
    a.sums = sums.as<float>();
    for (int64_t at = 0; at < nbkv; at += chunk) {
      a.bkv0 = (int)at;
      a.nbkv = (int)(nbkv - at < chunk ? nbkv - at : chunk);
      const int64_t keys =
          (int64_t)a.nbkv * (a.nsb * a.nslice + (a.nblk - a.nsb) * (int64_t)a.nsplit);
      TJH_ARG(keys < (int64_t(1) << 24), "tjh_window_backward: too large");
      switch (cdiv(D, 32)) {
        case 1: rc = launch_bwd<32>(a, (unsigned)keys, dq, strides[5]); break;
        case 2: rc = launch_bwd<64>(a, (unsigned)keys, dq, strides[5]); break;
        case 3: rc = launch_bwd<96>(a, (unsigned)keys, dq, strides[5]); break;
        default: rc = launch_bwd<128>(a, (unsigned)keys, dq, strides[5]); break;
      }
      if (rc != TJH_OK) return rc;
    }
    return TJH_OK;
  }
}

}  // extern "C"
