// One row of floats per workgroup, held in registers, with the block-wide
// counts, scans and the selection of its largest values that the vocabulary
// operators (topk.hip, sample_logits.hip, distill.hip) share.  Device only.
//
// Layout: the row's 16-byte aligned chunks of four go round the threads, so
// every load is a whole chunk whatever the row's alignment and chunk order is
// index order; the up to three elements before the first chunk and after the
// last one are an extra element of the first six threads.  Rows that outgrow
// the registers (NV == 0) are read again on every pass, from the L2s only
// while the rows in flight fit them.
#pragma once

#include "common.h"
#include "wave.h"

namespace tjh {
namespace rowreg {

typedef unsigned long long u64;

// Unsigned integer in the order of the floats, -0 and +0 equal; NaN has the
// key `nan`, above or below all others.
constexpr uint32_t kNanFirst = 0xffffffffu, kNanLast = 1u;
__device__ __forceinline__ uint32_t order_key(float x, uint32_t nan = kNanFirst) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes +0
  const uint32_t k = (u >> 31) ? ~u : (u | 0x80000000u);
  return x != x ? nan : k;
}
// the float of a number's key
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

// (value, index) as one integer: larger values first, of equal ones the
// lower index.
__device__ __forceinline__ u64 composite(uint32_t key, int i) {
  return ((u64)key << 32) | (uint32_t)~(uint32_t)i;
}
__device__ __forceinline__ int index_of(u64 c) { return (int)~(uint32_t)c; }

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
constexpr int kBufferFlags = 0x00020000;  // 32-bit data, raw addressing (gfx9)
constexpr uint32_t kNegInf = 0xff800000u;

template <int T, int NV>
struct Row {
  float v[NV > 0 ? 4 * NV : 1];
  float edge;      // the extra element
  int edge_index;  // and its place in the row
  const float* p;
  uint32_t sign;   // flipped in every element: 0x80000000 looks for the smallest
  int n, head, n4; // elements, of them before the first chunk; chunks

  __device__ __forceinline__ float at(int i) const {
    return __uint_as_float(__float_as_uint(p[i]) ^ sign);
  }

  // `any` alignment: chunks from the first element on, so that what a thread
  // holds goes by the elements' places alone (equal rows sum to equal bits)
  __device__ __forceinline__ void load(const float* row, int cols, uint32_t flip = 0,
                                       bool any = false) {
    p = row;
    n = cols;
    sign = flip;
    head = any ? 0 : min(cols, (int)((16 - ((uintptr_t)row & 15)) & 15) / 4);
    n4 = (n - head) >> 2;
    const int t = threadIdx.x, tail = (n - head) & 3;
    edge_index = t < 3 ? (t < head ? t : -1) : (t - 3 < tail ? head + 4 * n4 + t - 3 : -1);
    if constexpr (NV > 0) {
      // bounds-checked loads (chunks past the end give zeros), whose address
      // is one register for all of them
      const auto res = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<float*>(p + head), 0, 16 * n4, kBufferFlags);
      uint4v x[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j)
        x[j] = __builtin_amdgcn_raw_buffer_load_b128(res, 16 * t, 16 * j * T, 0);
      edge = edge_index >= 0 ? at(edge_index) : -INFINITY;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const uint32_t past = t + j * T < n4 ? 0u : kNegInf;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[4 * j + u] = __uint_as_float((x[j][u] ^ sign) | past);
      }
    } else {
      edge = edge_index >= 0 ? at(edge_index) : -INFINITY;
    }
  }

  // place in the row of element u of this thread's j-th chunk; j < 0: the
  // extra element's.  Not in [0, n): a place past the row.
  __device__ __forceinline__ int index(int j, int u) const {
    return j < 0 ? edge_index : head + 4 * ((int)threadIdx.x + j * T) + u;
  }
  __device__ __forceinline__ bool inside(int j, int u) const {
    return j < 0 ? edge_index >= 0 : (int)threadIdx.x + j * T < n4;
  }

  // f(j, u, x) for the extra element (j = -1), then for each element u of
  // this thread's j-th chunk; places past the row hold -infinity
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    f(-1, 0, edge);
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) f(j, u, v[4 * j + u]);
    } else {
      const int t = threadIdx.x;
      for (int j = 0; t + j * T < n4; j += 2) {  // two chunks' loads at a time
        const bool both = t + (j + 1) * T < n4;
        const uint4v x = *reinterpret_cast<const uint4v*>(p + head + 4 * (t + j * T));
        const uint4v y =
            *reinterpret_cast<const uint4v*>(p + head + 4 * (t + (both ? j + 1 : j) * T));
#pragma unroll
        for (int u = 0; u < 4; ++u) f(j, u, __uint_as_float(x[u] ^ sign));
        if (both) {
#pragma unroll
          for (int u = 0; u < 4; ++u) f(j + 1, u, __uint_as_float(y[u] ^ sign));
        }
      }
    }
  }
};

// Sum over the wave, in every lane.
template <int CTRL>
__device__ __forceinline__ u64 dpp_u64(u64 v) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xF, 0xF, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, 0xF, 0xF, false);
  return ((u64)(uint32_t)hi << 32) | (uint32_t)lo;
}
__device__ __forceinline__ u64 lane_u64(u64 v, int lane) {
  return ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
  v += dpp_u64<kDppXor1>(v);
  v += dpp_u64<kDppXor2>(v);
  v += dpp_u64<kDppRor4>(v);
  v += dpp_u64<kDppRor8>(v);
  return lane_u64(v, 0) + lane_u64(v, 16) + lane_u64(v, 32) + lane_u64(v, 48);
}

// Inclusive sums over the lanes by the DPP network: within rows of 16, then
// their last lanes' to the rows after them.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_shift(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_shift(u64 v) {
  const int lo = dpp_shift<CTRL, ROWS>((int)(uint32_t)v);
  const int hi = dpp_shift<CTRL, ROWS>((int)(v >> 32));
  return ((u64)(uint32_t)hi << 32) | (uint32_t)lo;
}
template <class V>
__device__ __forceinline__ V wave_scan(V v) {
  v += dpp_shift<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
  v += dpp_shift<0x112, 0xF>(v);
  v += dpp_shift<0x114, 0xF>(v);
  v += dpp_shift<0x118, 0xF>(v);
  v += dpp_shift<0x142, 0xA>(v);  // row_bcast:15 to rows 1 and 3
  v += dpp_shift<0x143, 0xC>(v);  // row_bcast:31 to rows 2 and 3
  return v;
}
__device__ __forceinline__ int last_lane(int v) { return __builtin_amdgcn_readlane(v, 63); }
__device__ __forceinline__ u64 last_lane(u64 v) { return lane_u64(v, 63); }

// Block-wide operations, one barrier each: consecutive ones use the two
// halves of `sm` in turn, so nobody writes a half that is still being read.
template <int T>
struct Block {
  static constexpr int W = T / 64;
  u64* sm;  // [2 * W]
  int half;
  __device__ __forceinline__ explicit Block(u64* s) : sm(s), half(0) {}

  // op over every wave's value, in wave order; the same in every thread
  template <class V, class C>
  __device__ __forceinline__ V across(V v, C op) {
    if (W == 1) return v;
    V* s = reinterpret_cast<V*>(sm + half * W);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    half ^= 1;
    V r = s[0];
#pragma unroll
    for (int i = 1; i < W; ++i) r = op(r, s[i]);
    return r;
  }
  __device__ __forceinline__ float max(float v) { return across(wave_max(v), MaxOp{}); }
  __device__ __forceinline__ float sum(float v) { return across(wave_sum(v), AddOp{}); }
  __device__ __forceinline__ u64 sum64(u64 v) {
    return across(wave_sum_u64(v), [](u64 x, u64 y) { return x + y; });
  }
  __device__ __forceinline__ bool any(bool p) {
    return across((int)(__ballot(p) != 0), [](int x, int y) { return x | y; }) != 0;
  }
  __device__ __forceinline__ int sum_i(int v) {
    return across(last_lane(wave_scan(v)), [](int x, int y) { return x + y; });
  }
  // sum of v over the threads before this one; total in *all
  template <class V>
  __device__ __forceinline__ V before(V v, V* all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const V incl = wave_scan(v);
    if (W == 1) {
      *all = last_lane(incl);
      return incl - v;
    }
    V* s = reinterpret_cast<V*>(sm + half * W);
    if (lane == 63) s[w] = incl;
    __syncthreads();
    half ^= 1;
    V base = 0, tot = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i == w) base = tot;
      tot += s[i];
    }
    *all = tot;
    return base + incl - v;
  }
};

constexpr int kRank = 256;  // longest list sorted by counting

template <int N>
struct Int {
  static constexpr int value = N;
};

// LDS of a selection: a list of CAP composites, room for the short sort, and
// the block operations' slots.
template <int T, int CAP>
struct SelectLds {
  u64 list[CAP];
  u64 sorted[kRank];
  int rank[kRank];
  int count;
  u64 sm[2 * (T / 64)];
};

// list[0, c) in descending order in s.sorted, c <= 256: each thread counts the
// items above one of them (c * c / T comparisons, three barriers), eight of
// them read at a time: the list has room for 256 and is padded with zeros,
// which no item is below.
template <int T, int CAP>
__device__ __forceinline__ void sort_short(u64* list, int c, SelectLds<T, CAP>& s) {
  int pad = 64;
  while (pad < c) pad <<= 1;
  const int ng = T >= pad ? T / pad : 1;  // threads an item
  const int end = (c + 8 * ng - 1) / (8 * ng) * (8 * ng);  // <= 256
  for (int i = threadIdx.x; i < c; i += T) s.rank[i] = 0;
  for (int i = c + threadIdx.x; i < end; i += T) list[i] = 0;
  __syncthreads();  // ranks cleared, list written
  const auto above = [&](u64 me, int g) {
    int r = 0;
    for (int j = g; j < end; j += 8 * ng) {
      u64 x[8];
#pragma unroll
      for (int v = 0; v < 8; ++v) x[v] = list[j + v * ng];
#pragma unroll
      for (int v = 0; v < 8; ++v) r += x[v] > me;
    }
    return r;
  };
  if (T >= pad) {
    const int i = threadIdx.x & (pad - 1);
    if (i < c) {
      const int r = above(list[i], threadIdx.x / pad);
      if (ng > 1) atomicAdd(&s.rank[i], r);
      else s.rank[i] = r;
    }
  } else {
    for (int i = threadIdx.x; i < c; i += T) s.rank[i] = above(list[i], 0);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < c; i += T) s.sorted[s.rank[i]] = list[i];
  __syncthreads();
}

// s.list[0, c) in descending order in place, c <= min(T * M, 2048): runs of 64
// by counting, eight of them at a time into runs of 512, those into one.  An
// item's place is the number of items above it in each run, by bisection, a
// run's reads in flight with the others'.  Padded to whole 512s with numbers
// below every item, in order.
template <int M, int T, int CAP>
__device__ __forceinline__ void sort_runs(SelectLds<T, CAP>& s, int c) {
  u64* list = s.list;
  const int p = (c + 511) & ~511;
  for (int i = c + threadIdx.x; i < p; i += T) list[i] = p - i;
  __syncthreads();
  u64 x[M];
  int to[M];
  // rank(i, x): its place; those from c's run (of `run`) on stand already
  const auto pass = [&](int run, auto rank) {
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int i = threadIdx.x + m * T;
      if (i >= p || (i & ~(run - 1)) >= c) continue;
      x[m] = list[i];
      to[m] = rank(i, x[m]);
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int i = threadIdx.x + m * T;
      if (i < p && (i & ~(run - 1)) < c) list[to[m]] = x[m];
    }
    __syncthreads();
  };
  pass(64, [&](int i, u64 me) {
    int r = i & ~63;
    const u64* from = list + r;
#pragma unroll 1
    for (int j = 0; j < 64; j += 8) {
      u64 y[8];
#pragma unroll
      for (int v = 0; v < 8; ++v) y[v] = from[j + v];
#pragma unroll
      for (int v = 0; v < 8; ++v) r += y[v] > me;
    }
    return r;
  });
  const auto above = [&](auto runs, int first, int len, u64 me) {
    constexpr int G = decltype(runs)::value;
    int at[G];
#pragma unroll
    for (int v = 0; v < G; ++v) at[v] = first + v * len;
#pragma unroll 1
    for (int h = len >> 1; h > 0; h >>= 1) {
      u64 y[G];
#pragma unroll
      for (int v = 0; v < G; ++v) y[v] = list[at[v] + h - 1];
#pragma unroll
      for (int v = 0; v < G; ++v) at[v] += y[v] > me ? h : 0;
    }
    int r = first;
#pragma unroll
    for (int v = 0; v < G; ++v) r += at[v] - (first + v * len) + (list[at[v]] > me);
    return r;
  };
  pass(512, [&](int i, u64 me) { return above(Int<8>{}, i & ~511, 64, me); });
  if (p <= 512) return;
  pass(2048, [&](int, u64 me) {
    return p == 1024   ? above(Int<2>{}, 0, 512, me)
           : p == 1536 ? above(Int<3>{}, 0, 512, me)
                       : above(Int<4>{}, 0, 512, me);
  });
}

// s.list[0, c) in descending order: where it stands.  Up to 256 items
// by counting alone, up to 2048 of several waves by runs (300 items: 6 us
// less, 1400: 12); else by a bitonic network in place over the next power of
// two, padded with zeros, which no real item is below (c log^2 c / 4 T exchanges, log^2 c / 2 rounds).  Its pairs of a
// wave's 64 threads stay within 128 items while the distance is 64 or less,
// so that barriers stand only around the rounds of larger ones.
template <int T, int CAP>
__device__ __forceinline__ u64* sort_list(SelectLds<T, CAP>& s, int c) {
  static_assert((CAP & (CAP - 1)) == 0 && CAP >= 2 * kRank, "padded to a power of two");
  if (c <= kRank) {
    sort_short(s.list, c, s);
    return s.sorted;
  }
  if constexpr (T > 64) {
    if (c <= 2048) {
      sort_runs<2048 / T>(s, c);
      return s.list;
    }
  }
  int p = 2 * kRank;
  while (p < c) p <<= 1;  // <= CAP
  for (int i = c + threadIdx.x; i < p; i += T) s.list[i] = 0;
  __syncthreads();
  for (int len = 2; len <= p; len <<= 1) {
    for (int o = len >> 1; o >= 1; o >>= 1) {
      for (int q = threadIdx.x; q < p / 2; q += T) {
        const int i = 2 * q - (q & (o - 1));  // the pair (i, i + o)
        const u64 x = s.list[i], y = s.list[i + o];
        const bool down = (i & len) == 0;  // descending run
        if ((x < y) == down) {
          s.list[i] = y;
          s.list[i + o] = x;
        }
      }
      const int next = o > 1 ? o >> 1 : len;
      if (o > 64 || next > 64) {
        __syncthreads();
      } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
  return s.list;
}

// The elements for which in(j, u, x) holds into the list, in no order (it is
// sorted next): their number, of which the first CAP were stored.  The first
// barrier is for callers that chose this by reading s.count: all waves have
// read it before it is cleared.
template <int T, int CAP, class In>
__device__ __forceinline__ int gather_list(const Row<T, 0>& row, uint32_t nan, In in,
                                           SelectLds<T, CAP>& s) {
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  row.each([&](int j, int u, float x) {
    if (in(j, u, x) && row.inside(j, u)) {
      const int at = atomicAdd(&s.count, 1);
      if (at < CAP) s.list[at] = composite(order_key(x, nan), row.index(j, u));
    }
  });
  __syncthreads();
  return s.count;
}

// The same for the elements that are not below `bound`, some ten or hundred of
// the row, straight from the registers.
template <int T, int NV, int CAP>
__device__ __forceinline__ int gather_above(const Row<T, NV>& row, uint32_t nan, float bound,
                                            SelectLds<T, CAP>& s) {
  if constexpr (NV == 0) {
    return gather_list(row, nan, [&](int, int, float x) { return !(x < bound); }, s);
  } else {
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
    const auto put = [&](int j, int u, float x) {
      if (!(x < bound) && row.inside(j, u)) {
        const int to = atomicAdd(&s.count, 1);
        if (to < CAP) s.list[to] = composite(order_key(x, nan), row.index(j, u));
      }
    };
    put(-1, 0, row.edge);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      // the maximum that NaN is larger than everything for
      const float x = __builtin_elementwise_maximum(
          __builtin_elementwise_maximum(row.v[4 * j], row.v[4 * j + 1]),
          __builtin_elementwise_maximum(row.v[4 * j + 2], row.v[4 * j + 3]));
      if (!(x < bound)) {
#pragma unroll
        for (int u = 0; u < 4; ++u) put(j, u, row.v[4 * j + u]);
      }
    }
    __syncthreads();
    return s.count;
  }
}

// (x, index) as they are
__device__ __forceinline__ u64 pair_of(float x, int i) {
  return ((u64)__float_as_uint(x) << 32) | (uint32_t)i;
}
__device__ __forceinline__ float pair_value(u64 e) { return __uint_as_float((uint32_t)(e >> 32)); }
__device__ __forceinline__ int pair_index(u64 e) { return (int)(uint32_t)e; }

// Pairs of the elements that are not below `bound`, above -infinity, of a row
// without NaN into the list, if it holds them: their number.  They are counted
// first, so that each thread knows its places: an 11th of a row's elements
// would wait for each other's increments of one count.
template <int T, int NV, int CAP>
__device__ __forceinline__ int gather_pairs(const Row<T, NV>& row, float bound,
                                            SelectLds<T, CAP>& s, Block<T>& b) {
  int at = 0, total = 0;
  row.each([&](int, int, float x) { at += x >= bound; });
  at = b.before(at, &total);
  if (total > CAP) return total;
  asm volatile("" : "+v"(bound));  // compared anew: else every comparison's mask is kept
  const auto put = [&](int j, int u, float x) {
    if (x >= bound) s.list[at++] = pair_of(x, row.index(j, u));
  };
  if constexpr (NV == 0) {
    row.each(put);
  } else {
    put(-1, 0, row.edge);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float x = __builtin_elementwise_maximum(
          __builtin_elementwise_maximum(row.v[4 * j], row.v[4 * j + 1]),
          __builtin_elementwise_maximum(row.v[4 * j + 2], row.v[4 * j + 3]));
      if (x >= bound) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float x = row.v[4 * j + u];
          asm volatile("" : "+v"(x));  // a copy: else every value of the row takes half a pair
          put(j, u, x);
        }
      }
    }
  }
  __syncthreads();
  return total;
}

// The index of the need-th element (in index order, need >= 1) of those for
// which in(j, u, x) holds, by bisection: log2(n) passes.  Passes over memory
// here and below: over the registers they would keep an index and a mask of
// every element besides.
template <int T, class In>
__device__ __forceinline__ int nth_index(const Row<T, 0>& row, int need, In in, Block<T>& b) {
  int lo = 0;  // fewer than `need` of them lie before lo
  for (int bit = 31 - __builtin_clz((unsigned)row.n); bit >= 0; --bit) {
    const int c = lo + (1 << bit);
    if (c > row.n) continue;  // the same for every thread
    int m = 0;
    row.each([&](int j, int u, float x) {
      m += row.inside(j, u) && row.index(j, u) < c && in(j, u, x);
    });
    if (b.sum_i(m) < need) lo = c;
  }
  return lo;
}

// The composite of the row's k-th largest element (1 <= k <= n) by bisection
// over the keys, then over the indices of the elements that share the key:
// for rows with more near-ties than the list holds, and for any k.
template <int T>
__device__ __forceinline__ u64 kth_by_bisection(const Row<T, 0>& row, int k, uint32_t nan,
                                                Block<T>& b) {
  const auto key = [&](int j, int u, float x) {  // 0: no element
    return row.inside(j, u) ? order_key(x, nan) : 0u;
  };
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = t | (1u << bit);
    int m = 0;
    row.each([&](int j, int u, float x) { m += key(j, u, x) >= c; });
    if (b.sum_i(m) >= k) t = c;
  }
  int above = 0;
  row.each([&](int j, int u, float x) { above += key(j, u, x) > t; });
  const int need = k - b.sum_i(above);  // of the elements with key t, >= 1
  return composite(
      t, nth_index(row, need, [&](int j, int u, float x) { return key(j, u, x) == t; }, b));
}

// A bound that the row's k largest elements are not below and few others are
// either: the k-th largest of the threads' own maxima (four of each thread),
// to the 16 high bits of its key, found two at a time; -infinity where there
// are fewer maxima.  50 of 50257 random values leave about 55.
template <int T, int NV>
__device__ __forceinline__ float kth_bound(const Row<T, NV>& row, int k, Block<T>& b) {
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  // NaN takes no part: still a lower bound
  row.each([&](int, int u, float x) { mx[u] = fmaxf(mx[u], x); });
  uint32_t mk[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) mk[u] = order_key(mx[u]);
  uint32_t lo = 0;
#pragma unroll 1
  for (int bit = 30; bit >= 16; bit -= 2) {  // counts of three bounds a round
    u64 c = 0;
#pragma unroll
    for (int i = 3; i >= 1; --i) {
      const uint32_t bound = lo | ((uint32_t)i << bit);
      int n = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) n += __popcll(__ballot(mk[u] >= bound));
      c = (c << 20) | (u64)n;
    }
    c = b.across(c, [](u64 x, u64 y) { return x + y; });
    uint32_t digit = 0;
#pragma unroll
    for (int i = 1; i <= 3; ++i)
      if ((int)((c >> (20 * (i - 1))) & 0xfffff) >= k) digit = i;
    lo |= digit << bit;
  }
  return lo > 0x007fffffu ? key_value(lo) : -INFINITY;  // 0x007fffff: the key of -infinity
}

// The row's k largest elements in order, 1 <= k <= min(n, CAP): where they
// stand, given a bound that they are not below.
// Where more than CAP elements are above the bound (ties), the exact one
// comes from bisection.
template <int T, int NV, int CAP>
__device__ __forceinline__ u64* select_above(const Row<T, NV>& row, int k, float bound,
                                             uint32_t nan, SelectLds<T, CAP>& s, Block<T>& b) {
  const int c = gather_above(row, nan, bound, s);
  if (c > CAP) {
    Row<T, 0> again;
    again.load(row.p, row.n, row.sign);
    const u64 thr = kth_by_bisection(again, k, nan, b);
    gather_list(
        again, nan,
        [&](int j, int u, float x) {
          return composite(order_key(x, nan), again.index(j, u)) >= thr;
        },
        s);
  }
  return sort_list(s, c > CAP ? k : c);
}

template <int T, int NV, int CAP>
__device__ __forceinline__ u64* select_largest(const Row<T, NV>& row, int k, uint32_t nan,
                                               SelectLds<T, CAP>& s, Block<T>& b) {
  return select_above(row, k, kth_bound(row, k, b), nan, s, b);
}

}  // namespace rowreg
}  // namespace tjh
