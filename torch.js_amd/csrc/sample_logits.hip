// Sampling of one index a row from logits, with temperature, top-k, top-p and
// min-p, from given uniform numbers (F.sample_logits; beside
// Tensor.multinomial, src/tensor/Tensor.ts:271-359, which takes
// probabilities and the whole row).
//
// Definition.  m the row's largest logit, w_i = exp((x_i - m) / temperature).
// In the order of descending x (equal ones by ascending index) the kept
// elements are the first top_k; of these, the ones before which less than
// top_p of their weight lies; of these, the ones with x_i - m >= temperature
// * ln(min_p).  Each rule keeps a prefix of the order and each keeps the
// first element.  The draw is the first kept index (in index order) whose
// running sum of weights exceeds u times their sum.
// temperature that is not > 0: the first index of the largest logit.  A row
// with NaN, +infinity or nothing above -infinity draws -1.
//
// Weights are integers, w_i * 2^s with the row's sum below 2^62 (s = 46 at
// 50257 columns): sums are then the same in whatever order the atomics and
// the waves add them, exact, and finer than 32-bit floats by 2^22.  They are
// formed in 64 bits as 2^(k / 32) 2^(f / 32), |f| <= 1 / 2, from a table and
// the first six terms of the second (the seventh is below 2^-48): 32-bit ones
// would move one draw in some thousand over a border between two indices.  A
// weight below half of 2^-s counts as 0.
//
// One workgroup has a row, in registers (rowreg.h).  Wherever the elements
// that can be drawn fit (8192), they are moved into LDS and everything else
// happens on that list: the top_k largest; the elements above min_p's bound;
// the nucleus, which ends in a bin of a histogram of the weights over x (one
// pass in which every element's weight is formed).  Only the nucleus's last
// bin and the part of the list around the draw are sorted: lists longer than
// 256 are added up by parts of the index range first.  Larger sets are a
// bound on (x, index), and passes that add the kept weights up by runs of the
// index range, one a wave, and look into one.
//
// Bound by the work of a row on its one CU, far from memory (10 us for 256
// rows of 50257).  Up to 256 rows of 50257: greedy 7 us (the load and the
// maximum), top_k 50 15, min_p 0.01 16, no rule 27 (of it some 12 the
// weights, 31 instructions each on four SIMDs), top_k 1000 38, top_p 0.9 40; of
// 32001, top_p 0.9 32.  4096 rows of 4000: top_k 50 80 us, top_p 0.9 119.
// 256 rows of 128256, outside the registers: top_k 50 66 us, no rule 69, top_p
// 0.9 160.  A row with fewer than top_k logits above -infinity leaves the list
// for topk.hip's bisection: 302 us with 30 of 50257 and top_k 50.
#include "rowreg.h"

#include <float.h>
#include <math.h>

namespace tjh {
namespace {

using namespace rowreg;

constexpr int kMostK = 1024;  // top_k that is selected by the threads' maxima
constexpr int64_t kMaxCols = int64_t(1) << 20;

struct SampleArgs {
  const float* x;
  int64_t ld;
  int n;
  const float* u;
  // one value a row, or null and the same for all
  const float *temperature, *top_p, *min_p;
  const int32_t* top_k;
  double t0, p0, m0;
  int64_t k0;
  int32_t* out;
};

// kCap: elements of a list, kBins: of the nucleus's histogram.
template <int T, int kCap, int kBins>
struct SampleLds {
  SelectLds<T, kCap> s;
  u64 bins[kBins];
  u64 w[kCap];     // weights of the list
  u64 few[kRank];  // a part of the list
  double pow2[32];  // 2^(i / 32 + s)
  u64 edge_w[6];
  u64 first;
  int pick;
};

// Weights of a row: 2^(d * per_t + s) rounded to an integer, d = x - m <= 0
// (NaN: 0), s <= 51.  Constants are scalar registers of their own: literals
// would each be moved into vector registers for every weight.
struct Weights {
  double m, scale, lowest, magic, c1, c2, c3, c4, c5, top;
  const double* pow2;
  __device__ __forceinline__ Weights(double max, double per_t, const double* table)
      : m(max), scale(per_t * 32.0), pow2(table) {
    constexpr double l = 6.93147180559945286e-01 / 32;  // 2^(f / 32) = sum (l f)^k / k!
    lowest = -2048.0 / scale;      // 2^(51 - 64) is 0
    magic = 6755399441055744.0;    // 1.5 * 2^52: its low word takes the integer
    top = 4503599627370496.0;      // 2^52: the integer is in the low 52 bits
    c1 = l;
    c2 = l * l / 2;
    c3 = l * l * l / 6;
    c4 = l * l * l * l / 24;
    c5 = l * l * l * l * l / 120;
    asm volatile("" : "+s"(magic), "+s"(top), "+s"(c1), "+s"(c2), "+s"(c3), "+s"(c4), "+s"(c5));
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    const double d = fmax((double)x - m, lowest);
    const double kd = __builtin_fma(d, scale, magic);
    const int k = (int)__double_as_longlong(kd);
    const double f = __builtin_fma(d, scale, -(kd - magic));  // |f| <= 1 / 2
    const double tab = pow2[k & 31];
    double e = __builtin_fma(f, c5, c4);
    e = __builtin_fma(f, e, c3);
    e = __builtin_fma(f, e, c2);
    e = __builtin_fma(f, e, c1);
    e = __builtin_fma(tab * f, e, tab);
    // times 2^(k >> 5): normal numbers of 2^-14 to 2^52
    e = __hiloint2double(__double2hiint(e) + ((k & ~31) << 15), __double2loint(e)) + top;
    return (u64)__double_as_longlong(e) & 0xfffffffffffffull;
  }
};

// A float that is not above x, nor far below it.
__device__ __forceinline__ float float_below(double x) {
  const float f = (float)x;
  return f - (fabsf(f) * 2.4e-7f + FLT_MIN);
}

// f(x0, x1, x2, x3) for each chunk of the row and its extra element (with
// -infinity), a chunk's work kept together: that of all of them at once would
// take more registers than there are.
template <int T, int NV, class F>
__device__ __forceinline__ void each_four(const Row<T, NV>& row, F f) {
  f(row.edge, -INFINITY, -INFINITY, -INFINITY);
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      if (j * T < row.n4) f(row.v[4 * j], row.v[4 * j + 1], row.v[4 * j + 2], row.v[4 * j + 3]);
    }
    __builtin_amdgcn_sched_barrier(0);
  } else {
#pragma unroll 2
    for (int c = threadIdx.x; c < row.n4; c += T) {
      const float4 x = *reinterpret_cast<const float4*>(row.p + row.head + 4 * c);
      f(x.x, x.y, x.z, x.w);
    }
  }
}

// f(i, list[i]) for i < c, four of a thread's items at a time, their reads
// together.
template <int T, class F>
__device__ __forceinline__ void each_listed_of(const u64* list, int c, F f) {
  for (int i0 = threadIdx.x; i0 < c; i0 += 4 * T) {
    u64 e[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) e[v] = list[min(i0 + v * T, c - 1)];
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (i0 + v * T < c) f(i0 + v * T, e[v]);
  }
}

// (~index, place in the list) of a pair: in descending order by the index
__device__ __forceinline__ u64 by_index(u64 e, int i) {
  return ((u64)(uint32_t)~pair_index(e) << 32) | (uint32_t)i;
}

template <int T, int NV>
__global__ __launch_bounds__(T) void k_sample(SampleArgs a) {
  // rows of 4096 at most: two workgroups fit a CU
  constexpr int kCap = T == 256 ? 4096 : 8192, kBins = T == 256 ? 1024 : 2048;
  __shared__ SampleLds<T, kCap, kBins> lds;
  SelectLds<T, kCap>& s = lds.s;
  constexpr int W = T / 64;
  constexpr int kNone = 0x7fffffff;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  Block<T> b(s.sm);
  Row<T, NV> row;
  row.load(a.x + r * a.ld, a.n);
  const int n = a.n;

  const double temp = a.temperature ? (double)a.temperature[r] : a.t0;
  const int64_t top_k = a.top_k ? (int64_t)a.top_k[r] : a.k0;
  const double top_p = a.top_p ? (double)a.top_p[r] : a.p0;
  const double min_p = a.min_p ? (double)a.min_p[r] : a.m0;
  const double u = (double)a.u[r];
  const bool use_k = top_k > 0 && top_k < n, use_p = top_p < 1.0;
  const bool largest = use_k && top_k <= kMostK, cut = use_k && !largest;
  const bool nucleus = use_p && !largest;  // by the histogram

  float mx = -INFINITY, mn = INFINITY;  // mn: the smallest above -infinity, for the nucleus
  uint32_t mag = 0;                     // largest |x| as bits: above infinity's is NaN
  row.each([&](int, int, float x) {
    mx = fmaxf(mx, x);
    const uint32_t u = __float_as_uint(x) << 1;
    mag = u > mag ? u : mag;
  });
  if (nucleus) {
    row.each([&](int, int, float x) { mn = x > -INFINITY ? fminf(mn, x) : mn; });
    for (int i = t; i < kBins; i += T) lds.bins[i] = 0;
  }
  if (t < 32) lds.pow2[t] = ldexp(exp2((double)t / 32), min(51, 62 - (32 - __clz(n))));
  if (t == 0) lds.pick = kNone;
  mx = __ballot(mag > 0xff000000u) ? INFINITY : wave_max(mx);
  const float2 ends = b.across(make_float2(mx, wave_max(-mn)), [](float2 x, float2 y) {
    return make_float2(fmaxf(x.x, y.x), fmaxf(x.y, y.y));
  });
  mx = ends.x;
  mn = -ends.y;
  if (!(fabsf(mx) < INFINITY)) {
    if (t == 0) a.out[r] = -1;
    return;
  }
  if (!(temp > 0.0)) {
    row.each([&](int j, int u, float x) {
      if (x == mx && row.inside(j, u)) atomicMin(&lds.pick, row.index(j, u));
    });
    __syncthreads();
    if (t == 0) a.out[r] = lds.pick;
    return;
  }
  const double p = top_p > 0.0 ? top_p : 1e-300;  // the first element at least
  const double floor_z = min_p > 0.0 ? fmin(temp * log(min_p), 0.0) : -INFINITY;
  const double m = (double)mx;
  const double per_t = fmax(fmin(1.4426950408889634074 / temp, 1e300), 1e-300);
  const Weights weight(m, per_t, lds.pow2);

  // elements of the order up to (tx, ti) are kept
  float tx = -INFINITY;
  int ti = n;
  const auto in_order = [&](const auto& of, int j, int e, float x) {
    return x > tx || (x == tx && of.index(j, e) <= ti);
  };
  if (cut) {
    Row<T, 0> again;
    again.load(row.p, n);
    const u64 last = kth_by_bisection(again, (int)top_k, kNanFirst, b);
    tx = key_value((uint32_t)(last >> 32));
    ti = index_of(last);
  }
  // the elements that can be drawn are not below `bound`: where that is known
  float bound = -INFINITY;
  double limit = INFINITY;  // weight before an element that is in the nucleus
  const auto bin_of = [&](float per, float x) {  // nondecreasing as x falls
    return (int)fminf((mx - x) * per, (float)(kBins - 1));
  };
  float per = 0.f;
  int last = -1;
  u64 above = 0;  // weight of the bins before `last`
  if (nucleus) {
    // weights by bins of m - x, out to weights of e^-24 or the smallest x
    per = (float)(kBins / fmax(fmin(24.0 * temp, m - (double)mn), 1e-30));
    if (!cut) {
      each_four(row, [&](float x0, float x1, float x2, float x3) {
        const float x[4] = {x0, x1, x2, x3};
        u64 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = weight(x[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (w[e]) atomicAdd(&lds.bins[bin_of(per, x[e])], w[e]);
      });
    } else {
      Row<T, 0> again;
      again.load(row.p, n);
      again.each([&](int j, int e, float x) {
        const u64 w = in_order(again, j, e, x) ? weight(x) : 0;
        if (w) atomicAdd(&lds.bins[bin_of(per, x)], w);
      });
    }
    if (t == 0) lds.pick = -1;
    __syncthreads();
    // the last bin before which less than the limit lies
    constexpr int kEach = (kBins + T - 1) / T;
    u64 mine = 0, all;
#pragma unroll
    for (int i = 0; i < kEach; ++i) mine += lds.bins[t * kEach + i];
    above = b.before(mine, &all);
    limit = p * (double)all;
    int found = -1;
    u64 before = above;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const u64 w = lds.bins[t * kEach + i];
      if (w && (double)before < limit) {
        found = t * kEach + i;
        above = before;
      }
      before += w;
    }
    if (found >= 0) atomicMax(&lds.pick, found);
    __syncthreads();
    if (lds.pick == found) lds.first = above;  // one thread: the bins are its own
    __syncthreads();
    above = lds.first;
    last = lds.pick;
    // elements of later bins that are not below it do no harm
    if (last < kBins - 1) bound = float_below(m - (last + 1.01) / per);
  } else if (!largest && floor_z > -INFINITY) {
    bound = float_below(m + floor_z);
  }
  int c = -1;  // elements of the list, if there is one
  u64* list = s.list;
  if (bound > -INFINITY) c = gather_pairs(row, bound, s, b);
  if (c > kCap) c = -1;
  if (largest) {
    list = select_largest(row, (int)top_k, kNanFirst, s, b);
    c = (int)top_k;
  } else if (use_p) {
    // the nucleus ends in bin `last`: (tx, ti) from that bin's elements
    if (t == 0) s.count = 0;
    __syncthreads();
    each_listed_of<T>(s.list, c, [&](int, u64 e) {
      const float x = pair_value(e);
      if (bin_of(per, x) == last && (x > tx || (x == tx && pair_index(e) <= ti))) {
        const int at = atomicAdd(&s.count, 1);
        if (at < kRank) lds.few[at] = composite(order_key(x), pair_index(e));
      }
    });
    __syncthreads();
    int in = s.count;
    const u64* part = s.sorted;
    if (c >= 0 && in <= kRank) {
      sort_short(lds.few, in, s);
    } else {
      c = -1;  // no list: the bin alone
      Row<T, 0> again;
      again.load(row.p, n);
      in = gather_list(
          again, kNanFirst,
          [&](int j, int e, float x) {
            return bin_of(per, x) == last && x > -INFINITY && in_order(again, j, e, x);
          },
          s);
      if (in <= kCap) part = sort_list(s, in);
    }
    if (in <= kCap) {
      if (t == 0) lds.pick = 0;
      __syncthreads();
      u64 sum = above;
      for (int i0 = 0; i0 < in; i0 += T) {
        const int i = i0 + t;
        const u64 w = i < in ? weight(key_value((uint32_t)(part[i] >> 32))) : 0;
        u64 all;
        const u64 before = sum + b.before(w, &all);
        if (i < in && (double)before < limit) atomicMax(&lds.pick, i);
        sum += all;
      }
      __syncthreads();
      const u64 e = part[lds.pick];
      tx = key_value((uint32_t)(e >> 32));
      ti = index_of(e);
    } else {
      // more elements than the list holds.  All equal: as many of them as
      // there is room for, by index; else the largest composite with at
      // least the limit above it, bit by bit, is the first one outside
      Row<T, 0> again;
      again.load(row.p, n);
      float lo = INFINITY, hi = -INFINITY;
      again.each([&](int j, int e, float x) {
        if (bin_of(per, x) == last && x > -INFINITY && in_order(again, j, e, x)) {
          lo = fminf(lo, x);
          hi = fmaxf(hi, x);
        }
      });
      lo = -b.max(-lo);
      hi = b.max(hi);
      if (lo == hi) {
        // element i of them is in where above + i * w < limit
        const double w = (double)weight(lo);
        int q = (int)ceil((limit - (double)above) / w);
        q = q < 1 ? 1 : q > in ? in : q;
        while (q > 1 && !((double)above + (q - 1) * w < limit)) --q;
        while (q < in && (double)above + q * w < limit) ++q;
        ti = nth_index(
            again, q, [&](int j, int e, float x) { return x == lo && in_order(again, j, e, x); }, b);
        tx = lo;
      } else {
        u64 out = 0;
        for (int bit = 63; bit >= 0; --bit) {
          const u64 cand = out | (u64(1) << bit);
          u64 w = 0;
          again.each([&](int j, int e, float x) {
            if (again.inside(j, e) && in_order(again, j, e, x) &&
                composite(order_key(x), again.index(j, e)) > cand)
              w += weight(x);
          });
          if ((double)b.sum64(w) >= limit) out = cand;
        }
        // the kept elements are the composites above `out`; the last one's
        if (t == 0) lds.first = ~u64(0);
        __syncthreads();
        again.each([&](int j, int e, float x) {
          const u64 at = composite(order_key(x), again.index(j, e));
          if (again.inside(j, e) && at > out) atomicMin(&lds.first, at);
        });
        __syncthreads();
        tx = key_value((uint32_t)(lds.first >> 32));
        ti = index_of(lds.first);
      }
    }
    __syncthreads();  // bins and parts are free
  }

  if (c >= 0) {
    // the list's weights, none for elements that are not kept; those of more
    // than 256 by parts of the index range too
    constexpr int kParts = 1024, kEach = (kParts + T - 1) / T;
    const int shift = max(0, 32 - __clz(n - 1) - 10);  // 2^10 parts
    bool parts = !largest && c > kRank;
    const auto clear = [&]() {
      for (int i = t; i < kParts; i += T) lds.bins[i] = 0;
      if (t == 0) {
        lds.pick = kNone;
        s.count = 0;
      }
      __syncthreads();
    };
    if (parts) clear();
    u64 mine = 0;
    each_listed_of<T>(list, c, [&](int i, u64 e) {
      if (largest) list[i] = e = pair_of(key_value((uint32_t)(e >> 32)), index_of(e));
      const float x = pair_value(e);
      const bool in = largest || ((double)x - m >= floor_z &&
                                  (x > tx || (x == tx && pair_index(e) <= ti)));
      const u64 w = in ? weight(x) : 0;
      lds.w[i] = w;
      mine += w;
      if (parts && w) atomicAdd(&lds.bins[pair_index(e) >> shift], w);
    });
    u64 all = parts ? 0 : b.sum64(mine);
    int keep = c;
    if (largest && (use_p || floor_z > -INFINITY)) {  // a sorted list, to be cut
      if (use_p) limit = p * (double)all;
      int kept = 0;
      u64 sum = 0, mine_kept = 0;
      for (int i0 = 0; i0 < c; i0 += T) {
        const int i = i0 + t;
        const u64 w = i < c ? lds.w[i] : 0;
        u64 part;
        const u64 before = sum + b.before(w, &part);
        sum += part;
        const bool in =
            i < c && (double)before < limit && (double)pair_value(list[i]) - m >= floor_z;
        kept += in;
        mine_kept += in ? w : 0;
      }
      keep = b.sum_i(kept);
      all = b.sum64(mine_kept);
    }
    if (largest && keep > kRank) {
      parts = true;
      __syncthreads();
      clear();
      for (int i = t; i < keep; i += T)
        if (lds.w[i]) atomicAdd(&lds.bins[pair_index(list[i]) >> shift], lds.w[i]);
    }
    double target = u * (double)all;
    u64 sum = 0;  // weight of the indices before the ones looked into
    int in = keep;
    if (parts) {
      // the first part with the target, or, where u is 1 or more, the last of
      // any weight
      __syncthreads();
      u64 own = 0, total;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (T <= kParts || t < kParts) own += lds.bins[t * kEach + i];
      u64 before = b.before(own, &total);
      target = u * (double)total;
      int first = kNone, end = -1;
      u64 start = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const u64 w = lds.bins[t * kEach + i];
        if (w && first == kNone && (double)(before + w) > target) {
          first = t * kEach + i;
          start = before;
        }
        if (w) end = t * kEach + i;
        before += w;
      }
      if (first != kNone) atomicMin(&lds.pick, first);
      __syncthreads();
      int at = lds.pick;
      if (at == kNone) {
        __syncthreads();
        if (t == 0) lds.pick = -1;
        __syncthreads();
        atomicMax(&lds.pick, end);
        __syncthreads();
        at = lds.pick;
        if (end == at) lds.first = total - lds.bins[at];
      } else if (first == at) {
        lds.first = start;
      }
      each_listed_of<T>(list, keep, [&](int i, u64 e) {
        if (pair_index(e) >> shift == at && lds.w[i]) {
          const int put = atomicAdd(&s.count, 1);
          if (put < kRank) lds.few[put] = by_index(e, i);
        }
      });
      __syncthreads();
      sum = lds.first;
      in = s.count;
    } else {
      for (int i = t; i < keep; i += T) lds.few[i] = by_index(list[i], i);
    }
    if (in <= kRank) {
      // (index, place in the list), in ascending order of the index
      if (t == 0) lds.pick = kNone;
      sort_short(lds.few, in, s);
      int end = -1;
      for (int i0 = 0; i0 < in; i0 += T) {
        const int i = i0 + t;
        const u64 w = i < in ? lds.w[(uint32_t)s.sorted[i]] : 0;
        u64 here;
        const u64 before = sum + b.before(w, &here);
        sum += here;
        if (w && (double)(before + w) > target) atomicMin(&lds.pick, i);
        if (w) end = i;
      }
      __syncthreads();
      int at = lds.pick;
      if (at == kNone) {  // the last one of any weight
        __syncthreads();
        if (t == 0) lds.pick = -1;
        __syncthreads();
        atomicMax(&lds.pick, end);
        __syncthreads();
        at = lds.pick;
      }
      if (t == 0) a.out[r] = (int)~(uint32_t)(s.sorted[at] >> 32);
      return;
    }
    // more than 256 in one part: the pass over the row, down to the last kept
    if (largest) {
      const u64 e = list[keep - 1];
      tx = pair_value(e);
      ti = pair_index(e);
    }
    __syncthreads();
  }

  // index order: the head's elements, the chunks, the tail's elements.  The
  // chunks' weights are added up by runs, and the first run with the target is
  // looked into.  In registers a wave's 64 chunks of each round are a run;
  // otherwise each wave adds a run of the chunks up, and the one with the
  // target is cut into runs again, until one wave's lanes have a chunk each
  const auto in = [&](int i, float x) {
    return (x > tx || (x == tx && i <= ti)) && (double)x - m >= floor_z;
  };
  const auto kept = [&](int i, float x) -> u64 { return in(i, x) ? weight(x) : 0; };
  const int w = t >> 6, lane = t & 63;
  if (t < 6) lds.edge_w[t] = row.edge_index >= 0 ? kept(row.edge_index, row.edge) : 0;
  u64 base = 0, all = 0;
  double target = 0.0;
  int lo = 0, count = row.n4;
  // the head's weight and the target; whether an element of the head is drawn
  const auto in_head = [&](u64 chunks) {
    base = lds.edge_w[0] + lds.edge_w[1] + lds.edge_w[2];
    all = chunks + base + lds.edge_w[3] + lds.edge_w[4] + lds.edge_w[5];
    target = u * (double)all;
    if (!base || !((double)base > target)) return false;
    u64 cum = 0;
    int i = 0;
    for (; i < 2; ++i) {
      cum += lds.edge_w[i];
      if (lds.edge_w[i] && (double)cum > target) break;
    }
    if (t == 0) a.out[r] = i;
    return true;
  };
  if constexpr (NV > 0) {
    static_assert(NV * W <= T && NV * W <= kBins, "a run a thread");
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      u64 sum = 0;
      if (j * T < row.n4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = row.v[4 * j + e];  // past the row -infinity, of weight 0
          const u64 wx = weight(x);
          sum += in(row.index(j, e), x) ? wx : 0;
        }
        sum = wave_sum_u64(sum);
      }
      if (lane == 0) lds.bins[j * W + w] = sum;
    }
    __builtin_amdgcn_sched_barrier(0);
    if (t == 0) lds.pick = kNone;
    __syncthreads();
    const u64 mine = t < NV * W ? lds.bins[t] : 0;
    u64 chunks;
    const u64 before = b.before(mine, &chunks);
    if (in_head(chunks)) return;
    if (mine && (double)(base + before + mine) > target) atomicMin(&lds.pick, t);
    __syncthreads();
    const int run = lds.pick;
    if (run == kNone) {
      base += chunks;
      count = -1;
    } else {
      if (t == run) lds.first = base + before;
      __syncthreads();
      base = lds.first;
      lo = 64 * run;
      count = min(64, row.n4 - lo);
    }
  } else {
    for (bool whole = true; whole || count > 64; whole = false) {
      const int per = (count + W - 1) / W;
      const int c0 = lo + w * per, c1 = min(lo + count, c0 + per);
      u64 sum = 0;
      for (int c = c0 + lane; c < c1; c += 256) {
        float4 x[4];
#pragma unroll
        for (int v = 0; v < 4; ++v)  // past the run the last chunk, not counted
          x[v] = *reinterpret_cast<const float4*>(row.p + row.head + 4 * min(c + 64 * v, c1 - 1));
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int i = row.head + 4 * (c + 64 * v);
          const float e[4] = {x[v].x, x[v].y, x[v].z, x[v].w};
          bool k[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) k[y] = c + 64 * v < c1 && in(i + y, e[y]);
          if (__ballot(k[0] || k[1] || k[2] || k[3])) {  // four weights at a time, no branches
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const u64 wy = weight(e[y]);
              sum += k[y] ? wy : 0;
            }
          }
        }
      }
      sum = wave_sum_u64(sum);
      __syncthreads();  // the last round's runs are read, the edges written
      if (lane == 0) lds.bins[w] = sum;
      __syncthreads();
      if (whole) {
        u64 chunks = 0;
        for (int i = 0; i < W; ++i) chunks += lds.bins[i];
        if (in_head(chunks)) return;
      }
      int run = -1;
      for (int i = 0; i < W; ++i) {
        const u64 v = lds.bins[i];
        if (v && (double)(base + v) > target) {
          run = i;
          break;
        }
        base += v;
      }
      if (run < 0) {  // not among the chunks (in the first round)
        count = -1;
        break;
      }
      lo += run * per;
      count = min(per, count - run * per);
    }
  }
  if (count > 0) {
    if (w != 0) return;
    u64 wt[4] = {0, 0, 0, 0};
    const int i = row.head + 4 * (lo + lane);
    if (lane < count) {
#pragma unroll
      for (int e = 0; e < 4; ++e) wt[e] = kept(i + e, row.p[i + e]);
    }
    const u64 mine = wt[0] + wt[1] + wt[2] + wt[3];
    u64 incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    const unsigned long long hit = __ballot(mine && (double)(base + incl) > target);
    if (hit && lane == __ffsll(hit) - 1) {
      u64 cum = base + incl - mine;
      int e = 0, found = 0;
      for (; e < 4; ++e) {
        cum += wt[e];
        if (wt[e]) found = e;
        if (wt[e] && (double)cum > target) break;
      }
      a.out[r] = i + found;
    }
    return;
  }
  // among the tail's elements, or (u is 1 or more) the last one of any weight
  u64 cum = base;
  int got = -1;
  for (int i = 3; i < 6; ++i) {
    cum += lds.edge_w[i];
    if (got < 0 && lds.edge_w[i] && (double)cum > target) got = row.head + 4 * row.n4 + i - 3;
  }
  if (got < 0) {
    __syncthreads();
    if (t == 0) lds.pick = -1;
    __syncthreads();
    Row<T, 0> again;
    again.load(row.p, n);
    again.each([&](int j, int e, float x) {
      if (again.inside(j, e) && kept(again.index(j, e), x))
        atomicMax(&lds.pick, again.index(j, e));
    });
    __syncthreads();
    got = lds.pick;
  }
  if (t == 0) a.out[r] = got;
}

}  // namespace
}  // namespace tjh

using namespace tjh;

extern "C" int tjh_sample_logits(const float* logits, int64_t ld, int64_t rows, int64_t cols,
                                 const float* uniforms, const float* temperatures,
                                 const int32_t* top_ks, const float* top_ps, const float* min_ps,
                                 double temperature, int64_t top_k, double top_p, double min_p,
                                 int32_t* out) {
  TJH_REQUIRE_INIT();
  TJH_ARG(rows >= 0 && cols > 0 && ld >= cols, "tjh_sample_logits: bad sizes");
  TJH_ARG(rows < (int64_t(1) << 22), "tjh_sample_logits: too many rows");  // of a grid
  if (rows == 0) return TJH_OK;
  if (cols > kMaxCols)
    return set_error(TJH_ERR_UNSUPPORTED, "tjh_sample_logits: %lld columns, at most %lld",
                     (long long)cols, (long long)kMaxCols);
  TJH_ARG(logits && uniforms && out, "tjh_sample_logits: NULL pointer");
  const SampleArgs a{logits, ld,    (int)cols, uniforms, temperatures, top_ps, min_ps,
                     top_ks, temperature, top_p, min_p,    top_k,        out};
  KernelScope ks("sample_logits");
  const dim3 grid((unsigned)rows);
  if (cols <= 4096) tjh_launch(k_sample<256, 4>, grid, dim3(256), 0, stream(), a);
  else if (cols <= 16384) tjh_launch(k_sample<512, 8>, grid, dim3(512), 0, stream(), a);
  else if (cols <= 53248) tjh_launch(k_sample<512, 26>, grid, dim3(512), 0, stream(), a);
  else tjh_launch(k_sample<1024, 0>, grid, dim3(1024), 0, stream(), a);
  return check_launch("sample_logits");
}
