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
// formed in 64 bits as 2^t = 2^(k / 128) 2^f, |f| <= 1 / 256, from a table and
// the first five terms of 2^f (the sixth is below 2^-49): 32-bit ones would
// move one draw in some thousand over a border between two indices.
//
// One workgroup has a row, in registers (rowreg.h).  With top_k up to 256 the
// largest elements are sorted in LDS and everything else happens on that
// list.  Otherwise every element's weight is needed: a nucleus takes a pass
// for the weights' sum, one that adds the weights of the elements that can
// be in it to a histogram over x (an element of weight w_i is outside when
// even n elements of its weight are no more than 1 - top_p of the sum), and
// sorts the one bin that the nucleus ends in; then the draw adds the kept
// weights up by wave and chunk, which is index order, and looks into one.
#include "rowreg.h"

#include <math.h>

namespace tjh {
namespace {

using namespace rowreg;

constexpr int kCap = 4096;    // sorted elements
constexpr int kList = 256;    // top_k whose elements are drawn from in LDS
constexpr int kBins = 2048;   // of the nucleus's histogram
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

template <int T, int NV>
struct SampleLds {
  SelectLds<T, kCap> s;
  union {
    u64 bins[kBins];
    u64 seg[NV > 0 ? NV * (T / 64) : 4096];  // weight of each (chunk, wave)
    u64 w[kList];
  };
  double pow2[128];  // 2^(i / 128 + s)
  u64 edge_w[6];
  int pick;
};

// 2^(t + s) rounded to an integer, for t <= 0 (or NaN: 0) and s <= 51.
__device__ __forceinline__ u64 weight_of(double t, const double* pow2) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: its low word takes the integer
  constexpr double c1 = 6.93147180559945286e-01, c2 = 2.40226506959100694e-01,
                   c3 = 5.55041086648215762e-02, c4 = 9.61812910762847687e-03;  // ln(2)^k / k!
  t = fmax(t, -64.0);  // 2^(51 - 64) is 0
  const double kd = __builtin_fma(t, 128.0, kMagic);
  const int k = (int)__double_as_longlong(kd);
  const double f = __builtin_fma(kd - kMagic, -1.0 / 128, t);
  double e = __builtin_fma(f, c4, c3);
  e = __builtin_fma(f, e, c2);
  e = __builtin_fma(f, e, c1);
  const double tab = pow2[k & 127];
  e = __builtin_fma(tab * f, e, tab);
  e = ldexp(e, k >> 7) + 4503599627370496.0;  // 2^52: the integer is in the low 52 bits
  return (u64)__double_as_longlong(e) & 0xfffffffffffffull;
}

template <int T, int NV>
__global__ __launch_bounds__(T) void k_sample(SampleArgs a) {
  __shared__ SampleLds<T, NV> lds;
  SelectLds<T, kCap>& s = lds.s;
  constexpr int W = T / 64;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  Block<T> b(s.sm);
  Row<T, NV> row;
  row.load(a.x + r * a.ld, a.n);
  const int n = a.n;

  float mx = -INFINITY;
  uint32_t mag = 0;  // largest |x| as bits: above infinity's is NaN
  row.each([&](int, int, float x) {
    mx = fmaxf(mx, x);
    const uint32_t u = __float_as_uint(x) << 1;
    mag = u > mag ? u : mag;
  });
  mx = b.max(mx);
  if (b.any(mag > 0xff000000u) || !(fabsf(mx) < INFINITY)) {
    if (t == 0) a.out[r] = -1;
    return;
  }
  const double temp = a.temperature ? (double)a.temperature[r] : a.t0;
  if (t == 0) lds.pick = 0x7fffffff;
  if (!(temp > 0.0)) {
    __syncthreads();
    row.each([&](int j, int u, float x) {
      if (x == mx && row.inside(j, u)) atomicMin(&lds.pick, row.index(j, u));
    });
    __syncthreads();
    if (t == 0) a.out[r] = lds.pick;
    return;
  }
  const int64_t top_k = a.top_k ? (int64_t)a.top_k[r] : a.k0;
  const double top_p = a.top_p ? (double)a.top_p[r] : a.p0;
  const double min_p = a.min_p ? (double)a.min_p[r] : a.m0;
  const bool use_k = top_k > 0 && top_k < n, use_p = top_p < 1.0;
  const double p = top_p > 0.0 ? top_p : 1e-300;  // the first element at least
  const double floor_z = min_p > 0.0 ? fmin(temp * log(min_p), 0.0) : -INFINITY;
  const double m = (double)mx;
  const double per_t = fmin(1.4426950408889634074 / temp, 1e300);
  const double scale = ldexp(1.0, min(51, 62 - (32 - __clz(n))));
  const double u = (double)a.u[r];
  if (t < 128) lds.pow2[t] = exp2((double)t / 128) * scale;
  __syncthreads();
  const auto weight = [&](float x) { return weight_of(((double)x - m) * per_t, lds.pow2); };

  // elements of the order up to (tx, ti) are kept
  float tx = -INFINITY;
  int ti = n;
  if (use_k && top_k <= kCap / 4) {
    const int k = (int)top_k;
    select_largest(row, k, kNanFirst, s, b);
    if (k <= kList && k <= T) {
      const u64 c = t < k ? s.list[t] : 0;
      const float x = t < k ? key_value((uint32_t)(c >> 32)) : -INFINITY;
      const u64 w = weight(x);
      u64 all;
      const u64 before = b.before(w, &all);
      const bool keep = t < k && (!use_p || (double)before < p * (double)all) &&
                        (double)x - m >= floor_z;
      const u64 kept = b.sum64(keep ? w : 0);
      const bool one[1] = {keep};
      const int count = b.count(one);
      if (t < k) lds.w[t] = w;
      __syncthreads();
      const double target = u * (double)kept;
      if (keep && w) {
        const int me = index_of(c);
        u64 sum = 0;
        for (int j = 0; j < count; ++j) sum += index_of(s.list[j]) <= me ? lds.w[j] : 0;
        if ((double)sum > target) atomicMin(&lds.pick, me);
      }
      __syncthreads();
      if (lds.pick == 0x7fffffff) {  // u is 1 or more: the last one of any weight
        __syncthreads();
        if (t == 0) lds.pick = -1;
        __syncthreads();
        if (keep && w) atomicMax(&lds.pick, index_of(c));
        __syncthreads();
      }
      if (t == 0) a.out[r] = lds.pick;
      return;
    }
    const u64 c = s.list[k - 1];
    tx = key_value((uint32_t)(c >> 32));
    ti = index_of(c);
  } else if (use_k) {
    Row<T, 0> again;
    again.load(row.p, n);
    const u64 c = kth_by_bisection(again, (int)top_k, kNanFirst, b);
    tx = key_value((uint32_t)(c >> 32));
    ti = index_of(c);
  }
  const auto in_order = [&](const auto& of, int j, int e, float x) {
    return x > tx || (x == tx && of.index(j, e) <= ti);
  };

  if (use_p) {
    u64 mine = 0;
    row.each([&](int j, int e, float x) { mine += in_order(row, j, e, x) ? weight(x) : 0; });
    const u64 all = b.sum64(mine);
    const double limit = p * (double)all;  // weight before an element that is in
    // elements further than `far` below the maximum are outside
    const double far =
        fmax(temp * (log((double)n) - log1p(-p) - log((double)all / scale)) * 1.001, 0.0);
    const float per = (float)((kBins - 1) / far);
    for (int i = t; i < kBins; i += T) lds.bins[i] = 0;
    __syncthreads();
    const auto bin = [&](float x) {  // nondecreasing as x falls
      const float z = (float)(m - (double)x) * per;
      return z < (float)(kBins - 1) ? (int)z : kBins - 1;
    };
    row.each([&](int j, int e, float x) {
      if (m - (double)x <= far && in_order(row, j, e, x)) atomicAdd(&lds.bins[bin(x)], weight(x));
    });
    if (t == 0) lds.pick = -1;
    __syncthreads();
    // the last bin before which less than `limit` lies
    u64 run = 0;
    for (int i0 = 0; i0 < kBins; i0 += T) {
      const u64 w = lds.bins[i0 + t];
      u64 part;
      const u64 before = run + b.before(w, &part);
      if (w && (double)before < limit) {
        atomicMax(&lds.pick, i0 + t);
      }
      run += part;
    }
    __syncthreads();
    const int last = lds.pick;
    run = 0;
    for (int i0 = 0; i0 < kBins; i0 += T) run += i0 + t < last ? lds.bins[i0 + t] : 0;
    const u64 above = b.sum64(run);
    const int c = gather_list(
        row, kNanFirst,
        [&](int j, int e, float x) {
          return m - (double)x <= far && bin(x) == last && in_order(row, j, e, x);
        },
        s);
    if (c <= kCap) {
      sort_list(s, c);
      if (t == 0) lds.pick = 0;
      __syncthreads();
      u64 sum = above;
      for (int i0 = 0; i0 < c; i0 += T) {
        const int i = i0 + t;
        const u64 w = i < c ? weight(key_value((uint32_t)(s.list[i] >> 32))) : 0;
        u64 part;
        const u64 before = sum + b.before(w, &part);
        if (i < c && (double)before < limit) atomicMax(&lds.pick, i);
        sum += part;
      }
      __syncthreads();
      const u64 e = s.list[lds.pick];
      tx = key_value((uint32_t)(e >> 32));
      ti = index_of(e);
    } else {
      // more equal logits than the list holds: the largest composite with at
      // least `limit` above it, bit by bit, is the first one outside
      Row<T, 0> again;
      again.load(row.p, n);
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
      __syncthreads();
      if (t == 0) s.list[0] = ~u64(0);
      __syncthreads();
      again.each([&](int j, int e, float x) {
        const u64 c = composite(order_key(x), again.index(j, e));
        if (again.inside(j, e) && c > out) atomicMin(&s.list[0], c);
      });
      __syncthreads();
      tx = key_value((uint32_t)(s.list[0] >> 32));
      ti = index_of(s.list[0]);
    }
    __syncthreads();  // bins and list are free
  }

  // the kept weight of every wave's part of every chunk, in index order
  const auto kept = [&](const auto& of, int j, int e, float x) -> u64 {
    return in_order(of, j, e, x) && (double)x - m >= floor_z ? weight(x) : 0;
  };
  const int w = t >> 6, lane = t & 63;
  const int chunks = NV > 0 ? NV : (row.n4 + T - 1) / T;
  u64 part = 0;
  const auto flush = [&](int j) {
    if (__ballot(part != 0)) part = wave_sum_u64(part);
    if (lane == 0) lds.seg[j * W + w] = part;
    part = 0;
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) part += kept(row, j, e, row.v[4 * j + e]);
      flush(j);
    }
  } else {
    for (int j = 0; j < chunks; ++j) {
      const int c = t + j * T;
      if (c < row.n4) {
        const float4 x = *reinterpret_cast<const float4*>(row.p + row.head + 4 * c);
        part = kept(row, j, 0, x.x) + kept(row, j, 1, x.y) + kept(row, j, 2, x.z) +
               kept(row, j, 3, x.w);
      }
      flush(j);
    }
  }
  if (t < 6) lds.edge_w[t] = row.edge_index >= 0 ? kept(row, -1, 0, row.edge) : 0;
  if (t == 0) lds.pick = 0x7fffffff;
  __syncthreads();
  const u64 first = lds.edge_w[0] + lds.edge_w[1] + lds.edge_w[2];
  u64 sum = 0;
  for (int i = t; i < chunks * W; i += T) sum += lds.seg[i];
  const u64 inner = b.sum64(sum);
  const u64 all = first + inner + lds.edge_w[3] + lds.edge_w[4] + lds.edge_w[5];
  const double target = u * (double)all;
  // index order: the head's elements, the segments, the tail's elements
  u64 run = first;
  if ((double)first > target && first) {
    if (t == 0) {
      u64 c = 0;
      int i = 0;
      for (; i < 2; ++i) {
        c += lds.edge_w[i];
        if (lds.edge_w[i] && (double)c > target) break;
      }
      a.out[r] = i;
    }
    return;
  }
  for (int i0 = 0; i0 < chunks * W; i0 += T) {
    const int i = i0 + t;
    const u64 v = i < chunks * W ? lds.seg[i] : 0;
    u64 part_all;
    const u64 before = run + b.before(v, &part_all);
    if (v && (double)(before + v) > target) atomicMin(&lds.pick, i);
    run += part_all;
  }
  __syncthreads();
  const int seg = lds.pick;
  if (seg != 0x7fffffff) {
    // the weight before the segment, then the segment by itself
    u64 sum_before = 0;
    for (int i = t; i < seg; i += T) sum_before += lds.seg[i];
    const u64 base = first + b.sum64(sum_before);
    if (w != 0) return;
    const int j = seg / W, th = (seg % W) * 64 + lane, c = th + j * T;
    u64 wt[4] = {0, 0, 0, 0};
    const int i = row.head + 4 * c;
    if (c < row.n4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = row.p[i + e];
        const bool in = x > tx || (x == tx && i + e <= ti);
        wt[e] = in && (double)x - m >= floor_z ? weight(x) : 0;
      }
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
  u64 c = first + inner;
  int got = -1;
  for (int i = 3; i < 6; ++i) {
    c += lds.edge_w[i];
    if (got < 0 && lds.edge_w[i] && (double)c > target) got = row.head + 4 * row.n4 + i - 3;
  }
  if (got < 0) {
    if (t == 0) lds.pick = -1;
    __syncthreads();
    row.each([&](int j, int e, float x) {
      if (row.inside(j, e) && kept(row, j, e, x)) atomicMax(&lds.pick, row.index(j, e));
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
  TJH_ARG(rows < (int64_t(1) << 31), "tjh_sample_logits: too many rows");
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
  else if (cols <= 16384) tjh_launch(k_sample<1024, 4>, grid, dim3(1024), 0, stream(), a);
  else if (cols <= 53248) tjh_launch(k_sample<1024, 13>, grid, dim3(1024), 0, stream(), a);
  else tjh_launch(k_sample<1024, 0>, grid, dim3(1024), 0, stream(), a);
  return check_launch("sample_logits");
}
