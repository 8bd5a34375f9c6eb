// A beam search's step and the reordering of its caches (beside
// Tensor.multinomial, src/tensor/Tensor.ts:271-359: the next tokens of several
// kept sequences instead of one drawn from each).
//
// Step: of the continuations (w, v) with the scores s_w + x_wv - ln sum exp x_w,
// the `keep` largest.  Within a beam their order is that of the logits, so each
// workgroup of the first kernel takes the largest logits of a piece of a row, with
// the piece's maximum and sum of exponentials, and one workgroup a search then
// compares the scores of those in 64 bits.  Logits that differ by less than such a
// score holds keep their order within a beam, in which a piece hands them on: so the
// first continuations are the same for every `keep`.
#include "rowreg.h"

#include <math.h>

namespace tjh {
namespace {

using namespace rowreg;

struct BeamArgs {
  const float* x;
  const float* scores;
  const uint8_t* finished;
  float2* stats;  // [rows, S]: maximum, sum of exponentials from it
  u64* cand;      // [rows, S, keep]: composites, best first
  float* out_scores;
  int32_t *tokens, *parents;
  uint8_t* out_finished;
  int64_t ld;
  int W, V, S, per, keep, eos;
};

// exp(x) for x <= 0 to about a float's step: the rounding of x log2(e) goes back
// in behind the hardware's power of two (half of expf's instructions, of which a
// row has one each).
__device__ __forceinline__ float exp_near(float x) {
  constexpr float kLog2e = 1.44269502f, kLog2eLow = 1.92596299e-8f, kLn2 = 0.693147182f;
  const float y = fmaxf(x, -200.f) * kLog2e;  // below, 0 in any case
  const float low = __builtin_fmaf(x, kLog2eLow, __builtin_fmaf(x, kLog2e, -y));
  const float e = __builtin_amdgcn_exp2f(y);
  return x > -100.f ? __builtin_fmaf(e, low * kLn2, e) : x == x ? 0.f : x;
}

// A bound that a piece's k largest elements are not below, for small k: the k-th
// largest of a wave's 64 threads' maxima `top`, to the 16 high bits of its key
// (-infinity where fewer of them are above -infinity).  No barrier; the largest of
// the waves' bounds leaves some ten of the k more than a bound over all threads
// would, which takes eight barriers.
constexpr int kWaveBound = 16;
__device__ __forceinline__ float wave_bound(float top, int k) {
  const uint32_t key = order_key(top);
  uint32_t lo = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t c = lo | (1u << bit);
    if (__popcll(__ballot(key >= c)) >= k) lo = c;
  }
  return lo > 0x007fffffu ? key_value(lo) : -INFINITY;  // 0x007fffff: the key of -infinity
}

// A piece of a row: `per` columns, fewer at the end.  Bound for many rows by
// reading them and then selecting, in step on all CUs: 256 rows of 50257 (51 MB)
// 16.5 us, 12.5 of them without the selection; for few by latency, 6 us.
template <int T, int NV, int CAP>
__global__ __launch_bounds__(T, T == 512 ? 4 : 1) void k_beam_pieces(BeamArgs a) {
  __shared__ SelectLds<T, CAP> s;
  const int64_t r = blockIdx.x / a.S;
  if (a.finished && a.finished[r]) return;
  const int piece = blockIdx.x - (int)r * a.S, c0 = piece * a.per, n = min(a.per, a.V - c0);
  Block<T> b(s.sm);
  Row<T, NV> row;
  row.load(a.x + r * a.ld + c0, n, 0, true);
  float m = -INFINITY, sum = 0.f;
  row.each([&](int, int, float x) { m = fmaxf(m, x); });  // NaN takes no part here,
  const int k = min(a.keep, n);
  float bound = k <= kWaveBound ? wave_bound(m, k) : -INFINITY;
  {
    // both at once, as (larger first) halves
    u64 v = ((u64)order_key(wave_max(m)) << 32) | order_key(bound);
    v = b.across(v, [](u64 x, u64 y) {
      const uint32_t h = max((uint32_t)(x >> 32), (uint32_t)(y >> 32));
      return ((u64)h << 32) | max((uint32_t)x, (uint32_t)y);
    });
    m = key_value((uint32_t)(v >> 32));
    bound = key_value((uint32_t)v);
  }
  const float from = m == -INFINITY ? 0.f : m;
  row.each([&](int, int, float x) { sum += exp_near(x - from); });  // but in the sum
  sum = b.sum(sum);
  if (bound == -INFINITY) bound = kth_bound(row, k, b);
  const u64* best = select_above(row, k, bound, kNanFirst, s, b);
  u64* to = a.cand + blockIdx.x * (int64_t)a.keep;
  for (int i = threadIdx.x; i < k; i += T) {
    const u64 c = best[i];
    to[i] = composite((uint32_t)(c >> 32), c0 + index_of(c));
  }
  if (threadIdx.x == 0) a.stats[blockIdx.x] = make_float2(m, sum);
}

// Unsigned integer in the order of the scores; 0: no continuation.
__device__ __forceinline__ u64 score_key(double v) {
  if (!(v > -INFINITY)) return 0;
  const u64 u = (u64)__double_as_longlong(v + 0.0);
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double key_score(u64 k) {
  return __longlong_as_double((long long)((k >> 63) ? k & 0x7fffffffffffffffull : ~k));
}

constexpr int kMaxBeams = 64, kMaxEntries = kMaxBeams * kMaxBeams;
constexpr int kTokenBits = 20;

// The order of continuations of equal scores as one integer, the first one's the
// largest: ascending beams, then descending logits, then ascending tokens.
__device__ __forceinline__ u64 tie_of(int w, uint32_t logit, int v) {
  const uint32_t last = (1u << kTokenBits) - 1;
  return ((u64)(kMaxBeams - 1 - w) << (32 + kTokenBits)) | ((u64)logit << kTokenBits) | (last - v);
}
__device__ __forceinline__ int beam_of(u64 tie) {
  return kMaxBeams - 1 - (int)(tie >> (32 + kTokenBits));
}
__device__ __forceinline__ int token_of(u64 tie) {
  const uint32_t last = (1u << kTokenBits) - 1;
  return last - ((uint32_t)tie & last);
}
constexpr int kMergeThreads = 512;
constexpr int kEarly = 3;  // candidates a thread, read before anything else is known

// One workgroup a search.  The lists (a beam's pieces) are in order, so only the
// `keep` lists with the best heads matter, and of those only what is not below the
// last of these heads; some tens of entries, ranked by counting.  A chain of reads
// of what other CUs wrote, barriers and 64-bit logarithms: 5.7 us for one search
// with four beams, 5.9 us for 32 with eight.
__global__ __launch_bounds__(kMergeThreads) void k_beam_merge(BeamArgs a) {
  __shared__ double from[kMaxBeams];  // a beam's score less its logarithm of the sum
  __shared__ int state[kMaxBeams];    // 0 goes on, 1 finished, 2 has no continuation
  __shared__ int chosen[kMaxBeams];
  __shared__ u64 early[kEarly * kMergeThreads];
  __shared__ u64 key[kMaxEntries];  // the lists' heads, then the entries
  __shared__ u64 tie[kMaxEntries];
  __shared__ u64 bound;
  __shared__ int count;
  const int t = threadIdx.x, lists = a.W * a.S;
  const int64_t r0 = (int64_t)blockIdx.x * a.W;
  // Most of the time goes by reads one after the other of what other CUs have
  // just written: where there are few candidates they are all read at once (of
  // ended beams, whatever stands there).
  const u64* __restrict__ cand = a.cand + r0 * a.S * a.keep;
  const int all = lists * a.keep;
  const bool few = all <= kEarly * kMergeThreads;
  u64 pre[kEarly];
  if (few) {
#pragma unroll
    for (int i = 0; i < kEarly; ++i)
      if (t + kMergeThreads * i < all) pre[i] = cand[t + kMergeThreads * i];
  }
  if (t == 0) {
    bound = 0;
    count = 0;
  }
  if (t < kMaxBeams) chosen[t] = -1;
  // a wave a beam, its lanes the pieces, always added up in one order
  for (int w = t >> 6; w < a.W; w += kMergeThreads / 64) {
    const int lane = t & 63;
    const float2* p = a.stats + (r0 + w) * a.S;
    const float2 first = lane < a.S ? p[lane] : make_float2(-INFINITY, 0.f);
    const bool ended = a.finished && a.finished[r0 + w];
    const double s = a.scores[r0 + w];
    float m = first.x;
    for (int i = lane + 64; i < a.S; i += 64) m = fmaxf(m, p[i].x);
    m = wave_max(m);
    const auto term = [&](float2 x) {
      return x.x == -INFINITY ? (double)x.y : (double)x.y * exp((double)x.x - (double)m);
    };
    double sum = term(first);
    for (int i = lane + 64; i < a.S; i += 64) sum += term(p[i]);
    for (int o = 1; o < 64 && o < a.S; o <<= 1) sum += __shfl_xor(sum, o, 64);
    // NaN in the sum, +infinity as the maximum, or nothing above -infinity
    const bool ok = sum > 0.0 && sum < INFINITY && m < INFINITY && m > -INFINITY;
    if (lane == 0) {
      state[w] = !(s > -INFINITY) ? 2 : ended ? 1 : ok ? 0 : 2;
      from[w] = ended || !ok ? s : s - ((double)m + log(sum));
    }
  }
  if (few) {
#pragma unroll
    for (int i = 0; i < kEarly; ++i)
      if (t + kMergeThreads * i < all) early[t + kMergeThreads * i] = pre[i];
  }
  __syncthreads();
  const auto entry = [&](int list, int i, u64* at) -> u64 {  // the i-th of a list: key, tie
    const int w = list / a.S, piece = list - w * a.S;
    if (state[w] == 2) return 0;
    if (state[w] == 1) {
      *at = tie_of(w, 0, a.eos);
      return piece == 0 && i == 0 ? score_key(from[w]) : 0;
    }
    if (i >= min(a.keep, min(a.per, a.V - piece * a.per))) return 0;
    const u64 c = few ? early[list * a.keep + i] : cand[(int64_t)list * a.keep + i];
    *at = tie_of(w, (uint32_t)(c >> 32), index_of(c));
    return score_key(from[w] + (double)key_value((uint32_t)(c >> 32)));
  };
  // how many of the entries [0, n) come before the i-th; without a branch, so that
  // the reads go on: 4096 entries in 0.9 ms, with one 2.2 (3.4 where all are equal)
  const auto rank_of = [&](int i, int n) {
    const u64 me = key[i], mine = tie[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += (key[j] > me) | ((key[j] == me) & (tie[j] > mine));
    return rank;
  };
  u64 at = 0;
  for (int i = t; i < lists; i += kMergeThreads) {
    key[i] = entry(i, 0, &at);
    tie[i] = at;
  }
  __syncthreads();
  for (int i = t; i < lists; i += kMergeThreads) {
    if (key[i] == 0) continue;
    const int rank = rank_of(i, lists);
    if (rank < a.keep) chosen[rank] = i;
    if (rank == a.keep - 1) bound = key[i];
  }
  __syncthreads();
  for (int i = t; i < a.keep * a.keep; i += kMergeThreads) {
    const int list = chosen[i / a.keep];
    if (list < 0) continue;
    const u64 k = entry(list, i % a.keep, &at);
    if (k != 0 && k >= bound) {
      const int to = atomicAdd(&count, 1);
      key[to] = k;
      tie[to] = at;
    }
  }
  __syncthreads();
  const int n = count;
  const int64_t o = (int64_t)blockIdx.x * a.keep;
  for (int i = t; i < n; i += kMergeThreads) {
    const int rank = rank_of(i, n);
    if (rank >= a.keep) continue;
    const int w = beam_of(tie[i]), v = token_of(tie[i]);
    a.out_scores[o + rank] = (float)key_score(key[i]);
    a.tokens[o + rank] = v;
    a.parents[o + rank] = w;
    a.out_finished[o + rank] = v == a.eos || state[w] == 1;
  }
  for (int i = n + t; i < a.keep; i += kMergeThreads) {
    a.out_scores[o + i] = -INFINITY;
    a.tokens[o + i] = -1;
    a.parents[o + i] = min(i, a.W - 1);
    a.out_finished[o + i] = 1;
  }
}

// ---------------------------------------------------------------- reordering

constexpr int kTensors = 32;  // of a launch

struct Moved {
  char* p;
  int64_t row, stride;  // bytes of a row, from one block to the next
  int64_t units;        // 16, 4 or 1 bytes: of a block's moved part
  int first;            // workgroup of the launch (grid x) at which this tensor begins
  int per;              // workgroups a block
  int unit;
};
struct ReorderArgs {
  Moved t[kTensors];
  const int32_t* parents;
  int n, W;
};

// A thread has one unit's place in all beams of a search: it reads what its
// beams become, then writes those that change, so no other thread's units are
// touched in between.  Bound by memory: half of 64 beams' 4-bit caches of 4000
// positions (1.1 GB read and written) 196 us, 5.7 TB/s; 24 float caches of 700
// positions (206 MB, from the caches in part) 34 us.
template <int W, class U>
__device__ __forceinline__ void move_units(char* p, int64_t row, int n, const int* parent) {
  U v[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int from = __builtin_amdgcn_readfirstlane(parent[i]);
    if (i < n && from != i) v[i] = *reinterpret_cast<const U*>(p + from * row);
  }
#pragma unroll
  for (int i = 0; i < W; ++i)
    if (i < n && __builtin_amdgcn_readfirstlane(parent[i]) != i)
      *reinterpret_cast<U*>(p + i * row) = v[i];
}

template <int W>
__global__ __launch_bounds__(256) void k_reorder(ReorderArgs a) {
  __shared__ int parent[W];
  const int b = blockIdx.y;
  if (threadIdx.x < W) {
    const int i = threadIdx.x;
    int p = i < a.W ? a.parents[(int64_t)b * a.W + i] : i;
    parent[i] = p >= 0 && p < a.W ? p : i;
  }
  __syncthreads();
  int k = 0;
  while (k + 1 < a.n && (int)blockIdx.x >= a.t[k + 1].first) ++k;
  const Moved& t = a.t[k];
  const int at = blockIdx.x - t.first, block = at / t.per;
  const int64_t unit = (int64_t)(at - block * t.per) * 256 + threadIdx.x;
  if (unit >= t.units) return;
  char* p = t.p + (int64_t)b * a.W * t.row + block * t.stride + unit * t.unit;
  typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
  if (t.unit == 16) move_units<W, uintx4>(p, t.row, a.W, parent);
  else if (t.unit == 4) move_units<W, uint32_t>(p, t.row, a.W, parent);
  else move_units<W, uint8_t>(p, t.row, a.W, parent);
}

}  // namespace
}  // namespace tjh

using namespace tjh;

extern "C" {

int tjh_beam_step(const float* logits, int64_t ld, const float* scores, const uint8_t* finished,
                  int64_t B, int64_t W, int64_t V, int64_t keep, int64_t eos, float* out_scores,
                  int32_t* tokens, int32_t* parents, uint8_t* out_finished) {
  TJH_REQUIRE_INIT();
  TJH_ARG(B >= 0 && W > 0 && V > 0 && keep >= 0 && ld >= V && eos < V && (!finished || eos >= 0),
          "tjh_beam_step: bad sizes");
  if (W > kMaxBeams || keep > kMaxBeams || V > (1 << 20))
    return set_error(TJH_ERR_UNSUPPORTED,
                     "tjh_beam_step: %lld beams of %lld tokens, %lld kept (at most %d, 2^20, %d)",
                     (long long)W, (long long)V, (long long)keep, kMaxBeams, kMaxBeams);
  TJH_ARG(keep <= W * V, "tjh_beam_step: %lld kept of %lld", (long long)keep, (long long)(W * V));
  if (B == 0 || keep == 0) return TJH_OK;
  TJH_ARG(logits && scores && out_scores && tokens && parents && out_finished,
          "tjh_beam_step: NULL pointer");
  TJH_ARG(B < (1 << 20), "tjh_beam_step: too many searches");
  // pieces of a row: as small as one load of each thread while the lists and
  // the workgroups stay few
  const int64_t rows = B * W;
  int per = 53248 - 4;
  for (const int size : {1024 - 4, 4096 - 4, 16384 - 4, 26624 - 4}) {
    const int64_t S = cdiv(V, size);
    if (S == 1 || (W * S <= 64 && rows * S <= 2 * num_cus())) {
      per = size;
      break;
    }
  }
  BeamArgs a{logits, scores, finished, nullptr, nullptr, out_scores, tokens, parents, out_finished,
             ld, (int)W, (int)V, (int)cdiv(V, per), per, (int)keep, eos < 0 ? -1 : (int)eos};
  const int64_t pieces = rows * a.S;
  TJH_ARG(pieces < (1 << 21), "tjh_beam_step: too many searches");
  Scratch s((size_t)pieces * (sizeof(float2) + keep * sizeof(u64)));
  if (!s.ok()) return set_error(TJH_ERR_OOM, "tjh_beam_step: no scratch");
  a.cand = s.as<u64>();
  a.stats = reinterpret_cast<float2*>(a.cand + pieces * keep);
  KernelScope ks("beam_step");
  const dim3 grid((unsigned)pieces);
  if (per < 1024)
    tjh_launch(k_beam_pieces<256, 1, 1024>, grid, dim3(256), 0, stream(), a);
  else if (per < 4096)
    tjh_launch(k_beam_pieces<256, 4, 4096>, grid, dim3(256), 0, stream(), a);
  else if (per < 16384)
    tjh_launch(k_beam_pieces<512, 8, 4096>, grid, dim3(512), 0, stream(), a);
  else if (per < 26624)
    tjh_launch(k_beam_pieces<512, 13, 4096>, grid, dim3(512), 0, stream(), a);
  else
    tjh_launch(k_beam_pieces<512, 26, 4096>, grid, dim3(512), 0, stream(), a);
  const int rc = check_launch("beam_pieces");
  if (rc != TJH_OK) return rc;
  tjh_launch(k_beam_merge, dim3((unsigned)B), dim3(kMergeThreads), 0, stream(), a);
  return check_launch("beam_merge");
}

int tjh_cache_reorder(int n, void* const* tensors, const int64_t* outers, const int64_t* strides,
                      const int64_t* sizes, int64_t B, int64_t W, const int32_t* parents) {
  TJH_REQUIRE_INIT();
  TJH_ARG(n >= 0 && B >= 0 && W >= 0, "tjh_cache_reorder: bad sizes");
  if (W > 64)
    return set_error(TJH_ERR_UNSUPPORTED, "tjh_cache_reorder: %lld beams, at most 64",
                     (long long)W);
  if (n == 0 || B == 0 || W < 2) return TJH_OK;
  TJH_ARG(tensors && outers && strides && sizes && parents, "tjh_cache_reorder: NULL pointer");
  TJH_ARG(B < 65536, "tjh_cache_reorder: too many searches");
  for (int i = 0; i < n; ++i)
    TJH_ARG(outers[i] >= 0 && sizes[i] >= 0 && strides[i] >= sizes[i] &&
                (tensors[i] || outers[i] * sizes[i] == 0),
            "tjh_cache_reorder: bad tensor %d", i);
  // all of them before the first launch: a call moves everything or nothing
  const auto unit_of = [&](int i) {
    const uint64_t bits = (uint64_t)(uintptr_t)tensors[i] | (uint64_t)strides[i] | (uint64_t)sizes[i];
    return (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : 1;
  };
  for (int i = 0; i < n; ++i)
    TJH_ARG(cdiv(sizes[i] / unit_of(i), 256) * outers[i] < (int64_t(1) << 23),
            "tjh_cache_reorder: tensor %d is too large", i);
  KernelScope ks("cache_reorder");
  int i = 0;
  while (i < n) {
    ReorderArgs a{};
    a.parents = parents;
    a.W = (int)W;
    int64_t groups = 0;
    for (; i < n && a.n < kTensors; ++i) {
      if (outers[i] * sizes[i] == 0) continue;
      Moved& t = a.t[a.n];
      t.p = static_cast<char*>(tensors[i]);
      t.row = outers[i] * strides[i];
      t.stride = strides[i];
      t.unit = unit_of(i);
      t.units = sizes[i] / t.unit;
      const int64_t per = cdiv(t.units, 256);
      if (groups + per * outers[i] >= (int64_t(1) << 23)) break;  // the next launch's
      t.per = (int)per;
      t.first = (int)groups;
      groups += per * outers[i];
      ++a.n;
    }
    if (a.n == 0) continue;
    const int64_t most = (int64_t(1) << 23) / groups;  // searches of a launch
    for (int64_t b = 0; b < B; b += most) {
      const dim3 grid((unsigned)groups, (unsigned)(B - b < most ? B - b : most));
      ReorderArgs part = a;
      part.parents = parents + b * W;
      for (int j = 0; j < a.n; ++j) part.t[j].p += b * W * a.t[j].row;
      if (W <= 4) tjh_launch(k_reorder<4>, grid, dim3(256), 0, stream(), part);
      else if (W <= 8) tjh_launch(k_reorder<8>, grid, dim3(256), 0, stream(), part);
      else if (W <= 16) tjh_launch(k_reorder<16>, grid, dim3(256), 0, stream(), part);
      else if (W <= 32) tjh_launch(k_reorder<32>, grid, dim3(256), 0, stream(), part);
      else tjh_launch(k_reorder<64>, grid, dim3(256), 0, stream(), part);
    }
  }
  return check_launch("cache_reorder");
}

}  // extern "C"
