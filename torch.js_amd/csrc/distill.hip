// Distillation from a teacher's largest logits (F.distillation_loss), beside
// the cross entropy of norm.hip (src/nn/losses.ts:129-168).
//
// A row has `cols` student logits x and K teacher entries (v_k, id_k); an
// entry whose id is outside [0, cols) is none, and a row is valid when some
// entry above -infinity is left.  With T the temperature, p = softmax(v / T)
// over the row's entries and q = softmax(x / T) over the columns,
//   loss_row = T^2 sum_k p_k (ln p_k - ln q[id_k])
//   d loss_row / d x_j = T (q_j - sum_k p_k [id_k = j])
// (an entry given twice counts twice); invalid rows have loss 0 and gradient
// 0.  Reductions as the cross entropy's: none, the mean over valid rows, the
// sum, the sum over the number of rows.
//
// Bound by reading the logits once and, for a gradient, writing it once
// (8 bytes an element): a workgroup keeps its row in registers (rowreg.h)
// between the two, takes maximum and sum from there, and forms the row's loss
// and gradient in the same pass.  (2048, 50257) with 64 entries: 179 us, 4.6
// TB/s, where a large copy moves 5.2; (509, 32001): 29 us, 4.4.  Rows of more
// than 53248 are read three times ((1024, 128256): 318 us a call, 3.3 TB/s of
// one read and the write; the loss alone 165).
#include "rowreg.h"

#include <math.h>

namespace tjh {
namespace {

using namespace rowreg;

constexpr int kMaxK = 1024;
constexpr int kPairs = 64;     // entries whose duplicates are found by comparing all
constexpr int kHash = 2 * kMaxK;
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
  const float* x;
  int64_t ld;
  int n, k;
  const float* v;     // [rows, K]
  const int32_t* ids; // [rows, K]
  float temp;
  int reduction;
  const float* gout;   // upstream gradient (null: 1)
  const float* denom;  // what mean and batchmean divide by (null: 1), or
  const float* valid;  // each row's 0 or 1, whose sum it is
  int64_t rows;
  float* loss_rows;    // or null
  float* d;            // [rows, ldd] or null
  int64_t ldd;
};

// Per row 1 where it is valid, one wave a row.
__global__ __launch_bounds__(256) void k_distill_valid(const float* __restrict__ v,
                                                       const int32_t* __restrict__ ids,
                                                       int64_t rows, int n, int k,
                                                       float* __restrict__ valid) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  bool any = false;
  for (int i = threadIdx.x & 63; i < k; i += 64)
    any |= (unsigned)ids[r * k + i] < (unsigned)n && v[r * k + i] != -INFINITY;
  any = __ballot(any) != 0;
  if ((threadIdx.x & 63) == 0) valid[r] = any ? 1.f : 0.f;
}

// out = sum of x[0, n), over denom[0] or over the sum of valid[0, n) where
// one of them is given: one workgroup, each thread adding every 1024th in
// order.
__global__ __launch_bounds__(1024) void k_distill_sum(const float* __restrict__ x, int64_t n,
                                                      const float* __restrict__ denom,
                                                      const float* __restrict__ valid,
                                                      float* __restrict__ out) {
  __shared__ u64 sm[32];
  Block<1024> b(sm);
  float s = 0.f, c = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    s += x[i];
    c += valid ? valid[i] : 0.f;
  }
  s = b.sum(s);
  c = b.sum(c);
  if (threadIdx.x == 0) out[0] = s / (valid ? c : denom ? denom[0] : 1.f);
}

template <int T, int NV>
__global__ __launch_bounds__(T, T == 512 ? 4 : 1) void k_distill(DistillArgs a) {
  __shared__ u64 sm[2 * (T / 64)];
  __shared__ float p[kMaxK];
  __shared__ int32_t id[kMaxK];
  // rows of one wave compare all entries: a table would halve their waves
  constexpr bool kTable = T > 64;
  __shared__ int32_t seen[kTable ? kHash : 1];
  __shared__ int twice;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x, K = a.k;
  Block<T> b(sm);
  Row<T, NV> row;
  row.load(a.x + r * a.ld, a.n);
  // the teacher's entries, while the row is on its way
  float mt = -INFINITY;
  bool bad = false;
  for (int i = t; i < K; i += T) {
    const int32_t c = a.ids[r * K + i];
    const float v = a.v[r * K + i];
    const bool in = (unsigned)c < (unsigned)a.n;
    id[i] = in ? c : -1;
    p[i] = in ? v : -INFINITY;
    mt = in ? fmaxf(mt, v) : mt;  // NaN takes no part
    bad |= in && v != v;
  }
  float count = 0.f;  // of valid rows, this thread's part
  if (a.valid && a.d)
    for (int64_t i = t; i < a.rows; i += T) count += a.valid[i];
  mt = b.max(mt);
  const bool valid = b.any(bad) || mt > -INFINITY;
  if (!valid) {
    if (t == 0 && a.loss_rows) a.loss_rows[r] = 0.f;
    if (a.d) {
      float* d = a.d + r * a.ldd;
      for (int i = t; i < a.n; i += T) d[i] = 0.f;
    }
    return;
  }
  float c2 = kLog2e / a.temp;
  const float inv_t = 1.0f / a.temp;
  float st = 0.f;
  for (int i = t; i < K; i += T) {
    const float e = __builtin_amdgcn_exp2f((p[i] - mt) * c2);
    st += e;
  }
  // an entry of NaN or +infinity makes this NaN, and by the factor of every
  // exponent the row's loss and whole gradient, as q_j times the sum of the
  // probabilities would be.  In a scalar register: chosen at the gradient, it
  // cost 3.5 of 190 us at 2048 rows of 50257
  st = b.sum(st);
  c2 = __uint_as_float(
      __builtin_amdgcn_readfirstlane(__float_as_uint(st == st ? c2 : NAN)));
  const float lst = logf(st), ist = 1.0f / st;
  // the student's
  float mx = -INFINITY;
  row.each([&](int, int, float x) { mx = fmaxf(mx, x); });
  mx = b.max(mx);
  float s = 0.f;
  row.each([&](int, int, float x) { s += __builtin_amdgcn_exp2f((x - mx) * c2); });
  s = b.sum(s);
  const float ls = logf(s);
  float loss = 0.f;
  for (int i = t; i < K; i += T) {
    const float z = (p[i] - mt) * inv_t;
    const float e = __builtin_amdgcn_exp2f((p[i] - mt) * c2) * ist;
    if (id[i] >= 0 && e != 0.f)
      loss += e * ((z - lst) - ((row.p[id[i]] - mx) * inv_t - ls));
    p[i] = e;
  }
  if (a.loss_rows) {
    loss = b.sum(loss);
    if (t == 0) a.loss_rows[r] = loss * (a.temp * a.temp);
  }
  if (!a.d) return;
  float g = a.gout ? a.gout[a.reduction == 0 ? r : 0] : 1.f;
  if (a.valid) g /= b.sum(count);
  else if (a.denom) g /= a.denom[0];
  g *= a.temp;
  const float gq = g / s;
  float* __restrict__ d = a.d + r * a.ldd;
  const auto grad = [&](float x) { return __builtin_amdgcn_exp2f((x - mx) * c2) * gq; };
  if (row.edge_index >= 0) d[row.edge_index] = grad(row.edge);
  const bool al = (((uintptr_t)(d + row.head)) & 15) == 0;
  const auto put = [&](int c, float x0, float x1, float x2, float x3) {
    float* to = d + row.head + 4 * c;
    const float4 o = make_float4(grad(x0), grad(x1), grad(x2), grad(x3));
    if (al) {
      st_nt(to, o);
    } else {
      to[0] = o.x;
      to[1] = o.y;
      to[2] = o.z;
      to[3] = o.w;
    }
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (t + j * T < row.n4)
        put(t + j * T, row.v[4 * j], row.v[4 * j + 1], row.v[4 * j + 2], row.v[4 * j + 3]);
  } else {
    for (int c = t; c < row.n4; c += T) {
      const float4 x = *reinterpret_cast<const float4*>(row.p + row.head + 4 * c);
      put(c, x.x, x.y, x.z, x.w);
    }
  }
  // the teacher's columns once more, with their probabilities.  Whether a
  // column is given twice: up to 64 entries by comparing, more by a table
  if (kTable && K > kPairs) {
    for (int i = t; i < kHash; i += T) seen[i] = -1;
    if (t == 0) twice = 0;
    __syncthreads();
    for (int i = t; i < K; i += T) {
      const int32_t c = id[i];
      if (c < 0) continue;
      unsigned h = ((unsigned)c * 2654435761u) >> 21;  // one of 2048 places
      for (;;) {
        const int32_t was = atomicCAS(&seen[h], -1, c);
        if (was == -1) break;
        if (was == c) {
          twice = 1;
          break;
        }
        h = (h + 1) & (kHash - 1);
      }
    }
  }
  __threadfence_block();
  __syncthreads();  // p complete, the row written
  const bool compare = !kTable || K <= kPairs || twice;
  for (int i = t; i < K; i += T) {
    const int32_t c = id[i];
    if (c < 0) continue;
    float sum = p[i];
    if (compare) {
      bool first = true;
      sum = 0.f;
      for (int j = 0; j < K; ++j) {  // in entry order: the same on every run
        if (id[j] == c) {
          first &= j >= i;
          sum += p[j];
        }
      }
      if (!first) continue;
    }
    d[c] = grad(row.p[c]) - g * sum;
  }
}

}  // namespace
}  // namespace tjh

using namespace tjh;

extern "C" int tjh_distill(const float* logits, int64_t ld, int64_t rows, int64_t cols,
                           const float* teacher, const int32_t* ids, int64_t k, float temperature,
                           int reduction, const float* grad_out, float* loss_rows, float* out,
                           float* dlogits, int64_t ldd) {
  TJH_REQUIRE_INIT();
  TJH_ARG(rows >= 0 && cols > 0 && k > 0 && ld >= cols, "tjh_distill: bad sizes");
  TJH_ARG(rows < (int64_t(1) << 31) && cols < (int64_t(1) << 30), "tjh_distill: too large");
  const int threads = cols <= 1024 ? 64 : cols <= 4096 ? 256 : cols <= 53248 ? 512 : 1024;
  TJH_ARG(rows * threads < (int64_t(1) << 32), "tjh_distill: too many rows");  // of a grid
  TJH_ARG(reduction >= 0 && reduction <= 3, "tjh_distill: reduction %d", reduction);
  // 1 / T and T^2 are numbers
  TJH_ARG(temperature >= 1e-18f && temperature <= 1e18f,
          "tjh_distill: temperature must be positive, from 1e-18 to 1e18");
  if (k > kMaxK)
    return set_error(TJH_ERR_UNSUPPORTED, "tjh_distill: %lld teacher entries a row, at most %d",
                     (long long)k, kMaxK);
  TJH_ARG(!out || (reduction && loss_rows), "tjh_distill: a reduced loss needs loss_rows");
  TJH_ARG(!dlogits || ldd >= cols, "tjh_distill: ldd");
  TJH_ARG(!(dlogits && reduction == 0 && !grad_out), "tjh_distill: row gradients are needed");
  if (rows == 0) {
    if (out) return tjh_fill_f32(out, 1, reduction == 2 ? 0.f : NAN);
    return TJH_OK;
  }
  TJH_ARG(logits && teacher && ids && (loss_rows || dlogits), "tjh_distill: NULL pointer");
  KernelScope ks("distill");
  const bool mean = reduction == 1, batch = reduction == 3;
  Scratch sc(mean ? (size_t)(rows + 1) * sizeof(float) : batch ? sizeof(float) : 0);
  float* denom = nullptr;
  if (mean || batch) {
    if (!sc.ok()) return set_error(TJH_ERR_OOM, "tjh_distill: no scratch");
    denom = sc.as<float>();
  }
  // the count of valid rows: up to two per thread every workgroup adds their
  // flags up itself, which saves a launch (2 of 40 us at 509 rows; at 2048 the
  // launch is 4 us faster)
  const float* valid = mean && rows <= 2 * threads ? denom + 1 : nullptr;
  int rc = TJH_OK;
  if (batch) {
    rc = tjh_fill_f32(denom, 1, (float)rows);
  } else if (mean) {
    tjh_launch(k_distill_valid, dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, stream(), teacher, ids,
               rows, (int)cols, (int)k, denom + 1);
    if (!valid)
      tjh_launch(k_distill_sum, dim3(1), dim3(1024), 0, stream(), (const float*)(denom + 1), rows,
                 (const float*)nullptr, (const float*)nullptr, denom);
    rc = check_launch("distill_valid");
  }
  if (rc != TJH_OK) return rc;
  const DistillArgs a{logits,   ld,    (int)cols, (int)k, teacher,   ids,     temperature, reduction,
                      grad_out, denom, valid,     rows,   loss_rows, dlogits, ldd};
  const dim3 grid((unsigned)rows);
  if (cols <= 1024) tjh_launch(k_distill<64, 4>, grid, dim3(64), 0, stream(), a);
  else if (cols <= 4096) tjh_launch(k_distill<256, 4>, grid, dim3(256), 0, stream(), a);
  else if (cols <= 16384) tjh_launch(k_distill<512, 8>, grid, dim3(512), 0, stream(), a);
  else if (cols <= 53248) tjh_launch(k_distill<512, 26>, grid, dim3(512), 0, stream(), a);
  else tjh_launch(k_distill<1024, 0>, grid, dim3(1024), 0, stream(), a);
  rc = check_launch("distill");
  if (rc != TJH_OK || !out) return rc;
  tjh_launch(k_distill_sum, dim3(1), dim3(1024), 0, stream(), (const float*)loss_rows, rows,
             (const float*)denom, valid, out);
  return check_launch("distill_sum");
}
