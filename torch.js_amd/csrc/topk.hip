// The k largest (or smallest) values of each row with their indices:
// Tensor.topk (src/tensor/Tensor.ts:3048-3178, which sorts the whole row on
// the host), and its backward.
//
// Order: value descending (ascending for the smallest), NaN counted as the
// largest, equal values by ascending index, so the result is one and the
// same on every run.
//
// Bound by reading the rows once: a workgroup keeps its row in registers,
// takes a lower bound of the k-th value from the threads' maxima, moves the
// few elements above it into LDS and sorts those (rowreg.h).  64 of each of
// 2048 rows of 50257: 75 us, 5.5 TB/s; 20 of one row: 9 us, a chain of loads,
// rounds of the bound and the sort on one CU.  Rows of more than 53248 are read
// twice (1024 of 128256: 162 us, 3.2 TB/s counted once).  A row with fewer than
// k elements above -infinity has no bound, and is longer than the list: some 50
// passes of the bisection (50 of 50257, 30 of them above it: 311 us, not 10).
#include "rowreg.h"

namespace tjh {
namespace {

using namespace rowreg;

template <int T, int NV, int CAP>
__global__ __launch_bounds__(T, T == 512 ? 4 : 1) void k_topk(const float* __restrict__ x, int64_t ld, int n, int k,
                                            int largest, float* __restrict__ values,
                                            int32_t* __restrict__ indices) {
  __shared__ SelectLds<T, CAP> s;
  const int64_t r = blockIdx.x;
  Block<T> b(s.sm);
  Row<T, NV> row;
  row.load(x + r * ld, n, largest ? 0u : 0x80000000u);
  const u64* best = select_largest(row, k, largest ? kNanFirst : kNanLast, s, b);
  for (int i = threadIdx.x; i < k; i += T) {
    const int at = index_of(best[i]);
    indices[r * k + i] = at;
    values[r * k + i] = row.p[at];
  }
}

// dx = 0 but dx[r, indices[r, i]] = g[r, i]: the row's zeros, then its k
// values, one workgroup a row.  (4099, 1000), 8 values: 5.1 us, 3.2 TB/s.
__global__ __launch_bounds__(256) void k_topk_bwd(const float* __restrict__ g,
                                                  const int32_t* __restrict__ indices, int n, int k,
                                                  float* __restrict__ dx) {
  const int64_t r = blockIdx.x;
  float* __restrict__ d = dx + r * n;
  const int head = min(n, (int)((16 - ((uintptr_t)d & 15)) & 15) / 4);
  const int n4 = (n - head) / 4;
  for (int i = threadIdx.x; i < head; i += 256) d[i] = 0.f;
  for (int i = threadIdx.x; i < n4; i += 256)
    *reinterpret_cast<float4*>(d + head + 4 * i) = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = head + 4 * n4 + threadIdx.x; i < n; i += 256) d[i] = 0.f;
  __syncthreads();
  for (int i = threadIdx.x; i < k; i += 256) {
    const int c = indices[r * k + i];
    if ((unsigned)c < (unsigned)n) d[c] = g[r * k + i];
  }
}

constexpr int kMaxK = 1024;
constexpr int64_t kGrid = 1 << 21;  // workgroups of a launch: a grid has less than 2^32 threads

}  // namespace
}  // namespace tjh

using namespace tjh;

extern "C" {

int tjh_topk_forward(const float* x, int64_t ld, int64_t rows, int64_t cols, int64_t k, int largest,
                     float* values, int32_t* indices) {
  TJH_REQUIRE_INIT();
  TJH_ARG(rows >= 0 && cols >= 0 && k >= 0 && ld >= cols, "tjh_topk_forward: bad sizes");
  TJH_ARG(k <= cols, "tjh_topk_forward: k = %lld of %lld columns", (long long)k, (long long)cols);
  if (rows == 0 || k == 0) return TJH_OK;
  if (k > kMaxK)
    return set_error(TJH_ERR_UNSUPPORTED, "tjh_topk_forward: k = %lld, at most %d are sorted",
                     (long long)k, kMaxK);
  TJH_ARG(rows < (int64_t(1) << 31) && cols < (int64_t(1) << 30), "tjh_topk_forward: too large");
  TJH_ARG(x && values && indices, "tjh_topk_forward: NULL pointer");
  KernelScope ks("topk");
  const int n = (int)cols, kk = (int)k;
  // The fewest threads that hold the row, but with enough of their maxima for
  // the k: with too few the bound lets most of the row into the list.  (4096,
  // 1000), k 64: one wave 16 us, four 27; 256: 124, 49.  Few rows leave the
  // CUs idle anyway: (64, 1000), k 32: 6, 6; 64: 8, 6.  (2048, 4000), k 500:
  // four waves 52 us, eight 66; 1000: 211, 87.
  for (int64_t at = 0; at < rows; at += kGrid) {
    const dim3 grid((unsigned)(rows - at < kGrid ? rows - at : kGrid));
    const float* p = x + at * ld;
    float* v = values + at * k;
    int32_t* ix = indices + at * k;
    if (n <= 1024 - 3 && kk <= (rows < 1024 ? 32 : 128))
      tjh_launch(k_topk<64, 4, 1024>, grid, dim3(64), 0, stream(), p, ld, n, kk, largest, v, ix);
    else if (n <= 4096 - 3 && kk <= 512)
      tjh_launch(k_topk<256, 4, 4096>, grid, dim3(256), 0, stream(), p, ld, n, kk, largest, v, ix);
    else if (n <= 16384 - 3)
      tjh_launch(k_topk<512, 8, 8192>, grid, dim3(512), 0, stream(), p, ld, n, kk, largest, v, ix);
    else if (n <= 53248 - 3)
      tjh_launch(k_topk<512, 26, 8192>, grid, dim3(512), 0, stream(), p, ld, n, kk, largest, v, ix);
    else
      tjh_launch(k_topk<1024, 0, 8192>, grid, dim3(1024), 0, stream(), p, ld, n, kk, largest, v, ix);
  }
  return check_launch("topk");
}

int tjh_topk_backward(const float* g, const int32_t* indices, int64_t rows, int64_t cols, int64_t k,
                      float* dx) {
  TJH_REQUIRE_INIT();
  TJH_ARG(rows >= 0 && cols >= 0 && k >= 0 && k <= cols, "tjh_topk_backward: bad sizes");
  if (rows == 0 || cols == 0) return TJH_OK;
  TJH_ARG(rows < (int64_t(1) << 31) && cols < (int64_t(1) << 30), "tjh_topk_backward: too large");
  TJH_ARG(dx && (k == 0 || (g && indices)), "tjh_topk_backward: NULL pointer");
  KernelScope ks("topk_bwd");
  for (int64_t at = 0; at < rows; at += kGrid)
    tjh_launch(k_topk_bwd, dim3((unsigned)(rows - at < kGrid ? rows - at : kGrid)), dim3(256), 0,
               stream(), g + at * k, indices + at * k, (int)cols, (int)k, dx + at * cols);
  return check_launch("topk_bwd");
}

}  // extern "C"
