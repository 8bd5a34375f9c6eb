// Register and LDS layouts of the attention kernels (flash.hip, window.hip):
// 32x32 products on the fp32 matrix cores (v_mfma_f32_32x32x2_f32) over head
// dims padded to HD in {32, 64, 96, 128}.  flash.hip's header describes the
// layouts.  Device only.
#pragma once

#include "common.h"
#include "wave.h"

namespace tjh {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int HD_MAX = 128;   // largest head dim handled here
constexpr int TILE = 32;      // rows per wave and per streamed block
constexpr int WAVES = 4;      // waves per workgroup
constexpr int ROWS = WAVES * TILE;  // 128 rows (queries or keys) per workgroup
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kXcds = 8;

// Shape constants of a padded head dim HD.
template <int HD>
struct Hd {
  static_assert(HD % 32 == 0 && HD >= 32 && HD <= HD_MAX, "head dim");
  static constexpr int NC = HD / 32;   // 32-column blocks (accumulators of a [HD,32] result)
  static constexpr int RUN = HD / 2;   // contraction values per lane
  static constexpr int W = HD + 4;     // padded LDS row length (floats)
  static constexpr int F4 = HD / 4;    // float4 per row
};

// Workgroups per CU each kernel is compiled for: the LDS tiles grow with
// HD (the paired key kernel's 43 KB at HD 64 allows three per CU, 76 KB at
// HD 128 two), and so do the register-resident rows (the forward at HD 128
// and the four-product kernels above HD 64 would spill at two).
template <int HD> constexpr int occ_fwd() { return HD <= 96 ? 2 : 1; }
template <int HD> constexpr int occ_main() { return HD <= 64 ? 2 : 1; }
template <int HD> constexpr int occ_pair() { return HD <= 64 ? 3 : 2; }

struct Strides3 {
  int64_t b, h, t;
};

// Column of key offset ko (0..31) inside a dS block row: the query-block
// kernel's lane (query row, h) reads its 16 keys kappa(j, h), j = 0..15, as
// one contiguous run at h*16, so key kappa(j, h) sits at h*16 + j.
__device__ __forceinline__ int ds_col(int ko) {
  return ((ko >> 2) & 1) * 16 + (((ko >> 3) << 2) | (ko & 3));
}

// Cost rank of the item a workgroup processes (rank 0 = most expensive).
// Workgroup w runs on XCD w % 8, and the j-th workgroup an XCD receives
// lands on its CU j % cus (one "round" per cus workgroups; the rounds are
// co-resident when the kernel's occupancy allows).  Ranks go round-robin
// over the XCDs, and within an XCD each round is laid over the CUs in
// alternating direction, so every CU holds one long, one middle and one
// short causal block instead of three of the same length.
__device__ __forceinline__ int balanced_rank(int bid, int n, int cus) {
  const int x = bid % kXcds, j = bid / kXcds;
  const int cnt = (n - x + kXcds - 1) / kXcds;  // items on this XCD
  const int round = j / cus, c = j % cus;
  const int in_round = min(cus, cnt - round * cus);
  const int p = round * cus + ((round & 1) ? in_round - 1 - c : c);
  return p * kXcds + x;
}

__device__ __forceinline__ int kappa(int s, int h) { return 8 * (s >> 2) + 4 * h + (s & 3); }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ floatx16 mfma(float a, float b, const floatx16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ floatx16 zero16() {
  floatx16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// Loads rows [r0, r0+32) x HD of a strided [T, D] matrix, HD/32 float4 per
// lane of a 256-lane workgroup.  GUARD: rows >= T and columns >= D read as
// zero.
template <int HD, bool GUARD>
__device__ __forceinline__ void load_tile(const float* __restrict__ base, int64_t st, int r0, int T,
                                          int D, floatx4 (&reg)[Hd<HD>::NC], int tid = -1) {
  if (tid < 0) tid = threadIdx.x;
#pragma unroll
  for (int i = 0; i < Hd<HD>::NC; ++i) {
    const int f = tid + 256 * i;
    const int row = f / Hd<HD>::F4, c4 = f % Hd<HD>::F4;
    const int r = r0 + row;
    if (!GUARD || (r < T && c4 * 4 < D))
      reg[i] = *reinterpret_cast<const floatx4*>(base + (int64_t)r * st + c4 * 4);
    else
      reg[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
}

template <int HD>
__device__ __forceinline__ void store_tile(float* __restrict__ S, const floatx4 (&reg)[Hd<HD>::NC],
                                           int tid = -1) {
  if (tid < 0) tid = threadIdx.x;
#pragma unroll
  for (int i = 0; i < Hd<HD>::NC; ++i) {
    const int f = tid + 256 * i;
    const int row = f / Hd<HD>::F4, c4 = f % Hd<HD>::F4;
    *reinterpret_cast<floatx4*>(S + row * Hd<HD>::W + c4 * 4) = reg[i];
  }
}

// The RUN operand values row[h*RUN ..] of an LDS tile row.
template <int HD, int RUN>
__device__ __forceinline__ void lds_run(const float* __restrict__ S, int row, int h,
                                        float (&x)[RUN]) {
  const floatx4* p = reinterpret_cast<const floatx4*>(S + row * Hd<HD>::W + h * RUN);
#pragma unroll
  for (int i = 0; i < RUN / 4; ++i) {
    const floatx4 v = p[i];
    x[4 * i] = v.x;
    x[4 * i + 1] = v.y;
    x[4 * i + 2] = v.z;
    x[4 * i + 3] = v.w;
  }
}

// The same run from global memory (rows >= T are zero; with GUARD, columns
// >= D too), times `mul`.
template <int HD, bool GUARD, int RUN>
__device__ __forceinline__ void gl_run(const float* __restrict__ base, int64_t st, int r, int T,
                                       int D, int h, float mul, float (&x)[RUN]) {
  if (r < T) {
    const floatx4* p =
        reinterpret_cast<const floatx4*>(base + (int64_t)r * st + h * RUN);
#pragma unroll
    for (int i = 0; i < RUN / 4; ++i) {
      floatx4 v = floatx4{0.f, 0.f, 0.f, 0.f};
      if (!GUARD || h * RUN + 4 * i < D) v = p[i];
      x[4 * i] = v.x * mul;
      x[4 * i + 1] = v.y * mul;
      x[4 * i + 2] = v.z * mul;
      x[4 * i + 3] = v.w * mul;
    }
  } else {
#pragma unroll
    for (int i = 0; i < RUN; ++i) x[i] = 0.f;
  }
}

// Operands of a transposed product X^T . P for a 32-row LDS tile X [r][d]:
// in step s the lane contributes X[kappa(s,h)][c*32 + l32] to block c.
template <int HD>
__device__ __forceinline__ void lds_cols(const float* __restrict__ S, int l32, int h,
                                         float (&x)[Hd<HD>::NC][16]) {
#pragma unroll
  for (int s = 0; s < 16; ++s)
#pragma unroll
    for (int c = 0; c < Hd<HD>::NC; ++c) x[c][s] = S[kappa(s, h) * Hd<HD>::W + c * 32 + l32];
}

// acc = offset-step + sum over RUN steps of a[s] * b[s].  The offset step
// adds off_a[m] * off_b[n] through the h = 0 lanes (a rank-1 update).
template <int HD, int RUN>
__device__ __forceinline__ floatx16 chain(float off_a, float off_b,
                                          const float (&a)[RUN],
                                          const float (&b)[RUN]) {
  floatx16 acc = mfma(off_a, off_b, zero16());
#pragma unroll
  for (int s = 0; s < RUN; ++s) acc = mfma(a[s], b[s], acc);
  return acc;
}

template <int HD, int RUN>
__device__ __forceinline__ floatx16 chain0(const float (&a)[RUN],
                                           const float (&b)[RUN]) {
  floatx16 acc = mfma(a[0], b[0], zero16());
#pragma unroll
  for (int s = 1; s < RUN; ++s) acc = mfma(a[s], b[s], acc);
  return acc;
}

// Writes transposed accumulators acc[c][j] = X[row = l32][d] (d = c*32 +
// 8(j/4)+4h+j%4) for the wave's 32 rows through LDS (buf, 32 x W floats)
// into dst rows r0.. (stride st, columns < D), times `mul`.  BLOCK: every wave
// of the workgroup calls this the same number of times (one barrier);
// otherwise each wave by itself.
template <int HD, bool BLOCK = true>
__device__ __forceinline__ void write_rows(float* __restrict__ buf,
                                           const floatx16 (&acc)[Hd<HD>::NC], float mul,
                                           float* __restrict__ dst, int64_t st, int r0, int T,
                                           int D, int l32, int h, int lane) {
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int c = 0; c < Hd<HD>::NC; ++c)
      buf[l32 * Hd<HD>::W + c * 32 + 8 * (j >> 2) + 4 * h + (j & 3)] = acc[c][j] * mul;
  if constexpr (BLOCK) __syncthreads();
  else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // one wave's LDS accesses are in order
  // 32 rows x HD/4 float4: HD/8 float4 per lane
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) {
    const int f = lane + 64 * i;
    const int row = f / Hd<HD>::F4, c4 = f % Hd<HD>::F4;
    const int r = r0 + row;
    if (r < T && c4 * 4 < D)
      *reinterpret_cast<floatx4*>(dst + (int64_t)r * st + c4 * 4) =
          *reinterpret_cast<const floatx4*>(buf + row * Hd<HD>::W + c4 * 4);
  }
}

template <int NC>
__device__ __forceinline__ void zero_acc(floatx16 (&acc)[NC]) {
#pragma unroll
  for (int c = 0; c < NC; ++c) acc[c] = zero16();
}

}  // namespace

// dsum[b, h, q] = sum over d of dout * o, both [B, H, Tq, D] (flash.hip).
int attn_dsum(const float* dout, const float* o, const int64_t* gs, const int64_t* os, int64_t B,
              int64_t H, int64_t Tq, int64_t D, float* dsum);

}  // namespace tjh
