/*
 * torchjs_hip_lm.h — entry points of libtorchjs_hip.so around a language
 * model's attention and vocabulary: attention over a sliding window, the
 * largest values of a row, distillation from a teacher's largest logits, and
 * sampling from truncated distributions.  torch.js has Tensor.topk
 * (src/tensor/Tensor.ts:3048-3178, on the host) of these.
 *
 * The conventions are those of torchjs_hip.h: int status, the library's one
 * stream, asynchronous, float32 and int32, strides in elements.  All can be
 * captured into a HIP graph.
 */
#ifndef TORCHJS_HIP_LM_H
#define TORCHJS_HIP_LM_H

#include "torchjs_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The k largest (largest == 0: smallest) values of each row of x [rows,
 * cols] at row stride ld >= cols: values [rows, k] in descending (ascending)
 * order and indices [rows, k]; NaN counts as the largest, equal values stand
 * by ascending index.  k <= cols; k > 1024 is TJH_ERR_UNSUPPORTED. */
int tjh_topk_forward(const float* x, int64_t ld, int64_t rows, int64_t cols, int64_t k,
                     int largest, float* values, int32_t* indices);
/* dx [rows, cols] = 0 but dx[r, indices[r, i]] = g[r, i] (indices of
 * tjh_topk_forward: distinct in a row; one outside [0, cols) is skipped). */
int tjh_topk_backward(const float* g, const int32_t* indices, int64_t rows, int64_t cols,
                      int64_t k, float* dx);

/* Distillation: each row has logits x [cols] (row stride ld) and k teacher
 * entries (teacher[r, i], ids[r, i]), contiguous, of which the ones with an
 * id outside [0, cols) are none.  With T the temperature,
 * p = softmax(teacher / T) over the row's entries, q = softmax(x / T):
 *   loss_row = T^2 sum_i p_i (ln p_i - ln q[ids_i])
 *   dlogits[r, j] = s_r T (q_j - sum_i p_i [ids_i == j])
 * A row with no entry above -infinity has loss 0 and gradient 0 and is not
 * counted by the mean; one with an entry of NaN or +infinity is NaN.
 * reduction and s_r (from grad_out, NULL: 1) as tjh_cross_entropy_backward's.
 * Each of loss_rows [rows], out (the reduced loss; needs loss_rows) and
 * dlogits (row stride ldd) may be NULL; with several the logits are read once
 * (rows of up to 53248).  temperature from 1e-18 to 1e18; k <= 1024,
 * else TJH_ERR_UNSUPPORTED. */
int tjh_distill(const float* logits, int64_t ld, int64_t rows, int64_t cols,
                const float* teacher, const int32_t* ids, int64_t k, float temperature,
                int reduction, const float* grad_out, float* loss_rows, float* out,
                float* dlogits, int64_t ldd);

/* One index of each row of logits [rows, cols] (row stride ld), drawn with
 * uniforms [rows].  With m the row's maximum, w_i = exp((x_i - m) /
 * temperature), in the order of descending logits (equal ones by ascending
 * index): kept are the first top_k (0 or less, or cols or more: all); of
 * these the ones before which less than top_p of their weight lies (1 or
 * more: all); of these the ones with x_i - m >= temperature * ln(min_p) (0
 * or less: all); always the first one.  out[r] is the first kept index, in
 * index order, whose running sum of weights exceeds uniforms[r] times their
 * sum (the last kept one if none does).  A temperature that is not above 0
 * takes the first index of the maximum.  A row with NaN, +infinity or no
 * logit above -infinity gives -1.  temperatures, top_ks, top_ps, min_ps
 * [rows]: a setting of each row in place of the number, or NULL.  cols up
 * to 2^20, else TJH_ERR_UNSUPPORTED. */
int tjh_sample_logits(const float* logits, int64_t ld, int64_t rows, int64_t cols,
                      const float* uniforms, const float* temperatures, const int32_t* top_ks,
                      const float* top_ps, const float* min_ps, double temperature,
                      int64_t top_k, double top_p, double min_p, int32_t* out);

/* Attention over a sliding window with sinks.  q [B,H,Tq,D], k/v
 * [B,Hkv,Tk,D], H a multiple of Hkv (query head h reads head h / (H / Hkv)),
 * Tk >= Tq: the queries are the last Tq of the Tk positions, and the one at
 * position i sees the keys j <= i with j > i - window or j < sinks (window >=
 * 1).  o = softmax(scale q k^T over those) v; strides (elements) for the B, H
 * and T axes, D contiguous, as tjh_sdpa_forward's.  lse [B,H,Tq],
 * the logarithm to base 2 of a query's sum of exponentials, is saved for the
 * backward, or NULL.  Keys and values that a query does not see have no
 * part in its output, whatever they hold.  Head dims up to 128 that are
 * multiples of 4, rows 16-byte aligned and less than 2^23 elements apart (else
 * TJH_ERR_UNSUPPORTED).  B H times Tq / 32, rounded up, below 2^24; with up to
 * 4 queries B H Tq below 2^23 (else TJH_ERR_INVALID). */
int tjh_window_forward(const float* q, const float* k, const float* v, float* o, float* lse,
                       int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t D,
                       const int64_t* q_strides, const int64_t* k_strides,
                       const int64_t* v_strides, const int64_t* o_strides, float scale,
                       int64_t window, int64_t sinks);
/* dq [B,H,Tq,D], dk/dv [B,Hkv,Tk,D] written (not accumulated; with Tq == 0
 * nothing is), summed over the query heads of a key head.  Scratch of some Tq
 * (window + sinks) floats a query head, at least for all that read one key
 * head (TJH_ERR_OOM where they do not fit).  strides[0..7] = q, k, v, o, do_,
 * dq, dk, dv as tjh_sdpa_backward's. */
int tjh_window_backward(const float* q, const float* k, const float* v, const float* o,
                        const float* do_, const float* lse, float* dq, float* dk, float* dv,
                        int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t D,
                        const int64_t* const* strides, float scale, int64_t window,
                        int64_t sinks);

#ifdef __cplusplus
}
#endif
#endif /* TORCHJS_HIP_LM_H */
