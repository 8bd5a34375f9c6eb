/*
 * torchjs_hip_decode.h — entry points of libtorchjs_hip.so for decoding in
 * four bits and with beams: products with 4-bit weights, a key / value cache
 * held in 4 bits with the attention that reads it, a beam search's step and
 * the reordering of its caches.  torch.js has none of these; they stand beside
 * its Linear, scaled_dot_product_attention and multinomial.
 *
 * The conventions are those of torchjs_hip.h: int status, the library's one
 * stream, asynchronous, strides in elements.  All can be captured into a HIP
 * graph.
 *
 * Four bits: a code is a sign (8) and the number of a step of 0, 0.5, 1, 1.5,
 * 2, 3, 4, 6, and stands for that step times the float32 scale of the values
 * that it shares one with.  The scale is their largest magnitude over 6,
 * rounded to float32; a code is the step nearest to value / scale, of two that
 * are as near the one with the even number, decided exactly.  Values whose
 * largest magnitude is under 2^-100 are held as zeros; where one is NaN or
 * infinite all that share its scale stand for NaN.
 */
#ifndef TORCHJS_HIP_DECODE_H
#define TORCHJS_HIP_DECODE_H

#include "torchjs_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Weights w [N, K] (row stride ld >= K) in 4 bits, `group` (32, 64 or 128)
 * columns to a scale.  With nb = ceil(K / 128): codes [N, 64 nb] bytes, 16-byte
 * aligned, scales [N, nb 128 / group], zeros past K.  A row's 64 bytes of 128
 * columns hold column 32 t + 8 j + e in the 4 bits e of 32-bit word 4 j + t
 * (t, j < 4, e < 8): what a lane of the matrix cores takes is 16 bytes. */
int tjh_fp4_quantize(const float* w, int64_t ld, int64_t N, int64_t K, int64_t group,
                     uint8_t* codes, float* scales);
/* out [N, K] (row stride ldo >= K) = the values that codes and scales stand for. */
int tjh_fp4_dequantize(const uint8_t* codes, const float* scales, int64_t N, int64_t K,
                       int64_t group, float* out, int64_t ldo);
/* y [M, N] (row stride ldy) = x [M, K] (row stride ldx) times the transpose of
 * such weights, plus bias [N] (or NULL); sums are float32.  y does not overlap
 * x.  M below 2^31, N and K below 2^26. */
int tjh_fp4_linear(const float* x, int64_t ldx, int64_t M, int64_t N, int64_t K,
                   const uint8_t* codes, const float* scales, int64_t group, const float* bias,
                   float* y, int64_t ldy);

/* A cache of keys and values: each codes [B, H, L, P] with P = 16 ceil(D / 32)
 * bytes a position (column d in the low (d even) or high 4 bits of byte d / 2,
 * zeros past D) and one scale a position, scales [B, H, L]; all contiguous,
 * codes 16-byte aligned.  D up to 128, L below 2^24, else
 * TJH_ERR_UNSUPPORTED.
 *
 * Writes k and v [B, H, T, D] (strides of the four axes) to positions [pos,
 * pos + T), or from positions[b] on in sequence b; given those, positions
 * outside [0, L) are not written. */
int tjh_fp4_cache_append(const float* k, const float* v, const int64_t* k_strides,
                         const int64_t* v_strides, uint8_t* k_codes, float* k_scales,
                         uint8_t* v_codes, float* v_scales, int64_t B, int64_t H, int64_t T,
                         int64_t D, int64_t L, int64_t pos, const int32_t* positions);
/* out [B, H, n, D], contiguous = the values at positions [start, start + n) of
 * one of keys or values, and out2 those of the other (codes2 NULL: none). */
int tjh_fp4_cache_read(const uint8_t* codes, const float* scales, const uint8_t* codes2,
                       const float* scales2, int64_t B, int64_t H, int64_t L, int64_t D,
                       int64_t start, int64_t n, float* out, float* out2);
/* Causal attention of q [B, H, Tq, D] over such a cache of Hkv heads (H a
 * multiple of Hkv; query head h reads head h / (H / Hkv)): the queries are the
 * last Tq of the first `length` positions, or of lengths[b] (taken into [0, L])
 * of sequence b.  The query at position i sees the keys j <= i; one that sees
 * none (at a position before the first) gives zeros; one all of whose scores are
 * -infinity has no distribution and gives NaN.  o = softmax(scale q k^T) v
 * [B, H, Tq, D]; strides of q and o for the B, H and T axes, D contiguous.  What
 * positions past a sequence's length hold has no part in it.  Sums are float32:
 * a key's before its scale, for |q| under 2^118; a row's, of weights up to 2^10
 * times the values of up to 2^24 positions, before it is divided by the sum of
 * the weights, for values under 2^94. */
int tjh_fp4_attention(const float* q, const uint8_t* k_codes, const float* k_scales,
                      const uint8_t* v_codes, const float* v_scales, float* o, int64_t B,
                      int64_t H, int64_t Hkv, int64_t Tq, int64_t L, int64_t D,
                      const int64_t* q_strides, const int64_t* o_strides, int64_t length,
                      const int32_t* lengths, float scale);

/* One step of a beam search: of the continuations (w, v) of a search's W beams
 * by V tokens, with scores[b, w] + x[v] - ln sum exp x (x the beam's row of
 * logits [B, W, V] at row stride ld), the `keep` largest in descending order,
 * equal ones by ascending w, of a beam by descending x, then by ascending v:
 * scores, tokens, parents (w), all [B, keep].  A
 * beam with finished[b, w] != 0 (finished may be NULL) goes on as (eos, its
 * score) alone.  out_finished: the parent's flag, or 1 where the token is eos
 * (eos < 0: no such token, finished must be NULL).  A beam whose score is
 * -infinity or NaN, or whose row holds NaN or +infinity or nothing above
 * -infinity, has no continuation, nor has a token of -infinity; where fewer
 * than `keep` are there, the rest has score -infinity, token -1, parent
 * min(place, W - 1) and flag 1.  Scores are compared in 64 bits and rounded at
 * the end.  W and keep up to 64, V up to 2^20, keep <= W V; else
 * TJH_ERR_UNSUPPORTED (TJH_ERR_INVALID). */
int tjh_beam_step(const float* logits, int64_t ld, const float* scores, const uint8_t* finished,
                  int64_t B, int64_t W, int64_t V, int64_t keep, int64_t eos, float* out_scores,
                  int32_t* tokens, int32_t* parents, uint8_t* out_finished);
/* In place, for each of n tensors: row b W + i becomes row b W + parents[b, i]
 * as it was (parents [B, W] int32; one outside [0, W) leaves its row).  Tensor t
 * has B W rows of outers[t] blocks of strides[t] bytes each, of whose every one
 * the first sizes[t] bytes are moved.  The tensors do not overlap.  W up to 64,
 * else TJH_ERR_UNSUPPORTED. */
int tjh_cache_reorder(int n, void* const* tensors, const int64_t* outers, const int64_t* strides,
                      const int64_t* sizes, int64_t B, int64_t W, const int32_t* parents);

#ifdef __cplusplus
}
#endif
#endif /* TORCHJS_HIP_DECODE_H */
