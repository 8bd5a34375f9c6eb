"""Decoding in four bits and with beams (torch.nn.functional exports these):
products with 4-bit weights beside linear (src/nn/linear.ts:43-66), a key /
value cache in 4 bits with the attention that reads it beside
scaled_dot_product_attention (src/nn/functional.ts:866-890), and a beam
search's step beside Tensor.multinomial (src/tensor/Tensor.ts:271-359);
torch.js has none of them.

Four bits stand for 0, 0.5, 1, 1.5, 2, 3, 4, 6 or their negatives, times a
float32 scale: the largest magnitude of the values that share it over 6.  Each
value becomes the nearest step, of two that are as near the one whose number is
even.  Values whose largest magnitude is under 2^-100 are held as zeros; where
one is NaN or infinite, all that share its scale become NaN."""
import ctypes
import functools

import numpy as np

from . import _lib as L
from . import tensor as _T
from .tensor import (Storage, Tensor, _empty_padded, _gemm, _k_contiguous, _numel, _record, empty,
                     reshape_raw)

GROUPS = (32, 64, 128)


def _group(who, group_size):
    if group_size not in GROUPS:
        raise ValueError("%s: group_size must be one of %s, got %r"
                         % (who, list(GROUPS), group_size))
    return int(group_size)


def _weight_shapes(n, k, group):
    """Shapes of a [n, k] weight's codes and scales: whole blocks of 128."""
    blocks = (k + 127) // 128
    return (n, 64 * blocks), (n, blocks * 128 // group)


def _weights(who, codes, scales, k, group):
    """Checks 4-bit weights of k columns; (number of rows, pointer of the codes,
    of the scales)."""
    if not (isinstance(codes, Tensor) and isinstance(scales, Tensor)):
        raise TypeError("%s: codes and scales must be tensors" % who)
    n = _weight_rows(who, codes._shape, codes._strides, codes._dtype, scales._shape,
                     scales._strides, scales._dtype, k, group)
    p = codes.data_ptr()
    if p & 15:
        raise ValueError("%s: codes must be 16-byte aligned" % who)
    return n, p, scales.data_ptr()


@functools.lru_cache(maxsize=1024)
def _weight_rows(who, cs, cst, cd, ss, sst, sd, k, group):
    if len(cs) != 2 or cd != "uint8" or sd != "float32":
        raise TypeError("%s: codes must be a 2-D uint8 tensor and scales a float32 one" % who)
    if (cs, ss) != _weight_shapes(cs[0], k, group):
        raise ValueError("%s: codes %s and scales %s do not hold %d columns in groups of %d"
                         % (who, list(cs), list(ss), k, group))
    if not (_contiguous(cs, cst) and _contiguous(ss, sst)):
        raise ValueError("%s: codes and scales must be contiguous" % who)
    return cs[0]


def _contiguous(shape, strides):
    return not _numel(shape) or all(
        a == b for a, b, n in zip(strides, _T._contig_strides(shape), shape) if n != 1)


@functools.lru_cache(maxsize=1024)
def _strides(st):
    """Strides as the C entry points take them."""
    return L.i64arr(st)


def quantize_fp4(weight, group_size=64):
    """(codes, scales) of weight [N, K] in 4 bits, group_size (32, 64 or 128)
    columns of a row to a scale, laid out for linear_fp4: codes uint8
    [N, 64 ceil(K / 128)], scales float32 [N, 128 / group_size ceil(K / 128)]."""
    g = _group("quantize_fp4", group_size)
    if weight.ndim != 2:
        raise ValueError("quantize_fp4: expected a [N, K] weight, got shape %s"
                         % (list(weight.shape),))
    w = weight.detach()
    w = w if w.dtype == "float32" else w.float()
    w, pw, ld, n, k = _T._rows_2d(w)
    cs, ss = _weight_shapes(n, k, g)
    codes, scales = empty(cs, "uint8"), empty(ss)
    L.check(L.lib().tjh_fp4_quantize(pw, ld, n, k, g, codes.data_ptr(), scales.data_ptr()),
            "quantize_fp4")
    return codes, scales


def dequantize_fp4(codes, scales, in_features, group_size=64):
    """The float32 weight [N, in_features] that quantize_fp4's codes and scales
    stand for."""
    g = _group("dequantize_fp4", group_size)
    k = int(in_features)
    n, pc, ps = _weights("dequantize_fp4", codes, scales, k, g)
    out = empty((n, k))
    L.check(L.lib().tjh_fp4_dequantize(pc, ps, n, k, g, out.data_ptr(), k), "dequantize_fp4")
    return out


def linear_fp4(x, codes, scales, bias=None, group_size=64):
    """y = x W^T + b for x [..., K] and the 4-bit weight [N, K] of
    quantize_fp4, summed in float32 (a group before its scale: for x under 2^118 in
    magnitude).  The gradient goes to x (through the float weight, formed for it)
    and to bias; the weight has none."""
    g = _group("linear_fp4", group_size)
    if not x._shape:
        raise ValueError("linear_fp4: x has no dimensions")
    if x._dtype != "float32":
        x = x.float()
    k, lead = x._shape[-1], x._shape[:-1]
    n, pc, ps = _weights("linear_fp4", codes, scales, k, g)
    b = bias
    if b is not None:
        if b._shape != (n,):
            raise ValueError("linear_fp4: bias of shape %s for %d outputs" % (list(b._shape), n))
        if b._dtype != "float32" or b._strides != (1,):
            b = b.detach().float().contiguous()
    # the tensor that holds x's rows lives until the launch is queued
    xd, px, ld, m, _ = _T._rows_2d(x)
    pb = b.data_ptr() if b is not None else None
    y = _empty_padded(m, n) if n % 4 else Tensor(Storage(max(1, m * n) * 4), (m, n))
    L.check(L.lib().tjh_fp4_linear(px, ld, m, n, k, pc, ps, g, pb, y.data_ptr(),
                                   max(y._strides[0], n)), "linear_fp4")
    out = reshape_raw(y, lead + (n,)) if len(lead) != 1 else y
    if not _T._recorded(x, bias):
        return out
    rx, rb = x.requires_grad, bias is not None and bias.requires_grad

    def bwd(gr):
        g2 = reshape_raw(gr, (m, n))
        dx = db = None
        if rx:
            dx = reshape_raw(_gemm(g2, dequantize_fp4(codes, scales, k, g)), lead + (k,))
        if rb:
            gc = g2 if g2.is_contiguous() else _k_contiguous(g2)
            db = _T._view_raw(_T._k_reduce("sum", gc, [0]), (n,))
        return [dx, db]

    def gbwd(gr):  # linear in the gradient: a product with a constant
        g2 = _T.reshape(gr, (m, n))
        dx = db = None
        if rx:
            dx = _T.reshape(_T.matmul(g2, dequantize_fp4(codes, scales, k, g)), lead + (k,))
        if rb:
            db = _T.reduce_sum(g2, 0)
        return [dx, db]
    return _record(out, "LinearFP4", [x, bias], bwd, gfn=gbwd)


# ------------------------------------------------------------------ cache


def cache_row_bytes(head_dim):
    """Bytes of a cached position's codes: half of head_dim, in whole 16s."""
    return (int(head_dim) + 31) // 32 * 16


def _cache(who, codes, scales, d):
    """Checks a cache of one of keys or values: its (B, H, L), its pointers."""
    if not (isinstance(codes, Tensor) and isinstance(scales, Tensor)):
        raise TypeError("%s: a cache's codes and scales must be tensors" % who)
    shape = _cache_shape(who, codes._shape, codes._strides, codes._dtype, scales._shape,
                         scales._strides, scales._dtype, d)
    p = codes.data_ptr()
    if p & 15:
        raise ValueError("%s: a cache's codes must be 16-byte aligned" % who)
    return shape, p, scales.data_ptr()


@functools.lru_cache(maxsize=1024)
def _cache_shape(who, cs, cst, cd, ss, sst, sd, d):
    if cd != "uint8" or sd != "float32":
        raise TypeError("%s: a cache's codes must be uint8 and its scales float32" % who)
    if len(cs) != 4 or cs[3] != cache_row_bytes(d) or ss != cs[:3]:
        raise ValueError("%s: codes %s and scales %s do not hold heads of %d columns"
                         % (who, list(cs), list(ss), d))
    if not (_contiguous(cs, cst) and _contiguous(ss, sst)):
        raise ValueError("%s: a cache must be contiguous" % who)
    return cs[:3]


def _per_sequence(who, name, value, b):
    """(number, pointer or None, tensor) of a whole number, or of one of each
    of b sequences."""
    if type(value) is int and 0 <= value < 1 << 62:
        return value, None, None
    if isinstance(value, Tensor) or np.ndim(value):
        t = value
        if not isinstance(t, Tensor):
            a = np.asarray(value)
            if a.dtype.kind not in "iu":
                raise TypeError("%s: %s must be whole numbers" % (who, name))
            t = _T.tensor(np.clip(a, -2 ** 31, 2 ** 31 - 1).astype(np.int32), dtype="int32")
        if t.dtype != "int32":
            raise TypeError("%s: %s must be an int32 tensor, got %s" % (who, name, t.dtype))
        if t.shape != (b,):
            raise ValueError("%s: %s of shape %s for %d sequences"
                             % (who, name, list(t.shape), b))
        t = t.contiguous()
        return 0, t.data_ptr(), t
    n = int(value)
    if n != value or n < 0:
        raise ValueError("%s: %s must be a whole number, got %r" % (who, name, value))
    return min(n, 1 << 62), None, None


def cache_append_fp4(k_codes, k_scales, v_codes, v_scales, key, value, pos):
    """Writes key and value [B, H, T, D] in 4 bits, one scale a position and
    head, to positions [pos, pos + T) of a cache: codes uint8
    [B, H, L, cache_row_bytes(D)], scales float32 [B, H, L].  pos may be an int32
    tensor [B], where each sequence's new positions begin; positions outside
    [0, L) are then not written.  D up to 128."""
    who = "cache_append_fp4"
    ks = key._shape
    if len(ks) != 4 or ks != value._shape:
        raise ValueError("%s: key %s and value %s must be [B, H, T, D] alike"
                         % (who, list(ks), list(value._shape)))
    B, H, T, D = ks
    if not 0 < D <= 128:
        raise NotImplementedError("%s: head dims up to 128, got %d" % (who, D))
    shape, pkc, pks = _cache(who, k_codes, k_scales, D)
    vshape, pvc, pvs = _cache(who, v_codes, v_scales, D)
    if vshape != shape or shape[:2] != (B, H):
        raise ValueError("%s: key %s does not fit caches %s and %s"
                         % (who, list(ks), list(k_codes._shape), list(v_codes._shape)))
    if (pkc == pvc or pks == pvs) and _numel(shape):
        raise ValueError("%s: keys and values are one cache" % who)
    n, p, _keep = _per_sequence(who, "pos", pos, B)
    if p is None and n + T > shape[2]:
        raise RuntimeError("KV cache: position %d beyond its length %d" % (n + T, shape[2]))
    if key._dtype != "float32":
        key = key.float()
    if value._dtype != "float32":
        value = value.float()
    pk, pv = key.data_ptr(), value.data_ptr()
    _T._before_write(k_codes, k_scales, v_codes, v_scales)
    L.check(L.lib().tjh_fp4_cache_append(
        pk, pv, _strides(key._strides), _strides(value._strides), pkc, pks, pvc, pvs, B, H, T, D,
        shape[2], n, p), who)


def cache_read_fp4(codes, scales, head_dim, start, stop, other=None):
    """The float32 values [B, H, stop - start, head_dim] that positions
    [start, stop) of a cache's keys or values stand for; with `other`, the
    (codes, scales) of the other of the two, both as a pair."""
    who = "cache_read_fp4"
    d = int(head_dim)
    if not 0 < d <= 128:
        raise NotImplementedError("%s: head dims up to 128, got %d" % (who, d))
    shape, pc, ps = _cache(who, codes, scales, d)
    pc2 = ps2 = None
    if other is not None:
        shape2, pc2, ps2 = _cache(who, other[0], other[1], d)
        if shape2 != shape:
            raise ValueError("%s: caches of shapes %s and %s"
                             % (who, list(codes._shape), list(other[0]._shape)))
    B, H, n = shape
    if not 0 <= start <= stop <= n or start != int(start) or stop != int(stop):
        raise ValueError("%s: positions [%s, %s) of %d" % (who, start, stop, n))
    rows = int(stop) - int(start)
    size, sh = B * H * rows * d, (B, H, rows, d)
    # both in one allocation, the second one 16-byte aligned
    second = (size + 3) & ~3
    st = Storage(max(1, 2 * second if pc2 is not None else size) * 4)
    L.check(L.lib().tjh_fp4_cache_read(pc, ps, pc2, ps2, B, H, n, d, int(start), rows, st.ptr,
                                       st.ptr + 4 * second), who)
    out = Tensor(st, sh)
    return out if pc2 is None else (out, Tensor(st, sh, None, second))


def attention_fp4(query, k_codes, k_scales, v_codes, v_scales, length, scale=None):
    """Causal attention of query [B, H, Tq, D] over a cache in 4 bits of Hkv
    heads (cache_append_fp4), H a multiple of Hkv (query head h reads head
    h // (H // Hkv)).  The queries are the last Tq of the cache's first `length`
    positions (already in the cache), or of length[b] of sequence b (an int32
    tensor [B], taken into [0, L]); one that sees no key, before the first
    position, gives zeros, and one all of whose scores are -infinity NaN.  What
    later positions hold has no part in the result.
    Sums are float32 (a key's before its scale: for queries under 2^118 in
    magnitude; a row's before its weights are divided by their sum: for values
    under 2^94 in the cache); D up to 128.  For inference: a query that needs a
    gradient is refused."""
    who = "attention_fp4"
    qs = query._shape
    if len(qs) != 4:
        raise ValueError("%s: expected a [B, H, Tq, D] query, got shape %s" % (who, list(qs)))
    if _T._recorded(query):
        raise RuntimeError("%s: no gradient is taken through a cache in 4 bits; run it under "
                           "no_grad()" % who)
    B, H, Tq, D = qs
    if not 0 < D <= 128:
        raise NotImplementedError("%s: head dims up to 128, got %d" % (who, D))
    shape, pkc, pks = _cache(who, k_codes, k_scales, D)
    vshape, pvc, pvs = _cache(who, v_codes, v_scales, D)
    if vshape != shape or shape[0] != B:
        raise ValueError("%s: query %s does not fit caches %s and %s"
                         % (who, list(qs), list(k_codes._shape), list(v_codes._shape)))
    Hkv, n = shape[1:]
    if (Hkv == 0) != (H == 0) or (Hkv and H % Hkv):
        raise RuntimeError("%s: %d query heads over %d of keys" % (who, H, Hkv))
    count, p, _keep = _per_sequence(who, "length", length, B)
    if p is None:
        if count > n:
            raise ValueError("%s: length %d of a cache of %d" % (who, count, n))
        if Tq > count:
            raise RuntimeError("%s: %d queries are not the last of %d positions"
                               % (who, Tq, count))
    q = query if query._dtype == "float32" else query.float()
    if q._strides[3] != 1 and D > 1:
        q = _k_contiguous(q)
    o = Storage(max(1, B * Tq * H * D) * 4)
    st = (Tq * H * D, D, H * D, 1)
    L.check(L.lib().tjh_fp4_attention(
        q.data_ptr(), pkc, pks, pvc, pvs, o.ptr, B, H, Hkv, Tq, n, D, _strides(q._strides),
        _strides(st), count, p, float(scale) if scale is not None else D ** -0.5), who)
    return Tensor(o, qs, st)


# ------------------------------------------------------------------ beams


def beam_step(logits, scores, beams=None, finished=None, eos=None):
    """One step of a beam search over B sequences with W beams each: logits
    [B, W, V] (or [B * W, V]) of the beams' next tokens and their scores [B, W],
    sums of logarithms of probabilities.  Of the continuations (w, v), which
    have score scores[w] + log_softmax(logits[w])[v], takes the `beams` (W
    unless given) largest.  Scores are compared in 64 bits; equal ones go by
    ascending w, of a beam by descending logit, then by ascending v, whatever
    `beams` is.  Returns (scores,
    tokens, parents, finished), each [B, beams]: int32 tokens and the beams that
    they continue, and whether the new beam has ended, as its token is `eos` or
    its parent had ended.  finished [B, W] (bool): a beam that has ended goes on
    only as itself, by the token eos.

    A beam of score -infinity (or NaN), or whose logits hold NaN, +infinity or
    nothing above -infinity, has no continuation, nor has a token of -infinity;
    places that remain empty get score -infinity, token -1, the parent of their
    own number (the last beam's at most), and count as ended.  W and beams up to
    64, V up to 2^20.  No gradient."""
    who = "beam_step"
    if not isinstance(scores, Tensor):
        scores = _T.tensor(np.asarray(scores, dtype=np.float32))
    ss, ls = scores._shape, logits._shape
    if len(ss) != 2 or ss[1] == 0:
        raise ValueError("%s: expected scores [B, W], got shape %s" % (who, list(ss)))
    B, W = ss
    if len(ls) not in (2, 3) or ls[-1] == 0 or \
            (ls[:-1] != ss if len(ls) == 3 else ls[0] != B * W):
        raise ValueError("%s: logits of shape %s for scores %s" % (who, list(ls), [B, W]))
    V = ls[-1]
    keep = W if beams is None else int(beams)
    if keep < 1 or keep != (W if beams is None else beams) or keep > W * V:
        raise ValueError("%s: %r beams of %d continuations" % (who, beams, W * V))
    if eos is not None and not (eos == int(eos) and 0 <= eos < V):
        raise ValueError("%s: eos %r of %d tokens" % (who, eos, V))
    if finished is not None:
        if eos is None:
            raise ValueError("%s: ended beams go on by eos, which is not given" % who)
        if not isinstance(finished, Tensor):
            finished = _T.tensor(np.asarray(finished, dtype=np.bool_))
        if finished.dtype not in ("bool", "uint8"):
            raise TypeError("%s: finished must be bool, got %s" % (who, finished.dtype))
        if finished.shape != (B, W):
            raise ValueError("%s: finished of shape %s for scores %s"
                             % (who, list(finished.shape), [B, W]))
        finished = finished.contiguous()
    x = logits if logits._dtype == "float32" else logits.float()
    if scores._dtype != "float32":
        scores = scores.float()
    if not scores.is_contiguous():
        scores = scores.detach().contiguous()
    xd, px, ld, _, _ = _T._rows_2d(x)
    # all four in one allocation
    n, shape = B * keep, (B, keep)
    st = Storage(max(1, 13 * n))
    out, tokens = Tensor(st, shape), Tensor(st, shape, None, n, "int32")
    parents, done = Tensor(st, shape, None, 2 * n, "int32"), Tensor(st, shape, None, 12 * n, "bool")
    p = st.ptr
    L.check(L.lib().tjh_beam_step(px, ld, scores.data_ptr(),
                                  finished.data_ptr() if finished is not None else None, B, W, V,
                                  keep, -1 if eos is None else int(eos), p, p + 4 * n, p + 8 * n,
                                  p + 12 * n), who)
    return out, tokens, parents, done


def cache_reorder_(tensors, parents, length=None):
    """In place, for each of `tensors` [B * W, ...]: row b * W + i becomes row
    b * W + parents[b, i] as it was, for parents [B, W] (beam_step's; an entry
    outside [0, W) leaves its row).  With `length`, tensors are
    [B * W, H, L, ...] and only the first `length` positions of L are moved.  They
    must be contiguous, share no memory, and need no gradient.  W up to 64."""
    who = "cache_reorder_"
    if isinstance(tensors, Tensor):
        tensors = [tensors]
    tensors = list(tensors)
    if not isinstance(parents, Tensor):
        a = np.asarray(parents)
        if a.dtype.kind not in "iu":
            raise TypeError("%s: parents must be whole numbers" % who)
        parents = _T.tensor(np.clip(a, -2 ** 31, 2 ** 31 - 1).astype(np.int32), dtype="int32")
    if parents.dtype != "int32":
        raise TypeError("%s: parents must be int32, got %s" % (who, parents.dtype))
    if parents.ndim != 2:
        raise ValueError("%s: expected parents [B, W], got shape %s"
                         % (who, list(parents.shape)))
    B, W = parents.shape
    if length is not None and length != int(length):
        raise ValueError("%s: %r positions" % (who, length))
    for t in tensors:
        if t.requires_grad:
            raise RuntimeError("%s: a tensor that requires grad is changed in place" % who)
    geometry = _reorder_geometry(tuple([(t._shape, t._strides, t._dtype) for t in tensors]), B * W,
                                 None if length is None else int(length))
    ptrs = [t.data_ptr() for t in tensors]
    parents = parents.contiguous()
    spans = list(zip(ptrs, geometry[0]))
    spans.append((parents.data_ptr(), 4 * parents.numel()))
    spans.sort()
    end = 0
    for p, size in spans:
        if size:
            if p < end:
                raise ValueError("%s: tensors share memory" % who)
            end = p + size
    _T._before_write(*tensors)
    L.check(L.lib().tjh_cache_reorder(len(ptrs), (ctypes.c_void_p * max(1, len(ptrs)))(*ptrs),
                                      *geometry[1:], B, W, parents.data_ptr()), who)


@functools.lru_cache(maxsize=256)
def _reorder_geometry(kinds, rows, length):
    """(bytes of each tensor, blocks a row, bytes of a block, of them moved), the
    last three as the library takes them, for tensors of these shapes, strides and
    types."""
    who = "cache_reorder_"
    total, outers, strides, sizes = [], [], [], []
    for sh, st, dtype in kinds:
        if not sh or sh[0] != rows:
            raise ValueError("%s: a tensor of shape %s for %d rows" % (who, list(sh), rows))
        if any(a != b for a, b, n in zip(st, _T._contig_strides(sh), sh) if n != 1) and _numel(sh):
            raise ValueError("%s: a tensor of shape %s is not contiguous" % (who, list(sh)))
        item = _T._DT[dtype][0]
        if length is None:
            outer, size = 1, _numel(sh[1:]) * item
            part = size
        else:
            if len(sh) < 3 or not 0 <= length <= sh[2]:
                raise ValueError("%s: %d positions of a tensor of shape %s"
                                 % (who, length, list(sh)))
            outer, size = sh[1], _numel(sh[2:]) * item
            part = length * _numel(sh[3:]) * item
        total.append(rows * outer * size)
        outers.append(outer)
        strides.append(size)
        sizes.append(part)
    return total, L.i64arr(outers), L.i64arr(strides), L.i64arr(sizes)
