"""That 4-bit products and attention keep the 24 bits of their float operands: errors
in the 2-norm against 64 bits, under bounds that are shown, without a GPU, to fail
where an operand is cut to two of its three bfloat16 parts.

A bound element by element has to allow that all roundings add up; the 2-norm goes by
how they add up at random, against the size of a sum whose terms have random signs,
sqrt(sum of squares).  In units of U, half a step: a matrix instruction adds 32
products and cuts each off below a step (2 U) of the sum, 2 / sqrt(3) sqrt(32) = 6.5 in
all; a chain of c float additions, each U / sqrt(3) of a sum that grows to the whole,
sqrt(c / 6)."""
import numpy as np
import pytest

from test_gpu_decode_ops import (ATTEND, LINEAR, SOME, U, _filled, _linear_case, _weight, held,
                                 held_weight)

gpu = pytest.mark.gpu
PRODUCTS = sorted(set(LINEAR + SOME))


def _linear_bound(k):
    """Products of 32 columns, the chain of their sums, and three roundings each of
    the parts', the waves' and slices' and the bias's."""
    return (6.5 + (k / 32 / 6) ** 0.5 + 3) * U


def _linear_size(x, v, b=None):
    size = (x.astype(np.float64) ** 2) @ (v.T ** 2)
    return np.sqrt(size + (0 if b is None else b.astype(np.float64) ** 2))


# The weights: a score t (in powers of two, random size up to 1.5 with these inputs,
# up to 8 from the maximum) is off by 6.5 of its size, one of it, one of its distance;
# times ln 2, and two for the exponential.  Products with the values 6.5, sums over the
# keys and roundings of the weights 3.
ATTENTION_BOUND = (0.6932 * (6.5 * 1.5 + 1.5 + 8) + 2 + 6.5 + 3) * U


def _attend(q, k, v, cut_q=None, cut_p=None):
    """Causal attention in 64 bits of queries at the end of all keys, and the random
    size of its sums; cut_q and cut_p are applied to the scaled queries and to the
    weights before they are divided by their sum."""
    b, h, tq, d = q.shape
    group, n = h // k.shape[1], k.shape[2]
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    unseen = np.arange(n)[None, :] > np.arange(n - tq, n)[:, None]
    for i in range(b):
        for j in range(h):
            kk, vv = k[i, j // group], v[i, j // group]
            f = q[i, j].astype(np.float64) * np.float32(d ** -0.5)
            s = (cut_q(f).astype(np.float64) if cut_q else f) @ kk.T
            s[unseen] = -np.inf
            p = np.exp(s - s.max(-1, keepdims=True))
            den = p.sum(-1, keepdims=True)
            if cut_p:
                p = cut_p(p).astype(np.float64)
            out[i, j] = p @ vv / den
            size[i, j] = np.sqrt((p / den) ** 2 @ vv ** 2)
    return out, size


def two_parts(x):
    """A float cut to its first 16 bits: two bfloat16 parts of eight bits each."""
    return (np.asarray(x, np.float32).view(np.uint32) & np.uint32(0xffffff00)).view(np.float32)


def _norm(x):
    return np.linalg.norm(np.asarray(x, np.float64).ravel())


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_products_keep_24_bits(torch, m, k, n, group):
    x, b, codes, scales, want, _ = _linear_case(torch, m, k, n, group, n % 2 == 1, 7)
    v = torch.functional.dequantize_fp4(codes, scales, k, group).numpy().astype(np.float64)
    y = torch.functional.linear_fp4(torch.tensor(x), codes, scales,
                                    torch.tensor(b) if b is not None else None, group).numpy()
    size = _linear_size(x, v, b)
    assert _norm(y - want) <= _linear_bound(k) * _norm(size)
    # and so in each sixteenth of the rows and columns, which a wrong tile would fill
    err = (y - want) ** 2
    for axis in (0, 1):
        for part in np.array_split(np.arange(y.shape[axis]), 16):
            if part.size * y.shape[1 - axis] >= 64:
                e, s = err.take(part, axis).sum(), (size.take(part, axis) ** 2).sum()
                assert e <= (2 * _linear_bound(k)) ** 2 * s


@gpu
@pytest.mark.parametrize("b,h,hkv,tq,n,d", ATTEND)
def test_attention_keeps_24_bits(torch, b, h, hkv, tq, n, d):
    rng = np.random.default_rng(b * n + d + 1)
    cache, k, v = _filled(torch, b, hkv, n, d, rng, 0.3)
    q = rng.standard_normal((b, h, tq, d)).astype(np.float32)
    y = torch.functional.attention_fp4(torch.tensor(q), *cache, n).numpy()
    want, size = _attend(q, k, v)
    assert _norm(y - want) <= ATTENTION_BOUND * _norm(size)


@pytest.mark.parametrize("m,k,n", [c for c in PRODUCTS if c[1] * min(c[2], 300) < 1 << 22])
def test_bound_of_products_tells_two_parts(m, k, n):
    rng = np.random.default_rng(7)
    v = held_weight(_weight(rng, min(n, 300), k), 64)[2]
    x = rng.standard_normal((min(m, 64), k)).astype(np.float32)
    if m * k < 64:  # of so few numbers one may end in zeros: some others
        x = rng.standard_normal((64, k)).astype(np.float32)
    err = _norm((x - two_parts(x).astype(np.float64)) @ v.T)
    assert err > 3 * _linear_bound(k) * _norm(_linear_size(x, v))


@pytest.mark.parametrize("b,h,hkv,tq,n,d", [c for c in ATTEND if c[4] >= 20 and c[0] * c[1] * c[3] < 2000])
@pytest.mark.parametrize("which", ["queries", "weights"])
def test_bound_of_attention_tells_two_parts(b, h, hkv, tq, n, d, which):
    rng = np.random.default_rng(b * n + d + 1)
    k, v = rng.standard_normal((2, b, hkv, n, d)).astype(np.float32)
    k *= np.exp(0.3 * rng.standard_normal((1, hkv, 1, d))).astype(np.float32)
    q = rng.standard_normal((b, h, tq, d)).astype(np.float32)
    k, v = held(k)[2], held(v)[2]
    want, size = _attend(q, k, v)
    got, _ = _attend(q, k, v, **{"cut_q" if which == "queries" else "cut_p": two_parts})
    assert _norm(got - want) > 2 * ATTENTION_BOUND * _norm(size)
