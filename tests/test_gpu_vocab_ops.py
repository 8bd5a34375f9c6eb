"""Tensor.topk, F.distillation_loss and F.sample_logits against plain numpy in
64 bits."""
import math
import sys
import types

import numpy as np
import pytest

gpu = pytest.mark.gpu
U = 2.0 ** -24  # half a step of float32, relative


# ------------------------------------------------------------------- oracles


def topk_ref(x, k, largest=True):
    """Indices [rows, k]: NaN the largest, equal values by ascending index."""
    n = x.shape[1]
    x = x.astype(np.float64) + 0.0
    nan = np.isnan(x)
    v = np.where(nan, 0.0, x)
    idx = np.broadcast_to(np.arange(n), x.shape)
    order = np.lexsort((idx, -v, ~nan) if largest else (idx, v, nan), axis=1)
    return order[:, :k]


def sample_ref(x, u, t=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row's index by the definition, each rule over the sorted row."""
    x = x.astype(np.float64)
    m = x.max()
    if np.isnan(x).any() or not math.isfinite(m):
        return -1
    if not t > 0:
        return int(np.argmax(x == m))
    order = np.lexsort((np.arange(x.size), -x))
    z = x[order] - m
    with np.errstate(invalid="ignore"):
        w = np.exp(np.where(np.isinf(z), -np.inf, z / t))
    keep = np.ones(x.size, bool)
    if 0 < top_k < x.size:
        keep &= np.arange(x.size) < top_k
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(np.where(keep, w, 0.0))[:-1]])
        keep &= before < max(top_p, 1e-300) * np.where(keep, w, 0.0).sum()
    if min_p > 0:
        keep &= z >= min(t * math.log(min_p), 0.0)
    keep[0] = True
    w = np.where(keep, w, 0.0)
    kept = np.zeros(x.size)
    kept[order] = w
    cum = np.cumsum(kept)
    hit = np.nonzero((cum > u * cum[-1]) & (kept > 0))[0]
    return int(hit[0]) if hit.size else int(np.nonzero(kept > 0)[0][-1])


def distill_ref(x, v, ids, t):
    """(per-row loss, per-row gradient of it, valid rows, the sizes that
    float32 roundings scale with: of the loss and of the gradient)."""
    x, v = x.astype(np.float64), v.astype(np.float64)
    rows, n = x.shape
    loss, grad, valid = np.zeros(rows), np.zeros((rows, n)), np.zeros(rows, bool)
    lsize, gsize = np.zeros(rows), np.zeros((rows, n))
    for r in range(rows):
        lq = x[r] / t - x[r].max() / t
        lq = lq - np.log(np.exp(lq).sum())
        at = [i for i in range(ids.shape[1]) if 0 <= ids[r, i] < n and v[r, i] > -np.inf]
        if not at:
            continue
        valid[r] = True
        lp = v[r, at] / t - v[r, at].max() / t
        lp = lp - np.log(np.exp(lp).sum())
        p = np.exp(lp)
        loss[r] = t * t * (p * (lp - lq[ids[r, at]])).sum()
        lsize[r] = t * t * (p * (np.abs(lp) + np.abs(lq[ids[r, at]]) + 1)).sum()
        grad[r] = t * np.exp(lq)
        gsize[r] = grad[r] * (1 + np.abs(lq))
        np.add.at(grad[r], ids[r, at], -t * p)
        np.add.at(gsize[r], ids[r, at], t * p * (1 + np.abs(lp)))
    return loss, grad, valid, lsize, gsize


# --------------------------------------------------------------------- top-k


NS = [1, 2, 3, 5, 6, 7, 63, 255, 1000, 1023, 1024, 1025, 1029, 4096, 4097, 16384, 16387, 50257,
      53248, 53249, 70001]


@gpu
@pytest.mark.parametrize("n", NS)
def test_topk(torch, n):
    rng = np.random.default_rng(n)
    for k in sorted({1, 2, 20, 64, 255, 257, 1024, n // 2, n}):
        if not 0 < k <= min(n, 1024):
            continue
        for largest in (True, False):
            x = rng.standard_normal((3, n)).astype(np.float32) * 3
            v, i = torch.tensor(x).topk(k, largest=largest)
            ref = topk_ref(x, k, largest)
            assert i.dtype == "int32" and v.shape == i.shape == (3, k)
            np.testing.assert_array_equal(i.numpy(), ref, err_msg="k=%d %s" % (k, largest))
            np.testing.assert_array_equal(v.numpy(), np.take_along_axis(x, ref, 1))


@gpu
@pytest.mark.parametrize("n", [6, 500, 3000, 9000, 50257, 60000])
@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "nan", "infinite", "masked", "sorted"])
def test_topk_ties_and_specials(torch, n, kind):
    rng = np.random.default_rng(n)
    x = rng.standard_normal((2, n)).astype(np.float32)
    if kind == "equal":
        x[:] = 1.5
    elif kind == "few":
        x = rng.integers(-2, 3, (2, n)).astype(np.float32)
    elif kind == "zeros":
        x = np.where(rng.random((2, n)) < 0.5, np.float32(0.0), np.float32(-0.0))
    elif kind == "nan":
        x[:, :: 3] = np.nan
    elif kind == "infinite":
        x[:, :: 4], x[:, 1 :: 4] = np.inf, -np.inf
    elif kind == "masked":
        x[:, 5:] = -np.finfo(np.float32).max
        x[1] = -np.inf
    elif kind == "sorted":
        x = np.sort(x, axis=1)
    for k in (1, 3, min(n, 40), min(n, 700)):
        for largest in (True, False):
            v, i = torch.tensor(x).topk(k, largest=largest)
            ref = topk_ref(x, k, largest)
            np.testing.assert_array_equal(i.numpy(), ref, err_msg="k=%d %s" % (k, largest))
            np.testing.assert_array_equal(v.numpy(), np.take_along_axis(x, ref, 1))


@gpu
def test_topk_layouts(torch):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((4, 37, 11)).astype(np.float32)
    t = torch.tensor(x)
    for dim in (0, 1, 2, -1, -2):
        v, i = t.topk(3, dim=dim)
        ref = np.argsort(-x, axis=dim, kind="stable").take(range(3), axis=dim)
        np.testing.assert_array_equal(i.numpy(), ref)
        np.testing.assert_array_equal(v.numpy(), np.take_along_axis(x, ref, dim))
    # rows at every alignment, and rows wider apart than they are long
    w = rng.standard_normal((5, 1234)).astype(np.float32)
    for lo in range(5):
        view = torch.tensor(w)[:, lo:lo + 1001]
        np.testing.assert_array_equal(view.topk(9)[1].numpy(), topk_ref(w[:, lo:lo + 1001], 9))
    one = torch.tensor(w[0])
    np.testing.assert_array_equal(one.topk(5)[1].numpy(), topk_ref(w[:1], 5)[0])
    v, i = torch.tensor(np.float32(3.0).reshape(())).topk(1)
    assert v.shape == i.shape == () and v.item() == 3.0 and i.item() == 0
    assert torch.tensor(w).topk(0)[0].shape == (5, 0)
    assert torch.zeros(0, 7).topk(2)[1].shape == (0, 2)
    ints = torch.tensor(np.array([[3, 9, 9, 1]], np.int32))
    assert ints.topk(2)[1].numpy().tolist() == [[1, 2]]


@gpu
@pytest.mark.parametrize("shape,k,dim", [((5, 1000), 8, -1), ((3, 50257), 64, -1), ((2, 6, 7), 3, 1),
                                         ((1, 3), 3, -1)])
def test_topk_gradient(torch, shape, k, dim):
    rng = np.random.default_rng(k)
    x = rng.standard_normal(shape).astype(np.float32)
    t = torch.tensor(x, requires_grad=True)
    v, i = t.topk(k, dim=dim)
    g = rng.standard_normal(v.shape).astype(np.float32)
    v.backward(torch.tensor(g))
    ref = np.zeros(shape, np.float32)
    np.put_along_axis(ref, i.numpy().astype(np.int64), g, dim)
    np.testing.assert_array_equal(t.grad.numpy(), ref)
    # through a differentiable backward: d/dx of (d sum v^2 / dx)^2
    t2 = torch.tensor(x, requires_grad=True)
    v2, _ = t2.topk(k, dim=dim)
    (d,) = torch.autograd.grad((v2 * v2).sum(), t2, create_graph=True)
    (dd,) = torch.autograd.grad((d * d).sum(), t2)
    ref = np.zeros(shape, np.float32)
    np.put_along_axis(ref, i.numpy().astype(np.int64), 8 * v.numpy(), dim)
    np.testing.assert_allclose(dd.numpy(), ref, rtol=8 * U)


# ------------------------------------------------------------------ sampling


def _settings():
    for top_k in (0, 1, 2, 50, 300, 2000):
        for top_p in (1.0, 0.9, 0.3, 0.0):
            for min_p in (0.0, 0.05, 1.0):
                yield top_k, top_p, min_p


@gpu
@pytest.mark.parametrize("n", [1, 2, 3, 5, 7, 200, 1027, 4096, 4097, 4101, 16384, 16391, 50257, 53252,
                               53253, 70001])
def test_sample_logits(torch, n):
    rng = np.random.default_rng(n)
    rows = 4
    for i, (top_k, top_p, min_p) in enumerate(_settings()):
        t = (1.0, 0.7, 1.3)[i % 3]
        x = (rng.standard_normal((rows, n)) * 2.5).astype(np.float32)
        u = rng.random(rows).astype(np.float32)
        got = torch.functional.sample_logits(torch.tensor(x), torch.tensor(u), t, top_k, top_p, min_p)
        ref = [sample_ref(x[r], float(u[r]), t, top_k, top_p, min_p) for r in range(rows)]
        assert got.dtype == "int32" and got.numpy().tolist() == ref, (top_k, top_p, min_p, t)


@gpu
@pytest.mark.parametrize("n", [5, 900, 5000, 50257, 60001])
@pytest.mark.parametrize("kind", ["equal", "few", "one", "masked", "lowest", "flat", "sharp"])
def test_sample_logits_ties_and_masks(torch, n, kind):
    rng = np.random.default_rng(n)
    rows = 3
    x = rng.standard_normal((rows, n)).astype(np.float32)
    if kind == "equal":
        x[:] = -2.25
    elif kind == "few":
        x = rng.integers(0, 3, (rows, n)).astype(np.float32)
    elif kind == "one":
        x[:] = -np.inf
        x[np.arange(rows), [0, n // 2, n - 1]] = 0.5
    elif kind == "masked":
        x[:, ::2] = -np.inf
    elif kind == "lowest":
        x[:, ::3] = -np.finfo(np.float32).max
        x[1] = -np.finfo(np.float32).max
    elif kind == "flat":
        x *= 1e-4
    elif kind == "sharp":
        x *= 1e30
    for top_k, top_p, min_p in ((0, 1.0, 0.0), (0, 0.7, 0.0), (3, 1.0, 0.0), (400, 0.5, 0.0),
                                (1500, 0.9, 0.0), (0, 1.0, 0.5), (4, 0.6, 0.2)):
        u = rng.random(rows).astype(np.float32)
        got = torch.functional.sample_logits(torch.tensor(x), torch.tensor(u), 1.0, top_k, top_p, min_p)
        ref = [sample_ref(x[r], float(u[r]), 1.0, top_k, top_p, min_p) for r in range(rows)]
        assert got.numpy().tolist() == ref, (top_k, top_p, min_p)


@gpu
@pytest.mark.parametrize("n", [9, 4099, 50257, 60001])
def test_sample_logits_ends(torch, n):
    """The smallest and largest uniforms, greedy rows, extreme temperatures
    and rows without a distribution."""
    F = torch.functional
    rng = np.random.default_rng(n)
    x = rng.uniform(-3, 3, (6, n)).astype(np.float32)
    for kw in ({}, {"top_k": 5}, {"top_p": 0.5}, {"min_p": 0.3}):
        # u = 1 is past every running sum: the last kept index
        for u in (0.0, 0.99999994, 1.0):
            got = F.sample_logits(torch.tensor(x), np.full(6, u, np.float32), **kw)
            ref = [sample_ref(r, float(np.float32(u)), 1.0, **kw) for r in x]
            assert got.numpy().tolist() == ref, (kw, u)
    y = x.copy()
    y[:, [n // 3, n - 1]] = 4.0
    assert F.sample_logits(torch.tensor(y), np.zeros(6, np.float32), 0.0).numpy().tolist() == [n // 3] * 6
    u = rng.random(6).astype(np.float32)
    for t in (1e-30, 1e-6, 1e30, math.inf):
        for top_p in (1.0, 0.4):
            got = F.sample_logits(torch.tensor(x), u, t, top_p=top_p).numpy().tolist()
            assert got == [sample_ref(x[r], float(u[r]), t, top_p=top_p) for r in range(6)], (t, top_p)
    bad = x.copy()
    bad[0, n - 1], bad[1, 0], bad[2] = np.nan, np.inf, -np.inf
    got = F.sample_logits(torch.tensor(bad), u, top_k=3, top_p=0.9).numpy().tolist()
    assert got[:3] == [-1] * 3
    assert got[3:] == [sample_ref(x[r], float(u[r]), 1.0, 3, 0.9) for r in range(3, 6)]


@gpu
@pytest.mark.parametrize("n", [50, 4099, 50257, 60001])
def test_sample_logits_settings_of_each_row(torch, n):
    rng = np.random.default_rng(n)
    rows = 12
    x = (rng.standard_normal((rows, n)) * 2.5).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    t = np.array([0.5, 1, 2, 0, -1, np.nan, 1, 1, 1, 0.9, 1, 1], np.float32)
    k = np.array([0, 1, 20, 3, 3, 3, -5, n, 10 ** 6, 300, 1400, 7], np.int32)
    p = np.array([1, 0.5, 0.9, 1, 1, 1, 2, np.nan, 0.9, -1, 0.8, 1], np.float32)
    m = np.array([0, 0, 0.1, 0, 0, 0, -1, np.nan, 2, 0, 0, 0.2], np.float32)
    got = torch.functional.sample_logits(torch.tensor(x), torch.tensor(u), torch.tensor(t), k, p, m)
    ref = [sample_ref(x[r], float(u[r]), float(t[r]), int(k[r]), float(p[r]), float(m[r]))
           for r in range(rows)]
    assert got.numpy().tolist() == ref


@gpu
@pytest.mark.parametrize("n", [50257, 60001])
def test_sample_logits_nucleus_in_one_bin(torch, n):
    """One far outlier below: the whole nucleus falls into one bin of the
    histogram, more different logits than a list holds."""
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((3, n)) * 1e-4).astype(np.float32)
    x[0, 5], x[1, n - 1], x[2, n // 2] = -100, -100, -np.finfo(np.float32).max
    u = rng.random(3).astype(np.float32)
    for kw in (dict(top_p=0.7), dict(top_p=0.05), dict(top_p=0.6, top_k=20000), dict(top_p=0.9, min_p=0.9999)):
        got = torch.functional.sample_logits(torch.tensor(x), torch.tensor(u), **kw)
        assert got.numpy().tolist() == [sample_ref(x[r], float(u[r]), **kw) for r in range(3)], kw


@gpu
@pytest.mark.parametrize("n", [1500, 4000, 16001, 50257, 60001])
def test_sample_logits_nucleus_ends_among_ties(torch, n):
    """Logits of a few values: a list holds what can be drawn, and the bin in
    which the nucleus ends holds more than the short sort takes."""
    rng = np.random.default_rng(n)
    rows = 64
    x = np.full((rows, n), -40, np.float32)
    for r in range(rows):
        at = rng.permutation(n)[:min(n, 3900)]
        x[r, at] = -0.7 * rng.integers(0, 3, at.size)
    u = rng.random(rows).astype(np.float32)
    for kw in (dict(top_p=0.35), dict(top_p=0.77), dict(top_p=0.97), dict(top_p=0.6, min_p=0.3),
               dict(top_p=0.8, top_k=1200)):
        ref = [sample_ref(x[r], float(u[r]), **kw) for r in range(rows)]
        for _ in range(2):
            got = torch.functional.sample_logits(torch.tensor(x), torch.tensor(u), **kw)
            assert got.numpy().tolist() == ref, kw


@gpu
@pytest.mark.parametrize("n", [9001, 600000, 2 ** 20])
def test_sample_logits_of_neighbours(torch, n):
    """All that can be drawn stands side by side."""
    rng = np.random.default_rng(n)
    x = np.full((4, n), -8, np.float32) + rng.random((4, n)).astype(np.float32) / 8
    for r, at in enumerate((0, 5001, n - 2000, n // 2)):
        x[r, at:at + 2000] = rng.standard_normal(min(2000, n - at)) / 10
    for kw in (dict(min_p=0.2), dict(top_p=0.6), dict(top_k=900), dict(top_k=1500), dict(top_k=1000, top_p=0.9),
               dict(top_p=0.8, min_p=0.9)):
        for u in (rng.random(4).astype(np.float32), np.zeros(4, np.float32), np.ones(4, np.float32)):
            got = torch.functional.sample_logits(torch.tensor(x), torch.tensor(u), **kw)
            assert got.numpy().tolist() == [sample_ref(x[r], float(u[r]), **kw) for r in range(4)], (kw, u)


@gpu
def test_sample_logits_layouts_and_frequencies(torch):
    F = torch.functional
    rng = np.random.default_rng(3)
    w = (rng.standard_normal((5, 6000)) * 2).astype(np.float32)
    u = rng.random(5).astype(np.float32)
    for lo in range(5):  # rows at every alignment
        x = w[:, lo:lo + 5003]
        got = F.sample_logits(torch.tensor(w)[:, lo:lo + 5003], u, 0.9, 0, 0.8)
        assert got.numpy().tolist() == [sample_ref(x[r], float(u[r]), 0.9, 0, 0.8) for r in range(5)]
    got = F.sample_logits(torch.tensor(np.ascontiguousarray(w.T)).T, u)
    assert got.numpy().tolist() == [sample_ref(w[r], float(u[r])) for r in range(5)]
    one = F.sample_logits(torch.tensor(w[0]), np.float32(0.3), top_k=4)
    assert one.shape == () and one.item() == sample_ref(w[0], float(np.float32(0.3)), 1.0, 4)
    assert F.sample_logits(torch.zeros(0, 5), torch.zeros(0)).shape == (0,)
    # drawn from the seeded stream: the same again, and in the right shares
    x = np.log(np.array([0.5, 0.25, 0.125, 0.125], np.float32))
    rows = torch.tensor(np.broadcast_to(x, (20000, 4)).copy())
    torch.manual_seed(5)
    a = F.sample_logits(rows).numpy()
    torch.manual_seed(5)
    assert (F.sample_logits(rows).numpy() == a).all()
    share = np.bincount(a, minlength=4) / a.size
    # five standard deviations of 20000 draws
    assert (np.abs(share - np.exp(x)) < 5 * np.sqrt(np.exp(x) * (1 - np.exp(x)) / a.size)).all()


@gpu
def test_sample_logits_in_a_graph(torch):
    F = torch.functional
    rng = np.random.default_rng(8)
    x, u = torch.zeros(3, 5003), torch.zeros(3)

    def call():
        return (F.sample_logits(x, u, 0.8, top_k=40, top_p=0.9), F.sample_logits(x, u, top_p=0.9),
                x.topk(7)[1])
    call()
    g = torch.hip.Graph()
    with torch.hip.graph(g):
        got = call()
    for _ in range(3):
        hx = (rng.standard_normal((3, 5003)) * 2).astype(np.float32)
        hu = rng.random(3).astype(np.float32)
        x.copy_(torch.tensor(hx))
        u.copy_(torch.tensor(hu))
        torch.zeros(1000).add(1.0).numpy()  # work of the program's own between the replays
        g.replay()
        torch.synchronize()
        assert got[0].numpy().tolist() == [sample_ref(hx[r], float(hu[r]), 0.8, 40, 0.9) for r in range(3)]
        assert got[1].numpy().tolist() == [sample_ref(hx[r], float(hu[r]), 1.0, 0, 0.9) for r in range(3)]
        np.testing.assert_array_equal(got[2].numpy(), topk_ref(hx, 7))


# -------------------------------------------------------------- distillation


def _distill_inputs(rng, rows, n, k, spread=2.5):
    x = (rng.standard_normal((rows, n)) * spread).astype(np.float32)
    v = (rng.standard_normal((rows, k)) * 3).astype(np.float32)
    ids = np.stack([rng.permutation(max(n, k))[:k] for _ in range(rows)]).astype(np.int32)
    return x, v, ids


def _bounds(n, threads_terms):
    """Half steps that a row's sums and exponentials can be off: the longest
    chain of additions a thread makes (`threads_terms`), the tree over the
    block, and the roundings of an exponential, a logarithm, a division and
    the products around them; arguments of exponentials are off by two half
    steps of their own size, which the sizes of distill_ref carry."""
    return (threads_terms + 40) * U


def _check_distill(torch, x, v, ids, t, reduction):
    rows, n = x.shape
    loss, grad, valid, lsize, gsize = distill_ref(x, v, ids, t)
    c = _bounds(n, 4 * math.ceil(n / (4 * 64 if n <= 1024 else 4 * 256)) + 4)
    den = {"mean": valid.sum(), "sum": 1, "batchmean": rows, "none": 1}[reduction]
    tx = torch.tensor(x, requires_grad=True)
    out = torch.functional.distillation_loss(tx, torch.tensor(v), torch.tensor(ids), t, reduction)
    if reduction == "none":
        assert (np.abs(out.numpy() - loss) <= c * lsize).all()
        g = np.random.default_rng(1).standard_normal(rows).astype(np.float32)
        out.backward(torch.tensor(g))
        scale = g.astype(np.float64)[:, None]
    else:
        assert abs(out.item() - loss.sum() / den) <= (c + (rows / 1024 + 20) * U) * lsize.sum() / den
        out.backward()
        scale = np.full((rows, 1), 1.0 / den)
    got = tx.grad.numpy()
    assert got.shape == x.shape
    assert (np.abs(got - grad * scale) <= c * gsize * np.abs(scale)).all()
    assert (got[~valid] == 0).all()


@gpu
@pytest.mark.parametrize("n,k", [(1, 1), (2, 3), (6, 2), (7, 5), (1000, 8), (1021, 64), (1024, 100),
                                 (1025, 65), (4096, 7), (4099, 300), (16385, 1024), (32001, 37),
                                 (50257, 64), (53248, 1), (53261, 200)])
def test_distillation_loss(torch, n, k):
    rng = np.random.default_rng(n)
    for t in (1.0, 2.5):
        x, v, ids = _distill_inputs(rng, 5, n, k)
        ids[ids >= n] = -1
        ids[1, k // 2:] = -1
        ids[2] = n  # no entry
        ids[3, 0] = -2 ** 31
        if (ids[[0, 1, 3, 4]] >= 0).any():
            for reduction in ("mean", "sum", "batchmean", "none"):
                _check_distill(torch, x, v, ids, t, reduction)


@gpu
@pytest.mark.parametrize("n", [10, 900, 3000, 50257])
@pytest.mark.parametrize("k", [5, 64, 130])
def test_distillation_columns_given_twice(torch, n, k):
    rng = np.random.default_rng(k)
    x, v, _ = _distill_inputs(rng, 4, n, k)
    ids = rng.integers(0, min(n, 9), (4, k)).astype(np.int32)
    ids[3] = n - 1
    for reduction in ("mean", "none"):
        _check_distill(torch, x, v, ids, 1.5, reduction)
    # the same bits on every run
    def grads():
        tx = torch.tensor(x, requires_grad=True)
        torch.functional.distillation_loss(tx, torch.tensor(v), torch.tensor(ids)).backward()
        return tx.grad.numpy()
    np.testing.assert_array_equal(grads(), grads())


@gpu
def test_distillation_masks(torch):
    """Logits and teacher entries of -infinity and of the lowest float."""
    F = torch.functional
    rng = np.random.default_rng(2)
    x, v, ids = _distill_inputs(rng, 4, 5000, 20)
    x[:, 3000:] = -np.inf
    x[:, 2000:3000] = -np.finfo(np.float32).max
    ids %= 2000
    v[0, 10:], v[1, 5] = -np.inf, -np.finfo(np.float32).max
    v[2] = -np.inf  # no entry above -infinity
    _, grad, valid, _, gsize = distill_ref(x[:, :2000], v, ids, 1.0)
    assert valid.tolist() == [True, True, False, True]
    tx = torch.tensor(x, requires_grad=True)
    out = F.distillation_loss(tx, torch.tensor(v), torch.tensor(ids), reduction="sum")
    out.backward()
    got = tx.grad.numpy()
    assert math.isfinite(out.item()) and (got[:, 2000:] == 0).all()
    assert (np.abs(got[:, :2000] - grad) <= _bounds(5000, 24) * gsize).all()
    # a teacher's column that the student rules out costs without end
    x[0, ids[0, 0]] = -np.inf
    assert F.distillation_loss(torch.tensor(x), torch.tensor(v), torch.tensor(ids)).item() == math.inf
    v[1, 0] = np.nan
    per = F.distillation_loss(torch.tensor(x), torch.tensor(v), torch.tensor(ids), reduction="none")
    assert np.isnan(per.numpy()).tolist() == [False, True, False, False]
    none = F.distillation_loss(torch.tensor(x), torch.tensor(v), np.full((4, 20), -1, np.int32))
    assert math.isnan(none.item())


@gpu
def test_distillation_shapes_and_differences(torch):
    F = torch.functional
    rng = np.random.default_rng(4)
    x, v, ids = _distill_inputs(rng, 6, 77, 5)
    want = F.distillation_loss(torch.tensor(x), torch.tensor(v), torch.tensor(ids), 2.0).item()
    x3 = torch.tensor(x.reshape(2, 3, 77), requires_grad=True)
    out = F.distillation_loss(x3, torch.tensor(v.reshape(2, 3, 5)), ids.reshape(2, 3, 5), 2.0)
    assert out.item() == want
    out.backward()
    assert x3.grad.shape == (2, 3, 77)
    mod = torch.nn.DistillationLoss(2.0)
    assert mod(torch.tensor(x), torch.tensor(v), torch.tensor(ids)).item() == want
    one = F.distillation_loss(torch.tensor(x[0]), torch.tensor(v[0]), torch.tensor(ids[0]), reduction="none")
    assert one.shape == ()
    # against central differences of the oracle's loss
    h, g = 1e-4, x3.grad.numpy().reshape(6, 77)
    for r, j in ((0, ids[0, 0]), (3, 5), (5, 76)):
        lo, hi = x.astype(np.float64), x.astype(np.float64)
        lo[r, j] -= h
        hi[r, j] += h
        d = (distill_ref(hi, v, ids, 2.0)[0].sum() - distill_ref(lo, v, ids, 2.0)[0].sum()) / (2 * h) / 6
        # h^2 / 6 times a third derivative of at most 1 / T, and float32
        assert abs(g[r, j] - d) <= h * h + 60 * U
    # upstream gradients other than one, and twice through one graph
    tx = torch.tensor(x, requires_grad=True)
    out = F.distillation_loss(tx, torch.tensor(v), torch.tensor(ids), 2.0)
    out.backward(torch.tensor(np.float32(3.0).reshape(())), retain_graph=True)
    np.testing.assert_allclose(tx.grad.numpy(), 3 * g, rtol=4 * U, atol=0)
    out.backward()
    np.testing.assert_allclose(tx.grad.numpy(), 4 * g, rtol=8 * U, atol=0)


@gpu
@pytest.mark.parametrize("n", [50, 3000, 50257])
def test_distillation_of_many_rows(torch, n):
    """The count of rows with entries, where a launch of its own takes it."""
    rng = np.random.default_rng(n)
    rows = 1500
    x, v, ids = _distill_inputs(rng, rows, n, 7)
    ids[rng.random(rows) < 0.3] = -1
    _check_distill(torch, x, v, ids, 1.5, "mean")


@gpu
def test_rows_of_a_padded_output(torch):
    """Logits [B, T, C] whose rows are padded, as a linear layer's output of
    an odd width, are read where they stand."""
    F = torch.functional
    rng = np.random.default_rng(1)
    b, t, n = 2, 3, 1003
    w = rng.standard_normal((b, t, n + 5)).astype(np.float32)
    x = np.ascontiguousarray(w[:, :, :n])
    _, v, ids = _distill_inputs(rng, b * t, n, 6)
    v, ids = v.reshape(b, t, 6), ids.reshape(b, t, 6)
    for pick in (np.s_[:, :], np.s_[:, 1:2], np.s_[1:, :], np.s_[:, 1]):
        tx, tw = torch.tensor(x, requires_grad=True), torch.tensor(w, requires_grad=True)
        tv, ti = v[pick], ids[pick]
        for y in (tx, tw):
            z = y[:, :, :n][pick]
            F.distillation_loss(z, torch.tensor(np.ascontiguousarray(tv)), np.ascontiguousarray(ti)).backward()
        np.testing.assert_allclose(tw.grad.numpy()[:, :, :n], tx.grad.numpy(), rtol=0, atol=60 * U)
        assert (tw.grad.numpy()[:, :, n:] == 0).all()
        val, idx = tw.detach()[:, :, :n][pick].topk(5)
        flat = x[pick].reshape(-1, n)
        ref = topk_ref(flat, 5)
        np.testing.assert_array_equal(idx.numpy().reshape(-1, 5), ref)
        np.testing.assert_array_equal(val.numpy().reshape(-1, 5), np.take_along_axis(flat, ref, 1))


@gpu
@pytest.mark.parametrize("n,ks", [(300, (33, 100, 128, 300)), (1000, (90, 128, 129, 700)), (1021, (64, 1021)),
                                  (4093, (512, 513)), (16000, (250, 640))])
def test_topk_of_many_rows(torch, n, ks):
    """Sizes at which the rows' number and k choose between kernels and ways
    to sort, and lists much longer than k."""
    rng = np.random.default_rng(n)
    for spread in (False, True):
        x = rng.standard_normal((1025, n)).astype(np.float32)
        if spread:  # a few values: ties by index
            x = np.rint(x * 3).astype(np.float32)
        tx = torch.tensor(x)
        for k in ks:
            for largest in (True, False):
                v, i = tx.topk(k, largest=largest)
                ref = topk_ref(x, k, largest)
                np.testing.assert_array_equal(i.numpy(), ref)
                np.testing.assert_array_equal(v.numpy(), np.take_along_axis(x, ref, 1))


@gpu
def test_topk_of_more_rows_than_a_grid(torch):
    rng = np.random.default_rng(3)
    rows = 2 ** 21 + 3
    x = rng.integers(0, 50, (rows, 5)).astype(np.float32)
    tx = torch.tensor(x, requires_grad=True)
    v, i = tx.topk(2)
    ref = topk_ref(x, 2)
    np.testing.assert_array_equal(i.numpy(), ref)
    v.backward(torch.tensor(np.arange(2 * rows, dtype=np.float32).reshape(rows, 2)))
    want = np.zeros_like(x)
    np.put_along_axis(want, ref, np.arange(2 * rows, dtype=np.float32).reshape(rows, 2), 1)
    np.testing.assert_array_equal(tx.grad.numpy(), want)


@gpu
def test_distillation_second_derivative(torch):
    rng = np.random.default_rng(6)
    x, v, ids = _distill_inputs(rng, 3, 9, 4)
    ids[1, 2:] = -1
    w = rng.standard_normal((3, 9)).astype(np.float32)
    for red in ("mean", "none"):
        tx = torch.tensor(x, requires_grad=True)
        out = torch.functional.distillation_loss(tx, torch.tensor(v), torch.tensor(ids), 1.5, red)
        (d,) = torch.autograd.grad(out.sum(), tx, create_graph=True)
        (dd,) = torch.autograd.grad((d * torch.tensor(w)).sum(), tx)
        s = 1 / 3 if red == "mean" else 1.0
        q = np.exp(x / 1.5 - x.max(1, keepdims=True) / 1.5).astype(np.float64)
        q /= q.sum(1, keepdims=True)
        ref = s * q * (w - (q * w).sum(1, keepdims=True))
        # a dozen float32 operations on values of at most 4
        assert np.abs(dd.numpy() - ref).max() <= 100 * U


@gpu
def test_distillation_in_a_graph(torch):
    F = torch.functional
    rng = np.random.default_rng(9)
    x = torch.zeros(6, 3001).requires_grad_(True)
    v = torch.tensor(rng.standard_normal((6, 8)).astype(np.float32))
    ids = torch.tensor(rng.integers(0, 3001, (6, 8)).astype(np.int32))

    def call():
        x.grad = None
        loss = F.distillation_loss(x, v, ids, 2.0)
        loss.backward()
        return loss, x.grad
    call()
    g = torch.hip.Graph()
    with torch.hip.graph(g):
        loss, grad = call()
    for _ in range(3):
        hx = rng.standard_normal((6, 3001)).astype(np.float32)
        x.detach().copy_(torch.tensor(hx))
        g.replay()
        torch.synchronize()
        got = loss.item(), grad.numpy().copy()
        e = torch.tensor(hx, requires_grad=True)
        want = F.distillation_loss(e, v, ids, 2.0)
        want.backward()
        assert got[0] == want.item()
        np.testing.assert_array_equal(got[1], e.grad.numpy())


class _Memory:
    """A library that computes nothing: it hands out and takes back addresses
    and notes the logits that tjh_distill is given."""

    def __init__(self):
        self.live, self.at, self.read = {}, 1 << 20, []

    def __getattr__(self, name):
        return lambda *args: 0

    def tjh_malloc(self, n, out):
        self.at += 1 << 20
        self.live[self.at] = n
        out._obj.value = self.at
        return 0

    def tjh_free(self, p):
        del self.live[p]
        return 0

    def tjh_distill(self, px, *args):
        self.read.append(any(p <= px < p + n for p, n in self.live.items()))
        return 0


@pytest.mark.parametrize("view", ["shifted", "transposed", "columns"])
def test_distillation_reads_memory_of_its_own(pkg, monkeypatch, view):
    """Logits that had to be copied are there until the last backward."""
    from torchjs_amd import _lib as L
    mem = _Memory()
    with monkeypatch.context() as m:
        m.setattr(L, "_lib", mem)
        m.setitem(sys.modules["torchjs_amd.tensor"]._state, "init", True)
        v, ids = pkg.empty((2, 3, 4)), pkg.empty((2, 3, 4), "int32")
        for reduction in ("none", "mean"):
            w = pkg.empty({"shifted": (2, 4, 9), "transposed": (2, 9, 3), "columns": (2, 3, 18)}[view])
            y = w.requires_grad_(True)
            z = {"shifted": lambda: y[:, :3], "transposed": lambda: y.transpose(1, 2),
                 "columns": lambda: y.view(2, 3, 9, 2)[:, :, :, 0]}[view]()
            assert z.shape == (2, 3, 9)
            out = pkg.functional.distillation_loss(z, v, ids, reduction=reduction)
            del z
            g = pkg.empty(out.shape)
            out.backward(g, retain_graph=True)
            out.backward(g)
            del out, y, w, g
        del v, ids
        assert mem.read == [True] * 6


@gpu
@pytest.mark.parametrize("view", ["shifted", "transposed", "columns", "one column apart"])
def test_distillation_of_logits_that_are_copied(torch, view):
    """Views whose rows are not evenly spaced or not dense, with upstream
    gradients that the forward could not know and other tensors of the
    copy's size made and dropped before the backward."""
    F = torch.functional
    rng = np.random.default_rng(4)
    b, t, n = 2, 5, 3001
    full = (rng.standard_normal((b, t + 1, n + 1)) * 2).astype(np.float32)
    pick = {"shifted": lambda y: y[:, :-1, :n], "transposed": lambda y: y.transpose(1, 2)[:, :, :t],
            "columns": lambda y: y.view(b, t + 1, (n + 1) // 2, 2)[:, :, :, 0],
            "one column apart": lambda y: y[:, 1:, 1:]}[view]
    host = {"shifted": lambda y: y[:, :-1, :n], "transposed": lambda y: y.swapaxes(1, 2)[:, :, :t],
            "columns": lambda y: y[:, :, ::2], "one column apart": lambda y: y[:, 1:, 1:]}[view]
    x = np.ascontiguousarray(host(full))
    rows, c = x.shape[0] * x.shape[1], x.shape[2]
    v = (rng.standard_normal(x.shape[:2] + (4,)) * 2).astype(np.float32)
    ids = rng.integers(0, c, v.shape).astype(np.int32)
    up = rng.standard_normal(x.shape[:2]).astype(np.float32)

    def grads(y, z, reduction, twice):
        out = F.distillation_loss(z, torch.tensor(v), torch.tensor(ids), 2.0, reduction)
        del z
        for _ in range(4):  # takes a freed copy's memory, if there is one
            torch.full(x.shape, 1e9)
        if reduction == "none":
            out.backward(torch.tensor(up))
        elif twice:
            out.backward(retain_graph=True)
            torch.full(x.shape, 1e9)
            out.backward()
        else:
            (out * 0.5 + (y * y).sum() * 0.25).backward()
        return y.grad.numpy()
    for reduction, twice in (("none", False), ("mean", False), ("sum", True)):
        tf, tx = torch.tensor(full, requires_grad=True), torch.tensor(x, requires_grad=True)
        got = host(grads(tf, pick(tf), reduction, twice))
        want = grads(tx, tx, reduction, twice)
        assert got.shape == want.shape and np.isfinite(want).all()
        # both are off from the formula by at most _bounds times T (q (1 + |ln
        # q|) + sum p (1 + |ln p|)) <= 2 (2 + ln 4), a row's factor and twice
        # that where two gradients are added, and by a rounding of the sum
        # with the other loss's share
        tol = 2 * _bounds(c, 16) * 6.8 * max(1, np.abs(up).max()) * (2 if twice else 1)
        assert np.abs(got - want).max() <= tol + 2 * U * np.abs(want).max(), (reduction, twice)


@gpu
@pytest.mark.parametrize("n,k", [(9, 3), (900, 70), (900, 200), (3000, 300), (50257, 600), (60001, 5)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_distillation_teacher_of_nan_or_infinity(torch, n, k, value):
    """Such an entry makes its row's loss and whole gradient NaN wherever it
    stands, and leaves the other rows and entries that are none alone."""
    rng = np.random.default_rng(k)
    x, v, _ = _distill_inputs(rng, 6, n, k)
    ids = rng.integers(0, n, (6, k)).astype(np.int32)
    v[0, 0] = v[1, k - 1] = v[2, 0] = value
    v[2, 1:] = -np.inf  # and nothing else
    v[3, 0] = value
    ids[3, 0] = n  # none
    want = distill_ref(x[3:], v[3:], ids[3:], 1.5)
    tx = torch.tensor(x, requires_grad=True)
    call = lambda red: torch.functional.distillation_loss(tx, torch.tensor(v), torch.tensor(ids), 1.5, red)
    out = call("none")
    out.backward(torch.tensor(np.ones(6, np.float32)))
    got, grad = out.numpy(), tx.grad.numpy()
    assert np.isnan(got[:3]).all() and np.isnan(grad[:3]).all()
    c = _bounds(n, 4 * math.ceil(n / (4 * 64 if n <= 1024 else 4 * 256)) + 4)
    assert (np.abs(got[3:] - want[0]) <= c * want[3]).all()
    assert (np.abs(grad[3:] - want[1]) <= c * want[4]).all()
    assert math.isnan(call("mean").item())
    (d,) = torch.autograd.grad(call("sum"), tx, create_graph=True)
    d = d.detach().numpy()
    assert np.isnan(d[:3]).all() and np.isfinite(d[3:]).all()


@gpu
def test_distillation_second_derivative_beside_masked_logits(torch):
    """Logits of -infinity where the teacher has no probability: entries that
    are none stand for column 0, others are -infinity or underflow."""
    rng = np.random.default_rng(16)
    x, v, ids = _distill_inputs(rng, 3, 9, 4)
    x[:, 0] = x[2, 7] = -np.inf
    ids[:] = [[1, -1, 5, 9], [0, 2, 3, 4], [7, 1, 2, 8]]
    v[1, 0] = -np.inf
    v[2, 0] = -1000
    w = rng.standard_normal((3, 9)).astype(np.float32)
    fin = x > -np.inf
    q = np.where(fin, np.exp(np.where(fin, x, 0.0).astype(np.float64)), 0.0)
    q /= q.sum(1, keepdims=True)
    h = np.where((ids >= 0) & (ids < 9), v.astype(np.float64), -np.inf)
    p = np.exp(h - h.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    first = q.copy()
    for r in range(3):
        np.add.at(first[r], np.clip(ids[r], 0, 8), -p[r])
    for red in ("sum", "none"):
        tx = torch.tensor(x, requires_grad=True)
        out = torch.functional.distillation_loss(tx, torch.tensor(v), torch.tensor(ids), 1.0, red)
        assert np.isfinite(out.numpy()).all()
        (d,) = torch.autograd.grad(out.sum(), tx, create_graph=True)
        # a dozen float32 operations on values of at most 4, here and below
        assert np.abs(d.detach().numpy() - first).max() <= 100 * U
        (dd,) = torch.autograd.grad((d * torch.tensor(w)).sum(), tx)
        assert np.abs(dd.numpy() - q * (w - (q * w).sum(1, keepdims=True))).max() <= 100 * U


# ------------------------------------------------------------------ refusals


def _fake(pkg, *shape, dtype="float32"):
    """A tensor without a device: the checks come before anything reads it."""
    return pkg.Tensor(types.SimpleNamespace(ptr=4096), shape, None, 0, dtype)


def test_refusals(pkg):
    F = pkg.functional
    x = _fake(pkg, 4, 10)
    for k in (-1, 11):
        with pytest.raises(ValueError, match="topk"):
            x.topk(k)
    with pytest.raises(IndexError):
        x.topk(1, dim=2)
    u = _fake(pkg, 4)
    for kw in (dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1), dict(top_p=1.5),
               dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=math.nan)):
        with pytest.raises(ValueError, match="must lie in"):
            F.sample_logits(x, u, **kw)
    with pytest.raises(ValueError, match="whole number"):
        F.sample_logits(x, u, top_k=0.5)
    with pytest.raises(ValueError, match="uniforms"):
        F.sample_logits(x, _fake(pkg, 3))
    with pytest.raises(ValueError, match="has shape"):
        F.sample_logits(x, u, temperature=_fake(pkg, 5))
    for bad in (_fake(pkg, 2, 3, 4), _fake(pkg), _fake(pkg, 3, 0)):
        with pytest.raises(ValueError, match="expected logits"):
            F.sample_logits(bad, u)
    v, ids = _fake(pkg, 4, 3), _fake(pkg, 4, 3, dtype="int32")
    for t in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            F.distillation_loss(x, v, ids, t)
    with pytest.raises(ValueError, match="reduction"):
        F.distillation_loss(x, v, ids, reduction="max")
    for bv, bi in ((_fake(pkg, 3, 3), ids), (v, _fake(pkg, 4, 2, dtype="int32")),
                   (_fake(pkg, 4, 0), _fake(pkg, 4, 0, dtype="int32")),
                   (_fake(pkg, 3), _fake(pkg, 3, dtype="int32"))):
        with pytest.raises(ValueError, match="do not fit"):
            F.distillation_loss(x, bv, bi)
    with pytest.raises(ValueError, match="no classes"):
        F.distillation_loss(_fake(pkg, 4, 0), v, ids)


def test_distillation_temperatures_without_float32_powers(pkg):
    v, ids = _fake(pkg, 4, 3), _fake(pkg, 4, 3, dtype="int32")
    for t in (1e-40, 9e-19, 1.1e18, 1e30):
        with pytest.raises(ValueError, match="temperature"):
            pkg.functional.distillation_loss(_fake(pkg, 4, 10), v, ids, t)


def test_fractions_are_no_counts(pkg):
    """They were cut off: of numpy's numbers, of lists, of topk's k."""
    x, u = _fake(pkg, 4, 10), _fake(pkg, 4)
    for k in (2.5, np.float32(2.5), np.float64(0.5), [2, 2.5, 3, 4], np.array([1, 2, np.nan, 4]),
              [1, math.inf, 2, 0.5]):
        with pytest.raises(ValueError, match="whole number"):
            pkg.functional.sample_logits(x, u, top_k=k)
    for k in (math.inf, math.nan, 2 ** 31):
        with pytest.raises(ValueError, match="must lie in"):
            pkg.functional.sample_logits(x, u, top_k=k)
    for k in (2.5, np.float32(0.5)):
        with pytest.raises(ValueError, match="whole number"):
            x.topk(k)


@gpu
@pytest.mark.parametrize("t", [1e-18, 1e18])
def test_distillation_at_the_ends_of_the_temperatures(torch, t):
    x, v, ids = _distill_inputs(np.random.default_rng(3), 4, 1500, 6)
    for reduction in ("mean", "none"):
        _check_distill(torch, x, v, ids, t, reduction)
    from torchjs_amd import _lib as L
    p = torch.zeros(4, 10).data_ptr()
    for bad in (1e-40, 9e-19, 1.1e18, math.inf, math.nan):
        assert L.lib().tjh_distill(p, 10, 2, 10, p, p, 1, bad, 1, None, p, p, None, 0) == 1


@gpu
@pytest.mark.parametrize("dtype", [np.int8, np.uint8, np.int16, np.int64, np.uint64, np.float16, np.float32])
def test_counts_of_any_type(torch, dtype):
    rng = np.random.default_rng(2)
    x, u = rng.standard_normal((3, 40)).astype(np.float32), rng.random(3).astype(np.float32)
    got = torch.functional.sample_logits(torch.tensor(x), u, top_k=np.array([4, 0, 1], dtype))
    assert got.numpy().tolist() == [sample_ref(x[r], float(u[r]), top_k=(4, 0, 1)[r]) for r in range(3)]


@gpu
def test_counts_past_32_bits(torch):
    """A top_k of a row that int32 does not hold is no rule."""
    rng = np.random.default_rng(2)
    x, u = rng.standard_normal((3, 40)).astype(np.float32), rng.random(3).astype(np.float32)
    for k in (np.array([2 ** 32 + 1, -2 ** 40, 3]), [2.0 ** 40, -1.0, 3.0], [2 ** 31, 0, 3]):
        got = torch.functional.sample_logits(torch.tensor(x), u, top_k=k)
        assert got.numpy().tolist() == [sample_ref(x[r], float(u[r]), top_k=(0, 0, 3)[r]) for r in range(3)]


@gpu
def test_refusals_of_the_library(torch):
    from torchjs_amd import _lib as L
    x = torch.zeros(2, 2000)
    with pytest.raises(L.HipError, match="at most 1024"):
        x.topk(1025)
    with pytest.raises(L.HipError, match="at most 1024"):
        torch.functional.distillation_loss(x, torch.zeros(2, 1025), np.zeros((2, 1025), np.int32))
    big = torch.zeros(1).expand(1, 2 ** 20 + 1)
    with pytest.raises(L.HipError, match="at most"):
        torch.functional.sample_logits(big, torch.zeros(1))
    lib, p = L.lib(), x.data_ptr()
    assert lib.tjh_topk_forward(p, 1, 2, 2000, 1, 1, p, p) == 1
    assert lib.tjh_topk_forward(None, 2000, 2, 2000, 1, 1, p, p) == 1
    assert lib.tjh_topk_backward(p, p, 2, 5, 6, p) == 1
    assert lib.tjh_sample_logits(p, 2000, 2 ** 22, 2000, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p) == 1
    assert lib.tjh_distill(p, 2000, 2 ** 24, 2000, p, p, 1, 1.0, 1, None, p, p, None, 0) == 1
    assert lib.tjh_sample_logits(p, 2000, 2, 2000, None, None, None, None, None, 1.0, 0, 1.0, 0.0, p) == 1
    assert lib.tjh_distill(p, 2000, 2, 2000, p, p, 1, 1.0, 7, None, p, None, None, 0) == 1
    assert lib.tjh_distill(p, 2000, 2, 2000, p, p, 1, 1.0, 0, None, None, None, p, 2000) == 1
    assert lib.tjh_distill(p, 2000, 2, 2000, p, p, 1, 0.0, 1, None, p, p, None, 0) == 1
