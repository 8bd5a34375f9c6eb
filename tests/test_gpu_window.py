"""F.sliding_window_attention against plain numpy in 64 bits."""
import math
import types

import numpy as np
import pytest

gpu = pytest.mark.gpu
U = 2.0 ** -24  # half a step of float32, relative


def visible(tq, tk, window, sinks):
    i, j = np.arange(tk - tq, tk)[:, None], np.arange(tk)
    return (j <= i) & ((j > i - window) | (j < sinks))


def reference(q, k, v, window, sinks, g=None, scale=None):
    """Output and gradients with, for each, how far float32 can be off: every
    product over n terms by n + 2 half steps of the sum of its terms' sizes,
    an exponential by the error of its argument and a few half steps, and
    what follows from those."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    b, h, tq, d = q.shape
    hkv, tk = k.shape[1:3]
    grp = h // hkv
    sc = d ** -0.5 if scale is None else scale
    kk, vv = np.repeat(k, grp, 1), np.repeat(v, grp, 1)
    seen = visible(tq, tk, window, sinks)
    n = int(seen.sum(1).max()) + 64  # terms of a sum over keys, and of its joins
    m = int(seen.sum(0).max()) * grp + 64  # terms of a sum over queries

    def mm(x, y):
        return np.matmul(x, y)

    def t(x):
        return x.swapaxes(-1, -2)
    s = np.where(seen, mm(q, t(kk)) * sc, -np.inf)
    top = s.max(-1, keepdims=True)
    p = np.exp(s - top)
    p /= p.sum(-1, keepdims=True)
    o = mm(p, vv)
    # relative error of a probability
    es = (d + 4) * U * mm(abs(q), t(abs(kk))) * abs(sc) + 4 * U * np.where(seen, abs(s - top), 0) + 8 * U
    e = es + (p * es).sum(-1, keepdims=True) + n * U
    eo = mm(p * e, abs(vv)) + n * U * mm(p, abs(vv))
    if g is None:
        return o, eo
    g = g.astype(np.float64)
    dp = mm(g, t(vv))
    dd = (g * o).sum(-1, keepdims=True)
    ds = p * (dp - dd)
    eds = p * (e * abs(dp - dd) + (d + 4) * U * mm(abs(g), t(abs(vv))) +
               (d + 4) * U * (abs(g) * abs(o)).sum(-1, keepdims=True) + (abs(g) * eo).sum(-1, keepdims=True)
               ) + 4 * U * abs(ds)

    def heads(x):
        return x.reshape(b, hkv, grp, tk, d).sum(2)
    dq, edq = sc * mm(ds, kk), abs(sc) * (mm(eds, abs(kk)) + n * U * mm(abs(ds), abs(kk)))
    dk, edk = heads(sc * mm(t(ds), q)), heads(abs(sc) * (mm(t(eds), abs(q)) + m * U * mm(t(abs(ds)), abs(q))))
    dv, edv = heads(mm(t(p), g)), heads(mm(t(p * e), abs(g)) + m * U * mm(t(p), abs(g)))
    return (o, dq, dk, dv), (eo, edq, edk, edv)


def near(got, want, bound, name):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= bound + 1e-30)
    assert not bad.any(), "%s: %d of %d off, first %s: %r for %r (bound %.3g)" % (
        name, bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], want[bad][0], bound[bad][0])


def inputs(seed, b, h, hkv, tq, tk, d):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal(s).astype(np.float32)
            for s in ((b, h, tq, d), (b, hkv, tk, d), (b, hkv, tk, d), (b, h, tq, d))]


CASES = [
    # b, h, hkv, tq, tk, d, window, sinks
    (1, 1, 1, 1, 1, 4, 1, 0), (1, 2, 1, 1, 1, 64, 5, 3), (2, 3, 3, 5, 5, 32, 1, 0),
    (1, 1, 1, 7, 7, 4, 2, 1), (1, 4, 2, 33, 33, 8, 7, 5), (2, 2, 1, 64, 64, 64, 32, 32),
    (1, 2, 2, 65, 97, 40, 30, 0), (1, 3, 1, 129, 300, 80, 64, 33), (1, 2, 2, 257, 257, 96, 100, 70),
    (1, 2, 1, 300, 300, 128, 1000, 4), (1, 1, 1, 160, 640, 128, 31, 129), (1, 2, 2, 513, 513, 64, 33, 1),
    (1, 4, 1, 700, 700, 48, 40, 65), (2, 4, 4, 1, 700, 64, 256, 4), (1, 8, 2, 3, 1500, 128, 600, 10),
    (1, 1, 1, 4, 2500, 64, 2100, 5), (1, 2, 1, 93, 701, 80, 300, 1), (1, 1, 1, 40, 3001, 64, 2000, 64),
    (1, 1, 1, 5, 5, 5, 3, 1), (1, 2, 1, 70, 81, 30, 9, 2), (1, 1, 1, 64, 64, 66, 20, 0),
    (1, 1, 1, 3, 300, 127, 50, 7), (1, 12, 12, 6, 1000, 64, 1, 0), (1, 2, 2, 320, 320, 64, 64, 96),
]


@gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_gradients(torch, case):
    b, h, hkv, tq, tk, d, window, sinks = case
    q, k, v, g = inputs(sum(case), b, h, hkv, tq, tk, d)
    want, bound = reference(q, k, v, window, sinks, g)
    f = torch.functional.sliding_window_attention
    with torch.no_grad():
        o = f(torch.tensor(q), torch.tensor(k), torch.tensor(v), window, sinks)
    near(o.numpy(), want[0], bound[0], "without a gradient")
    ts = [torch.tensor(x, requires_grad=True) for x in (q, k, v)]
    o = f(*ts, window, sinks)
    near(o.numpy(), want[0], bound[0], "output")
    o.backward(torch.tensor(g))
    for name, t, w, e in zip(("dq", "dk", "dv"), ts, want[1:], bound[1:]):
        near(t.grad.numpy(), w, e, name)


@gpu
@pytest.mark.parametrize("case", [(1, 1, 1, 900, 900, 64, 700, 3), (1, 2, 1, 301, 777, 128, 400, 70),
                                  (2, 1, 1, 270, 270, 20, 256, 0), (1, 1, 1, 2, 1300, 64, 1200, 1)], ids=str)
def test_slices_with_gradients(torch, case):
    """Few heads: keys in slices forward, steps in slices backward; the same
    bits on every run and with or without a gradient."""
    b, h, hkv, tq, tk, d, window, sinks = case
    q, k, v, g = inputs(sum(case), b, h, hkv, tq, tk, d)
    want, bound = reference(q, k, v, window, sinks, g)
    f = torch.functional.sliding_window_attention
    runs = []
    for _ in range(2):
        ts = [torch.tensor(x, requires_grad=True) for x in (q, k, v)]
        o = f(*ts, window, sinks)
        o.backward(torch.tensor(g))
        runs.append([o.numpy()] + [t.grad.numpy() for t in ts])
    for name, a, again, w, e in zip(("output", "dq", "dk", "dv"), *runs, want, bound):
        near(a, w, e, name)
        np.testing.assert_array_equal(a, again)
    with torch.no_grad():
        np.testing.assert_array_equal(f(*ts, window, sinks).numpy(), runs[0][0])


@gpu
@pytest.mark.parametrize("case", [(1, 2, 2, 100, 100, 64), (2, 4, 2, 77, 77, 32)], ids=str)
def test_equals_full_attention_where_the_window_holds_all(torch, case):
    b, h, hkv, tq, tk, d = case
    q, k, v, g = inputs(1, *case)
    kk, vv = np.repeat(k, h // hkv, 1), np.repeat(v, h // hkv, 1)
    o = torch.functional.sliding_window_attention(*map(torch.tensor, (q, k, v)), tk, 3)
    full = torch.functional.scaled_dot_product_attention(*map(torch.tensor, (q, kk, vv)), is_causal=True)
    _, bound = reference(q, k, v, tk, 0)
    near(o.numpy(), full.numpy().astype(np.float64), 2 * bound, "output")


@gpu
@pytest.mark.parametrize("d", [64, 80])
def test_what_is_not_seen_may_hold_anything(torch, d):
    """Infinities and NaN in keys and values: no part in the output or the
    gradient of a query that does not see them."""
    f = torch.functional.sliding_window_attention
    b, h, hkv, window, sinks = 1, 2, 1, 37, 5
    # a part of a prompt and single tokens over a cache: positions that no
    # query of the call sees
    for tq, tk in ((50, 300), (1, 300), (4, 97), (1, 2000)):
        q, k, v, g = inputs(d, b, h, hkv, tq, tk, d)
        clean = [x.copy() for x in (k, v)]
        hidden = ~visible(tq, tk, window, sinks).any(0)
        assert hidden.any()
        for i, bad in enumerate((np.nan, np.inf, -np.inf, 3e38)):
            k[:, :, np.nonzero(hidden)[0][i::4]] = bad
            v[:, :, np.nonzero(hidden)[0][i::4]] = bad
        want, bound = reference(q, *clean, window, sinks, g)
        with torch.no_grad():
            near(f(*map(torch.tensor, (q, k, v)), window, sinks).numpy(), want[0], bound[0], "output")
        ts = [torch.tensor(x, requires_grad=True) for x in (q, k, v)]
        o = f(*ts, window, sinks)
        near(o.numpy(), want[0], bound[0], "output")
        o.backward(torch.tensor(g))
        near(ts[0].grad.numpy(), want[1], bound[1], "dq")
        for t, w, e in zip(ts[1:], want[2:], bound[2:]):
            near(t.grad.numpy(), w, e, "dk, dv")
            assert (t.grad.numpy()[:, :, hidden] == 0).all()
    # one position that some queries see and others do not
    q, k, v, g = inputs(d, b, h, hkv, 200, 200, d)
    want, bound = reference(q, k, v, window, sinks, g)
    at = 70
    blind = ~visible(200, 200, window, sinks)[:, at]
    for bad in (np.nan, np.inf, -np.inf):
        for which in (1, 2):
            x = [q, k.copy(), v.copy()]
            x[which][:, :, at, :: 3] = bad
            ts = [torch.tensor(y, requires_grad=True) for y in x]
            o = f(*ts, window, sinks)
            near(o.numpy()[:, :, blind], want[0][:, :, blind], bound[0][:, :, blind], "output")
            if which == 2:  # its column of the ones that see it
                got = o.numpy()[:, :, ~blind][..., :: 3]
                assert (np.isnan(got) | np.isinf(got)).all()
            o.backward(torch.tensor(g))
            near(ts[0].grad.numpy()[:, :, blind], want[1][:, :, blind], bound[1][:, :, blind], "dq")


@gpu
def test_layouts(torch):
    f = torch.functional.sliding_window_attention
    b, t, h, d, window, sinks = 2, 75, 3, 32, 20, 4
    rng = np.random.default_rng(0)
    x = rng.standard_normal((b, t, 3 * h * d)).astype(np.float32)
    parts = [x[..., i * h * d:(i + 1) * h * d].reshape(b, t, h, d).transpose(0, 2, 1, 3) for i in range(3)]
    g = rng.standard_normal((b, h, t, d)).astype(np.float32)
    want, bound = reference(*parts, window, sinks, g)
    # the heads of one projection, as a layer has them
    tx = torch.tensor(x, requires_grad=True)
    views = [y.view(b, t, h, d).transpose(1, 2) for y in tx.split(h * d, dim=2)]
    o = f(*views, window, sinks)
    near(o.numpy(), want[0], bound[0], "output")
    o.backward(torch.tensor(g))
    grad = tx.grad.numpy()
    for i in range(3):
        got = grad[..., i * h * d:(i + 1) * h * d].reshape(b, t, h, d).transpose(0, 2, 1, 3)
        near(got, want[1 + i], bound[1 + i], "projection %d" % i)
    # gradients that arrive transposed, and rows that are not 16-byte aligned
    wide = [np.concatenate([np.zeros((b, h, t, 1), np.float32), y, np.zeros((b, h, t, 2), np.float32)], -1)
            for y in parts]
    ts = [torch.tensor(y, requires_grad=True) for y in wide]
    o = f(*[y.narrow(-1, 1, d) for y in ts], window, sinks)
    near(o.numpy(), want[0], bound[0], "unaligned rows")
    gt = torch.tensor(np.ascontiguousarray(g.transpose(0, 1, 3, 2))).transpose(2, 3)
    o.backward(gt)
    for y, w, e in zip(ts, want[1:], bound[1:]):
        near(y.grad.numpy()[..., 1:1 + d], w, e, "unaligned gradients")
    # columns apart, rows apart, and a cache's prefix
    odd = [torch.tensor(np.ascontiguousarray(y.transpose(0, 1, 3, 2))).transpose(2, 3) for y in parts]
    near(f(*odd, window, sinks).numpy(), want[0], bound[0], "columns apart")
    caches = [torch.zeros(b, h, 200, d) for _ in range(2)]
    for c, y in zip(caches, parts[1:]):
        c[:, :, :t].copy_(torch.tensor(y))
    o = f(torch.tensor(parts[0][:, :, -1:]), caches[0][:, :, :t], caches[1][:, :, :t], window, sinks)
    near(o.numpy(), want[0][:, :, -1:], bound[0][:, :, -1:], "cache")
    # 3-D
    q3, k3, v3 = (y[:, 0] for y in parts)
    ts = [torch.tensor(np.ascontiguousarray(y), requires_grad=True) for y in (q3, k3, v3)]
    o = f(*ts, window, sinks)
    assert o.shape == (b, t, d)
    w3, b3 = reference(*[y[:, :1] for y in parts], window, sinks, g[:, :1])
    near(o.numpy(), w3[0][:, 0], b3[0][:, 0], "3-D")
    o.backward(torch.tensor(g[:, 0]))
    for y, w, e in zip(ts, w3[1:], b3[1:]):
        near(y.grad.numpy(), w[:, 0], e[:, 0], "3-D gradients")
    # nothing
    e = [torch.zeros(2, 3, n, 8).requires_grad_(True) for n in (0, 5, 5)]
    o = f(*e, 3)
    assert o.shape == (2, 3, 0, 8)
    o.sum().backward()
    assert (e[1].grad.numpy() == 0).all() and e[0].grad.shape == (2, 3, 0, 8)
    # a scale of one's own
    w, bd = reference(*parts, window, sinks, scale=-0.3)
    near(f(*[torch.tensor(np.ascontiguousarray(y)) for y in parts], window, sinks, -0.3).numpy(), w, bd,
         "scale")


@gpu
def test_gradients_against_differences(torch):
    q, k, v, g = inputs(5, 1, 2, 1, 9, 12, 8)
    ts = [torch.tensor(x, requires_grad=True) for x in (q, k, v)]
    torch.functional.sliding_window_attention(*ts, 4, 2).backward(torch.tensor(g))
    h = 1e-5
    for which, at in ((0, (0, 1, 3, 2)), (1, (0, 0, 1, 5)), (1, (0, 0, 6, 0)), (2, (0, 0, 0, 7)), (2, (0, 0, 11, 1))):
        ends = []
        for sign in (1, -1):
            x = [y.astype(np.float64) for y in (q, k, v)]
            x[which][at] += sign * h
            ends.append((reference(*x, 4, 2)[0] * g).sum())
        d = (ends[0] - ends[1]) / (2 * h)
        # h^2 times third derivatives of some tens, and float32 over some hundred terms
        assert abs(ts[which].grad.numpy()[at] - d) <= 100 * h * h + 1000 * U


@gpu
def test_second_derivative(torch):
    q, k, v, g = inputs(6, 1, 2, 1, 6, 6, 8)
    ts = [torch.tensor(x, requires_grad=True) for x in (q, k, v)]
    f = torch.functional.sliding_window_attention
    grads = torch.autograd.grad((f(*ts, 3, 1) * torch.tensor(g)).sum(), ts, create_graph=True)
    loss = sum(((x * x).sum() for x in grads[1:]), (grads[0] * grads[0]).sum())
    dd = torch.autograd.grad(loss, ts)
    h = 1e-5
    for which, at in ((0, (0, 1, 3, 2)), (1, (0, 0, 1, 5)), (2, (0, 0, 4, 1))):
        ends = []
        for sign in (1, -1):
            x = [y.astype(np.float64) for y in (q, k, v)]
            x[which][at] += sign * h
            want, _ = reference(*x, 3, 1, g)
            ends.append(sum((y * y).sum() for y in want[1:]))
        d = (ends[0] - ends[1]) / (2 * h)
        # values of some tens over some hundred terms of float32
        assert abs(dd[which].numpy()[at] - d) <= 1e-6 * abs(d) + 10000 * U


@gpu
@pytest.mark.parametrize("tq,tk", [(70, 70), (1, 900)])
def test_in_a_graph(torch, tq, tk):
    f = torch.functional.sliding_window_attention
    rng = np.random.default_rng(2)
    train = tq == tk
    ts = [torch.zeros(1, 2, n, 64).requires_grad_(train) for n in (tq, tk, tk)]
    g = torch.tensor(rng.standard_normal((1, 2, tq, 64)).astype(np.float32))

    def call():
        for t in ts:
            t.grad = None
        o = f(*ts, 30, 3)
        if train:
            o.backward(g)
        return [o] + [t.grad for t in ts if train]
    call()
    graph = torch.hip.Graph()
    with torch.hip.graph(graph):
        got = call()
    for _ in range(3):
        hx = [rng.standard_normal(t.shape).astype(np.float32) for t in ts]
        for t, x in zip(ts, hx):
            t.detach().copy_(torch.tensor(x))
        graph.replay()
        torch.synchronize()
        got_np = [t.numpy().copy() for t in got]
        es = [torch.tensor(x, requires_grad=train) for x in hx]
        o = f(*es, 30, 3)
        if train:
            o.backward(g)
        for a, e in zip(got_np, [o] + [t.grad for t in es if train]):
            np.testing.assert_array_equal(a, e.numpy())


@gpu
def test_one_tensor_as_queries_keys_and_values(torch):
    x, _, _, g = inputs(8, 2, 2, 2, 45, 45, 16)
    want, bound = reference(x, x, x, 10, 2, g)
    t = torch.tensor(x, requires_grad=True)
    for n in (1, 2):  # and a second pass adds to the first one's gradient
        o = torch.functional.sliding_window_attention(t, t, t, 10, 2)
        near(o.numpy(), want[0], bound[0], "output")
        o.backward(torch.tensor(g))
        # three parts in two additions a pass, each off by half a step of the sum
        size = n * sum(np.abs(w) for w in want[1:])
        near(t.grad.numpy(), n * sum(want[1:]), n * sum(bound[1:]) + 3 * n * U * size, "gradient")


@gpu
@pytest.mark.parametrize("row", [2 ** 23 - 8, 2 ** 23])
def test_rows_far_apart(torch, row):
    """Offsets past 32 bits, and rows farther apart than the kernels take."""
    n, d, window, sinks = 300, 8, 40, 3
    q, k, v, g = (x[0] for x in inputs(9, 1, 2, 2, n, n, d))
    want, bound = reference(q[None], k[None], v[None], window, sinks, g[None])
    ts = []
    for i, x in enumerate((q, k, v)):
        if i == 1:
            base = torch.zeros(n, row)
            y = base[:, 4:4 + 2 * d]
            y.copy_(torch.tensor(np.ascontiguousarray(x.transpose(1, 0, 2).reshape(n, 2 * d))))
            y = y.view(n, 2, d).transpose(0, 1)
            assert y.stride() == (d, row, 1)
        else:
            y = torch.tensor(x)
        ts.append(y.requires_grad_(True))
    f = torch.functional.sliding_window_attention
    o = f(*ts, window, sinks)
    near(o.numpy(), want[0][0], bound[0][0], "output")
    o.backward(torch.tensor(g))
    for name, t, w, e in zip(("dq", "dk", "dv"), ts, want[1:], bound[1:]):
        near(t.grad.numpy(), w[0], e[0], name)
    o = f(ts[0].detach()[:, -1:], ts[1].detach(), ts[2].detach(), window, sinks)
    near(o.numpy(), want[0][0][:, -1:], bound[0][0][:, -1:], "last position")


@gpu
@pytest.mark.parametrize("h,hkv", [(260, 260), (320, 160)])
def test_backward_in_parts_of_the_heads(torch, h, hkv):
    """More heads than the backward's memory takes at once."""
    n, d, window, sinks = 2048, 4, 2040, 1
    q, k, v, g = inputs(10, 1, h, hkv, n, n, d)
    ts = [torch.tensor(x, requires_grad=True) for x in (q, k, v)]
    torch.functional.sliding_window_attention(*ts, window, sinks).backward(torch.tensor(g))
    grads = [t.grad.numpy() for t in ts]
    grp = h // hkv
    for kv in (0, hkv // 2, hkv - 1):
        a, b = slice(kv * grp, (kv + 1) * grp), slice(kv, kv + 1)
        want, bound = reference(q[:, a], k[:, b], v[:, b], window, sinks, g[:, a])
        for name, got, w, e in zip(("dq", "dk", "dv"), (grads[0][:, a], grads[1][:, b], grads[2][:, b]),
                                   want[1:], bound[1:]):
            near(got, w, e, "%s of key head %d" % (name, kv))


@gpu
def test_graphs_and_eager_work_between(torch):
    """Two captured graphs and eager calls share the library's workspaces."""
    f = torch.functional.sliding_window_attention
    q, k, v, g = inputs(12, 1, 4, 2, 200, 200, 64)
    hosts = [(q, k, v), tuple(np.ascontiguousarray(x[:, :, ::-1]) for x in (q, k, v))]
    tg = torch.tensor(g)

    def call(ts):
        for t in ts:
            t.grad = None
        o = f(*ts, 70, 5)
        o.backward(tg)
        return [o] + [t.grad for t in ts]

    leaves = [[torch.tensor(x, requires_grad=True) for x in xs] for xs in hosts]
    want = [[t.numpy().copy() for t in call(ts)] for ts in leaves]
    long = torch.tensor(np.random.default_rng(1).standard_normal((1, 1, 4000, 64)).astype(np.float32))
    one = f(long[:, :, -1:], long, long, 4000).numpy()
    graphs, got = [], []
    for ts in leaves:
        graph = torch.hip.Graph()
        with torch.hip.graph(graph):
            got.append(call(ts))
        graphs.append(graph)
    for order in ((0, 1), (1, 0), (0, 1)):
        for i in order:
            graphs[i].replay()
            np.testing.assert_array_equal(f(long[:, :, -1:], long, long, 4000).numpy(), one)
        for i in (0, 1):
            for a, w in zip(got[i], want[i]):
                np.testing.assert_array_equal(a.numpy(), w)


@gpu
@pytest.mark.parametrize("hkv", [1, 2])
def test_second_derivative_beside_what_is_not_seen(torch, hkv):
    """Keys and values that no query sees may hold anything there too."""
    q, k, v, g = inputs(16, 1, 2, hkv, 4, 12, 8)
    f = torch.functional.sliding_window_attention
    hidden = ~visible(4, 12, 3, 2).any(0)
    assert hidden.sum() == 4

    def derivatives(fill):
        x = [q, k.copy(), v.copy()]
        for y in x[1:]:
            y[:, :, hidden] = fill
        ts = [torch.tensor(y, requires_grad=True) for y in x]
        grads = torch.autograd.grad((f(*ts, 3, 2) * torch.tensor(g)).sum(), ts, create_graph=True)
        loss = sum(((y * y).sum() for y in grads[1:]), (grads[0] * grads[0]).sum())
        return [y.detach().numpy() for y in list(grads) + list(torch.autograd.grad(loss, ts))]
    want = derivatives(0.0)
    for fill in (np.nan, np.inf, -np.inf, 3e38):
        for a, w in zip(derivatives(fill), want):
            assert np.isfinite(w).all()
            np.testing.assert_array_equal(a, w)


# ------------------------------------------------------------------ refusals


def _fake(pkg, *shape):
    """A tensor without a device: the checks come before anything reads it."""
    return pkg.Tensor(types.SimpleNamespace(ptr=4096), shape, None, 0, "float32")


def test_refusals(pkg):
    f = pkg.functional.sliding_window_attention
    x = _fake(pkg, 2, 4, 10, 8)
    for window in (0, -1, 2.5):
        with pytest.raises(ValueError, match="window"):
            f(x, x, x, window)
    for sinks in (-1, 0.5):
        with pytest.raises(ValueError, match="sinks"):
            f(x, x, x, 3, sinks)
    for q, k, v in ((x, _fake(pkg, 2, 3, 10, 8), _fake(pkg, 2, 3, 10, 8)),
                    (x, _fake(pkg, 2, 4, 9, 8), _fake(pkg, 2, 4, 9, 8)),
                    (x, x, _fake(pkg, 2, 4, 11, 8)), (x, _fake(pkg, 1, 4, 10, 8), _fake(pkg, 1, 4, 10, 8)),
                    (x, _fake(pkg, 2, 4, 10, 12), _fake(pkg, 2, 4, 10, 12)),
                    (x, _fake(pkg, 2, 10, 8), _fake(pkg, 2, 10, 8)), (_fake(pkg, 10, 8),) * 3,
                    (x, _fake(pkg, 2, 0, 10, 8), _fake(pkg, 2, 0, 10, 8))):
        with pytest.raises(RuntimeError, match="sliding_window_attention"):
            f(q, k, v, 3)
    for d in (129, 256):
        with pytest.raises(NotImplementedError, match="up to 128"):
            f(*(_fake(pkg, 1, 1, 4, d),) * 3, 2)


@gpu
def test_refusals_of_the_library(torch):
    from torchjs_amd import _lib as L
    x = torch.zeros(1, 2, 8, 8)
    p, st = x.data_ptr(), L.i64arr((128, 64, 8))
    lib = L.lib()

    def forward(h=2, hkv=2, tq=8, tk=8, d=8, window=3, sinks=0, ptr=p, strides=st, scale=1.0):
        return lib.tjh_window_forward(ptr, p, p, p, None, 1, h, hkv, tq, tk, d, strides, st, st, st,
                                      scale, window, sinks)
    assert forward(window=0) == 1 and forward(sinks=-1) == 1 and forward(tk=7) == 1
    assert forward(hkv=0) == 1 and forward(h=3) == 1 and forward(ptr=None) == 1
    assert forward(strides=None) == 1 and forward(d=0) == 1
    assert forward(d=6) == 5 and forward(d=132) == 5 and forward(ptr=p + 4) == 5
    assert forward(strides=L.i64arr((128, 64, 9))) == 5
    assert forward(tq=0, ptr=None) == 0


@gpu
def test_rows_whose_grid_does_not_fit_are_refused(torch):
    """2^32 threads or more, by sizes alone: nothing is launched or read."""
    from torchjs_amd import _lib as L
    x = torch.zeros(1, 1, 8, 8)
    p, st = x.data_ptr(), L.i64arr((0, 0, 8))
    sts = (L.P_i64 * 8)(*[L.ctypes.cast(st, L.P_i64)] * 8)

    def calls(b, h, tq):
        f = L.lib().tjh_window_forward(p, p, p, p, None, b, h, h, tq, 8, 8, st, st, st, st, 1.0, 3, 0)
        g = L.lib().tjh_window_backward(p, p, p, p, p, p, p, p, p, b, h, h, tq, 8, 8, sts, 1.0, 3, 0)
        return f, g
    # a query takes 512 threads where there are at most four, a tile of up to
    # 32 takes 256
    for b, h, tq in ((2 ** 23, 1, 1), (1, 2 ** 23 + 1, 1), (2 ** 22, 1, 2), (2 ** 21, 2, 4),
                     (1398102, 2, 3), (2 ** 24, 1, 5), (2 ** 12, 2 ** 12, 8), (2 ** 29, 2 ** 29, 8)):
        assert calls(b, h, tq) == (1, 1), (b, h, tq)
        assert b"too large" in L.lib().tjh_last_error()
