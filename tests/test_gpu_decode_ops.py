"""4-bit weights and caches, a beam search's step and the reordering of caches
against plain numpy in 64 bits."""
import ctypes

import numpy as np
import pytest

gpu = pytest.mark.gpu
U = 2.0 ** -24  # half a step of float32, relative
STEPS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


# ------------------------------------------------------------------- oracles


def held(x):
    """x [..., n] float32 that share a scale along the last axis: (codes [..., n],
    scales [...] float32, the values they stand for in 64 bits)."""
    x = x.astype(np.float32)
    top = np.abs(x).max(-1) if x.shape[-1] else np.zeros(x.shape[:-1], np.float32)
    with np.errstate(invalid="ignore"):
        scale = np.where(np.isfinite(top), top / np.float32(6), np.float32(np.nan))
    scale = np.where(top < 2.0 ** -100, np.float32(0), scale).astype(np.float32)
    s = scale.astype(np.float64)[..., None]
    a = np.abs(x.astype(np.float64))
    code = np.zeros(x.shape, np.int64)
    for i, border in enumerate((STEPS[1:] + STEPS[:-1]) / 2):
        with np.errstate(invalid="ignore"):  # both sides are exact
            code += (a > border * s) if i % 2 == 0 else (a >= border * s)
    code = np.where(s > 0, code, 0)
    return code + 8 * (x < 0), scale, value(code + 8 * (x < 0), scale)


def value(code, scale):
    v = STEPS[code & 7] * np.where(code & 8, -1.0, 1.0)
    return v * scale.astype(np.float64)[..., None]


def held_weight(w, group):
    """The values of a weight [N, K] held by groups of columns."""
    k = w.shape[1]
    w = np.pad(w, ((0, 0), (0, -k % 128)))
    code, scale, v = held(w.reshape(w.shape[0], -1, group))
    return code.reshape(w.shape), scale, v.reshape(w.shape)[:, :k]


def packed_weight(code):
    """A weight's codes as tjh_fp4_quantize lays them out."""
    n, k = code.shape
    c = code.reshape(n, k // 128, 4, 4, 8).transpose(0, 1, 3, 2, 4)  # t, j -> j, t
    c = c.reshape(n, k // 2, 2)
    return (c[..., 0] | c[..., 1] << 4).astype(np.uint8)


def packed_rows(code):
    d = code.shape[-1]
    code = np.pad(code, [(0, 0)] * (code.ndim - 1) + [(0, -d % 32)])
    return (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8)


def attend_ref(q, k, v, lengths, scale):
    """(result, tolerance) of causal attention, the queries at the end of each
    sequence's keys."""
    b, h, tq, d = q.shape
    q, group = q.astype(np.float64), h // k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(b):
        n = int(np.clip(lengths[i], 0, k.shape[2]))
        for j in range(h):
            kk, vv = k[i, j // group, :n], v[i, j // group, :n]
            for t in range(tq):
                see = n - tq + t + 1
                if see <= 0:
                    continue
                s = kk[:see] @ q[i, j, t] * scale
                size = np.abs(kk[:see]) @ np.abs(q[i, j, t]) * abs(scale)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, j, t] = p @ vv[:see]
                # a score is off by D products' and sums' roundings and four more,
                # and by one of its distance from the maximum; then the exponential,
                # the weight and the sums over the keys that one lane group, or one
                # tile of 32, adds up, numerator and denominator
                off = ((d + 4) * size + 4 * np.abs(s).max()) * U
                terms = 2 * (see / 8 + 64) * U
                tol[i, j, t] = p * (2 * off.max() + terms) @ np.abs(vv[:see])
    return out, tol


def beam_ref(x, scores, keep, finished=None, eos=None):
    """Scores in 64 bits, tokens, parents, flags, and all candidates [B, W V]."""
    b, w, n = x.shape
    x = x.astype(np.float64)
    cand = np.full((b, w, n), -np.inf)
    for i in range(b):
        for j in range(w):
            s = float(scores[i, j])
            if not s > -np.inf:
                continue
            if finished is not None and finished[i, j]:
                cand[i, j, eos] = s
                continue
            m = x[i, j].max()
            if not np.isfinite(m):
                continue
            cand[i, j] = s + (x[i, j] - m - np.log(np.exp(x[i, j] - m).sum()))
    flat = cand.reshape(b, -1)
    order = np.argsort(-flat, axis=1, kind="stable")[:, :keep]
    best = np.take_along_axis(flat, order, 1)
    none = best == -np.inf
    tokens = np.where(none, -1, order % n)
    parents = np.where(none, np.minimum(np.arange(keep), w - 1), order // n)
    done = none.copy()
    if finished is not None:
        done |= np.take_along_axis(finished, parents, 1)
    if eos is not None:
        done |= tokens == eos
    return best, tokens, parents, done, flat


def test_oracle_of_four_bits():
    """Every step stands for itself, halves go to the even step."""
    x = np.concatenate([STEPS, -STEPS, [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]]).astype(np.float32)
    code, scale, v = held(x)
    assert scale == 1
    assert v[:16].tolist() == x[:16].tolist()
    assert v[16:].tolist() == [0, 1, 1, 2, 2, 4, 4]
    assert code[16:].tolist() == [0, 2, 2, 4, 4, 6, 6]
    assert held(np.zeros(3))[1] == 0 and np.isnan(held(np.array([1, np.inf]))[1])


# ------------------------------------------------------------------- weights


def _weight(rng, n, k):
    return (rng.standard_normal((n, k)) * np.exp(rng.standard_normal((n, 1)))).astype(np.float32)


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (5, 128), (17, 129), (64, 768), (33, 1000)])
def test_quantize(torch, n, k, group):
    F, rng = torch.functional, np.random.default_rng(n * k)
    w = _weight(rng, n, k)
    w[0, :min(k, 7)] = [6, 0.25, 0.75, -1.25, 1.75, -2.5, 5][:min(k, 7)]  # halves, if 6 is the largest
    if n > 2:
        w[1] = 0
        w[2] *= 2.0 ** -103
    code, scale, v = held_weight(w, group)
    codes, scales = F.quantize_fp4(torch.tensor(w), group)
    assert (scales.numpy() == scale).all()
    assert (codes.numpy() == packed_weight(code)).all()
    got = F.dequantize_fp4(codes, scales, k, group).numpy()
    assert (got == v.astype(np.float32)).all()


@gpu
def test_quantize_views_and_no_numbers(torch):
    F, rng = torch.functional, np.random.default_rng(0)
    w = _weight(rng, 40, 300)
    for view in (lambda t: t.T, lambda t: t[:, 7:260], lambda t: t[3:33:1]):
        x = torch.tensor(w)
        codes, scales = F.quantize_fp4(view(x), 32)
        code, scale, _ = held_weight(view(w), 32)
        assert (scales.numpy() == scale).all() and (codes.numpy() == packed_weight(code)).all()
    w[5, 40], w[6, 299], w[7, 0] = np.nan, np.inf, -np.inf
    codes, scales = F.quantize_fp4(torch.tensor(w), 64)
    bad = np.isnan(scales.numpy())
    assert bad.sum() == 3 and bad[5, 0] and bad[6, 4] and bad[7, 0]
    assert np.isnan(F.dequantize_fp4(codes, scales, 300, 64).numpy()[5, :64]).all()


def _linear_case(torch, m, k, n, group, bias, seed=0):
    rng = np.random.default_rng(seed)
    w = _weight(rng, n, k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32) if bias else None
    _, _, v = held_weight(w, group)
    want = x.astype(np.float64) @ v.T + (0 if b is None else b)
    size = np.abs(x.astype(np.float64)) @ np.abs(v.T) + (0 if b is None else np.abs(b))
    # an instruction adds 32 products, each cut off below a full step of the sum;
    # then K / 32 sums of 32 columns, and those of at most 16 waves, three parts
    # and the bias
    tol = (64 + k / 32 + 52) * U * size
    codes, scales = torch.functional.quantize_fp4(torch.tensor(w), group)
    return x, b, codes, scales, want, tol


LINEAR = [(1, 1, 1), (1, 31, 3), (2, 128, 16), (3, 129, 17), (5, 768, 2304), (6, 768, 50),
          (10, 300, 65), (16, 1000, 100), (17, 515, 77), (32, 640, 40), (33, 256, 129), (64, 1024, 64),
          (100, 96, 500), (129, 384, 257), (300, 200, 1030), (1, 4100, 5000), (4, 260, 33000),
          (7, 1300, 17000), (30, 700, 9000), (70, 33, 33000), (1100, 160, 4000), (2050, 300, 1900),
          (1900, 100, 1000), (26, 300, 70), (16, 140, 16400), (21, 140, 16400), (26, 140, 16400),
          (32, 140, 16400)]


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear(torch, m, k, n, group):
    x, b, codes, scales, want, tol = _linear_case(torch, m, k, n, group, n % 2 == 1)
    y = torch.functional.linear_fp4(torch.tensor(x), codes, scales,
                                    torch.tensor(b) if b is not None else None, group)
    assert y.shape == (m, n)
    assert (np.abs(y.numpy() - want) <= tol).all()


# some rows by every width and height of tiles, with x cut beforehand or not, and
# with the columns of x in slices: tiles 16 high by 16, 32, 64 wide, 32 and 64 high,
# rows that do not fill the last one, slices of unlike lengths, K inside a block
SOME = [(9, 500, 2000), (9, 500, 6001), (9, 301, 12000), (9, 301, 17000), (40, 300, 5000),
        (31, 300, 16500), (50, 297, 16000), (6, 4003, 50), (3, 9000, 40), (1, 31993, 17),
        (7, 8200, 300), (40, 2100, 300), (33, 1153, 1000), (60, 16000, 500), (100, 16001, 1000),
        (300, 16000, 1000), (700, 5000, 70)]


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,k,n", SOME)
def test_linear_of_some_rows(torch, m, k, n, group):
    x, b, codes, scales, want, tol = _linear_case(torch, m, k, n, group, n % 2 == 0, 3)
    tx, tb = torch.tensor(x), torch.tensor(b) if b is not None else None
    y = torch.functional.linear_fp4(tx, codes, scales, tb, group).numpy()
    # as in test_linear; a wave's and a slice's sums are fewer than there
    assert (np.abs(y - want) <= tol).all()
    again = torch.functional.linear_fp4(tx, codes, scales, tb, group).numpy()
    assert np.array_equal(y, again)
    # rows of a wider tensor, and a row's result does not go by its place
    wide = torch.tensor(np.concatenate([np.full((m, 1), np.nan, np.float32), x[::-1]], 1))
    y2 = torch.functional.linear_fp4(wide[:, 1:], codes, scales, tb, group).numpy()
    assert np.array_equal(y2[::-1], y)


@gpu
@pytest.mark.parametrize("m", [2, 9, 70])
def test_linear_takes_rows_where_they_stand(torch, m):
    x, _, codes, scales, want, tol = _linear_case(torch, 2 * m, 203, 30, 64, False)
    big = torch.tensor(np.concatenate([np.full((2 * m, 3), np.nan, np.float32), x,
                                       np.full((2 * m, 2), np.inf, np.float32)], 1))
    y = torch.functional.linear_fp4(big[:, 3:206], codes, scales)
    assert (np.abs(y.numpy() - want) <= tol).all()
    y = torch.functional.linear_fp4(torch.tensor(x).view(2, m, 203).transpose(0, 1), codes, scales)
    assert y.shape == (m, 2, 30)
    assert (np.abs(y.numpy().transpose(1, 0, 2).reshape(2 * m, 30) - want) <= tol).all()
    one = torch.functional.linear_fp4(torch.tensor(x[0]), codes, scales)
    assert one.shape == (30,) and (np.abs(one.numpy() - want[0]) <= tol[0]).all()
    none = torch.functional.linear_fp4(torch.zeros(0, 203), codes, scales)
    assert none.shape == (0, 30)
    empty, bias = torch.functional.quantize_fp4(torch.zeros(30, 0)), torch.randn(30)
    y = torch.functional.linear_fp4(torch.zeros(m, 0), *empty, bias)
    assert (y.numpy() == bias.numpy()).all()


@gpu
@pytest.mark.parametrize("m", [1, 8, 65])
def test_linear_of_extreme_values(torch, m):
    """Large and small floats keep their three parts; what is no number stays in
    its row."""
    x, _, codes, scales, want, tol = _linear_case(torch, m, 256, 40, 64, False)
    for f in (2.0 ** 100, 2.0 ** -90):
        y = torch.functional.linear_fp4(torch.tensor((x * np.float32(f)).astype(np.float32)), codes,
                                        scales).numpy()
        assert (np.abs(y.astype(np.float64) / f - want) <= tol).all()
    x = np.concatenate([x, x])
    x[0, 5], x[m, 9] = np.nan, 3e38
    y = torch.functional.linear_fp4(torch.tensor(x), codes, scales).numpy()
    assert np.isnan(y[0]).all()
    rest = [i for i in range(2 * m) if i not in (0, m)]
    assert (np.abs(y - np.concatenate([want, want])) <= np.concatenate([tol, tol]))[rest].all()
    # an infinity gives what it gives in floats: NaN by a zero, else an infinity
    x[m, 9] = np.inf
    y = torch.functional.linear_fp4(torch.tensor(x), codes, scales).numpy()[m]
    w = torch.functional.dequantize_fp4(codes, scales, 256, 64).numpy()[:, 9]
    with np.errstate(invalid="ignore"):
        assert np.array_equal(y, np.float32(np.inf) * w, equal_nan=True)


@gpu
@pytest.mark.parametrize("m,k,n", [(1, 40, 33), (7, 300, 64), (70, 129, 50)])
def test_linear_gradients(torch, m, k, n):
    F = torch.functional
    x, b, codes, scales, _, _ = _linear_case(torch, m, k, n, 64, True)
    w = F.dequantize_fp4(codes, scales, k, 64).numpy().astype(np.float64)
    rng = np.random.default_rng(1)
    g = rng.standard_normal((m, n)).astype(np.float32)
    tx, tb = torch.tensor(x, requires_grad=True), torch.tensor(b, requires_grad=True)
    y = F.linear_fp4(tx, codes, scales, tb, 64)
    y.backward(torch.tensor(g))
    # products of n, sums of m terms
    assert (np.abs(tx.grad.numpy() - g @ w) <= (n + 2) * U * (np.abs(g) @ np.abs(w))).all()
    assert (np.abs(tb.grad.numpy() - g.sum(0, dtype=np.float64)) <= m * U * np.abs(g).sum(0)).all()
    # against differences, along one direction
    d = rng.standard_normal((m, k)).astype(np.float32)
    with torch.no_grad():
        hi, lo = [(F.linear_fp4(torch.tensor(x + s * d), codes, scales, tb, 64).numpy()
                   .astype(np.float64) * g).sum() for s in (1, -1)]
    size = (np.abs(g) * ((np.abs(x) + np.abs(d)).astype(np.float64) @ np.abs(w.T) + np.abs(b))).sum()
    want = (tx.grad.numpy().astype(np.float64) * d).sum()
    # x + d rounds once; each side as test_linear's; the gradient's own
    assert abs((hi - lo) / 2 - want) <= (64 + k / 32 + 52 + n + 4) * U * size
    # the gradient's gradient: linear in what comes in
    tx, tg = torch.tensor(x, requires_grad=True), torch.tensor(g, requires_grad=True)
    (dx,) = torch.autograd.grad(F.linear_fp4(tx, codes, scales), tx, tg, create_graph=True)
    (dg,) = torch.autograd.grad(dx, tg, torch.tensor(d))
    assert (np.abs(dg.numpy() - d @ w.T) <= (k + 2) * U * (np.abs(d) @ np.abs(w.T))).all()


@gpu
def test_linear_of_more_rows_than_are_split_at_once(torch):
    """A GB of x's parts: the rows before and behind its end."""
    rng = np.random.default_rng(0)
    m, k, n = 1398144 + 70, 128, 70
    w = _weight(rng, n, k)
    codes, scales = torch.functional.quantize_fp4(torch.tensor(w))
    v = held_weight(w, 64)[2]
    torch.manual_seed(1)
    x = torch.randn(m, k)
    y = torch.functional.linear_fp4(x, codes, scales)
    for a, b in ((0, 100), (m - 200, m), (m // 2, m // 2 + 50)):
        xs, ys = x[a:b].numpy().astype(np.float64), y[a:b].numpy()
        tol = (64 + k / 32 + 52) * U * (np.abs(xs) @ np.abs(v.T))
        assert (np.abs(ys - xs @ v.T) <= tol).all()


@gpu
def test_linear_gradients_in_a_graph(torch):
    """A captured forward and backward beside a graph of the same leaves that
    is still alive; replays follow new values."""
    F, rng = torch.functional, np.random.default_rng(3)
    codes, scales = F.quantize_fp4(torch.tensor(_weight(rng, 48, 100)))
    x, b = torch.randn(9, 100, requires_grad=True), torch.randn(48, requires_grad=True)

    def loss():
        y = F.linear_fp4(x, codes, scales, b)
        return (y * y).sum()

    def grads():
        x.grad = b.grad = None
        loss().backward()
        return x.grad, b.grad
    grads()
    alive = loss()
    g = torch.hip.Graph()
    with torch.hip.graph(g):
        captured = grads()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(9, 100))
        g.replay()
        got = [t.numpy().copy() for t in captured]
        for a, w in zip(got, grads()):
            assert (a == w.numpy()).all()
    alive.backward()
    g.reset()


@gpu
def test_linear_module(torch):
    torch.manual_seed(3)
    nn = torch.nn
    lin = nn.Linear(100, 60)
    four = nn.LinearFP4.of(lin, 32)
    x = torch.randn(4, 100)
    v = held_weight(lin.weight.numpy(), 32)[2]
    want = x.numpy().astype(np.float64) @ v.T + lin.bias.numpy()
    size = np.abs(x.numpy()) @ np.abs(v.T) + np.abs(lin.bias.numpy())
    assert (np.abs(four(x).numpy() - want) <= 200 * U * size).all()
    other = nn.LinearFP4(100, 60, group_size=32)
    state = four.state_dict()
    assert sorted(state) == ["bias", "codes", "scales"]
    other.load_state_dict(state)
    assert (other(x).numpy() == four(x).numpy()).all()
    other = nn.LinearFP4(100, 60, group_size=32)
    other.load_state_dict({n: t.numpy() for n, t in state.items()})
    assert (other(x).numpy() == four(x).numpy()).all()
    # an optimizer passes over what has no gradient
    opt = torch.optim.Adam(other.parameters(), lr=0.1)
    before = other.codes.numpy()
    (other(x) * other(x)).sum().backward()
    opt.step()
    assert (other.codes.numpy() == before).all()
    assert (other.bias.numpy() != four.bias.numpy()).any()


# --------------------------------------------------------------------- cache


def _new_cache(torch, b, h, n, d, fill=0):
    F = torch.functional
    row = F.cache_row_bytes(d)
    return [torch.tensor(np.full((b, h, n, row), fill, np.uint8), dtype="uint8"),
            torch.tensor(np.full((b, h, n), fill, np.float32)),
            torch.tensor(np.full((b, h, n, row), fill, np.uint8), dtype="uint8"),
            torch.tensor(np.full((b, h, n), fill, np.float32))]


DIMS = [1, 4, 30, 32, 40, 64, 80, 96, 100, 127, 128]


@gpu
@pytest.mark.parametrize("d", DIMS)
def test_append_and_read(torch, d):
    F, rng = torch.functional, np.random.default_rng(d)
    b, h, n, t, pos = 2, 3, 23, 9, 5
    cache = _new_cache(torch, b, h, n, d, 77)
    k, v = rng.standard_normal((2, b, h, t, d)).astype(np.float32)
    k[0, 1, 2] = 0
    k[1, 0, 3] *= 2.0 ** -104
    v[0, 0, 4, 0] = np.nan
    F.cache_append_fp4(*cache, torch.tensor(k), torch.tensor(v), pos)
    for x, codes, scales in ((k, *cache[:2]), (v, *cache[2:])):
        code, scale, val = held(x)
        c, s = codes.numpy(), scales.numpy()
        assert np.array_equal(s[:, :, pos:pos + t], scale, equal_nan=True)
        finite = np.isfinite(scale)
        assert (c[:, :, pos:pos + t][finite] == packed_rows(code)[finite]).all()
        # the other positions as they were
        assert (c[:, :, :pos] == 77).all() and (c[:, :, pos + t:] == 77).all()
        assert (s[:, :, :pos] == 77).all() and (s[:, :, pos + t:] == 77).all()
        got = F.cache_read_fp4(codes, scales, d, pos, pos + t).numpy()
        assert np.array_equal(got, np.where(finite[..., None], val, np.nan).astype(np.float32),
                              equal_nan=True)
    assert F.cache_read_fp4(*cache[:2], d, 3, 3).shape == (b, h, 0, d)
    both = F.cache_read_fp4(*cache[:2], d, pos, pos + t, cache[2:])
    for x, one in zip(both, (cache[:2], cache[2:])):
        assert np.array_equal(x.numpy(), F.cache_read_fp4(*one, d, pos, pos + t).numpy(), equal_nan=True)


@gpu
@pytest.mark.parametrize("d", [40, 64])
def test_append_of_views(torch, d):
    """The heads of a projection, as a layer has them; a part of wider rows."""
    F, rng = torch.functional, np.random.default_rng(d)
    b, h, t = 2, 3, 6
    qkv = rng.standard_normal((b, t, 3 * h * d)).astype(np.float32)
    _, k, v = [y.view(b, t, h, d).transpose(1, 2)
               for y in torch.tensor(qkv).split(h * d, dim=2)]
    cache = _new_cache(torch, b, h, 8, d)
    F.cache_append_fp4(*cache, k, v, 1)
    want = held(qkv[:, :, h * d:2 * h * d].reshape(b, t, h, d).transpose(0, 2, 1, 3))[2]
    got = F.cache_read_fp4(*cache[:2], d, 1, 7).numpy()
    assert (got == want.astype(np.float32)).all()
    wide = rng.standard_normal((b, h, t, d + 3)).astype(np.float32)
    x = torch.tensor(wide)[:, :, :, 1:d + 1]
    F.cache_append_fp4(*cache, x, x, 0)
    want = held(wide[..., 1:d + 1])[2].astype(np.float32)
    for c in (cache[:2], cache[2:]):
        assert (F.cache_read_fp4(*c, d, 0, t).numpy() == want).all()


@gpu
def test_append_where_each_sequence_ends(torch):
    F, rng = torch.functional, np.random.default_rng(5)
    b, h, n, t, d = 5, 2, 12, 4, 32
    cache = _new_cache(torch, b, h, n, d, 9)
    k, v = rng.standard_normal((2, b, h, t, d)).astype(np.float32)
    pos = np.array([0, 8, 10, -2, 50], np.int32)  # two of them in part, one not at all
    F.cache_append_fp4(*cache, torch.tensor(k), torch.tensor(v), torch.tensor(pos, dtype="int32"))
    for x, codes, scales in ((k, *cache[:2]), (v, *cache[2:])):
        want = np.full(scales.shape, 9, np.float32)
        rows = np.full(codes.shape, 9, np.uint8)
        code, scale, _ = held(x)
        for i in range(b):
            for j in range(t):
                if 0 <= pos[i] + j < n:
                    want[i, :, pos[i] + j] = scale[i, :, j]
                    rows[i, :, pos[i] + j] = packed_rows(code)[i, :, j]
        assert (scales.numpy() == want).all() and (codes.numpy() == rows).all()
    other = _new_cache(torch, b, h, n, d, 9)
    F.cache_append_fp4(*other, torch.tensor(k), torch.tensor(v), [int(p) for p in pos])
    assert all((x.numpy() == y.numpy()).all() for x, y in zip(other, cache))


def _filled(torch, b, hkv, n, d, rng, spread=1.0):
    """A cache of n positions and the values it stands for."""
    cache = _new_cache(torch, b, hkv, n, d)
    k, v = rng.standard_normal((2, b, hkv, n, d)).astype(np.float32)
    k *= np.exp(spread * rng.standard_normal((1, hkv, 1, d))).astype(np.float32)
    if n:
        torch.functional.cache_append_fp4(*cache, torch.tensor(k), torch.tensor(v), 0)
    return cache, held(k)[2], held(v)[2]


ATTEND = [  # b, h, hkv, tq, keys, d
    (1, 1, 1, 1, 1, 64), (2, 3, 3, 1, 5, 64), (1, 2, 1, 1, 130, 32), (2, 4, 4, 1, 300, 64),
    (1, 6, 2, 1, 257, 128), (2, 8, 1, 1, 100, 80), (1, 12, 12, 1, 1000, 64), (1, 2, 2, 2, 2, 40),
    (1, 4, 2, 3, 70, 96), (2, 2, 2, 7, 7, 64), (1, 3, 3, 33, 33, 64), (1, 4, 4, 31, 90, 128),
    (1, 4, 1, 64, 200, 80), (1, 2, 2, 65, 65, 32), (2, 2, 1, 100, 133, 64), (1, 1, 1, 129, 400, 128),
    (1, 2, 2, 40, 40, 30), (1, 2, 2, 3, 20, 1), (1, 2, 1, 50, 60, 127), (1, 16, 1, 1, 513, 64),
    (1, 5, 5, 200, 200, 64),
    # keys in slices; a wave for each 16 rows; both
    (1, 4, 2, 1, 1500, 64), (2, 2, 2, 3, 1300, 80), (1, 2, 1, 40, 1100, 32), (3, 8, 1, 1, 2100, 128),
    (32, 16, 16, 17, 30, 64), (1, 16, 1, 1024, 1030, 32)]


@gpu
@pytest.mark.parametrize("b,h,hkv,tq,n,d", ATTEND)
def test_attention(torch, b, h, hkv, tq, n, d):
    rng = np.random.default_rng(b * n + d)
    cache, k, v = _filled(torch, b, hkv, n, d, rng, 0.3)
    q = rng.standard_normal((b, h, tq, d)).astype(np.float32)
    y = torch.functional.attention_fp4(torch.tensor(q), *cache, n)
    assert y.shape == q.shape
    want, tol = attend_ref(q, k, v, [n] * b, np.float32(d ** -0.5))
    assert (np.abs(y.numpy() - want) <= tol).all()


@gpu
@pytest.mark.parametrize("n", [150, 1200])
@pytest.mark.parametrize("tq", [1, 3, 40])
@pytest.mark.parametrize("h,hkv,d", [(4, 2, 64), (3, 3, 128)])
def test_attention_of_ragged_sequences(torch, tq, h, hkv, d, n):
    """A length each: none, fewer than there are queries, some, all, and more and
    less than there can be.  Later positions hold NaN."""
    rng = np.random.default_rng(tq)
    lengths = np.array([0, 1, 2, 39, 41, n, 9999, -3, n - 1], np.int32)
    b = len(lengths)
    cache, k, v = _filled(torch, b, hkv, n, d, rng, 0.3)
    for i, length in enumerate(lengths):
        for s in (cache[1], cache[3]):
            if 0 <= length < n:
                s[i, :, int(length):].fill_(float("nan"))
    q = rng.standard_normal((b, h, tq, d)).astype(np.float32)
    y = torch.functional.attention_fp4(torch.tensor(q), *cache, torch.tensor(lengths, dtype="int32"))
    want, tol = attend_ref(q, k, v, lengths, np.float32(d ** -0.5))
    assert (np.abs(y.numpy() - want) <= tol).all()
    again = torch.functional.attention_fp4(torch.tensor(q), *cache, list(map(int, lengths)))
    assert (again.numpy() == y.numpy()).all()


@gpu
@pytest.mark.parametrize("tq,n,d", [(1, 700, 64), (2, 90, 80), (50, 260, 64), (70, 70, 128)])
def test_attention_far_from_even(torch, tq, n, d):
    """Scores far apart, rising and falling along the keys: running maxima that
    change often; a scale given; queries as a layer lays them out."""
    rng = np.random.default_rng(n)
    b, h = 2, 3
    cache = _new_cache(torch, b, h, n + 7, d)
    slope = np.linspace(-4, 4, n)[None, None, :, None] * np.array([1, -1, 3])[None, :, None, None]
    u = rng.standard_normal((1, 1, 1, d))
    k = (u * slope + 0.1 * rng.standard_normal((b, h, n, d))).astype(np.float32)
    v = rng.standard_normal((b, h, n, d)).astype(np.float32)
    torch.functional.cache_append_fp4(*cache, torch.tensor(k), torch.tensor(v), 0)
    q = (np.ones((b, h, tq, 1)) * u / d + 0.1 * rng.standard_normal((b, h, tq, d)) / d).astype(np.float32)
    rows = torch.tensor(np.ascontiguousarray(q.transpose(0, 2, 1, 3))).transpose(1, 2)
    y = torch.functional.attention_fp4(rows, *cache, n, scale=2.5)
    want, tol = attend_ref(q, held(k)[2], held(v)[2], [n] * b, 2.5)
    assert (np.abs(y.numpy() - want) <= tol).all()


@gpu
@pytest.mark.parametrize("tq", [1, 40])
def test_attention_of_no_numbers(torch, tq):
    """NaN in a key reaches the queries that see it; in a query its own row."""
    rng = np.random.default_rng(2)
    cache, k, v = _filled(torch, 1, 2, 64, 64, rng, 0.3)
    q = rng.standard_normal((1, 2, tq, 64)).astype(np.float32)
    q[0, 1, tq - 1, 3] = np.nan
    y = torch.functional.attention_fp4(torch.tensor(q), *cache, 64).numpy()
    want, tol = attend_ref(q, k, v, [64], np.float32(0.125))
    assert np.isnan(y[0, 1, tq - 1]).all()
    ok = ~np.isnan(want)
    assert (np.abs(y - want)[ok] <= tol[ok]).all()
    at = 64 - tq // 2 - 1
    cache[1][0, 0, at].fill_(float("nan"))
    y = torch.functional.attention_fp4(torch.tensor(q), *cache, 64).numpy()
    first = max(0, at - (64 - tq))
    assert np.isnan(y[0, 0, first:]).all() and not np.isnan(y[0, 0, :first]).any()


@gpu
def test_attention_without_keys_or_queries(torch):
    F = torch.functional
    cache = _new_cache(torch, 2, 2, 0, 64)
    y = F.attention_fp4(torch.ones(2, 4, 3, 64), *cache, torch.zeros(2, dtype="int32"))
    assert (y.numpy() == 0).all()
    cache = _new_cache(torch, 2, 2, 5, 64)
    assert F.attention_fp4(torch.ones(2, 4, 0, 64), *cache, 5).shape == (2, 4, 0, 64)
    F.cache_append_fp4(*cache, torch.ones(2, 2, 0, 64), torch.ones(2, 2, 0, 64), 5)
    assert (cache[1].numpy() == 0).all()


# --------------------------------------------------------------------- beams


def _check_beams(torch, x, scores, keep=None, finished=None, eos=None):
    w = scores.shape[1]
    f = torch.tensor(finished, dtype="bool") if finished is not None else None
    got = torch.functional.beam_step(torch.tensor(x), torch.tensor(scores), keep, f, eos)
    best, tokens, parents, done, flat = beam_ref(x, scores, keep or w, finished, eos)
    s, t, p, e = [y.numpy() for y in got]
    none = best == -np.inf
    assert (s[none] == -np.inf).all() and (t[none] == -1).all()
    assert (p[none] == parents[none]).all() and e[none].all()
    # the logarithm of a float sum: a chain of some 130 roundings and the
    # exponentials', then the score's own
    tol = 140 * U + 2 * U * np.abs(np.where(none, 0, best))
    assert (np.abs(np.where(none, 0, s) - np.where(none, 0, best)) <= tol).all()
    for i in range(x.shape[0]):
        for j in range(s.shape[1]):
            if none[i, j]:
                continue
            c = p[i, j] * x.shape[2] + t[i, j]
            # another one only where the two are as near as that
            if c != parents[i, j] * x.shape[2] + tokens[i, j]:
                assert abs(flat[i, c] - best[i, j]) <= 2 * tol[i, j]
                assert p[i, j] != parents[i, j]
            ends = (eos is not None and t[i, j] == eos) or \
                (finished is not None and finished[i, p[i, j]])
            assert bool(e[i, j]) == ends
        pairs = [(a, b) for a, b, m in zip(p[i], t[i], none[i]) if not m]
        assert len(set(pairs)) == len(pairs)


def _beams(b, w, n, seed=0):
    rng = np.random.default_rng(seed)
    x = (2.5 * rng.standard_normal((b, w, n))).astype(np.float32)
    return rng, x, (-10 - 3 * np.abs(rng.standard_normal((b, w)))).astype(np.float32)


@gpu
@pytest.mark.parametrize("b,w,n,keep", [(1, 1, 1, 1), (1, 1, 50, 4), (2, 4, 1, 3), (1, 4, 1019, None),
                                        (3, 2, 1021, 5), (1, 4, 50257, None), (2, 3, 50257, 64),
                                        (5, 16, 4093, 32), (40, 8, 3001, None), (70, 8, 16385, None),
                                        (1, 64, 20000, 64), (33, 8, 50257, 8), (2, 2, 131072, 10)])
def test_beam_step(torch, b, w, n, keep):
    _, x, scores = _beams(b, w, n, n)
    _check_beams(torch, x, scores, keep)


@gpu
@pytest.mark.parametrize("w,n", [(2, 7), (8, 1500), (5, 50257)])
def test_beam_step_with_ended_beams(torch, w, n):
    rng, x, scores = _beams(6, w, n, w)
    finished = rng.random((6, w)) < 0.5
    finished[0], finished[1] = True, False
    for eos in (0, n - 1):
        _check_beams(torch, x, scores, None, finished, eos)
        _check_beams(torch, x, scores, min(2 * w, 64), finished, eos)
    _check_beams(torch, x, scores, None, None, n // 2)


@gpu
@pytest.mark.parametrize("n", [9, 1030, 33000])
def test_beam_step_of_rows_without_a_distribution(torch, n):
    _, x, scores = _beams(6, 3, n)
    x[0, 1, 4] = np.nan
    x[1, 0, n - 1] = np.inf
    x[2, 2] = -np.inf
    x[3, :, 2:] = -np.inf  # two tokens a beam
    x[4] = -np.inf
    scores[5] = [-np.inf, -12, np.nan]
    _check_beams(torch, x, scores, 7)


@gpu
@pytest.mark.parametrize("n", [5, 1025, 4097, 50257])
@pytest.mark.parametrize("rows", [1, 60])
def test_beam_step_of_equal_continuations(torch, n, rows):
    """Equal beams have equal scores to the last bit, however their rows are
    aligned: the first beam's come first; of equal logits the first tokens."""
    rng = np.random.default_rng(n)
    row = rng.standard_normal(n).astype(np.float32)
    x = np.broadcast_to(row, (rows, 4, n)).copy()
    scores = np.full((rows, 4), -3.0, np.float32)
    s, t, p, _ = [y.numpy() for y in torch.functional.beam_step(torch.tensor(x), torch.tensor(scores), 6)]
    order = np.argsort(-row, kind="stable")
    assert (t == [order[0]] * 4 + [order[1]] * 2).all()
    assert (p == [0, 1, 2, 3, 0, 1]).all()
    assert (s[:, :4] == s[:1, :1]).all()
    x[:] = 1.5
    s, t, p, _ = [y.numpy() for y in torch.functional.beam_step(torch.tensor(x), torch.tensor(scores), 5)]
    assert (t == [0, 1, 2, 3, 4]).all() and (p == 0).all()


@gpu
def test_beam_step_where_logits_stand(torch):
    """Rows of a padded layer's output, one position of several, [B W, V] and
    other types."""
    _, x, scores = _beams(2, 3, 77)
    F = torch.functional
    want = [y.numpy() for y in F.beam_step(torch.tensor(x), torch.tensor(scores))]
    wide = np.full((6, 5, 80), np.nan, np.float32)
    wide[:, 2, 1:78] = x.reshape(6, 77)
    got = F.beam_step(torch.tensor(wide)[:, 2, 1:78], torch.tensor(scores))
    for a, b in zip(want, got):
        assert (a == b.numpy()).all()
    for a, b in zip(want, F.beam_step(torch.tensor(x), scores.tolist())):
        assert (a == b.numpy()).all()
    whole = (4 * x).astype(np.int32)
    a = F.beam_step(torch.tensor(whole), torch.tensor(scores))
    b = F.beam_step(torch.tensor(whole.astype(np.float32)), torch.tensor(scores))
    assert all((p.numpy() == q.numpy()).all() for p, q in zip(a, b))


# ---------------------------------------------------------------- reordering


def _reordered(x, parents, length):
    b, w = parents.shape
    y = x.reshape(b, w, *x.shape[1:])
    out = y.copy()
    for i in range(b):
        for j in range(w):
            if 0 <= parents[i, j] < w:
                if length is None:
                    out[i, j] = y[i, parents[i, j]]
                else:
                    out[i, j, :, :length] = y[i, parents[i, j], :, :length]
    return out.reshape(x.shape)


@gpu
@pytest.mark.parametrize("b,w", [(1, 1), (1, 2), (3, 4), (2, 7), (5, 8), (1, 13), (2, 32), (1, 64)])
@pytest.mark.parametrize("length", [0, 1, 5, 16, 19])
def test_reorder(torch, b, w, length):
    rng = np.random.default_rng(b * w + length)
    parents = rng.integers(0, w, (b, w)).astype(np.int32)
    if b > 1:
        parents[0] = np.roll(np.arange(w), 1)  # nobody stays
        parents[1, 0], parents[1, w - 1] = -1, w
    xs = [rng.standard_normal((b * w, 3, 19, 8)).astype(np.float32),
          rng.integers(0, 256, (b * w, 2, 19, 16)).astype(np.uint8),
          rng.standard_normal((b * w, 3, 19)).astype(np.float32),
          rng.integers(0, 256, (b * w, 1, 19, 3)).astype(np.uint8),
          rng.integers(-9, 9, (b * w, 1, 19, 1, 2)).astype(np.int32)]
    ts = [torch.tensor(x, dtype=str(x.dtype)) for x in xs]
    torch.functional.cache_reorder_(ts, torch.tensor(parents, dtype="int32"), length)
    for x, t in zip(xs, ts):
        assert (t.numpy() == _reordered(x, parents, length)).all()


@gpu
def test_reorder_whole_rows_and_many_tensors(torch):
    rng = np.random.default_rng(0)
    parents = rng.integers(0, 4, (2, 4)).astype(np.int32)
    xs = [rng.standard_normal((8, 1 + i % 5, 3)).astype(np.float32) for i in range(70)]
    xs.append(rng.integers(0, 99, 8).astype(np.int32))
    xs.append(np.zeros((8, 0), np.float32))
    ts = [torch.tensor(x, dtype=str(x.dtype)) for x in xs]
    torch.functional.cache_reorder_(ts, parents)
    for x, t in zip(xs, ts):
        assert (t.numpy() == _reordered(x, parents, None)).all()
    x = rng.standard_normal((8, 40000)).astype(np.float32)  # blocks of several workgroups
    t = torch.tensor(x)
    torch.functional.cache_reorder_(t, parents)
    assert (t.numpy() == _reordered(x, parents, None)).all()
    # rows of a larger tensor, and a tensor beside them
    big = torch.tensor(x)
    torch.functional.cache_reorder_([big[0:4], big[4:8]], parents[:1])
    assert (big.numpy()[:4] == _reordered(x[:4], parents[:1], None)).all()
    assert (big.numpy()[4:] == _reordered(x[4:], parents[:1], None)).all()


@gpu
def test_numbers_past_32_bits_are_taken_as_they_are(torch):
    """Parents of 2^32 are outside [0, W), not 0; a library caller's -2^32 is no
    token, not the token 0."""
    x = np.arange(6, dtype=np.float32).reshape(3, 2)
    t = torch.tensor(x)
    torch.functional.cache_reorder_(t, np.array([[1, 2 ** 32, -2 ** 32]]))
    assert (t.numpy() == x[[1, 1, 2]]).all()
    logits, scores = torch.tensor(np.float32([[2, 1, 0]])), torch.zeros(1, 1)
    s, d = torch.zeros(1, 2), torch.zeros(1, 2, dtype="uint8")
    tok, par = torch.zeros(1, 2, dtype="int32"), torch.zeros(1, 2, dtype="int32")
    lib = torch._lib
    lib.check(lib.lib().tjh_beam_step(logits.data_ptr(), 3, scores.data_ptr(), None, 1, 1, 3, 2,
                                      -2 ** 32, s.data_ptr(), tok.data_ptr(), par.data_ptr(),
                                      d.data_ptr()), "beam_step")
    assert tok.numpy().tolist() == [[0, 1]] and d.numpy().tolist() == [[0, 0]]


# ------------------------------------------------------------------- graphs


@gpu
def test_captured_and_replayed(torch):
    """All of them in one graph: replays follow new inputs, with other work and
    another graph of the same calls between them."""
    F, rng = torch.functional, np.random.default_rng(4)
    b, w, h, d, n, vocab = 2, 3, 2, 32, 40, 500
    weight = torch.tensor(_weight(rng, 3 * h * d, h * d))
    head = torch.tensor(_weight(rng, vocab, h * d))
    four, four_head = F.quantize_fp4(weight), F.quantize_fp4(head)

    def fresh():
        r = np.random.default_rng(8)
        return [torch.tensor(r.integers(0, 256, (b * w, h, n, 16)).astype(np.uint8), dtype="uint8"),
                torch.tensor(r.random((b * w, h, n)).astype(np.float32)),
                torch.tensor(r.integers(0, 256, (b * w, h, n, 16)).astype(np.uint8), dtype="uint8"),
                torch.tensor(r.random((b * w, h, n)).astype(np.float32))]

    def step(x, scores, cache):
        with torch.no_grad():
            qkv = F.linear_fp4(x, *four)
            q, k, v = [t.view(b * w, 1, h, d).transpose(1, 2) for t in qkv.split(h * d, dim=2)]
            F.cache_append_fp4(*cache, k, v, 20)
            y = F.attention_fp4(q, *cache, 21).transpose(1, 2).contiguous().view(b * w, h * d)
            out = F.beam_step(F.linear_fp4(y, *four_head), scores, None, None, 3)
            F.cache_reorder_(cache, out[2], 21)
        return [y] + list(out)

    inputs = [(rng.standard_normal((b * w, 1, h * d)).astype(np.float32),
               -rng.random((b, w)).astype(np.float32)) for _ in range(4)]
    x, scores = (torch.tensor(a) for a in inputs[0])
    graphs = []
    for _ in range(2):
        cache = fresh()
        step(x, scores, cache)
        g = torch.hip.Graph()
        with torch.hip.graph(g):
            out = step(x, scores, cache)
        graphs.append((g, cache, out))
    for i, (a, s) in enumerate(inputs + inputs):
        x.copy_(torch.tensor(a))
        scores.copy_(torch.tensor(s))
        for g, cache, out in graphs[::1 if i % 2 else -1]:
            for c, f in zip(cache, fresh()):
                c.copy_(f)
            g.replay()
        want_cache = fresh()
        want = step(x, scores, want_cache)
        torch.synchronize()
        for g, cache, out in graphs:
            for p, q in zip(out + cache, want + want_cache):
                assert np.array_equal(p.numpy(), q.numpy(), equal_nan=True)
    for g, _, _ in graphs:
        g.reset()


# ------------------------------------------------------------------ refusals


class _Memory:
    """Stands for a device allocation where only shapes are looked at."""

    def __init__(self, ptr=4096):
        self.ptr, self.nbytes = ptr, 1 << 40


def _shape_only(pkg, *shape, dtype="float32", ptr=4096, strides=None):
    from torchjs_amd.tensor import Tensor
    return Tensor(_Memory(ptr), shape, strides, 0, dtype)


def _refusals(t):
    """(error, call) of each refusal by shapes and numbers; `t` makes a tensor."""
    u8 = dict(dtype="uint8")
    codes, scales = t(6, 128, **u8), t(6, 4)
    cache = [t(2, 2, 9, 32, **u8), t(2, 2, 9), t(2, 2, 9, 32, ptr=1 << 20, **u8), t(2, 2, 9, ptr=1 << 21)]
    kv, q = t(2, 2, 3, 64), t(2, 4, 3, 64)
    ids = dict(dtype="int32")
    return [
        (ValueError, lambda F: F.quantize_fp4(t(6, 200), 16)),
        (ValueError, lambda F: F.quantize_fp4(t(6, 200), None)),
        (ValueError, lambda F: F.quantize_fp4(t(200))),
        (ValueError, lambda F: F.dequantize_fp4(codes, scales, 300)),
        (ValueError, lambda F: F.linear_fp4(t(3, 300), codes, scales)),
        (ValueError, lambda F: F.linear_fp4(t(3, 200), codes, scales, None, 32)),
        (ValueError, lambda F: F.linear_fp4(t(3, 200), codes, scales, t(5))),
        (ValueError, lambda F: F.linear_fp4(t(), codes, scales)),
        (TypeError, lambda F: F.linear_fp4(t(3, 200), t(6, 128), scales)),
        (TypeError, lambda F: F.linear_fp4(t(3, 200), codes, t(6, 4, **ids))),
        (ValueError, lambda F: F.linear_fp4(t(3, 200), t(6, 128, strides=(1, 6), **u8), scales)),
        (ValueError, lambda F: F.linear_fp4(t(3, 200), t(6, 128, ptr=4104, **u8), scales)),
        (ValueError, lambda F: F.cache_append_fp4(*cache, kv, t(2, 2, 4, 64), 0)),
        (RuntimeError, lambda F: F.cache_append_fp4(*cache, kv, kv, 7)),
        (ValueError, lambda F: F.cache_append_fp4(*cache, kv, kv, -1)),
        (ValueError, lambda F: F.cache_append_fp4(*cache, kv, kv, 1.5)),
        (ValueError, lambda F: F.cache_append_fp4(*cache, kv, kv, t(3, **ids))),
        (TypeError, lambda F: F.cache_append_fp4(*cache, kv, kv, t(2))),
        (ValueError, lambda F: F.cache_append_fp4(*cache, t(2, 3, 3, 64), t(2, 3, 3, 64), 0)),
        (ValueError, lambda F: F.cache_append_fp4(*cache, t(2, 2, 3, 65), t(2, 2, 3, 65), 0)),
        (ValueError, lambda F: F.cache_append_fp4(*cache[:2], *cache[:2], kv, kv, 0)),
        (NotImplementedError, lambda F: F.cache_append_fp4(*cache, t(2, 2, 3, 129), t(2, 2, 3, 129), 0)),
        (ValueError, lambda F: F.cache_read_fp4(*cache[:2], 64, 3, 10)),
        (ValueError, lambda F: F.cache_read_fp4(*cache[:2], 64, 5, 4)),
        (ValueError, lambda F: F.cache_read_fp4(*cache[:2], 70, 0, 4)),
        (ValueError, lambda F: F.cache_read_fp4(*cache[:2], 64, 0, 4, (t(2, 2, 8, 32, **u8), t(2, 2, 8)))),
        (ValueError, lambda F: F.attention_fp4(t(2, 3, 64), *cache, 9)),
        (RuntimeError, lambda F: F.attention_fp4(t(2, 3, 3, 64), *cache, 9)),
        (ValueError, lambda F: F.attention_fp4(q, *cache, 10)),
        (RuntimeError, lambda F: F.attention_fp4(q, *cache, 2)),
        (ValueError, lambda F: F.attention_fp4(t(3, 4, 3, 64), *cache, 9)),
        (ValueError, lambda F: F.attention_fp4(t(2, 4, 3, 80), *cache, 9)),
        (NotImplementedError, lambda F: F.attention_fp4(t(2, 4, 3, 130), *cache, 9)),
        (RuntimeError, lambda F: F.attention_fp4(t(2, 4, 3, 64).requires_grad_(), *cache, 9)),
        (ValueError, lambda F: F.attention_fp4(q, cache[0], t(2, 2, 8), *cache[2:], 9)),
        (ValueError, lambda F: F.beam_step(t(2, 3, 50), t(3, 2))),
        (ValueError, lambda F: F.beam_step(t(5, 50), t(2, 3))),
        (ValueError, lambda F: F.beam_step(t(2, 3, 50), t(2, 3), 0)),
        (ValueError, lambda F: F.beam_step(t(2, 3, 50), t(2, 3), 151)),
        (ValueError, lambda F: F.beam_step(t(2, 3, 50), t(2, 3), 2.5)),
        (ValueError, lambda F: F.beam_step(t(2, 3, 50), t(2, 3), 3, t(2, 3, dtype="bool"))),
        (ValueError, lambda F: F.beam_step(t(2, 3, 50), t(2, 3), 3, t(3, 2, dtype="bool"), 4)),
        (TypeError, lambda F: F.beam_step(t(2, 3, 50), t(2, 3), 3, t(2, 3), 4)),
        (ValueError, lambda F: F.beam_step(t(2, 3, 50), t(2, 3), 3, None, 50)),
        (ValueError, lambda F: F.beam_step(t(2, 3, 50), t(2, 3), 3, None, -1)),
        (ValueError, lambda F: F.cache_reorder_(t(6, 2, 9, 4), t(6, **ids))),
        (ValueError, lambda F: F.cache_reorder_(t(6, 2, 9, 4), t(2, 4, **ids))),
        (TypeError, lambda F: F.cache_reorder_(t(6, 2, 9, 4), t(2, 3))),
        (ValueError, lambda F: F.cache_reorder_(t(6, 2, 9, 4), t(2, 3, ptr=1 << 30, **ids), 10)),
        (ValueError, lambda F: F.cache_reorder_(t(6, 9), t(2, 3, ptr=1 << 30, **ids), 3)),
        (ValueError, lambda F: F.cache_reorder_(t(6, 2, 9, 4), t(2, 3, ptr=4100, **ids), 3)),
        (ValueError, lambda F: F.cache_reorder_([t(6, 2), t(6, 2)], t(2, 3, ptr=1 << 30, **ids))),
        (ValueError, lambda F: F.cache_reorder_(t(6, 2, strides=(1, 6)), t(2, 3, ptr=1 << 30, **ids))),
        (RuntimeError, lambda F: F.cache_reorder_(t(6, 2).requires_grad_(), t(2, 3, ptr=1 << 30, **ids))),
    ]


@pytest.mark.parametrize("i", range(54))
def test_refusals(pkg, i):
    """Refused by shapes alone, before the library is called."""
    from torchjs_amd import _lib

    class Closed:
        def __getattr__(self, name):
            raise AssertionError("%s was called" % name)
    cases = _refusals(lambda *s, **k: _shape_only(pkg, *s, **k))
    assert len(cases) == 54
    error, call = cases[i]
    real, _lib.lib = _lib.lib, lambda: Closed()
    try:
        with pytest.raises(error):
            call(pkg.functional)
    finally:
        _lib.lib = real


@gpu
def test_library_refusals(torch):
    """What the library itself refuses, before any launch."""
    from torchjs_amd import _lib as L
    lib = L.lib()
    st = L.i64arr((1, 1, 1, 1))
    p = torch.zeros(64).data_ptr()
    assert lib.tjh_fp4_quantize(p, 4, 1, 4, 48, p, p) == 1
    assert lib.tjh_fp4_quantize(p, 3, 1, 4, 32, p, p) == 1
    assert lib.tjh_fp4_linear(p, 4, 1, 1, 4, p, p, 16, None, p, 1) == 1
    assert lib.tjh_fp4_linear(p, 4, 1, 1, 4, p + 4, p, 32, None, p, 1) == 1
    assert lib.tjh_fp4_cache_append(p, p, st, st, p, p, p, p, 1, 1, 2, 4, 3, 2, None) == 1
    assert lib.tjh_fp4_cache_append(p, p, st, st, p, p, p, p, 1, 1, 2, 129, 3, 0, None) == 5
    assert lib.tjh_fp4_cache_read(p, p, None, None, 1, 1, 3, 4, 2, 2, p, None) == 1
    assert lib.tjh_fp4_cache_read(p, p, p, None, 1, 1, 3, 4, 0, 2, p, p) == 1
    assert lib.tjh_fp4_attention(p, p, p, p, p, p, 1, 3, 2, 1, 4, 4, st, st, 4, None, 1.0) == 1
    assert lib.tjh_fp4_attention(p, p, p, p, p, p, 1, 2, 2, 1, 4, 4, st, st, 5, None, 1.0) == 1
    assert lib.tjh_fp4_attention(p, p, p, p, p, p, 1, 2, 2, 1, 4, 200, st, st, 4, None, 1.0) == 5
    assert lib.tjh_beam_step(p, 4, p, None, 1, 65, 4, 1, -1, p, p, p, p) == 5
    assert lib.tjh_beam_step(p, 4, p, None, 1, 2, 4, 9, -1, p, p, p, p) == 1
    assert lib.tjh_beam_step(p, 4, p, p, 1, 2, 4, 2, -1, p, p, p, p) == 1
    one = L.i64arr((1,))
    t = (ctypes.c_void_p * 1)(p)
    assert lib.tjh_cache_reorder(1, t, one, one, L.i64arr((2,)), 1, 2, p) == 1
    assert lib.tjh_cache_reorder(1, t, one, one, one, 1, 65, p) == 5
