"""Where decoding's operators meet their limits: sums over many thousands of keys,
infinities, values near the ends of floats, scores that differ by less than 64 bits
hold, and what a program may put in the place of a model's parts."""
import numpy as np
import pytest

from test_gpu_decode_ops import U, _new_cache, _shape_only, held

gpu = pytest.mark.gpu


@pytest.fixture
def large(torch):
    """For tests of large tensors: their memory does not stay in the allocator's
    cache, whose blocks others' workspaces would be counted by."""
    yield
    torch.hip.empty_cache()


def _attend_some(q, k, v, scale, picks):
    """Causal attention in 64 bits of the queries (head, number) of q [H, Tq, D] over
    k, v [Hkv, n, D], and each result's sum of weighted magnitudes and largest score."""
    group, tq, n = q.shape[0] // k.shape[0], q.shape[1], k.shape[1]
    out, size, far = [], [], []
    for h, t in picks:
        see = n - tq + t + 1
        s = k[h // group, :see] @ q[h, t].astype(np.float64) * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out.append(p @ v[h // group, :see])
        size.append(p @ np.abs(v[h // group, :see]))
        far.append(np.abs(s).max())
    return np.array(out), np.array(size), np.array(far)


# a wave with 16 rows and all keys; four waves that share them; slices of them
LONG = [(16, 1, 1024, 32768, 32), (16, 1, 1024, 32768, 64), (16, 1, 1024, 32768, 80),
        (16, 1, 1024, 16384, 128), (400, 400, 1, 4096, 32), (400, 400, 1, 4096, 64),
        (400, 400, 1, 4096, 96), (400, 400, 1, 4096, 128), (2, 1, 3, 32768, 64)]


@gpu
@pytest.mark.parametrize("h,hkv,tq,n,d", LONG)
@pytest.mark.parametrize("values", ["even", "positive"])
def test_attention_sums_over_many_keys(torch, large, h, hkv, tq, n, d, values):
    """Values with a mean, whose sums over the keys grow with their number."""
    torch.manual_seed(n + d)
    cache = _new_cache(torch, 1, hkv, n, d)
    k, v = 0.3 * torch.randn(1, hkv, n, d), torch.randn(1, hkv, n, d)
    v = v * 0.01 + 1.0 if values == "even" else v.exp()
    torch.functional.cache_append_fp4(*cache, k, v, 0)
    q = torch.randn(1, h, tq, d)
    y = torch.functional.attention_fp4(q, *cache, n).numpy()[0]
    picks = [(i, t) for i in sorted({0, h // 2, h - 1}) for t in sorted({0, tq // 3, tq - 1})]
    kv = sorted({i * hkv // h for i, _ in picks})
    kh, vh = ({i: held(x[0, i].numpy())[2] for i in kv} for x in (k, v))
    qn, num, den = q.numpy()[0], 0.0, 0.0
    for i, t in picks:
        j = i * hkv // h
        want, _, _ = _attend_some(qn[i:i + 1], kh[j][None], vh[j][None], np.float32(d ** -0.5), [(0, t)])
        num += ((y[i, t] - want[0]) ** 2).sum()
        den += (want[0] ** 2).sum()
    # A sum of 16 tiles takes 48 instructions, each of which cuts off half a step (of
    # 2 U) on average of a sum that grows to the whole: 24 U.  The float additions
    # (of c tiles' sums, and of 128 weights before) round to either side: U / sqrt(3)
    # of a growing sum each, three standard deviations of both sums together.
    c = n / 512
    tol = (24 + 3 / 3 ** 0.5 * (2 * (c / 3) ** 0.5 + (128 / 3) ** 0.5)) * U
    assert np.sqrt(num / den) <= tol


@gpu
@pytest.mark.parametrize("h,hkv,tq,n,d", LONG[1:4] + LONG[5:])
@pytest.mark.parametrize("slope", [6, -6])
def test_attention_with_maxima_that_move_over_many_keys(torch, large, h, hkv, tq, n, d, slope):
    """Scores that rise along the keys raise the maxima of sums already put aside;
    falling ones leave them."""
    rng = np.random.default_rng(n + d)
    u = rng.standard_normal(d)
    k = (np.linspace(-slope, slope, n)[:, None] * u + 0.1 * rng.standard_normal((n, d))).astype(np.float32)
    v = rng.standard_normal((n, d)).astype(np.float32)
    q = (u / d * rng.uniform(1, 3, (h, tq, 1)) + 0.1 / d * rng.standard_normal((h, tq, d))).astype(np.float32)
    cache = _new_cache(torch, 1, hkv, n, d)
    tk, tv = (torch.tensor(np.broadcast_to(x, (1, hkv, n, d)).copy()) for x in (k, v))
    torch.functional.cache_append_fp4(*cache, tk, tv, 0)
    y = torch.functional.attention_fp4(torch.tensor(q[None]), *cache, n, scale=2.0).numpy()[0]
    kk, vv = held(k)[2][None], held(v)[2][None]
    for i in sorted({0, h // 2, h - 1}):
        for t in sorted({0, tq // 3, tq - 1}):
            want, size, far = _attend_some(q[i:i + 1], kk, vv, 2.0, [(0, t)])
            s = np.abs(kk[0]) @ np.abs(q[i, t].astype(np.float64)) * 2.0
            # a score's roundings, of its products and of its distance from the
            # maximum; the sums as above, no value's part off by more
            off = ((d + 4) * s.max() + 4 * far[0]) * U
            assert (np.abs(y[i, t] - want[0]) <= (2 * off + 2 * (48 + n / 512 + 128) * U) * size[0]).all()


@gpu
@pytest.mark.parametrize("b,h,hkv,tq,n,d", [
    (1, 1, 1, 1, 3, 1), (2, 3, 3, 5, 40, 64), (2, 4, 2, 1, 1500, 80), (1, 2, 2, 40, 1100, 32),
    (2, 16, 16, 512, 530, 32), (32, 16, 16, 17, 30, 128)])
def test_attention_of_infinite_queries(torch, b, h, hkv, tq, n, d):
    """Where all scores that a query sees are -infinity, or one is +infinity, there is
    no distribution: NaN.  A query that sees no key gives zeros all the same, and the
    other queries are what they are without it."""
    rng = np.random.default_rng(n)
    cache = _new_cache(torch, b, hkv, n, d)
    k, v = rng.standard_normal((2, b, hkv, n, d)).astype(np.float32)
    k[..., 0] = -1 - np.abs(k[..., 0])  # not held as zeros, beside values of up to some units
    assert (held(k)[2][..., 0] < 0).all()
    torch.functional.cache_append_fp4(*cache, torch.tensor(k), torch.tensor(v), 0)
    lengths = np.full(b, n, np.int32)
    lengths[b - 1] = n if b == 1 else tq // 2  # some queries there see nothing
    q = rng.standard_normal((b, h, tq, d)).astype(np.float32)
    plain = torch.functional.attention_fp4(torch.tensor(q), *cache, torch.tensor(lengths, dtype="int32")).numpy()
    assert not np.isnan(plain).any()
    sees = (lengths[:, None] - tq + np.arange(tq) >= 0)[:, None, :]
    for sign in (1, -1):
        odd = rng.random((b, h, tq)) < 0.5
        odd[0, 0, 0] = True
        q2 = q.copy()
        q2[..., 0] = np.where(odd, sign * np.float32(np.inf), q[..., 0])
        y = torch.functional.attention_fp4(torch.tensor(q2), *cache,
                                           torch.tensor(lengths, dtype="int32")).numpy()
        assert np.isnan(y[odd & sees]).all()
        assert (y[odd & ~sees] == 0).all()
        assert np.array_equal(y[~odd], plain[~odd])


@gpu
@pytest.mark.parametrize("far", [2.0 ** 94, 2.0 ** -99])
@pytest.mark.parametrize("n,tq", [(2 ** 24 - 1, 1), (32768, 1), (2000, 1), (4096, 20000)])
def test_attention_of_the_largest_and_smallest_values(torch, large, n, tq, far):
    """Values just inside the range, of one sign, over the longest cache: in every
    part of the keys the first tiles' scores are as far below the rest as leaves the
    running maximum where it is, so that weights are as large as they can be."""
    d = 32
    cache = _new_cache(torch, 1, 1, n, d)
    scale = np.float32(far * (1 - 2.0 ** -20) / 6)
    cache[0].fill_(0x22)  # every column 1
    cache[2].fill_(0x77)  # every column 6
    cache[3].fill_(float(scale))
    # scores of 9.75 in powers of two, but 0 at the start of each run of 512 keys
    # (slices are longer than that, and a wave's tiles 32 keys)
    k_scales = np.full(n + 512, 9.75 / 32 * np.log(2), np.float32)
    k_scales.reshape(-1)[:(n + 511) // 512 * 512].reshape(-1, 512)[::1 if tq > 1 else 8, :128] = 0
    cache[1].copy_(torch.tensor(k_scales[:n].reshape(1, 1, n)))
    q = torch.ones(1, 1, tq, d)
    y = torch.functional.attention_fp4(q, *cache, torch.tensor(np.full(1, n, np.int32), dtype="int32")
                                       if tq > n else n, scale=1.0).numpy()[0, 0]
    want = 6 * float(scale)
    assert np.isfinite(y).all()
    # equal values, so no error of a weight counts: cut-offs and float sums of 16
    # tiles, of up to 16 of those, and of up to 512 slices, numerator and denominator
    tol = 2 * (48 + 128 + 16 + 512) * U * want
    sees = np.arange(tq) - tq + n >= 0
    assert (np.abs(y[sees] - want) <= tol).all() and (y[~sees] == 0).all()


@gpu
@pytest.mark.parametrize("b,w,n", [(1, 1, 2), (1, 1, 3), (2, 3, 9), (1, 4, 2500), (40, 8, 1300),
                                   (2, 16, 50257), (1, 64, 5000)])
@pytest.mark.parametrize("levels", [5, 1000])
def test_beam_step_of_logits_nearer_than_a_score(torch, b, w, n, levels):
    """Logits that differ by less than the last bit of a 64-bit score: equal scores, by
    beam, then by logit, then by token; fewer beams are the first of more."""
    rng = np.random.default_rng(n)
    x = (np.float32(1e-20) * (rng.integers(0, levels, (b, w, n)) - levels // 2)).astype(np.float32)
    x[:, :, 1:n // 2:1 + n // 3] = rng.choice(np.float32([-2, 0, 1]), x[:, :, 1:n // 2:1 + n // 3].shape)
    x[:] = x[:, :1]  # equal rows: beams that tie
    scores = np.full((b, w), -2.0, np.float32)
    size = x + np.float32(1) - np.float32(1)  # as scores tell logits apart
    flat = [a.reshape(b, -1) for a in
            np.broadcast_arrays(-size, np.arange(w)[None, :, None], -x, np.arange(n)[None, None, :])]
    most = min(64, w * n)
    got = [a.numpy() for a in torch.functional.beam_step(torch.tensor(x), torch.tensor(scores), most)]
    for i in range(b):
        order = np.lexsort([a[i] for a in flat[::-1]])[:most]
        assert (got[1][i] == order % n).all() and (got[2][i] == order // n).all()
    for keep in sorted({1, 2, 5, w} & set(range(most))):
        few = torch.functional.beam_step(torch.tensor(x), torch.tensor(scores), keep)
        for a, c in zip(few, got):
            assert np.array_equal(a.numpy(), c[:, :keep])


# ------------------------------------------------- what a program puts in place


class _Closed:
    """The library where nothing is to be called."""

    def __getattr__(self, name):
        raise AssertionError("%s was called" % name)


@pytest.mark.parametrize("value,error", [
    (np.full((6, 64), 3.7, np.float32), TypeError), (np.full((6, 64), 3.0), TypeError),
    (np.full((6, 64), 256), ValueError), (np.full((6, 64), -1), ValueError),
    (np.full((6, 64), "a"), TypeError), ("float32", TypeError), ("int32", TypeError)])
def test_codes_of_another_type_are_not_converted(pkg, monkeypatch, value, error):
    from torchjs_amd import _lib
    m = pkg.nn.Module()
    m.register_parameter("codes", _shape_only(pkg, 6, 64, dtype="uint8"))
    if isinstance(value, str):
        value = _shape_only(pkg, 6, 64, dtype=value, ptr=8192)
    monkeypatch.setattr(_lib, "lib", _Closed)
    with pytest.raises(error):
        m.load_state_dict({"codes": value})


@gpu
def test_states_of_other_types(torch):
    """Whole numbers that a type holds, and any numbers for floats."""
    m = torch.nn.LinearFP4(70, 6, group_size=32)
    codes = np.random.default_rng(0).integers(0, 256, (6, 64))
    m.load_state_dict({"codes": codes, "scales": np.arange(24).reshape(6, 4), "bias": [1, 2, 3, 4, 5, 6]})
    assert (m.codes.numpy() == codes).all() and m.codes.dtype == "uint8"
    assert (m.scales.numpy() == np.arange(24).reshape(6, 4)).all() and m.scales.dtype == "float32"
    assert m.bias.numpy().tolist() == [1, 2, 3, 4, 5, 6]
    m.load_state_dict({"bias": torch.tensor(np.arange(6, dtype=np.int32)),
                       "scales": np.full((6, 4), 0.1)})
    assert m.bias.numpy().tolist() == list(range(6)) and (m.scales.numpy() == np.float32(0.1)).all()
    with pytest.raises(ValueError):
        m.load_state_dict({"codes": codes[:, :32]})


@gpu
def test_a_subclass_of_linear_keeps_the_fused_layers(torch, monkeypatch):
    """One that changes nothing takes the products with the GELU and the residual
    in them, forward and backward; one with a forward of its own is called."""
    from torchjs_amd import workloads as W
    F, nn = torch.functional, torch.nn
    mine = type("Mine", (nn.Linear,), {})
    twice = type("Twice", (nn.Linear,), {"forward": lambda self, x: nn.Linear.forward(self, x) * 2.0})
    x = np.random.default_rng(0).standard_normal((2, 9, 64)).astype(np.float32)
    seen = []
    for name in ("_linear_add", "_mlp_gelu"):
        real = getattr(F, name)
        monkeypatch.setattr(F, name, lambda *a, real=real, name=name: seen.append(name) or real(*a))

    def run(kind):
        torch.manual_seed(1)
        blk = W.Block(64, 2)
        if kind is not None:
            for m, part in ((blk.attn, "c_proj"), (blk.mlp, "c_fc"), (blk.mlp, "c_proj")):
                old = getattr(m, part)
                new = kind(old.in_features, old.out_features)
                new.load_state_dict(old.state_dict())
                setattr(m, part, new)
        del seen[:]
        t = torch.tensor(x, requires_grad=True)
        y = blk(t)
        (y * y).sum().backward()
        return [y.numpy(), t.grad.numpy()] + [p.grad.numpy() for p in blk.parameters()], list(seen)
    want, calls = run(None)
    assert calls == ["_linear_add", "_mlp_gelu"]
    got, same = run(mine)
    assert same == calls and all(np.array_equal(a, b) for a, b in zip(got, want))
    got, none = run(twice)
    assert none == [] and not np.array_equal(got[0], want[0])


@gpu
def test_quantized_model_with_subclasses_of_linear(torch):
    """One that changes nothing is held in 4 bits as nn.Linear is, one with a forward
    of its own stays."""
    from torchjs_amd import workloads as W
    nn = torch.nn
    mine = type("Mine", (nn.Linear,), {})
    twice = type("Twice", (nn.Linear,), {"forward": lambda self, x: nn.Linear.forward(self, x) * 2.0})
    m = W.GPT2(50, 8, 64, 2, 1)
    m.h[0].attn.c_attn, m.h[0].mlp.c_fc = mine(64, 192), twice(64, 256)
    want = m.h[0].attn.c_attn.weight.numpy()
    m.quantize_fp4(32)
    four = m.h[0].attn.c_attn
    assert type(four) is nn.LinearFP4 and type(m.h[0].mlp.c_fc) is twice
    got = torch.functional.dequantize_fp4(four.codes, four.scales, 64, 32).numpy()
    assert (got == held(want.reshape(192, 2, 32))[2].reshape(192, 64).astype(np.float32)).all()
    assert m(torch.tensor(np.zeros((1, 8), np.int32))).shape == (1, 8, 50)


def test_a_window_and_a_cache_in_four_bits(pkg, monkeypatch):
    """Refused before the library is called, wherever the two meet."""
    from torchjs_amd import _lib, workloads as W

    def make(kind, **kw):
        m = kind.__new__(kind)
        pkg.nn.Module.__init__(m)
        for name, value in kw.items():
            setattr(m, name, value)
        return m
    attn = make(W.CausalSelfAttention, window=8, sinks=0, d=64, heads=2, fused=True)
    blk = make(W.Block, attn=attn)
    model = make(W.GPT2, h=[make(W.Block, attn=make(W.CausalSelfAttention, window=None, d=64, heads=2)), blk],
                 ctx=16, vocab=50)
    cache = W.KVCacheFP4.__new__(W.KVCacheFP4)
    x, ids = _shape_only(pkg, 1, 4, 64), _shape_only(pkg, 1, 4, dtype="int32")
    monkeypatch.setattr(_lib, "lib", _Closed)
    for call in (lambda: model.new_cache(1, bits=4), lambda: model.forward_cached(ids, cache, 0),
                 lambda: blk.forward_cached(x, cache, 0, 0), lambda: attn.forward_cached(x, cache, 0, 0),
                 lambda: model.generate(ids, 3, cache_bits=4),
                 lambda: model.generate(ids, 3, beams=2, cache_bits=4)):
        with pytest.raises(NotImplementedError):
            call()


@gpu
def test_models_with_a_head_of_their_own(torch):
    """A subclass's `head`, a layer or a method, has no part in the model's logits, and
    it keeps it when its layers are held in 4 bits."""
    from torchjs_amd import workloads as W

    class Own(W.GPT2):
        def __init__(self, *a):
            super().__init__(*a)
            self.head = torch.nn.Linear(64, 3)

    class Method(W.GPT2):
        def head(self, ids):
            return 7

    def make(kind):
        torch.manual_seed(4)
        return kind(50, 16, 64, 2, 1)
    plain, own, method = make(W.GPT2), make(Own), make(Method)
    ids = torch.tensor(np.arange(8, dtype=np.int32).reshape(2, 4))
    assert method.head(ids) == 7
    for m in (own, method):
        assert np.array_equal(m(ids).numpy(), plain(ids).numpy())
        for kw in (dict(greedy=True), dict(beams=2)):
            assert np.array_equal(m.generate(ids, 5, **kw).numpy(), plain.generate(ids, 5, **kw).numpy())
        before = m.h[0].attn.c_attn
        with pytest.raises(ValueError):
            m.quantize_fp4()
        assert m.h[0].attn.c_attn is before
        m.quantize_fp4(head=False)
        assert np.array_equal(m(ids).numpy(), make(W.GPT2).quantize_fp4(head=False)(ids).numpy())
    assert type(own.head) is torch.nn.Linear and plain.head is None
    assert type(plain.quantize_fp4().quantize_fp4().head) is torch.nn.LinearFP4


@gpu
def test_a_model_with_caches_of_its_own(torch):
    """A new_cache that knows of no bits, as models had before there were any."""
    from torchjs_amd import workloads as W

    class Own(W.GPT2):
        def new_cache(self, batch, max_len=None):
            return W.KVCache(len(self.h), batch, 2, max_len, 32)

    def make(kind):
        torch.manual_seed(4)
        return kind(50, 16, 64, 2, 1)
    plain, own = make(W.GPT2), make(Own)
    ids = torch.tensor(np.arange(8, dtype=np.int32).reshape(2, 4))
    for kw in (dict(greedy=True), dict(top_k=1), dict(beams=2)):
        assert np.array_equal(own.generate(ids, 5, **kw).numpy(), plain.generate(ids, 5, **kw).numpy())
