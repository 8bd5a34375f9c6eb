"""A small GPT-2 with 4-bit weights that decodes over a 4-bit cache and is
searched with beams: the operators of decoding together, as a program uses
them."""
import numpy as np
import pytest

from test_gpu_decode_ops import beam_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24

VOCAB, CTX, D, HEADS, LAYERS = 211, 64, 96, 3, 2


def _model(torch, seed=11, **kw):
    from torchjs_amd import workloads as W
    torch.manual_seed(seed)
    m = W.GPT2(VOCAB, CTX, D, HEADS, LAYERS, **kw)
    with torch.no_grad():  # logits that differ by some units
        for p in (m.ln_f.weight, m.ln_f.bias):
            p.copy_(p + 0.1 * torch.randn(*p.shape))
        m.wte.weight.copy_(m.wte.weight * 0.3)
    return m


def _ids(torch, b, t, seed=0):
    return torch.tensor(np.random.default_rng(seed).integers(0, VOCAB, (b, t)).astype(np.int32))


def _float_copy(torch, four):
    """The same model with float layers of the values that the codes stand for;
    its logits come from `head`."""
    from torchjs_amd import workloads as W
    m = W.GPT2(VOCAB, CTX, D, HEADS, LAYERS)
    state = {n: t.numpy() for n, t in four.state_dict().items()}
    names = dict(m.named_parameters())
    m.load_state_dict({n: v for n, v in state.items() if n in names})
    F = torch.functional
    for a, b in zip(m.h, four.h):
        for x, y in ((a.attn.c_attn, b.attn.c_attn), (a.attn.c_proj, b.attn.c_proj),
                     (a.mlp.c_fc, b.mlp.c_fc), (a.mlp.c_proj, b.mlp.c_proj)):
            w = F.dequantize_fp4(y.codes, y.scales, y.in_features, y.group_size)
            x.load_state_dict({"weight": w, "bias": y.bias.numpy()})
    return m, F.dequantize_fp4(four.head.codes, four.head.scales, D, four.head.group_size)


def _hidden(m, ids):
    x = m._embed(ids, 0)
    for blk in m.h:
        x = blk(x)
    return m.ln_f(x)


@pytest.mark.parametrize("group", [32, 128])
def test_quantized_model(torch, group):
    """Logits, loss and gradients are those of the float model with the values
    that the codes stand for."""
    F = torch.functional
    four = _model(torch).quantize_fp4(group)
    same, head = _float_copy(torch, four)
    ids, targets = _ids(torch, 3, 40), _ids(torch, 3, 40, 1)
    with torch.no_grad():
        got, want = four(ids).numpy(), F.linear(_hidden(same, ids), head).numpy()
    # two float32 paths over sums of up to 4 D terms through two layers, each
    # step of a sum off by at most half a step
    assert np.linalg.norm(got - want) <= 2000 * U * np.linalg.norm(want)
    loss = four.loss(ids, targets)
    loss.backward()
    other = F.cross_entropy(F.linear(_hidden(same, ids), head).view(-1, VOCAB), targets.reshape(-1))
    other.backward()
    assert abs(loss.item() - other.item()) <= 2000 * U * abs(other.item())
    grads = dict(same.named_parameters())
    seen = 0
    for n, p in four.named_parameters():
        if n.endswith("codes") or n.endswith("scales"):
            assert p.grad is None
            continue
        w = grads[n].grad.numpy()
        assert np.linalg.norm(p.grad.numpy() - w) <= 4000 * U * np.linalg.norm(w), n
        seen += 1
    assert seen == 4 + 8 * LAYERS
    # quantized again it stays as it is
    before = four.h[0].attn.c_attn
    assert four.quantize_fp4(group).h[0].attn.c_attn is before


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("held", ["", "c_attn c_proj c_fc mlp", "c_fc", "c_proj"])
@pytest.mark.parametrize("B,T,C,heads", [(1, 1, 64, 2), (2, 37, 96, 3), (7, 20, 160, 2), (8, 300, 256, 4)])
def test_block_is_one_call(torch, monkeypatch, bits, held, B, T, C, heads):
    """Without a gradient a block with layers or a cache in 4 bits is one call,
    with bit for bit the values and the cache of its layers one by one; a layer
    or a cache that a program has replaced takes the layers."""
    from torchjs_amd import workloads as W
    nn = torch.nn
    torch.manual_seed(5)
    blk = W.Block(C, heads)
    for m, name, word in ((blk.attn, "c_attn", "c_attn"), (blk.attn, "c_proj", "c_proj"),
                          (blk.mlp, "c_fc", "c_fc"), (blk.mlp, "c_proj", "mlp")):
        if word in held.split():
            setattr(m, name, nn.LinearFP4.of(getattr(m, name), 32))
    kind = W.KVCacheFP4 if bits == 4 else W.KVCache
    x = torch.tensor(np.random.default_rng(1).standard_normal((B, T, C)).astype(np.float32))
    fast, calls = W.Block._infer, []
    monkeypatch.setattr(W.Block, "_infer", lambda self, *a: calls.append(fast(self, *a)) or calls[-1])

    def run():
        with torch.no_grad():
            cache = kind(1, B, heads, 2 * T + 3, C // heads)
            out = [blk(x), blk.forward_cached(x, cache, 0, 0),
                   blk.forward_cached(x[:, :1].contiguous(), cache, 0, T)]
            if bits == 4:
                out.append(blk.forward_cached(x, cache, 0, T + 1))
            with pytest.raises(RuntimeError):
                blk.forward_cached(x[:, :1].contiguous(), cache, 0, 2 * T + 3)
            return [a.numpy() for a in out + cache._tensors()]
    got = run()
    n = 4 if bits == 4 else 3
    assert all(c is not None for c in calls[:n]) and calls[n] is None
    with monkeypatch.context() as m:
        m.setattr(W.Block, "_infer", lambda self, *a: None)
        want = run()
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    with torch.no_grad():
        cache = kind(1, B, heads, T, C // heads)
        append, seen = cache.append, []
        cache.append = lambda *a: seen.append(a[3]) or append(*a)
        assert np.array_equal(blk.forward_cached(x, cache, 0, 0).numpy(), want[1]) and seen == [0]
        if held:
            blk.attn.c_attn = type("Mine", (type(blk.attn.c_attn),), {}).of(nn.Linear(C, 3 * C)) \
                if "c_attn" in held else type("Mine", (nn.Linear,), {})(C, 3 * C)
            blk(x)
            assert calls[-1] is None


@pytest.mark.parametrize("B,T", [(9, 1), (2, 8), (3, 17)])
def test_block_with_sums_in_slices(torch, monkeypatch, B, T):
    """The same where the MLP's last layer has 8192 columns, whose slices are added
    up before the residual, and replayed in a graph beside another one's workspace."""
    from torchjs_amd import workloads as W
    nn = torch.nn
    torch.manual_seed(6)
    blk = W.Block(2048, 16)
    blk.mlp.c_fc = nn.LinearFP4.of(blk.mlp.c_fc)
    blk.mlp.c_proj = nn.LinearFP4.of(blk.mlp.c_proj)
    x = torch.randn(B, T, 2048)
    graphs, outs = [torch.hip.Graph(), torch.hip.Graph()], []
    with torch.no_grad():
        blk(x)
        for g in graphs:
            with torch.hip.graph(g):
                outs.append(blk(x))
        for i in range(3):
            for g, out in zip(graphs, outs):
                x.copy_(torch.randn(B, T, 2048))
                want = blk(x).numpy()
                g.replay()
                assert np.array_equal(out.numpy(), want)
        x.copy_(torch.tensor(np.random.default_rng(2).standard_normal((B, T, 2048)).astype(np.float32)))
        got = blk(x).numpy()
        with monkeypatch.context() as m:
            m.setattr(W.Block, "_infer", lambda self, *a: None)
            assert np.array_equal(got, blk(x).numpy())
    for g in graphs:
        g.reset()


@pytest.mark.parametrize("parts", [(30,), (1,), (7, 1, 20), (33, 5)])
def test_cached_positions(torch, parts):
    """Each call's logits are those of explicit attention over what the cache
    holds of the positions seen."""
    F = torch.functional
    m = _model(torch)
    ids = _ids(torch, 2, sum(parts) + 4, 3)
    cache = m.new_cache(2, sum(parts) + 4, bits=4)
    hd = D // HEADS
    pos = 0
    with torch.no_grad():
        for n in list(parts) + [1] * 4:
            part = ids[:, pos:pos + n]
            got = m.forward_cached(part, cache, pos).numpy()
            x = m._embed(part, pos)
            mask = np.arange(pos + n)[None, :] <= np.arange(pos, pos + n)[:, None]
            for i, blk in enumerate(m.h):
                q = blk.attn.c_attn(blk.ln_1(x)).split(D, dim=2)[0]
                q = q.view(2, n, HEADS, hd).transpose(1, 2)
                k, v = cache.read(i, 0, pos + n)
                y = F.scaled_dot_product_attention(q, k, v, attn_mask=torch.tensor(mask))
                x = x + blk.attn.c_proj(y.transpose(1, 2).contiguous().view(2, n, D))
                x = x + blk.mlp.c_proj(F.gelu(blk.mlp.c_fc(blk.ln_2(x))))
            want = F.linear(m.ln_f(x), m.wte.weight).numpy()
            # other orders of sums of up to 64 and 4 D terms through two layers
            assert np.abs(got - want).max() <= 2000 * U * np.abs(want).max()
            pos += n


def _search_by_hand(torch, m, ids, count, w, eos, bits):
    """The search with the same calls of the model, everything else in numpy."""
    b, t = ids.shape
    with torch.no_grad():
        prompt = m.new_cache(b, t, bits)
        logits = m.forward_cached(ids, prompt, 0).numpy()[:, -1:, :]
        cache = m.new_cache(b * w, t + count, bits)
        for dst, src in zip(cache._tensors(), prompt._tensors()):
            a = dst.numpy()
            a[:, :, :t] = np.repeat(src.numpy(), w, 0)
            dst.copy_(torch.tensor(a, dtype=dst.dtype))
        scores, done = np.zeros((b, 1), np.float32), None
        seqs = np.zeros((b, 1, 0), np.int64)
        least = np.inf
        for i in range(count):
            best, tokens, parents, done, flat = beam_ref(logits, scores, w, done, eos)
            if eos is None:
                done = None
            order = -np.sort(-flat, 1)[:, :w + 1]
            least = min(least, np.min(-np.diff(order, axis=1)))
            scores = best.astype(np.float32)
            seqs = np.concatenate([np.take_along_axis(seqs, parents[..., None], 1), tokens[..., None]], 2)
            if i == count - 1:
                break
            if i:
                rows = (parents + w * np.arange(b)[:, None]).reshape(-1)
                for x in cache._tensors():
                    x.copy_(torch.tensor(x.numpy()[rows], dtype=x.dtype))
            logits = m.forward_cached(torch.tensor(tokens.reshape(-1, 1).astype(np.int32)), cache,
                                      t + i).numpy().reshape(b, w, -1)
    return seqs[:, 0], least


@pytest.mark.parametrize("bits", [32, 4])
@pytest.mark.parametrize("w", [2, 5])
@pytest.mark.parametrize("quantized", [False, True])
def test_search(torch, bits, w, quantized):
    m = _model(torch, 5)
    if quantized:
        m.quantize_fp4(32)
    ids = _ids(torch, 3, 9, 2)
    got = m.generate(ids, 12, beams=w, cache_bits=bits).numpy()
    assert got.shape == (3, 21) and (got[:, :9] == ids.numpy()).all()
    want, least = _search_by_hand(torch, m, ids, 12, w, None, bits)
    # no two of the scores that decide are as near as float sums of VOCAB terms
    # and scores of this size can be off
    assert least > 100 * U
    assert (got[:, 9:] == want).all()
    # a token that the search has chosen ends it
    eos = int(want[0, 3])
    got = m.generate(ids, 12, beams=w, eos=eos, cache_bits=bits).numpy()[:, 9:]
    want, least = _search_by_hand(torch, m, ids, 12, w, eos, bits)
    assert (got == want).all()
    for row in got:
        at = np.nonzero(row == eos)[0]
        assert not at.size or (row[at[0]:] == eos).all()


def test_search_with_a_window(torch):
    m = _model(torch, 5, window=6, sinks=1)
    ids = _ids(torch, 2, 9, 2)
    got = m.generate(ids, 12, beams=3).numpy()[:, 9:]
    want, least = _search_by_hand(torch, m, ids, 12, 3, None, 32)
    assert least > 100 * U
    assert (got == want).all()


def test_search_is_exhaustive_with_enough_beams(torch):
    """With as many beams as there are continuations the search is exhaustive."""
    from torchjs_amd import workloads as W
    torch.manual_seed(2)
    m = W.GPT2(6, 16, 32, 2, 1)
    ids = torch.tensor(np.array([[1, 2, 3]], np.int32))
    with pytest.raises(ValueError):
        m.generate(ids, 3, beams=36)  # more beams than the first step has tokens
    got = m.generate(ids, 2, beams=6).numpy()[0, 3:]
    every = np.array([[a, b] for a in range(6) for b in range(6)], np.int32)
    seqs = np.concatenate([np.repeat(ids.numpy(), 36, 0), every], 1)
    with torch.no_grad():
        lp = torch.functional.log_softmax(m(torch.tensor(seqs[:, :-1])), -1).numpy().astype(np.float64)
    total = sum(lp[np.arange(36), 2 + i, every[:, i]] for i in range(2))
    assert (got == every[np.argmax(total)]).all()


def test_generate_over_a_cache_in_four_bits(torch):
    m = _model(torch).quantize_fp4()
    ids = _ids(torch, 2, 10)
    a = m.generate(ids, 15, greedy=True, cache_bits=4).numpy()
    b = m.generate(ids, 15, temperature=0, cache_bits=4).numpy()
    assert a.shape == (2, 25) and (a == b).all()
    torch.manual_seed(1)
    c = m.generate(ids, 15, top_k=5, cache_bits=4).numpy()
    assert ((0 <= c) & (c < VOCAB)).all()


def test_generate_refusals(torch):
    from torchjs_amd import workloads as W
    m = _model(torch)
    ids = _ids(torch, 1, 10)
    for kw in (dict(beams=0), dict(beams=65), dict(beams=2, greedy=True), dict(beams=2, top_k=3),
               dict(beams=2, temperature=0.5), dict(eos=3), dict(cache_bits=8), dict(beams=2, eos=VOCAB),
               dict(beams=2, temperature=torch.ones(1))):
        with pytest.raises(ValueError):
            m.generate(ids, 5, **kw)
    with pytest.raises(ValueError):
        m.generate(ids, CTX, beams=2)
    assert (m.generate(ids, 0, beams=2).numpy() == ids.numpy()).all()
    windowed = W.GPT2(VOCAB, CTX, D, HEADS, LAYERS, window=8)
    with pytest.raises(NotImplementedError):
        windowed.generate(ids, 5, cache_bits=4)
