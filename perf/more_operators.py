"""Operators of decoding in four bits and with beams: products with 4-bit
weights, a key / value cache held in 4 bits with the attention that reads it, a
beam search's step, and the reordering of its caches.

Each has a plain form in elementary torch operations and, with `own`, the call
that a user of the 'hip' device makes.  Values are float32; four bits stand for
0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, times a float32 scale: the
largest magnitude of the values that share it over 6.  `listed()` holds fixed
sizes, `draw()` others of the same ranges."""
import math

import torch

own = False

VOCAB = 50257  # GPT-2's
STEPS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # one token through GPT-2 small's query, key and value projection
        dict(name="linear 1x768x2304", kind="linear", rows=1, cols=768, out=2304, group=64, bias=True),
        # the logits of four sequences' (or beams') next tokens
        dict(name="linear 4x768x50257", kind="linear", rows=4, cols=768, out=VOCAB, group=32, bias=False),
        # a prompt of an odd length through a wide layer
        dict(name="linear 2047x1600x6400", kind="linear", rows=2047, cols=1600, out=6400, group=64,
             bias=True),
        # one decoding step of four sequences of GPT-2 small's heads
        dict(name="attend 4x12, 1 of 1000", kind="attend", batch=4, heads=12, kv_heads=12, q=1, k=1000,
             dim=64, ragged=False),
        # one step of many sequences of different lengths, four query heads
        # to one of the cache
        dict(name="attend 32x32, 1 of 8192", kind="attend", batch=32, heads=32, kv_heads=8, q=1, k=8192,
             dim=128, ragged=True),
        # the next part of one prompt over a cache, an odd length and head size
        dict(name="attend 1x16, 1999 of 4095", kind="attend", batch=1, heads=16, kv_heads=4, q=1999,
             k=4095, dim=80, ragged=False),
        # the keys and values of one new token of many sequences
        dict(name="append 64x8, 1 at 1000", kind="append", batch=64, heads=8, t=1, pos=1000, dim=128),
        # and those of eight whole prompts of GPT-2 small's
        dict(name="append 8x12, 1024 at 0", kind="append", batch=8, heads=12, t=1024, pos=0, dim=64),
        # one search with four beams
        dict(name="beams 1x4x50257", kind="beam", batch=1, beams=4, vocab=VOCAB, keep=4, done=False),
        # many searches with eight, some of whose beams have ended
        dict(name="beams 32x8x50257", kind="beam", batch=32, beams=8, vocab=VOCAB, keep=8, done=True),
        # GPT-2 small's float caches of one search after 700 tokens
        dict(name="reorder 1x4, 700, float", kind="reorder", batch=1, beams=4, layers=12, heads=12,
             pos=700, length=1024, dim=64, four=False),
        # some layers' 4-bit caches of many searches over long prompts
        dict(name="reorder 16x4, 4000, 4 bits", kind="reorder", batch=16, beams=4, layers=4, heads=8,
             pos=4000, length=4096, dim=128, four=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "attend", "attend", "append", "beam", "reorder"])
    if kind == "linear":
        rows = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 64), _log(rng, 64, 4096)])
        cols = rng.choice([_log(rng, 96, 8192), 32 * _log(rng, 3, 256)])
        most = 2047 * 1600 * 6400 // (rows * cols)  # the largest listed case's products
        out = _log(rng, 100, max(101, min(65536, most, 2 ** 26 // cols)))
        return dict(kind=kind, rows=rows, cols=cols, out=out, group=rng.choice([32, 64, 128]),
                    bias=rng.random() < 0.5)
    if kind == "attend":
        kv = rng.randint(1, 12)
        heads = kv * rng.choice([1, 1, 2, 4, 8])
        one = rng.random() < 0.5
        k = _log(rng, 17, 32768 if one else 4096)
        q = 1 if one else rng.choice([min(k, _log(rng, 2, 16)), min(k, _log(rng, 16, 1024)), k])
        # no more scores and no more keys than the largest listed cases have
        batch = rng.randint(1, max(1, min(32, 16 * 1999 * 4095 // (heads * q * k), 32 * 8 * 8192 // (kv * k))))
        return dict(kind=kind, batch=batch, heads=heads, kv_heads=kv, q=q, k=k,
                    dim=rng.choice([32, 40, 64, 64, 80, 96, 128, 128]), ragged=rng.random() < 0.3)
    if kind == "append":
        t = rng.choice([1, _log(rng, 2, 2048)])
        heads = rng.randint(1, 16)
        return dict(kind=kind, batch=rng.randint(1, max(1, min(64, 8 * 12 * 1024 // (heads * t)))),
                    heads=heads, t=t, pos=rng.choice([0, _log(rng, 1, 2000)]),
                    dim=rng.choice([32, 40, 64, 80, 96]) if t > 1 else rng.choice([64, 80, 128]))
    if kind == "beam":
        beams, vocab = rng.randint(2, 16), _log(rng, 200, 131072)
        return dict(kind=kind, batch=_log(rng, 1, max(2, min(64, 32 * 8 * VOCAB // (beams * vocab)))),
                    beams=beams, vocab=vocab, keep=rng.choice([beams, beams, 2 * beams, rng.randint(1, 16)]),
                    done=rng.random() < 0.5)
    four = rng.random() < 0.5
    length, beams = _log(rng, 64, 4096), rng.choice([2, 4, 5, 6, 8])
    layers, heads = rng.randint(1, 4), rng.randint(1, 8)
    dim = rng.choice([32, 64, 80, 128]) if four else 64
    most = 16 * 4 * 4 * 8 * 4000 * 68 // (beams * layers * heads * length * (68 if four else 256))
    return dict(kind=kind, batch=_log(rng, 1, max(1, min(16, most))), beams=beams, layers=layers, heads=heads,
                pos=_log(rng, 1, length), length=length, dim=dim, four=four)


# --------------------------------------------------------------------- inputs


def _held(x):
    """What x [..., n] is held as: codes [..., n] (sign, then the step's number)
    and scales [...].  Borders are compared in 64 bits, where they are exact."""
    top = x.abs().amax(-1)
    # a quotient of tensors: one by a number would be a product with its inverse
    scale = torch.where(top < 2.0 ** -100, torch.zeros_like(top), top / torch.full_like(top, 6.0))
    s = scale.double().unsqueeze(-1)
    a = x.double().abs()
    code = torch.zeros(x.shape, dtype=torch.uint8, device=x.device)
    for i, mid in enumerate([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]):
        # halfway goes to the even step
        code += (a > mid * s) if i % 2 == 0 else (a >= mid * s)
    code = torch.where(s > 0, code, torch.zeros_like(code))
    return code + 8 * (x < 0).to(torch.uint8), scale


def _packed(code):
    """Two codes a byte, the first one in the low half."""
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _lengths(c):
    """Keys of each sequence; from half of the most on where they differ."""
    return [c["k"] - (b * (c["k"] - max(c["q"], c["k"] // 2)) // c["batch"] if c["ragged"] else 0)
            for b in range(c["batch"])]


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    def keys(b, h, t, d):  # some channels of a trained model's keys are larger than the rest
        return randn(b, h, t, d) * torch.exp(randn(1, h, 1, d, std=0.5))

    kind = c["kind"]
    if kind == "linear":
        x = {"x": randn(c["rows"], c["cols"]), "w": randn(c["out"], c["cols"], std=c["cols"] ** -0.5)}
        if c["bias"]:
            x["bias"] = randn(c["out"], std=0.1)
        return x
    if kind == "attend":
        b, kv, d = c["batch"], c["kv_heads"], c["dim"]
        x = {"q": randn(b, c["heads"], c["q"], d)}
        for n in "kv":
            held = []
            for _ in range(b):  # one sequence at a time: 64-bit copies of all would be large
                code, scale = _held(keys(1, kv, c["k"], d) if n == "k" else randn(1, kv, c["k"], d))
                held.append((_packed(code), scale))
            x[n], x[n + "_scale"] = (torch.cat(t) for t in zip(*held))
        if c["ragged"]:
            x["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
        return x
    if kind == "append":
        shape = (c["batch"], c["heads"], c["t"], c["dim"])
        return {"k": keys(*shape), "v": randn(*shape)}
    if kind == "beam":
        b, w, n = c["batch"], c["beams"], c["vocab"]
        # sums of the logarithms of some tokens, the best beam first
        x = {"x": randn(b, w, n, std=2.5), "scores": -torch.sort(randn(b, w).abs() * 3 + 10, dim=1)[0]}
        if c["done"]:
            x["done"] = torch.rand((b, w), generator=g, device="cuda") < 0.2
        return x
    b, w = c["batch"], c["beams"]
    # half of the beams stay in their places, the others become copies of
    # them: what a step is about to do, and the same however often it is done
    order = torch.argsort(torch.rand((b, w), generator=g, device="cuda"), dim=1)
    stay = (w + 1) // 2
    parents = torch.arange(w, device="cuda").repeat(b, 1)
    parents.scatter_(1, order[:, stay:], order[:, :w - stay])
    x = {"parents": parents.to(torch.int32)}
    shape = (b * w, c["heads"], c["length"])
    for i in range(c["layers"]):
        for n in "kv":
            name = "%s%d" % (n, i)
            if c["four"]:
                x[name] = torch.randint(0, 256, shape + (-(-c["dim"] // 32) * 16,), generator=g,
                                        device="cuda", dtype=torch.uint8)
                x[name + "_scale"] = randn(*shape).abs()
            else:
                x[name] = randn(*shape, c["dim"])
    return x


class _Array:
    """A library tensor's memory for torch.as_tensor, which keeps this object
    (and with it the memory) as long as the torch tensor lives."""

    def __init__(self, t):
        kind, size = {"float32": ("<f4", 4), "int32": ("<i4", 4), "uint8": ("|u1", 1),
                      "bool": ("|b1", 1)}[t.dtype]
        self.tensor = t
        self.__cuda_array_interface__ = {
            "shape": t.shape, "strides": tuple(size * s for s in t.stride()), "typestr": kind,
            "data": (t.data_ptr(), False), "version": 2}


def _view(t):
    return torch.as_tensor(_Array(t.detach()), device="cuda")


def _hip():
    import __graft_entry__ as graft
    return graft.load_package()


def _tensor(hip, x):
    """The same values in a tensor of the library."""
    kinds = {torch.float32: "float32", torch.int32: "int32", torch.uint8: "uint8", torch.bool: "bool"}
    t = hip.empty(tuple(x.shape), dtype=kinds[x.dtype])
    _view(t).copy_(x)
    return t


def prepare(case, seed):
    s = dict(case, **_inputs(case, seed))
    kind = case["kind"]
    if not own:
        if kind == "linear":
            # columns past the last group's end add nothing
            w = s.pop("w")
            w = torch.nn.functional.pad(w, (0, -case["cols"] % case["group"]))
            code, s["w_scale"] = _held(w.view(case["out"], -1, case["group"]))
            s["w"] = _packed(code)
        if kind == "append":
            _empty_cache(s)
        return s
    # the same values in tensors of the library, which has an allocator of its
    # own: a user's program holds them there from the start
    hip = s["hip"] = _hip()
    hip.init(0)
    F = hip.functional
    for name, x in s.items():
        if isinstance(x, torch.Tensor):
            if kind == "attend" and name in "kv":  # a row of the cache has whole groups of 32
                x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 16))
            s[name] = _tensor(hip, x)
    torch.cuda.synchronize()
    if kind == "linear":
        s["codes"], s["w_scale"] = F.quantize_fp4(s.pop("w"), case["group"])
    if kind == "append":
        from torchjs_amd import workloads
        s["cache"] = workloads.KVCacheFP4(1, case["batch"], case["heads"], case["pos"] + case["t"],
                                          case["dim"])
    if kind == "reorder":
        s["caches"] = [s[n] for n in s if n[0] in "kv" and n[1:2].isdigit()]
    hip.synchronize()
    return s


def _empty_cache(s):
    shape = (s["batch"], s["heads"], s["pos"] + s["t"])
    for n in "kv":
        s[n + "_codes"] = torch.zeros(shape + (s["dim"] // 2,), dtype=torch.uint8, device="cuda")
        s[n + "_scale"] = torch.zeros(shape, device="cuda")


# ----------------------------------------------------------------- one pass


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    hip, kind = s["hip"], s["kind"]
    F = hip.functional
    with hip.no_grad():
        if kind == "linear":
            bias = s["bias"] if s["bias"] is not False else None
            return _view(F.linear_fp4(s["x"], s["codes"], s["w_scale"], bias, s["group"]))
        if kind == "attend":
            return _view(F.attention_fp4(s["q"], s["k"], s["k_scale"], s["v"], s["v_scale"],
                                         s["lengths"] if s["ragged"] else s["k"].shape[2]))
        if kind == "append":
            # the new tokens' keys and values go in, and what is held of them comes back
            cache, pos, end = s["cache"], s["pos"], s["pos"] + s["t"]
            cache.append(0, s["k"], s["v"], pos)
            k, v = cache.read(0, pos, end)
            return {"k": _view(k), "v": _view(v)}
        if kind == "beam":
            done, last = (s["done"], s["vocab"] - 1) if s["done"] is not False else (None, None)
            scores, tokens, parents, done = F.beam_step(s["x"], s["scores"], s["keep"], done, last)
            return {"scores": _view(scores), "tokens": _view(tokens), "parents": _view(parents),
                    "done": _view(done)}
        F.cache_reorder_(s["caches"], s["parents"], s["pos"])
        return [_view(t) for t in s["caches"]]


def _run_plain(s):
    return {"linear": _linear, "attend": _attend, "append": _append, "beam": _beam,
            "reorder": _reorder}[s["kind"]](s)


def _values(packed, scale):
    """What packed codes [..., n / 2] with scales [...] stand for."""
    table = torch.tensor(STEPS + [-v for v in STEPS], device="cuda")
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    return table[code.int()] * scale.unsqueeze(-1)


def _linear(s):
    w = _values(s["w"], s["w_scale"]).view(s["out"], -1)[:, :s["cols"]].contiguous()
    y = torch.matmul(s["x"], w.t())
    return y + s["bias"] if s["bias"] is not False else y


def _attend(s):
    q, k, v = s["q"], _values(s["k"], s["k_scale"]), _values(s["v"], s["v_scale"])
    (b, h, tq, d), (kv, tk) = q.shape, k.shape[1:3]
    ends = s["lengths"] if s["ragged"] else torch.full((b,), tk, device="cuda")
    i = ends.view(b, 1, 1) - tq + torch.arange(tq, device="cuda").view(1, tq, 1)
    unseen = (torch.arange(tk, device="cuda") > i).view(b, 1, 1, tq, tk)
    qs = q.reshape(b, kv, h // kv * tq, d)  # the heads that share a key, one after the other
    p = torch.matmul(qs, k.transpose(-1, -2).contiguous()).view(b, kv, h // kv, tq, tk)
    p *= 1.0 / math.sqrt(d)
    p.masked_fill_(unseen, -math.inf)
    p -= p.amax(-1, keepdim=True)
    p = torch.exp_(p)
    p /= p.sum(-1, keepdim=True)
    return torch.matmul(p.view(b, kv, h // kv * tq, tk), v).view(q.shape)


def _append(s):
    out, pos, end = {}, s["pos"], s["pos"] + s["t"]
    for n in "kv":
        code, scale = _held(s[n])
        s[n + "_codes"][:, :, pos:end] = _packed(code)
        s[n + "_scale"][:, :, pos:end] = scale
        out[n] = _values(s[n + "_codes"][:, :, pos:end], s[n + "_scale"][:, :, pos:end])
    return out


def _beam(s):
    x = s["x"].double()
    b, w, n = x.shape
    x = x - x.amax(-1, keepdim=True)
    c = s["scores"].double().unsqueeze(-1) + (x - torch.log(torch.exp(x).sum(-1, keepdim=True)))
    done = s["done"] if isinstance(s["done"], torch.Tensor) else None
    if done is not None:
        # an ended beam goes on as it is, by the last token
        c.masked_fill_(done.unsqueeze(-1), -math.inf)
        c[:, :, n - 1] = torch.where(done, s["scores"].double(), c[:, :, n - 1])
    best, at = torch.sort(c.view(b, w * n), dim=1, descending=True, stable=True)
    best, at = best[:, :s["keep"]], at[:, :s["keep"]]
    tokens, parents = at % n, at // n
    none = best == -math.inf  # fewer continuations than asked for
    ended = none
    if done is not None:
        ended = none | torch.gather(done, 1, parents) | (tokens == n - 1)
    slots = torch.arange(s["keep"], device="cuda").clamp(max=w - 1)
    tokens, parents = torch.where(none, -1, tokens), torch.where(none, slots, parents)
    return {"scores": best.float(), "tokens": tokens.to(torch.int32), "parents": parents.to(torch.int32),
            "done": ended}


def _reorder(s):
    b, w = s["batch"], s["beams"]
    rows = (s["parents"].long() + w * torch.arange(b, device="cuda").unsqueeze(1)).flatten()
    out = []
    for name, t in s.items():
        if name[0] in "kv" and name[1:2].isdigit():
            t[:, :, :s["pos"]] = t[:, :, :s["pos"]][rows]
            out.append(t)
    return out


# ---------------------------------------------------------------- what it is


def work(c):
    kind = c["kind"]
    if kind == "linear":
        m, k, n = c["rows"], c["cols"], c["out"]
        held = n * (k / 2 + 4 * -(-k // c["group"]))
        return {"bytes": int(held) + 4 * (m * k + m * n + (n if c["bias"] else 0)), "flops": 2 * m * n * k}
    if kind == "attend":
        d, q = c["dim"], c["q"]
        keys = sum(_lengths(c))
        pairs = sum(n * q - q * (q - 1) // 2 for n in _lengths(c))
        return {"bytes": 2 * c["kv_heads"] * keys * (d // 2 + 4) + 8 * c["batch"] * c["heads"] * q * d,
                "flops": 4 * c["heads"] * pairs * d}
    if kind == "append":
        rows = 2 * c["batch"] * c["heads"] * c["t"]
        # read, held, and given back
        return {"bytes": rows * (8 * c["dim"] + c["dim"] // 2 + 4), "flops": 8 * rows * c["dim"]}
    if kind == "beam":
        b, w = c["batch"], c["beams"]
        return {"bytes": 4 * b * w * (c["vocab"] + 1) + 13 * b * c["keep"], "flops": 4 * b * w * c["vocab"]}
    moved = c["beams"] // 2
    row = (-(-c["dim"] // 32) * 16 + 4) if c["four"] else 4 * c["dim"]
    size = 2 * c["layers"] * c["heads"] * c["pos"] * row * c["batch"]
    # a beam that is copied is read once, its copy written once
    return {"bytes": 2 * size * moved + 4 * c["batch"] * c["beams"], "flops": size * moved // 4}


# -------------------------------------------------------- the same in 64 bits


def _number(code):
    """A code's value: one sign bit, two of an exponent, one of a fraction."""
    c = code.long()
    e, f = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e == 0, f / 2, torch.ldexp(1 + f / 2, (e - 1).double()))
    return torch.where(c >= 8, -v, v)


def _unpacked(packed):
    out = torch.empty(packed.shape[:-1] + (2 * packed.shape[-1],), dtype=torch.uint8, device="cuda")
    out[..., 0::2], out[..., 1::2] = packed % 16, packed // 16
    return out


def _nearest(x):
    """x [..., n] as it is held, by distances: of two steps that are as near the
    even one."""
    top = x.abs().amax(-1, keepdim=True).double()
    scale = (top / torch.full_like(top, 6.0)).float().double().masked_fill(top < 2.0 ** -100, 0.0)
    a = x.double().abs()
    best, far = torch.zeros_like(a), a.clone()
    for i, step in enumerate(STEPS[1:], 1):
        d = (a - step * scale).abs()
        nearer = (d < far) | ((d == far) & (i % 2 == 0))
        best = torch.where(nearer & (scale > 0), step * scale, best)
        far = torch.where(nearer, d, far)
    return torch.where(x < 0, -best, best)


def exact(case, seed):
    c = dict(case, **_inputs(case, seed))
    kind = case["kind"]
    if kind == "linear":
        g = case["group"]
        w = torch.zeros(c["out"], case["cols"], dtype=torch.float64, device="cuda")
        for k in range(0, case["cols"], g):
            w[:, k:k + g] = _nearest(c["w"][:, k:k + g])
        y = torch.matmul(c["x"].double(), w.t().contiguous())
        return y + c["bias"].double() if case["bias"] else y
    if kind == "attend":
        y = torch.empty(c["q"].shape, dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        for b, n in enumerate(_lengths(case)):
            row = torch.arange(n - case["q"], n, device="cuda").unsqueeze(1)
            for h in range(case["kv_heads"]):
                k, v = (_number(_unpacked(c[t][b, h, :n])) * c[t + "_scale"][b, h, :n, None].double()
                        for t in "kv")
                for i in range(h * group, (h + 1) * group):
                    p = torch.matmul(c["q"][b, i].double(), k.t().contiguous()) * case["dim"] ** -0.5
                    p = p.masked_fill(torch.arange(n, device="cuda") > row, -math.inf)
                    y[b, i] = torch.matmul(torch.softmax(p, -1), v)
        return y
    if kind == "append":
        return {n: _nearest(c[n]) for n in "kv"}
    if kind == "beam":
        lp = torch.log_softmax(c["x"].double(), -1) + c["scores"].double().unsqueeze(-1)
        if case["done"]:
            stop = torch.full_like(lp, -math.inf)
            stop[..., -1] = c["scores"].double()
            lp = torch.where(c["done"].unsqueeze(-1), stop, lp)
        best = torch.topk(lp.flatten(1), case["keep"], dim=1)[0]
        return {"scores": best, "tokens": None, "parents": None, "done": None}
    out = []
    for name, t in c.items():
        if name[0] in "kv" and name[1:2].isdigit():
            t = t.view((case["batch"], case["beams"]) + t.shape[1:])
            new = t.clone()
            for b in range(case["batch"]):
                for i, j in enumerate(c["parents"][b].tolist()):
                    new[b, i, :, :case["pos"]] = t[b, j, :, :case["pos"]]
            out.append(new.flatten(0, 1))
    return out
