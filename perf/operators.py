"""Operators around a language model's attention and vocabulary: attention over a
sliding window with sinks, the largest values of a row, distillation from a
teacher's largest logits, and sampling from truncated distributions.

Each has a plain form in elementary torch operations and, with `own`, the call
that a user of the 'hip' device makes.  Everything is float32 or int32, the
types that the device computes in.  `listed()` holds fixed sizes, `draw()`
others of the same ranges."""
import math

import torch

own = False

VOCAB = 50257  # GPT-2's


def listed():
    return [
        # one decoding step of four sequences of GPT-2 small's heads, whose
        # cache of 1000 positions is seen through a window with four sinks
        dict(name="window decode 4x12", kind="window", batch=4, heads=12, kv_heads=12, q=1, k=1000,
             dim=64, window=256, sinks=4, grad=False),
        # the next part of one prompt over a cache, an odd length and head
        # size, two query heads to one of the cache
        dict(name="window prompt 93 of 701", kind="window", batch=1, heads=16, kv_heads=8, q=93,
             k=701, dim=80, window=300, sinks=1, grad=False),
        # one layer of a GPT-2 small training step
        dict(name="window train 8x12x1024", kind="window", batch=8, heads=12, kv_heads=12, q=1024,
             k=1024, dim=64, window=256, sinks=4, grad=True),
        # a long sequence, four query heads to one head of keys and values
        dict(name="window train 16x8192", kind="window", batch=1, heads=16, kv_heads=4, q=8192,
             k=8192, dim=128, window=1024, sinks=16, grad=True),
        # the alternatives shown for one generated token
        dict(name="topk 1x50257", kind="topk", rows=1, cols=VOCAB, k=20, grad=False),
        # what a teacher's logits of two sequences are kept as
        dict(name="topk 2048x50257", kind="topk", rows=2048, cols=VOCAB, k=64, grad=False),
        # the best of many candidates' scores, with the gradient through them
        dict(name="topk grad 4099x1000", kind="topk", rows=4099, cols=1000, k=8, grad=True),
        # a student's loss and logits' gradient: one odd sequence, some of
        # the teacher's entries empty, and two whole sequences
        dict(name="distill 509x32001", kind="distill", rows=509, cols=32001, k=37, temperature=1.0),
        dict(name="distill 2048x50257", kind="distill", rows=2048, cols=VOCAB, k=64, temperature=2.0),
        # one sequence's next token with the usual settings
        dict(name="sample 1x50257", kind="sample", rows=1, cols=VOCAB, top_k=50, top_p=0.95,
             min_p=0.0, temperature=0.8, mixed=False),
        # many sequences at once, each with settings of its own
        dict(name="sample mixed 256x50257", kind="sample", rows=256, cols=VOCAB, top_k=40, top_p=0.9,
             min_p=0.05, temperature=1.0, mixed=True),
        # the nucleus alone of an odd vocabulary
        dict(name="sample nucleus 61x32001", kind="sample", rows=61, cols=32001, top_k=0, top_p=0.9,
             min_p=0.0, temperature=1.0, mixed=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "topk", "distill", "sample"])
    if kind == "window":
        kv = rng.randint(1, 12)
        heads = kv * rng.choice([1, 1, 2, 4])
        grad = rng.random() < 0.5
        one = not grad and rng.random() < 0.4
        k = _log(rng, 17, 32768 if one else 4096)
        q = 1 if one else k if grad else rng.choice([min(k, _log(rng, 2, 512)), k])
        # no more scores than the largest listed case has
        batch = rng.randint(1, max(1, min(8, 16 * 8192 * 8192 // (heads * q * k))))
        return dict(kind=kind, batch=batch, heads=heads, kv_heads=kv, q=q, k=k,
                    dim=rng.choice([32, 40, 64, 64, 80, 96, 128]), window=_log(rng, 1, 2048),
                    sinks=rng.choice([0, 1, 4, 16, rng.randint(0, 100)]), grad=grad)
    cols = _log(rng, 200, 131072)
    most = 2048 * VOCAB // cols
    if kind == "topk":
        return dict(kind=kind, rows=_log(rng, 1, min(most, 8192)), cols=cols,
                    k=_log(rng, 1, min(256, cols)), grad=rng.random() < 0.3)
    if kind == "distill":
        return dict(kind=kind, rows=_log(rng, 8, min(most, 4096)), cols=cols,
                    k=_log(rng, 1, min(256, cols)), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]))
    return dict(kind=kind, rows=_log(rng, 1, 512), cols=cols,
                top_k=rng.choice([0, _log(rng, 1, 200)]), top_p=rng.choice([1.0, rng.uniform(0.5, 0.99)]),
                min_p=rng.choice([0.0, rng.uniform(0.001, 0.2)]), temperature=rng.uniform(0.5, 1.5),
                mixed=rng.random() < 0.3)


# --------------------------------------------------------------------- inputs


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    if c["kind"] == "window":
        b, h, kv, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
        x = {"q": randn(b, h, c["q"], d), "k": randn(b, kv, c["k"], d), "v": randn(b, kv, c["k"], d)}
        if c["grad"]:
            x["g"] = randn(b, h, c["q"], d, std=1e-3)
        return x
    # logits of a trained model spread by some units, the best far above the rest
    r, n = c["rows"], c["cols"]
    x = {"x": randn(r, n, std=2.5)}
    if c["kind"] == "topk":
        if c["grad"]:
            x["g"] = randn(r, c["k"], std=1e-2)
        return x
    if c["kind"] == "distill":
        t = x["x"] + randn(r, n)
        t, ids = torch.topk(t, c["k"], dim=1)
        ids = ids.to(torch.int32)
        # rows of fewer entries, and rows of none, end in ids of -1
        lengths = torch.randint(0, c["k"] + 1, (r, 1), generator=g, device="cuda")
        short = torch.rand((r, 1), generator=g, device="cuda") < 0.1
        ids[short & (torch.arange(c["k"], device="cuda") >= lengths)] = -1
        x["t"], x["ids"] = t.contiguous(), ids
        return x
    x["u"] = torch.rand(r, generator=g, device="cuda")
    if c["mixed"]:
        def rows(lo, hi):
            return torch.rand(r, generator=g, device="cuda") * (hi - lo) + lo
        x["temperature"] = rows(0.5, 1.5)
        x["top_k"] = torch.randint(0, 2 * c["top_k"] + 2, (r,), generator=g, device="cuda", dtype=torch.int32)
        x["top_p"] = rows(0.5, 1.1)
        x["min_p"] = rows(-0.05, 0.2)
    return x


class _Array:
    """A library tensor's memory for torch.as_tensor, which keeps this object
    (and with it the memory) as long as the torch tensor lives."""

    def __init__(self, t):
        self.tensor = t
        self.__cuda_array_interface__ = {
            "shape": t.shape, "strides": tuple(4 * s for s in t.stride()),
            "typestr": "<f4" if t.dtype == "float32" else "<i4", "data": (t.data_ptr(), False),
            "version": 2}


def _view(t):
    return torch.as_tensor(_Array(t.detach()), device="cuda")


def _hip():
    import __graft_entry__ as graft
    return graft.load_package()


def prepare(case, seed):
    s = dict(case, **_inputs(case, seed))
    if own:
        # the same values in tensors of the library, which has an allocator of
        # its own: a user's program holds them there from the start
        hip = s["hip"] = _hip()
        hip.init(0)
        for name, x in s.items():
            if isinstance(x, torch.Tensor):
                t = hip.empty(tuple(x.shape), dtype="int32" if x.dtype == torch.int32 else "float32")
                _view(t).copy_(x)
                t.requires_grad = name in ("q", "k", "v", "x") and (case["kind"] == "distill"
                                                                   or bool(case.get("grad")))
                s[name] = t
        torch.cuda.synchronize()
    return s


# ----------------------------------------------------------------- one pass


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    hip, kind = s["hip"], s["kind"]
    F = hip.functional
    if kind == "window":
        ts = {n: s[n] for n in ("q", "k", "v")}
        if not s["grad"]:
            with hip.no_grad():
                return _view(F.sliding_window_attention(ts["q"], ts["k"], ts["v"], s["window"], s["sinks"]))
        for t in ts.values():
            t.grad = None
        y = F.sliding_window_attention(ts["q"], ts["k"], ts["v"], s["window"], s["sinks"])
        y.backward(s["g"])
        return dict({n: _view(t.grad) for n, t in ts.items()}, y=_view(y))
    x = s["x"]
    x.grad = None
    if kind == "topk":
        values, indices = x.topk(s["k"])
        out = {"values": _view(values), "indices": _view(indices)}
        if s["grad"]:
            values.backward(s["g"])
            out["x"] = _view(x.grad)
        return out
    if kind == "distill":
        loss = F.distillation_loss(x, s["t"], s["ids"], temperature=s["temperature"])
        loss.backward()
        return {"loss": _view(loss), "x": _view(x.grad)}
    return _view(F.sample_logits(x, s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                 top_p=s["top_p"], min_p=s["min_p"]))


def _run_plain(s):
    kind = s["kind"]
    if kind == "window":
        return _window(s)
    if kind == "topk":
        return _topk(s)
    if kind == "distill":
        return _distill(s)
    return _sample(s)


def _seen(tq, tk, window, sinks):
    """[tq, tk] truth values: which keys a query sees."""
    i = torch.arange(tk - tq, tk, device="cuda").unsqueeze(1)
    j = torch.arange(tk, device="cuda")
    return (j <= i) & ((j > i - window) | (j < sinks))


def _window(s):
    q, k, v = s["q"], s["k"], s["v"]
    (b, h, tq, d), (kv, tk) = q.shape, k.shape[1:3]
    seen = _seen(tq, tk, s["window"], s["sinks"])
    qs = q.reshape(b, kv, h // kv * tq, d)  # the heads that share a key, one after the other
    p = torch.matmul(qs, k.transpose(-1, -2).contiguous()).view(b, kv, h // kv, tq, tk)
    p *= 1.0 / math.sqrt(d)
    p.masked_fill_(~seen, -math.inf)
    p -= p.amax(-1, keepdim=True)
    p = torch.exp_(p)
    p /= p.sum(-1, keepdim=True)
    p = p.view(b, kv, h // kv * tq, tk)
    y = torch.matmul(p, v)
    if not s["grad"]:
        return y.view(q.shape)
    g = s["g"].reshape(y.shape)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), g)
    ds = torch.matmul(g, v.transpose(-1, -2).contiguous())
    ds -= (g * y).sum(-1, keepdim=True)
    ds *= p
    ds *= 1.0 / math.sqrt(d)
    return {"q": torch.matmul(ds, k).view(q.shape),
            "k": torch.matmul(ds.transpose(-1, -2).contiguous(), qs), "v": dv, "y": y.view(q.shape)}


def _topk(s):
    x, k = s["x"], s["k"]
    values, indices = torch.sort(x, dim=1, descending=True, stable=True)
    values, indices = values[:, :k].contiguous(), indices[:, :k]
    out = {"values": values, "indices": indices.to(torch.int32)}
    if s["grad"]:
        out["x"] = torch.zeros_like(x).scatter_(1, indices, s["g"])
    return out


def _distill(s):
    x, t = s["x"], s["temperature"]
    there = s["ids"] >= 0
    ids = s["ids"].long().clamp(min=0)
    valid = there.any(1)
    # the teacher's distribution over the entries that are there
    v = torch.where(there, s["t"] / t, torch.full_like(s["t"], -math.inf))
    v = v - torch.where(valid, v.amax(1), torch.zeros_like(v[:, 0])).unsqueeze(1)
    e = torch.exp(v)
    total = torch.where(valid, e.sum(1), torch.ones_like(v[:, 0])).unsqueeze(1)
    p = e / total
    lp = torch.where(there, v - torch.log(total), torch.zeros_like(v))
    # the student's over all
    z = x / t
    m = z.amax(1, keepdim=True)
    q = torch.exp(z - m)
    n = q.sum(1, keepdim=True)
    lq = torch.gather(z, 1, ids) - m - torch.log(n)
    rows = (p * (lp - lq)).sum(1) * (t * t)
    count = valid.sum()
    loss = torch.where(valid, rows, torch.zeros_like(rows)).sum() / count
    q /= n
    q.scatter_add_(1, ids, -p)
    q *= (valid * (t / count)).unsqueeze(1)
    return {"loss": loss, "x": q}


def _sample(s):
    x = s["x"].double()
    r, n = x.shape

    def rows(name):
        v = s[name]
        return v.double() if isinstance(v, torch.Tensor) else torch.full((r,), v, dtype=torch.float64, device="cuda")

    t, top_k, top_p, min_p = (rows(name).unsqueeze(1) for name in ("temperature", "top_k", "top_p", "min_p"))
    order = torch.sort(s["x"], dim=1, descending=True, stable=True)[1]
    z = torch.gather(x, 1, order)
    z = z - z[:, :1]
    w = torch.exp(z / t)
    w = w * ((top_k <= 0) | (torch.arange(n, device="cuda") < top_k))
    before = torch.cumsum(w, 1) - w
    w = w * ((top_p >= 1) | (before < top_p * w.sum(1, keepdim=True)))
    w = w * ((min_p <= 0) | (z >= t * torch.log(min_p)))
    w = torch.zeros_like(w).scatter_(1, order, w)  # back in the order of the vocabulary
    w = torch.cumsum(w, 1)
    ids = torch.searchsorted(w, s["u"].double().unsqueeze(1) * w[:, -1:], right=True)
    return ids.squeeze(1).clamp(max=n - 1).to(torch.int32)


# ---------------------------------------------------------------- what it is


def _pairs(c):
    """Queries times the keys that each sees."""
    total = 0
    for i in range(c["k"] - c["q"], c["k"]):
        first = max(0, i - c["window"] + 1)
        total += i + 1 - first + min(c["sinks"], first)
    return total


def _keys(c):
    """Keys that some query sees."""
    first = max(0, c["k"] - c["q"] - c["window"] + 1)
    return c["k"] - first + min(c["sinks"], first)


def work(c):
    if c["kind"] == "window":
        b, d = c["batch"], c["dim"]
        both = b * d * (c["heads"] * c["q"] + c["kv_heads"] * _keys(c))
        pairs = b * c["heads"] * _pairs(c) * d
        # q, k, v and o; with a gradient do, dq, dk and dv too
        return {"bytes": 4 * both * (4 if c["grad"] else 2), "flops": pairs * (14 if c["grad"] else 4)}
    r, n = c["rows"], c["cols"]
    if c["kind"] == "topk":
        return {"bytes": 4 * (r * n * (2 if c["grad"] else 1) + r * c["k"] * (3 if c["grad"] else 2)),
                "flops": r * n}
    if c["kind"] == "distill":
        return {"bytes": 4 * (2 * r * n + 2 * r * c["k"] + 1), "flops": 8 * r * n}
    return {"bytes": 4 * (r * n + r * (6 if c["mixed"] else 2)), "flops": 4 * r * n}


# -------------------------------------------------------- the same in 64 bits


def exact(case, seed):
    c = dict(case, **_inputs(case, seed))
    if c["kind"] == "window":
        return _window_exact(c, case)
    if c["kind"] == "topk":
        v, i = torch.topk(c["x"].double(), case["k"], dim=1)
        out = {"values": v, "indices": None}
        if case["grad"]:
            x = torch.zeros(c["x"].shape, dtype=torch.float64, device="cuda")
            out["x"] = x.index_put_((torch.arange(case["rows"], device="cuda").unsqueeze(1), i), c["g"].double())
        return out
    if c["kind"] == "distill":
        x, t, loss = c["x"].double().requires_grad_(True), case["temperature"], 0.0
        lq = torch.log_softmax(x / t, 1)
        there = c["ids"] >= 0
        count = int(there.any(1).sum())
        v = (c["t"].double() / t).masked_fill(~there, -1e30)
        lp = torch.log_softmax(v, 1)
        part = torch.exp(lp) * (lp - lq.gather(1, c["ids"].long().clamp(min=0)))
        loss = part[there].sum() * t * t / count
        loss.backward()
        return {"loss": loss.detach(), "x": x.grad}
    return None  # token numbers


def _window_exact(c, case):
    """Each kv head of each batch item by itself, queries in pieces that see a
    range of keys, gradients by autograd."""
    q, k, v = (c[n].double() for n in ("q", "k", "v"))
    tq, tk, d, kv = case["q"], case["k"], case["dim"], case["kv_heads"]
    group, off = case["heads"] // kv, case["k"] - case["q"]
    y = torch.empty_like(q)
    grads = {n: torch.zeros_like(t) for n, t in (("q", q), ("k", k), ("v", v))}
    step = max(64, case["window"])
    for b in range(case["batch"]):
        for n in range(kv):
            heads = slice(n * group, (n + 1) * group)
            for t0 in range(0, tq, step):
                t1 = min(tq, t0 + step)
                i = torch.arange(off + t0, off + t1, device="cuda")
                first = max(0, off + t0 - case["window"] + 1)
                j = torch.cat([torch.arange(0, min(case["sinks"], first), device="cuda"),
                               torch.arange(first, off + t1, device="cuda")])
                gap = i.unsqueeze(1) - j
                hidden = (gap < 0) | ((gap >= case["window"]) & (j >= case["sinks"]))
                a = [t.detach().requires_grad_(case["grad"])
                     for t in (q[b, heads, t0:t1], k[b, n, j], v[b, n, j])]
                s = torch.matmul(a[0], a[1].t().contiguous()) * d ** -0.5
                o = torch.matmul(torch.softmax(s.masked_fill(hidden, -math.inf), -1), a[2])
                y[b, heads, t0:t1] = o.detach()
                if case["grad"]:
                    o.backward(c["g"][b, heads, t0:t1].double())
                    grads["q"][b, heads, t0:t1] = a[0].grad
                    grads["k"][b, n].index_add_(0, j, a[1].grad)
                    grads["v"][b, n].index_add_(0, j, a[2].grad)
    return dict(grads, y=y) if case["grad"] else y
