"""The benchmark workloads as torch.js programs on the 'hip' device.

Each is written against this package's public API exactly as a torch.js
user would write it (nn modules, functional ops, backward(), optimizers):
  * MLP     Linear(784,256) -> ReLU -> Linear(256,10), cross_entropy, Adam
  * chain   (x + bias) -> GELU -> * y -> sum(0) -> mean
  * CNN     conv 3->32 3x3 p1 -> ReLU -> conv 32->64 3x3 s2 p1 -> ReLU ->
            global avg-pool -> Linear(64,10) -> cross_entropy
  * Block   pre-LN transformer block (causal SDPA, 4x GELU MLP)
  * GPT2    GPT-2 small with tied embeddings, next-token cross_entropy
"""
import ctypes
import math

import numpy as np

from . import _lib as L
from . import decode_ops
from . import functional as F
from . import nn
from .tensor import (Tensor, _before_write, arange, empty, from_numpy, is_grad_enabled, no_grad,
                     zeros)


def mlp():
    return nn.Sequential(nn.Linear(784, 256), nn.ReLU(), nn.Linear(256, 10))


def chain_loss(x, bias, y):
    return (F.gelu(x + bias) * y).sum(0).mean()


class CNN(nn.Module):
    """conv 3->32 3x3 p1, ReLU, conv 32->64 3x3 s2 p1, ReLU, average pool,
    Linear(64, 10).  `fused`: each conv and its ReLU as one op
    (F.conv2d_relu, bit for bit the two in sequence)."""

    def __init__(self, fused=True):
        super().__init__()
        self.conv1 = nn.Conv2d(3, 32, 3, padding=1)
        self.conv2 = nn.Conv2d(32, 64, 3, stride=2, padding=1)
        self.fc = nn.Linear(64, 10)
        self.fused = fused

    def forward(self, x):
        for conv in (self.conv1, self.conv2):
            if self.fused:
                x = F.conv2d_relu(x, conv.weight, conv.bias, conv.stride, conv.padding,
                                  conv.dilation, conv.groups)
            else:
                x = F.relu(conv(x))
        return self.fc(x.mean((2, 3)))


def _plain_linear(m):
    """Whether a layer computes what nn.Linear does: one, or a subclass's that
    leaves its forward as it is."""
    kind = type(m)
    return isinstance(m, nn.Linear) and kind.forward is nn.Linear.forward and \
        kind.__call__ is nn.Linear.__call__


def _check_cache(cache, *attns):
    """Refuses, before anything is launched, a cache that the attention layers do
    not read."""
    if isinstance(cache, KVCacheFP4) or cache is KVCacheFP4:
        if any(getattr(a, "window", None) is not None for a in attns):
            raise NotImplementedError("KV cache in 4 bits: not with a window")


class CausalSelfAttention(nn.Module):
    """With `window`, each position sees the last `window` positions and the
    first `sinks` ones (F.sliding_window_attention) in place of all earlier
    ones."""

    def __init__(self, d, heads, fused=True, window=None, sinks=0):
        super().__init__()
        self.d, self.heads, self.fused = d, heads, fused
        self.window, self.sinks = window, sinks
        self.c_attn = nn.Linear(d, 3 * d)
        self.c_proj = nn.Linear(d, d)

    def forward(self, x, residual=None):
        """attention(x), or residual + attention(x) (with `fused`, the add is
        done by the output projection's GEMM epilogue; without, it is the
        public `+`)."""
        B, T, C = x.shape
        hd = C // self.heads
        q, k, v = self.c_attn(x).split(C, dim=2)
        q = q.view(B, T, self.heads, hd).transpose(1, 2)
        k = k.view(B, T, self.heads, hd).transpose(1, 2)
        v = v.view(B, T, self.heads, hd).transpose(1, 2)
        if self.window is None:
            y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        else:
            y = F.sliding_window_attention(q, k, v, self.window, self.sinks)
        y = y.transpose(1, 2).contiguous().view(B, T, C)
        return self._project(y, residual)

    def forward_cached(self, x, cache, layer, pos, residual=None):
        """Attention of the new positions [pos, pos + T) of x against the
        cached keys / values of positions [0, pos) plus their own; the new
        keys and values are appended to the cache.  A prompt (pos 0) is
        causal over itself; a single new token attends to every cached
        position.  With a window, or a cache in 4 bits, a prompt may also
        come in parts."""
        _check_cache(cache, self)
        B, T, C = x.shape
        hd = C // self.heads
        q, k, v = self.c_attn(x).split(C, dim=2)
        q = q.view(B, T, self.heads, hd).transpose(1, 2)
        k = k.view(B, T, self.heads, hd).transpose(1, 2)
        v = v.view(B, T, self.heads, hd).transpose(1, 2)
        if isinstance(cache, KVCacheFP4):
            cache.append(layer, k, v, pos)
            y = cache.attend(layer, q, pos + T)
            y = y.transpose(1, 2).contiguous().view(B, T, C)
            return self._project(y, residual)
        keys, values = cache.append(layer, k, v, pos)
        if self.window is not None:
            y = F.sliding_window_attention(q, keys, values, self.window, self.sinks)
        elif pos == 0:
            y = F.scaled_dot_product_attention(q, keys, values, is_causal=True)
        elif T == 1:
            y = F.scaled_dot_product_attention(q, keys, values, is_causal=False)
        else:
            raise NotImplementedError("KV cache: prompts start at position 0, then one token "
                                      "per step")
        y = y.transpose(1, 2).contiguous().view(B, T, C)
        return self._project(y, residual)

    def _project(self, y, residual):
        if self.fused and _plain_linear(self.c_proj):
            return F._linear_add(y, self.c_proj.weight, self.c_proj.bias, residual)
        out = self.c_proj(y)
        return out if residual is None else residual + out


class MLPBlock(nn.Module):
    def __init__(self, d, fused=True):
        super().__init__()
        self.fused = fused
        self.c_fc = nn.Linear(d, 4 * d)
        self.c_proj = nn.Linear(4 * d, d)

    def forward(self, x, residual=None):
        if self.fused and _plain_linear(self.c_fc) and _plain_linear(self.c_proj):
            # c_proj(gelu(c_fc(x))) (+ residual) with GELU and the add fused
            # into the two GEMMs
            return F._mlp_gelu(x, self.c_fc.weight, self.c_fc.bias, self.c_proj.weight,
                               self.c_proj.bias, residual)
        out = self.c_proj(F.gelu(self.c_fc(x)))
        return out if residual is None else residual + out


class Block(nn.Module):
    """Pre-LayerNorm transformer block.  fused=False writes it with the
    public operators only (nn.Linear, F.gelu, `+`), as a torch.js program
    would; fused=True routes the GELU and the residual adds through the
    GEMM epilogues (the same values, bit for bit)."""

    def __init__(self, d, heads, fused=True, window=None, sinks=0):
        super().__init__()
        self.ln_1 = nn.LayerNorm(d)
        self.attn = CausalSelfAttention(d, heads, fused, window, sinks)
        self.ln_2 = nn.LayerNorm(d)
        self.mlp = MLPBlock(d, fused)

    def forward(self, x):
        # x + attn(ln_1(x)), then x + mlp(ln_2(x))
        if not is_grad_enabled():
            y = self._infer(x)
            if y is not None:
                return y
        x = self.attn(self.ln_1(x), residual=x)
        return self.mlp(self.ln_2(x), residual=x)

    def _infer(self, x, cache=None, layer=0, pos=0):
        """The block as one library call that issues the same launches (a
        decoding step's eight take 225 us of host time one by one), where no
        graph is recorded and the block is made of the plain layers in
        float32, or of their 4-bit forms, with a cache of either; None
        anywhere else."""
        at, mlp = self.attn, self.mlp
        if type(at) is not CausalSelfAttention or type(mlp) is not MLPBlock or \
                at.window is not None:
            return None
        mods = (self.ln_1, at, at.c_attn, at.c_proj, self.ln_2, mlp, mlp.c_fc, mlp.c_proj)
        kinds = tuple(map(type, mods))
        if kinds != _BLOCK_MODULES:  # some layers in 4 bits?
            if tuple([nn.Linear if k is nn.LinearFP4 else k for k in kinds]) != _BLOCK_MODULES:
                return None
        if not (at.fused and mlp.fused and x.ndim == 3 and x.dtype == "float32"):
            return None
        if any(k in m.__dict__ for m in mods for k in ("forward", "forward_cached", "_project")):
            return None
        B, T, C = x.shape
        hd = C // at.heads
        hid = mlp.c_fc.out_features if type(mlp.c_fc) is nn.LinearFP4 else mlp.c_fc.weight.shape[0]
        ln = ((C,), (C,))
        if not (x.numel() and C == at.d and C % at.heads == 0 and hd % 4 == 0 and
                hid % 4 == 0 and self.ln_1.normalized_shape == (C,) and
                self.ln_2.normalized_shape == (C,) and x.is_contiguous()):
            return None
        w, scales, groups = [], [], []
        for m, shapes in ((mods[0], ln), (mods[2], ((3 * C, C), (3 * C,))),
                          (mods[3], ((C, C), (C,))), (mods[4], ln),
                          (mods[6], ((hid, C), (hid,))), (mods[7], ((C, hid), (C,)))):
            ts = (m.bias,) if type(m) is nn.LinearFP4 else (m.weight, m.bias)
            if len(ts) == 1:
                try:
                    n, codes, sc = decode_ops._weights("block_infer", m.codes, m.scales,
                                                       shapes[0][1], m.group_size)
                except (TypeError, ValueError):
                    return None
                if n != shapes[0][0]:
                    return None
                w.append(codes)
                scales.append(sc)
                groups.append(m.group_size)
                shapes = shapes[1:]
            elif shapes is not ln:
                scales.append(None)
                groups.append(0)
            for t, shape in zip(ts, shapes):
                if t is None:  # a bias, or a norm without weights
                    w.append(None)
                    continue
                if t.shape != shape or t.dtype != "float32" or not t.is_contiguous():
                    return None
                w.append(t.data_ptr())
        kc = vc = four = None
        max_len = 0
        if cache is not None:
            four = type(cache) is KVCacheFP4
            if type(cache) not in (KVCache, KVCacheFP4) or "append" in cache.__dict__ or \
                    "attend" in cache.__dict__ or pos < 0 or (pos and T != 1 and not four):
                return None
            kc, vc = cache.k[layer], cache.v[layer]
            max_len = cache.max_len
            if pos + T > max_len:
                return None
            if four:
                if hd > 128:
                    return None
                try:
                    ks, vs = [decode_ops._cache("block_infer", c, s, hd)
                              for c, s in ((kc, cache.k_scales[layer]), (vc, cache.v_scales[layer]))]
                except (TypeError, ValueError):
                    return None
                if ks[0] != (B, at.heads, max_len) or vs[0] != ks[0]:
                    return None
                _before_write(kc, vc, cache.k_scales[layer], cache.v_scales[layer])
            else:
                for t in (kc, vc):
                    if t.shape != (B, at.heads, max_len, hd) or t.dtype != "float32" or \
                            not t.is_contiguous() or t.requires_grad:
                        return None
                _before_write(kc, vc)
        px = x.data_ptr()
        ptrs = w + [px] if cache is None else w + [px, kc.data_ptr(), vc.data_ptr()]
        if any(p is not None and p & 15 for p in ptrs):
            return None
        y = empty((B, T, C))
        ws = (ctypes.c_void_p * 12)(*w)
        sizes = (B, T, C, at.heads, hid, float(self.ln_1.eps), float(self.ln_2.eps),
                 1.0 / math.sqrt(hd))
        fc = (None, None) if kc is None or four else (kc.data_ptr(), vc.data_ptr())
        if four or any(groups):
            qc = (ks[1], ks[2], vs[1], vs[2]) if four else (None,) * 4
            rc = L.lib().tjh_block_infer_fp4(px, y.data_ptr(), ws, (ctypes.c_void_p * 4)(*scales),
                                             L.i64arr(groups), *sizes, *fc, *qc, max_len, pos)
        else:
            rc = L.lib().tjh_block_infer(px, y.data_ptr(), ws, *sizes, *fc, max_len, pos)
        if rc == L.ERR_OOM:  # no room for the workspace in one piece
            return None
        L.check(rc, "block_infer")
        return y

    def forward_cached(self, x, cache, layer, pos):
        _check_cache(cache, self.attn)
        if not is_grad_enabled():
            y = self._infer(x, cache, layer, pos)
            if y is not None:
                return y
        x = self.attn.forward_cached(self.ln_1(x), cache, layer, pos, residual=x)
        return self.mlp(self.ln_2(x), residual=x)


# the layers of a block that _infer stands for: ln_1, attn, its two
# projections, ln_2, mlp, its two layers
_BLOCK_MODULES = (nn.LayerNorm, CausalSelfAttention, nn.Linear, nn.Linear, nn.LayerNorm, MLPBlock,
                  nn.Linear, nn.Linear)


class KVCache:
    """Keys and values of every layer for positions [0, max_len): one
    [B, H, max_len, head_dim] buffer each, filled as positions arrive; the
    attention of a decoding step reads the prefix [0, pos] as a strided
    view (no copy)."""

    def __init__(self, layers, batch, heads, max_len, head_dim):
        self.max_len = max_len
        self.k = [zeros(batch, heads, max_len, head_dim) for _ in range(layers)]
        self.v = [zeros(batch, heads, max_len, head_dim) for _ in range(layers)]

    def append(self, layer, k, v, pos):
        T = k.shape[2]
        if pos + T > self.max_len:
            raise RuntimeError("KV cache: position %d beyond its length %d" % (pos + T,
                                                                              self.max_len))
        with no_grad():
            self.k[layer][:, :, pos:pos + T].copy_(k)
            self.v[layer][:, :, pos:pos + T].copy_(v)
        return self.k[layer][:, :, :pos + T], self.v[layer][:, :, :pos + T]

    def reorder(self, parents, length):
        """The first `length` positions of row b * W + i become those of row
        b * W + parents[b, i] (F.cache_reorder_), for a beam search whose W
        beams are neighbouring rows."""
        F.cache_reorder_(self._tensors(), parents, length)

    def spread(self, prompt, length):
        """Copies the first `length` positions of each of another cache's rows
        to as many neighbouring rows as this one has for it."""
        with no_grad():
            for dst, src in zip(self._tensors(), prompt._tensors()):
                n, rest = src.shape[0], dst.shape[1:]
                dst = dst.view(n, dst.shape[0] // n, *rest)
                src = src.view(n, 1, *src.shape[1:])[:, :, :, :length]
                dst = dst[:, :, :, :length]
                dst.copy_(src.expand(*dst.shape))

    def _tensors(self):
        return self.k + self.v


class KVCacheFP4(KVCache):
    """KVCache in 4 bits: codes k, v [B, H, max_len, bytes] and one float32
    scale a position and head (F.cache_append_fp4), a seventh of the float
    cache's memory at a head dim of 64.  A position's keys and values are held
    once they are appended, so attention reads them as they are held, a prompt's
    own among them."""

    def __init__(self, layers, batch, heads, max_len, head_dim):
        self.max_len, self.head_dim = max_len, head_dim
        shape = (batch, heads, max_len)
        row = (F.cache_row_bytes(head_dim),)
        self.k = [zeros(*(shape + row), dtype="uint8") for _ in range(layers)]
        self.v = [zeros(*(shape + row), dtype="uint8") for _ in range(layers)]
        self.k_scales = [zeros(*shape) for _ in range(layers)]
        self.v_scales = [zeros(*shape) for _ in range(layers)]

    def append(self, layer, k, v, pos):
        F.cache_append_fp4(self.k[layer], self.k_scales[layer], self.v[layer],
                           self.v_scales[layer], k, v, pos)

    def attend(self, layer, q, length, scale=None):
        """F.attention_fp4 over a layer's first `length` positions."""
        return F.attention_fp4(q, self.k[layer], self.k_scales[layer], self.v[layer],
                               self.v_scales[layer], length, scale)

    def read(self, layer, start, stop):
        """(keys, values) that positions [start, stop) stand for."""
        return F.cache_read_fp4(self.k[layer], self.k_scales[layer], self.head_dim, start, stop,
                                (self.v[layer], self.v_scales[layer]))

    def _tensors(self):
        return self.k + self.v + self.k_scales + self.v_scales


class GPT2(nn.Module):
    """GPT-2 with the LM head tied to the token embedding; with `window` and
    `sinks`, attention over a sliding window (CausalSelfAttention)."""

    head = None  # the LM head in 4 bits (quantize_fp4); a subclass's own is not used here

    def __init__(self, vocab=50257, ctx=1024, d=768, heads=12, layers=12, fused=True, window=None,
                 sinks=0):
        super().__init__()
        self.vocab, self.ctx = vocab, ctx
        self.fused = fused
        self.wte = nn.Embedding(vocab, d)
        self.wpe = nn.Embedding(ctx, d)
        self.h = nn.ModuleList([Block(d, heads, fused, window, sinks) for _ in range(layers)])
        self.ln_f = nn.LayerNorm(d)

    def quantize_fp4(self, group_size=64, head=True):
        """Holds the blocks' linear layers in 4 bits (nn.LinearFP4; a layer with a
        forward of its own stays as it is), and with `head` a 4-bit copy of the
        token table for the logits; the tables that tokens and positions are
        looked up in stay float."""
        if head and self.head is not None and not isinstance(self.head, nn.LinearFP4):
            raise ValueError("quantize_fp4: the model has another head; pass head=False")
        for blk in self.h:
            for m, name in ((blk.attn, "c_attn"), (blk.attn, "c_proj"), (blk.mlp, "c_fc"),
                            (blk.mlp, "c_proj")):
                if _plain_linear(getattr(m, name)):
                    setattr(m, name, nn.LinearFP4.of(getattr(m, name), group_size))
        if head:
            self.head = nn.LinearFP4.of(self.wte, group_size)
        return self

    def _logits(self, x):
        return self.head(x) if isinstance(self.head, nn.LinearFP4) else F.linear(x, self.wte.weight)

    def forward(self, ids):
        x = self._embed(ids, 0)
        for blk in self.h:
            x = blk(x)
        x = self.ln_f(x)
        return self._logits(x)

    def _embed(self, ids, pos0):
        """wte(ids) + wpe(positions pos0 .. pos0 + T - 1); with `fused` one
        kernel each way (F._embedding_pos), else the public lookups and +."""
        if self.fused:
            return F._embedding_pos(ids, self.wte.weight, self.wpe.weight, pos0)
        T = ids.shape[1]
        return self.wte(ids) + self.wpe(arange(pos0, pos0 + T, dtype="int32"))

    def loss(self, ids, targets):
        logits = self(ids)
        return F.cross_entropy(logits.view(-1, self.vocab), targets.reshape(-1))

    def distillation_loss(self, ids, teacher_logits, teacher_ids, temperature=1.0):
        """F.distillation_loss of this model's logits for ids [B, T] against a
        teacher's largest ones [B, T, K] (`teacher(ids).topk(K)`)."""
        return F.distillation_loss(self(ids), teacher_logits, teacher_ids, temperature)

    def new_cache(self, batch, max_len=None, bits=32):
        """A cache for `batch` rows: KVCache, or KVCacheFP4 with bits=4."""
        if bits not in (4, 32):
            raise ValueError("a KV cache holds 32 or 4 bits, got %r" % (bits,))
        blk = self.h[0].attn
        kind = KVCache if bits == 32 else KVCacheFP4
        _check_cache(kind, *[getattr(b, "attn", None) for b in self.h])
        return kind(len(self.h), batch, blk.heads, max_len or self.ctx, blk.d // blk.heads)

    def forward_cached(self, ids, cache, pos):
        """Logits of positions [pos, pos + T) of ids [B, T], the keys and
        values of earlier positions read from (and these appended to) the
        cache."""
        _check_cache(cache, *[getattr(b, "attn", None) for b in self.h])
        x = self._embed(ids, pos)
        for i, blk in enumerate(self.h):
            x = blk.forward_cached(x, cache, i, pos)
        x = self.ln_f(x)
        return self._logits(x)

    def generate(self, ids, max_new_tokens, temperature=1.0, greedy=False, top_k=0, top_p=1.0,
                 min_p=0.0, beams=1, eos=None, cache_bits=32):
        """Autoregressive decoding with a KV cache (the inference side of the
        GPT-2 path, tests/gpt2.test.ts): the prompt runs once, then each
        new token is one cached step; the next token is drawn by
        multinomial from softmax(logits / temperature) (or argmax when
        greedy).  With top_k, top_p or min_p, a temperature of 0, or one
        value a row of any of the four, it is drawn by F.sample_logits
        from the logits, without a readback in the loop; logits without a
        distribution (NaN) raise at the end.  With beams > 1, the most
        probable of the continuations that a search with so many beams keeps
        (F.beam_step), without drawing; one that ends with the token `eos` is
        filled up with it.  cache_bits=4 holds the cache in 4 bits.  Returns the
        [B, T + max_new_tokens] int32 ids."""
        from .tensor import cat
        if beams != 1:
            rules = (temperature, top_k, top_p, min_p)
            if greedy or any(isinstance(r, Tensor) or np.ndim(r) for r in rules) or \
                    rules != (1.0, 0, 1.0, 0.0):
                raise ValueError("generate: a beam search draws nothing; temperature, greedy, "
                                 "top_k, top_p and min_p do not apply")
            return self._search(ids, max_new_tokens, beams, eos, cache_bits)
        if eos is not None:
            raise ValueError("generate: eos ends a beam search's sequences; beams is 1")
        B, T = ids.shape
        total = T + max_new_tokens
        if total > self.ctx:
            raise ValueError("generate: %d positions exceed the context of %d" % (total, self.ctx))
        rules = (temperature, top_k, top_p, min_p)
        cut = any(isinstance(s, Tensor) or np.ndim(s) for s in rules) or \
            temperature == 0 or top_k != 0 or top_p != 1.0 or min_p != 0.0
        with no_grad():
            # (a model's own new_cache may know of no bits)
            cache = self.new_cache(B, total, *([] if cache_bits == 32 else [cache_bits]))
            logits = self.forward_cached(ids, cache, 0)
            out = [ids]
            pos = T
            for _ in range(max_new_tokens):
                last = logits[:, -1, :]
                if greedy:
                    nxt = last.argmax(-1, keepdim=True)
                elif cut:
                    nxt = F.sample_logits(last, None, temperature, top_k, top_p, min_p).view(B, 1)
                else:
                    probs = F.softmax(last * (1.0 / temperature), -1)
                    nxt = probs.multinomial(1)
                out.append(nxt)
                logits = self.forward_cached(nxt, cache, pos)
                pos += 1
            res = cat(out, 1)
            if cut and not greedy and (res.numpy()[:, T:] < 0).any():
                raise RuntimeError("generate: logits hold NaN, infinity or nothing to draw")
            return res

    def _search(self, ids, count, beams, eos, cache_bits):
        """generate's beam search: the prompt once, its cache copied to the
        beams, then a step, a reordering of the caches and one token of every
        beam at a time; the best beam's tokens are followed back at the end,
        after one readback."""
        B, T = ids.shape
        if not 1 < beams <= min(64, self.vocab) or beams != int(beams):
            raise ValueError("generate: %r beams of %d tokens (from 1 to 64)"
                             % (beams, self.vocab))
        beams = int(beams)
        if T + count > self.ctx:
            raise ValueError("generate: %d positions exceed the context of %d"
                             % (T + count, self.ctx))
        if not count:
            return ids if ids.dtype == "int32" else ids.to("int32")
        with no_grad():
            bits = [] if cache_bits == 32 else [cache_bits]
            prompt = self.new_cache(B, T, *bits)
            logits = self.forward_cached(ids, prompt, 0)[:, -1, :]
            cache = self.new_cache(B * beams, T + count, *bits)
            cache.spread(prompt, T)
            scores, tokens, parents, done = F.beam_step(logits, zeros(B, 1), beams, None, eos)
            steps = [(tokens, parents)]
            for pos in range(T, T + count - 1):
                if len(steps) > 1:
                    cache.reorder(parents, pos)
                logits = self.forward_cached(tokens.view(B * beams, 1), cache, pos)
                scores, tokens, parents, done = F.beam_step(
                    logits.view(B * beams, -1), scores, beams, done if eos is not None else None,
                    eos)
                steps.append((tokens, parents))
            at = np.zeros(B, np.int64)
            out = np.empty((B, count), np.int32)
            for i in range(count - 1, -1, -1):
                tokens, parents = (t.numpy() for t in steps[i])
                out[:, i] = tokens[np.arange(B), at]
                at = parents[np.arange(B), at]
            if (out < 0).any():
                raise RuntimeError("generate: logits hold NaN, infinity or nothing to choose")
            return from_numpy(np.concatenate([ids.numpy().astype(np.int32), out], 1))


def load_params(model, params):
    """Copies a {name: float32 array} dict into the model's parameters."""
    model.load_state_dict({k: from_numpy(v) for k, v in params.items()
                           if k in dict(model.named_parameters())})
    return model
