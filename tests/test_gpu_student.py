"""A small model with windowed attention that learns from a teacher's largest
logits and is sampled from: top-k, distillation, windowed attention and
sampling together, as a program uses them."""
import numpy as np
import pytest

from test_gpu_vocab_ops import sample_ref
from test_gpu_window import visible

pytestmark = pytest.mark.gpu
U = 2.0 ** -24

VOCAB, CTX, D, HEADS, LAYERS, WINDOW, SINKS = 503, 96, 64, 4, 2, 24, 3


def _models(torch):
    from torchjs_amd import workloads as W
    torch.manual_seed(11)
    teacher = W.GPT2(VOCAB, CTX, D, HEADS, LAYERS)
    student = W.GPT2(VOCAB, CTX, D, HEADS, LAYERS, window=WINDOW, sinks=SINKS)
    return teacher, student


def _ids(torch, b, t, seed=0):
    return torch.tensor(np.random.default_rng(seed).integers(0, VOCAB, (b, t)).astype(np.int32))


def _explicit(torch, student, ids, values, idx, temp):
    """The student's loss with masked attention over all scores and the
    distillation written out in recorded operations."""
    F = torch.functional
    b, t = ids.shape
    mask = torch.tensor(visible(t, t, WINDOW, SINKS))
    x = student._embed(ids, 0)
    for blk in student.h:
        h = blk.ln_1(x)
        q, k, v = [y.view(b, t, HEADS, D // HEADS).transpose(1, 2)
                   for y in blk.attn.c_attn(h).split(D, dim=2)]
        y = F.scaled_dot_product_attention(q, k, v, attn_mask=mask)
        x = x + blk.attn.c_proj(y.transpose(1, 2).contiguous().view(b, t, D))
        x = x + blk.mlp.c_proj(F.gelu(blk.mlp.c_fc(blk.ln_2(x))))
    logits = F.linear(student.ln_f(x), student.wte.weight)
    lq = F.log_softmax(logits * (1.0 / temp), -1).gather(-1, idx)
    lp = F.log_softmax(values * (1.0 / temp), -1)
    return (F.softmax(values * (1.0 / temp), -1) * (lp - lq)).sum() * (temp * temp / (b * t))


def test_training_step(torch):
    teacher, student = _models(torch)
    ids = _ids(torch, 3, 83)
    with torch.no_grad():
        values, idx = teacher(ids).topk(17)
    loss = student.distillation_loss(ids, values, idx, 2.0)
    loss.backward()
    got = {n: p.grad.numpy().copy() for n, p in student.named_parameters()}
    student.zero_grad()
    want = _explicit(torch, student, ids, values, idx, 2.0)
    want.backward()
    # two float32 paths over sums of up to VOCAB and 3 * 83 terms, each step of
    # a sum off by at most half a step: about 500 of them either way
    assert abs(loss.item() - want.item()) <= 1000 * U * abs(want.item())
    for n, p in student.named_parameters():
        w = p.grad.numpy()
        assert np.linalg.norm(got[n] - w) <= 1000 * U * np.linalg.norm(w), n
    # an optimizer's step on them moves every parameter
    before = {n: p.numpy().copy() for n, p in student.named_parameters()}
    torch.optim.AdamW(student.parameters(), lr=1e-3).step()
    assert all((p.numpy() != before[n]).any() for n, p in student.named_parameters() if n != "wpe.weight")


def test_teacher_is_matched_exactly(torch):
    """A student with the teacher's weights and a window that holds the whole
    sequence: nothing left to learn from all of the teacher's logits."""
    from torchjs_amd import workloads as W
    teacher, _ = _models(torch)
    same = W.GPT2(VOCAB, CTX, D, HEADS, LAYERS, window=CTX)
    same.load_state_dict(teacher.state_dict())
    ids = _ids(torch, 2, 40)
    with torch.no_grad():
        values, idx = teacher(ids).topk(VOCAB)
    loss = same.distillation_loss(ids, values, idx)
    # the difference of two logarithms that agree to some hundred half steps
    assert abs(loss.item()) <= 300 * U * np.log(VOCAB)


@pytest.mark.parametrize("parts", [(70,), (1,), (31, 32, 7), (24, 1, 45)])
def test_cached_positions_equal_the_whole_sequence(torch, parts):
    _, student = _models(torch)
    ids = _ids(torch, 2, 80, 3)
    with torch.no_grad():
        whole = student(ids).numpy()
        cache = student.new_cache(2, 80)
        pos, got = 0, []
        for n in list(parts) + [1] * (80 - sum(parts)):
            got.append(student.forward_cached(ids[:, pos:pos + n], cache, pos).numpy())
            pos += n
    got = np.concatenate(got, 1)
    # other orders of sums of at most 80 and 256 terms through two layers
    assert np.abs(got - whole).max() <= 2000 * U * np.abs(whole).max()


@pytest.mark.parametrize("kw", [dict(top_k=20, top_p=0.9), dict(top_p=0.8), dict(min_p=0.1),
                                dict(temperature=0.7, top_k=5, min_p=0.01)], ids=str)
def test_generate(torch, kw):
    _, student = _models(torch)
    prompt = _ids(torch, 2, 40, 5)
    torch.manual_seed(77)
    seq = student.generate(prompt, 30, **kw).numpy()
    assert seq.shape == (2, 70) and (seq[:, :40] == prompt.numpy()).all() and (seq >= 0).all()
    torch.manual_seed(77)
    t = kw.get("temperature", 1.0)
    rest = {k: v for k, v in kw.items() if k != "temperature"}
    with torch.no_grad():
        cache = student.new_cache(2, 70)
        logits = student.forward_cached(prompt, cache, 0)
        for pos in range(40, 70):
            x, u = logits[:, -1, :].numpy(), torch.rand(2).numpy()
            want = [sample_ref(x[r], float(u[r]), t, **rest) for r in range(2)]
            assert seq[:, pos].tolist() == want, pos
            logits = student.forward_cached(torch.tensor(seq[:, pos:pos + 1]), cache, pos)


def test_generate_says_when_there_is_nothing_to_draw(torch):
    _, student = _models(torch)
    student.ln_f.weight.detach().fill_(float("nan"))
    with pytest.raises(RuntimeError, match="nothing to draw"):
        student.generate(_ids(torch, 1, 5), 3, top_k=4)
    with pytest.raises(ValueError, match="top_p"):
        student.generate(_ids(torch, 1, 5), 3, top_p=2.0)


def test_generate_from_a_prompt_with_ids_out_of_range(torch):
    """A prompt's ids are clamped as the embedding does; only drawn ones of -1
    say that there was nothing to draw."""
    _, student = _models(torch)
    prompt = torch.tensor(np.array([[-1, 5, 9]], np.int32))
    seq = student.generate(prompt, 4, top_k=5).numpy()
    assert seq[0, :3].tolist() == [-1, 5, 9] and (seq[0, 3:] >= 0).all()


def test_generate_at_temperature_zero_is_greedy(torch):
    _, student = _models(torch)
    prompt = _ids(torch, 2, 20, 6)
    want = student.generate(prompt, 12, greedy=True).numpy()
    for kw in ({}, dict(top_k=3), dict(top_p=0.5), dict(top_k=[4, 0], min_p=0.1)):
        assert (student.generate(prompt, 12, 0, **kw).numpy() == want).all(), kw


def test_generate_with_settings_of_each_row(torch):
    """A number, a list, an array or a tensor for any of the settings."""
    _, student = _models(torch)
    prompt = _ids(torch, 2, 20, 7)
    settings = dict(temperature=[0.7, 1.2], top_k=[0, 9], top_p=[0.8, 1.0], min_p=[0.0, 0.02])
    one = {name: value[0] for name, value in settings.items()}
    for name, value in settings.items():
        dtype = np.int32 if name == "top_k" else np.float32
        kw = dict(one)
        kw[name] = np.array([value[0]] * 2, dtype)
        torch.manual_seed(3)
        want = student.generate(prompt, 10, **one).numpy()
        for v in (kw[name], kw[name].tolist(), torch.tensor(kw[name])):
            kw[name] = v
            torch.manual_seed(3)
            # float32 settings in place of Python's: one draw in millions differs
            assert (student.generate(prompt, 10, **kw).numpy() == want).all(), name
    torch.manual_seed(4)
    seq = student.generate(prompt, 10, **settings).numpy()
    torch.manual_seed(4)
    with torch.no_grad():
        cache = student.new_cache(2, 30)
        logits = student.forward_cached(prompt, cache, 0)
        for pos in range(20, 30):
            x, u = logits[:, -1, :].numpy(), torch.rand(2).numpy()
            want = [sample_ref(x[r], float(u[r]), float(np.float32(settings["temperature"][r])),
                               settings["top_k"][r], float(np.float32(settings["top_p"][r])),
                               float(np.float32(settings["min_p"][r]))) for r in range(2)]
            assert seq[:, pos].tolist() == want, pos
            logits = student.forward_cached(torch.tensor(seq[:, pos:pos + 1]), cache, pos)
