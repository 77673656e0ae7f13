"""Gradients of the losses over many classes as float32, and the layer that rounds them to integers.

Tolerance of a float32 gradient: that of test_gpu_vocab.py without the result's rounding to bfloat16 (2^-8 of the value)."""
import pytest
import torch

from oracle import niti_oracle as po
from oracle import vocab_oracle as vo
from test_gpu_vocab import call, exp_of, make, make_target, make_teacher

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return torch.device("cuda:0")


# few rows and many, one slice and several, features that are no multiple of four, operands that are copied, several pieces of the classes
@pytest.mark.parametrize("kind,n,f,v", [
    ("entropy", 1, 1, 1), ("distill", 1, 512, 1000), ("entropy", 17, 129, 333), ("distill", 31, 1024, 5000), ("entropy", 33, 66, 511), ("distill", 128, 256, 2000),
    ("entropy", 300, 1000, 777), ("distill", 1003, 997, 4100), ("entropy", 20000, 64, 300), ("entropy", 40, 64, 70000), ("distill", 16500, 48, 4097)])
def test_float32_gradients(dev, kind, n, f, v):
    from niti_amd import ops
    print("float32", kind, n, f, v, flush=True)
    act, w, ea, ew = make(dev, n, f, v, seed=n + f)
    t = 1.0 if kind == "entropy" else 2.0
    targets = {"target": make_target(dev, n, v)} if kind == "entropy" else dict(zip(("top_val", "top_idx"), make_teacher(dev, n, v, 6)))
    e = (exp_of(ea, dev), exp_of(ew, dev))
    state = call(kind, act, w, ea, ew, t, **targets)[2]
    for weight in (None, torch.full((1,), 1.0 / n, device=dev), torch.rand(n, device=dev)):
        wide = ops.vocab_backward(act, w, *e, state, weight, torch.float32)
        short = ops.vocab_backward(act, w, *e, state, weight)
        want = vo.backward(act, w, ea, ew, weight, t, **targets)
        for x, y, z, bound, terms in zip(wide, short, want[:2], want[2:], (v, n)):
            assert x.dtype == torch.float32 and y.dtype == torch.bfloat16 and x.shape == z.shape and x.is_contiguous()
            assert torch.equal(x.bfloat16(), y)          # the same sums
            assert bool(((x.double() - z).abs() <= (2.0 ** -9.9 + terms * 2.0 ** -24) * bound + 2.0 ** -38 * bound.max()).all())


def test_no_rows_and_refusals(dev):
    from niti_amd import ops
    act, w, ea, ew = make(dev, 2, 32, 50)
    e = (exp_of(ea, dev), exp_of(ew, dev))
    state = ops.vocab_loss(act[:0], w, *e, torch.empty(0, dtype=torch.int64, device=dev))[2]
    da, dw = ops.vocab_backward(act[:0], w, *e, state, None, torch.float32)
    assert da.shape == (0, 32) and da.dtype == dw.dtype == torch.float32 and bool((dw == 0).all())
    state = ops.vocab_loss(act, w, *e, torch.tensor([1, 2], device=dev))[2]
    for wrong in (torch.float16, torch.float64, None):
        with pytest.raises(RuntimeError, match="bfloat16 or float32"):
            ops.vocab_backward(act, w, *e, state, None, wrong)
    with pytest.raises(RuntimeError, match="state"):
        ops.vocab_backward(act[:1], w, *e, state, None, torch.float32)


def test_a_target_outside_of_the_classes(dev):
    from niti_amd import ops
    act, w, ea, ew = make(dev, 40, 64, 300)
    t = make_target(dev, 40, 300)
    t[2] = 300
    e = (exp_of(ea, dev), exp_of(ew, dev))
    da, dw = ops.vocab_backward(act, w, *e, ops.vocab_loss(act, w, *e, t)[2], None, torch.float32)
    assert bool(torch.isnan(da[2]).all()) and int(torch.isnan(da).any(1).sum()) == 1 and bool(torch.isnan(dw).all())


def _integers(d):
    """The layer's fixed point of a gradient, by the formula: (int32, exponent)."""
    m = float(d.abs().max())
    e = 0
    while m >= 2.0 ** e:
        e += 1
    while m < 2.0 ** (e - 1):
        e -= 1
    return torch.trunc(d.double() * 2.0 ** (24 - e)).to(torch.int32), e - 24


@pytest.mark.parametrize("mode", ["target", "teacher", "both"])
def test_layer_rounds_the_float32_sums(dev, mode):
    """The same calls of the kernels, then the reference's integer arithmetic, bit for bit."""
    from niti_amd import ops, ti_torch
    from niti_amd.ti_vocab import TiVocabHead
    n, f, v, t, alpha = 60, 96, 700, 2.0, 0.25
    torch.manual_seed(3)
    head = TiVocabHead(f, v)
    head.keep_grad = True
    act = torch.randint(-100, 101, (n, f), dtype=torch.int8, device=dev)
    target = make_target(dev, n, v)
    val, idx = make_teacher(dev, n, v, 5)
    before = head.weight.clone()
    e = (exp_of(-9, dev), exp_of(int(head.weight_exp), dev))
    what = {} if mode == "teacher" else {"target": target}
    if mode != "target":
        what.update(teacher=(val, idx), temperature=t, alpha=alpha)
    head.forward((act, -9), **what)
    err, err_exp = head.backward()
    grad = torch.full((1,), 1.0 / n, dtype=torch.float32, device=dev)
    calls = []
    if mode != "teacher":
        calls.append((1.0 if mode == "target" else alpha, ops.vocab_loss(act, before, *e, target)[2]))
    if mode != "target":
        calls.append((1.0 if mode == "teacher" else 1.0 - alpha, ops.vocab_distill(act, before, *e, val, idx, t)[2]))
    sums = None
    for share, state in calls:
        pair = ops.vocab_backward(act, before, *e, state, grad if share == 1.0 else grad * share, torch.float32)
        sums = pair if sums is None else tuple(a + b for a, b in zip(sums, pair))
    da, dw = (_integers(x.cpu()) for x in sums)
    y, shift = po.err_calc(da[0])
    assert torch.equal(err.cpu(), y) and int(err_exp) == da[1] + shift
    g, shift = po.grad_calc(dw[0], ti_torch.GRAD_BITWIDTH)
    assert torch.equal(head.grad.cpu(), g) and int(head.grad_exp) == dw[1] + shift
    assert torch.equal(head.weight.cpu(), po.weight_update(before.cpu(), g))


def test_mean_update_is_the_gradient(dev, monkeypatch):
    """Over many weights whose 64-bit gradient is about the same, the rounded update's mean is that gradient's: a rounding at random differs by less
    than 1 with a variance of 1/4 at most, so 6 standard deviations of the mean of N are 3 / sqrt(N); PstoShift knows a fraction to 2^-8; a gradient
    is within 2^-9.9 of its sum of magnitudes."""
    from niti_amd import ti_torch
    from niti_amd.ti_vocab import TiVocabHead
    assert ti_torch.GRAD_ROUND_METHOD is ti_torch.PstoShift
    monkeypatch.setattr(ti_torch, "DIV_MODE", "trunc")
    n, f, v = 64, 128, 4000
    torch.manual_seed(5)
    head = TiVocabHead(f, v)
    head.keep_grad = True
    act = torch.randint(-100, 101, (n, f), dtype=torch.int8, device=dev)
    target = make_target(dev, n, v)
    before, ew = head.weight.clone(), int(head.weight_exp)
    head.forward((act, -6), target=target)
    head.backward()
    _, exact, _, bound = (x * 2.0 ** -int(head.grad_exp) for x in vo.backward(act, before, -6, ew, torch.full((1,), 1.0 / n, device=dev), target=target))
    got = head.grad.double() * torch.sign(exact)
    size = exact.abs()
    asked = 0
    for i in range(-10, 2):
        at = (size >= 2.0 ** i) & (size < 2.0 ** (i + 1))
        count = int(at.sum())
        if count < 2000:
            continue
        asked += 1
        off = float(got[at].mean() - size[at].mean())
        print("2^%d: %d weights, %.4f" % (i, count, off), flush=True)
        assert abs(off) <= 3.0 / count ** 0.5 + 2.0 ** -8 + 2.0 ** -9.9 * float(bound[at].mean())
    assert asked >= 4


@pytest.mark.parametrize("shape", [(0, 96), (2, 0, 96)])
def test_layer_without_rows(dev, shape):
    from niti_amd.ti_vocab import TiVocabHead
    head = TiVocabHead(96, 700)
    before = head.weight.clone()
    act = torch.empty(shape, dtype=torch.int8, device=dev)
    target = torch.empty(shape[:-1], dtype=torch.int64, device=dev)
    teacher = (torch.empty(shape[:-1] + (4,), device=dev), torch.empty(shape[:-1] + (4,), dtype=torch.int64, device=dev))
    for what in ({"target": target}, {"teacher": teacher}, {"target": target, "teacher": teacher}):
        assert head.forward((act, -5), **what).shape == shape[:-1]
        err, exp = head.backward()
        assert err.shape == shape and err.dtype == torch.int8 and exp.shape == (1,) and torch.equal(head.weight, before)
