"""TiVocabHead (the layer over ops.vocab_*) and the example that trains with it; the kernels' paths that need larger calls than those of
test_gpu_vocab.py, whose tolerances these share."""
import pytest
import torch

from oracle import niti_oracle as po
from oracle import vocab_oracle as vo
from test_gpu_vocab import check_forward, check_gradients, exp_of, make, make_target, make_teacher, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return torch.device("cuda:0")


# tiles of 256 x 256, several in turn to a workgroup and partial ones at the edges; sums in one and in several parts; 128 x 128 tiles
@pytest.mark.parametrize("kind,n,f,v", [("entropy", 2100, 300, 9000), ("distill", 4100, 132, 5003), ("entropy", 8200, 128, 4090), ("distill", 2050, 1040, 8200),
                                        ("entropy", 1003, 260, 20011), ("entropy", 600, 2000, 1111), ("distill", 513, 72, 33000)])
def test_large_calls(dev, kind, n, f, v):
    print("large", kind, n, f, v, flush=True)
    weight = torch.rand(n, device=dev)
    run(kind, dev, n, f, v, t=2.0 if kind == "distill" else 1.0, k=9, seed=n, weight=weight)


@pytest.mark.parametrize("n", [3, 40, 300, 2100])
@pytest.mark.parametrize("f", [4, 20, 100, 136, 252])
def test_weights_at_multiples_of_four_bytes(dev, n, f):
    """Read in place: the last row's end is the end of the tensor, other rows are followed by other values."""
    from niti_amd import ops
    v = 260 if n < 2000 else 8200
    act, w, ea, ew = make(dev, n, f, v, seed=n + f)
    t = make_target(dev, n, v)
    wide = torch.full((v, f + 12), 127, dtype=torch.int8, device=dev)
    cut = wide[:, 4:4 + f]
    cut.copy_(w)
    base = None
    for b in (w, cut):
        got = ops.vocab_loss(act, b, exp_of(ea, dev), exp_of(ew, dev), t)
        check_forward(got, vo.forward(act, w, ea, ew, target=t), 1.0)
        grads = ops.vocab_backward(act, b, exp_of(ea, dev), exp_of(ew, dev), got[2])
        check_gradients(grads, vo.backward(act, w, ea, ew, target=t), n, v)
        if base is not None:
            assert torch.equal(base[0], grads[0]) and torch.equal(base[1], grads[1])
        base = grads


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
def test_layer(dev, mode):
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
    ea, ew = -9, int(head.weight_exp)
    e = (exp_of(ea, dev), exp_of(ew, dev))
    what = {} if mode == "teacher" else {"target": target}
    if mode != "target":
        what.update(teacher=(val, idx), temperature=t, alpha=alpha)
    loss = head.forward((act, ea), **what)
    hard = vo.forward(act, before, ea, ew, target=target)[0]
    soft = vo.forward(act, before, ea, ew, t, top_val=val, top_idx=idx)[0]
    want = {"target": hard, "teacher": soft, "both": alpha * hard + (1 - alpha) * soft}[mode]
    assert float((loss.double() - want).abs().max()) <= t * t * 2.0 ** -16 + 2.0 ** -20 * float(want.abs().max())
    err, err_exp = head.backward()
    # the same two calls of the kernels, then the reference's integer arithmetic
    grad = torch.full((1,), 1.0 / n, dtype=torch.float32, device=dev)
    calls = []
    if mode != "teacher":
        calls.append((1.0 if mode == "target" else alpha, ops.vocab_loss(act, before, *e, target)[2]))
    if mode != "target":
        calls.append((1.0 if mode == "teacher" else 1.0 - alpha, ops.vocab_distill(act, before, *e, val, idx, t)[2]))
    sums = None
    for share, state in calls:
        pair = ops.vocab_backward(act, before, *e, state, grad if share == 1.0 else grad * share)
        sums = pair if sums is None else tuple(a.float() + b.float() for a, b in zip(sums, pair))
    da, dw = (_integers(x.cpu()) for x in sums)
    y, shift = po.err_calc(da[0])
    assert torch.equal(err.cpu(), y) and int(err_exp) == da[1] + shift
    g, shift = po.grad_calc(dw[0], ti_torch.GRAD_BITWIDTH)
    assert torch.equal(head.grad.cpu(), g) and int(head.grad_exp) == dw[1] + shift
    assert torch.equal(head.weight.cpu(), po.weight_update(before.cpu(), g))
    with pytest.raises(RuntimeError, match="forward"):
        head.backward()
    with pytest.raises(RuntimeError, match="target or a teacher"):
        head.forward((act, ea))


def test_nothing_to_learn_leaves_the_weights(dev):
    from niti_amd.ti_vocab import TiVocabHead
    head = TiVocabHead(32, 50)
    act = torch.randint(-100, 101, (4, 32), dtype=torch.int8, device=dev)
    for wrong in (-100, 50):            # no row counts; every row's target is none of the classes
        before = head.weight.clone()
        loss = head.forward((act, -5), target=torch.full((4,), wrong, dtype=torch.int64, device=dev))
        assert bool((torch.isnan(loss) if wrong == 50 else loss == 0).all())
        err, _ = head.backward()
        assert bool((err == 0).all()) and torch.equal(head.weight, before)


def test_top_logits(dev):
    from niti_amd.ti_vocab import TiVocabHead
    head = TiVocabHead(64, 300)
    act = torch.randint(-100, 101, (5, 7, 64), dtype=torch.int8, device=dev)
    value, cls = head.top_logits((act, -4), 6, rows=16)
    assert value.shape == cls.shape == (5, 7, 6)
    z = (act.double() @ head.weight.double().t()) * 2.0 ** (-4 + int(head.weight_exp))
    assert torch.equal(value.double(), z.topk(6).values) and torch.equal(z.gather(2, cls), value.double())
    assert head.top_logits((act[:0], -4), 6)[0].shape == (0, 7, 6)


def test_example_learns(dev):
    """The example at a small size: the teacher's loss falls well below log(classes), the student gets nearer to the teacher."""
    from niti_amd import distill
    t0, t1, acc, s0, s1, _ = distill.run(classes=300, features=128, hidden=256, student=256, batch=128, steps=150, top=8, say=lambda line: print(line, flush=True))
    assert t0 > 4.0 and t1 < 0.5 * t0 and acc > 0.5 and s1 < 0.6 * s0
