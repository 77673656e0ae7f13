"""Losses over many classes at the ends of their ranges: teachers' values near a type's largest, rows that are all but sure of themselves."""
import pytest
import torch

from oracle import vocab_oracle as vo
from test_gpu_vocab import check_forward, check_gradients, exp_of, make, make_teacher

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return torch.device("cuda:0")


@pytest.mark.parametrize("value", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t", [0.25, 1.0, 3.0])
def test_teacher_values_over_a_temperature(dev, value, t):
    """A row of lowest values is a row of equal ones, whatever T; the largest value takes everything.  Tolerances of test_gpu_vocab.py; where
    weights are 1 / k or 1 the loss's terms are at most 30."""
    from niti_amd import ops
    n, f, v, k = 8, 64, 300, 4
    act, w, ea, ew = make(dev, n, f, v)
    e = (exp_of(ea, dev), exp_of(ew, dev))
    val, idx = make_teacher(dev, n, v, k, value=value)
    idx = torch.stack([torch.randperm(v, device=dev)[:k] for _ in range(n)])
    low, high = torch.finfo(value).min, torch.finfo(value).max
    val[0] = low
    val[1] = high
    val[2] = torch.tensor([low, high, low, high])
    val[3] = torch.tensor([low, low, -torch.inf, -torch.inf])
    val[4, 1] = high
    idx[5, 2:] = -1
    val[5] = low
    got = ops.vocab_distill(act, w, *e, val, idx, t)
    want = vo.forward(act, w, ea, ew, t, top_val=val, top_idx=idx)
    assert bool(torch.isfinite(want[0]).all())
    check_forward(got, want, t, 30.0)
    check_gradients(ops.vocab_backward(act, w, *e, got[2]), vo.backward(act, w, ea, ew, None, t, top_val=val, top_idx=idx), n, v)


@pytest.mark.parametrize("n", [1, 40, 200])
@pytest.mark.parametrize("v", [300000, 1000003])
def test_rows_that_are_all_but_sure(dev, n, v):
    """One class is ahead of many equal ones, and the loss is log(1 + (v - 1) 2^-31): what all the others come to.  Tiles' sums are float32 numbers.
    The largest class's own, just above 1, may lose the other classes of its tile, at most 255 2^-31 < 2^-23: an addition's rounding is no more than
    what is added.  The others keep 36 additions' 36 2^-24 of their value, their exponentials of 2^-31 31 ln 2 2^-23 + 2^-23, and the joined sum
    and its logarithm 2^-22 of what is beside the 1: 2^-16 in all."""
    from niti_amd import ops
    f = 16
    act = torch.zeros((n, f), dtype=torch.int8, device=dev)
    act[:, 0] = 64
    w = torch.zeros((v, f), dtype=torch.int8, device=dev)
    best = 12345
    w[best, 0] = 86                       # 5504 steps of 2^-8 ahead: e^-21.5 = 2^-31
    target = torch.full((n,), best, dtype=torch.int64, device=dev)
    loss, lse, _ = ops.vocab_loss(act, w, exp_of(-4, dev), exp_of(-4, dev), target)
    want = float(torch.log1p(torch.tensor((v - 1) * float(torch.exp(torch.tensor(-21.5, dtype=torch.float64))), dtype=torch.float64)))
    print(v, want, float(loss[0]), flush=True)
    assert bool(((loss.double() - want).abs() <= 2.0 ** -23 + 2.0 ** -16 * want).all())
    assert bool(((lse.double() - (21.5 + want)).abs() <= 2.0 ** -19).all())


@pytest.mark.parametrize("kind", ["entropy", "distill"])
@pytest.mark.parametrize("n", [1, 40, 200])
def test_gradients_of_rows_that_are_all_but_sure(dev, kind, n):
    """The same with 1 - p = 300000 e^-26.5 = 2^-20.  p - q of the target is within 2^-9.9 of its value like every other (see test_gpu_vocab.py),
    beside what the largest class's own tile may lose, 255 of the 300000 others; where a product has one term that counts, it is the result's
    error, with 2^-24 of the sum in float32."""
    from niti_amd import ops
    f, v, best = 16, 300000, 12345
    act = torch.zeros((n, f), dtype=torch.int8, device=dev)
    act[:, 0] = 64
    w = torch.zeros((v, f), dtype=torch.int8, device=dev)
    w[best, 0] = 106                      # 26.5
    e = (exp_of(-4, dev), exp_of(-4, dev))
    if kind == "entropy":
        state = ops.vocab_loss(act, w, *e, torch.full((n,), best, dtype=torch.int64, device=dev))[2]
    else:
        idx = torch.tensor([best, 17, best], device=dev).repeat(n, 1)
        state = ops.vocab_distill(act, w, *e, torch.tensor([1.0, -torch.inf, 1.0], device=dev).repeat(n, 1), idx)[2]
    da, dw = ops.vocab_backward(act, w, *e, state, torch.full((1,), 1.0 / n, device=dev), torch.float32)
    small = float(torch.exp(torch.tensor(-26.5, dtype=torch.float64)))
    rest = (v - 1) * small / (1.0 + (v - 1) * small)
    tol = 2.0 ** -9.9 + 255.0 / v + 2.0 ** -22
    print(kind, n, rest, float(dw[best, 0]) / -4.0, flush=True)
    assert abs(float(dw[best, 0]) / (-rest * 64 * 2.0 ** -4) - 1.0) <= tol
    assert bool((da[:, 0].double() / (-rest * 106 * 2.0 ** -4 / n) - 1.0).abs().max() <= tol)
    # a place of weight zero has its softmax
    if kind == "distill":
        assert abs(float(dw[17, 0]) / (small * 64 * 2.0 ** -4) - 1.0) <= 0.5 / 1.7      # 2^-38 is 1.7 of float16's last places here
