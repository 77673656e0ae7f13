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
