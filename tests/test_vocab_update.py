"""TiVocabHead's integer update and error against the gradients they are made of, on the CPU: the kernels' calls are replaced by the
oracles, the layer's own steps run as they are."""
import pytest
import torch

from oracle import niti_oracle as po


def grid(signs, seed=0):
    """(d_w [levels, samples], its unit): levels of 0.02 to 4 units of a gradient of 5 bits, every value within 5 % of its level, with all the
    bits that float64 has; the last row sets the unit by its magnitude, 31.9 units, and is one value, so no mean is asked of it."""
    g = torch.Generator().manual_seed(seed)
    levels = torch.tensor([0.0234375, 0.046875, 0.09375, 0.1875, 0.375, 0.75, 1.5, 2.94, 3.99], dtype=torch.float64)
    v = levels[:, None] * (0.95 + 0.1 * torch.rand((len(levels), 8192), generator=g, dtype=torch.float64))
    v = torch.cat([v, torch.full((1, 8192), 31.9, dtype=torch.float64)])
    if signs:
        v[:, 1::2] *= -1
    return v * 2.0 ** -17, 2.0 ** -17


@pytest.fixture()
def head_on_cpu(monkeypatch):
    """A layer whose kernels' results are given: (function of (d_act, d_w) in 64 bits) -> (layer, what it handed to the update and the error)."""
    from niti_amd import _lib, ops, ti_torch, ti_vocab
    monkeypatch.setattr(ti_torch, "GPU", "cpu")

    def make(da, dw):
        head = ti_vocab.TiVocabHead(dw.shape[1], dw.shape[0])
        head.keep_grad = True
        head.weight.zero_()
        state = object()
        monkeypatch.setattr(ops, "vocab_loss", lambda act, *a: (torch.zeros(act.shape[:-1]), torch.zeros(act.shape[:-1]), state))
        monkeypatch.setattr(ops, "vocab_backward", lambda act, w, ea, ew, s, grad=None, dtype=torch.bfloat16: (da.to(dtype), dw.to(dtype)))
        monkeypatch.setattr(ops, "absmax_i32", lambda x: torch.tensor([po.absmax(x)], dtype=torch.int32))

        def grad_update(g, w, absmax, mu, method, div_mode, bw_mode, rand, want_grad, exp_a, exp_out):
            y, shift = po.grad_calc(g, mu, method, div_mode, rand, bw_mode)
            exp_out.copy_(exp_a + shift)
            w.copy_(po.weight_update(w, y))
            return y, torch.tensor([shift], dtype=torch.int32)

        def requant(x, absmax, bits, method, div_mode, bw_mode, rand, relu, exp_a, exp_b, exp_out):
            y, shift = po.err_calc(x, method, div_mode, rand, bw_mode)
            exp_out.copy_(exp_a + shift)
            return y, torch.tensor([shift], dtype=torch.int32)

        monkeypatch.setattr(ops, "grad_update", grad_update)
        monkeypatch.setattr(ops, "requant", requant)
        return head

    return make


# The mean of many values rounded at random is their mean.  A sample of a fraction differs from it by less than 1 with a variance of 1/4 at most:
# 6 standard deviations of the mean of 8192 are 0.034.  PstoShift compares the high half of 17 and more dropped bits with the low half: the fraction
# is known to 2^-8, 0.004.
TOLERANCE = 6 * 0.5 / 8192 ** 0.5 + 2.0 ** -8


@pytest.mark.parametrize("div_mode,signs", [("floor", False), ("trunc", False), ("trunc", True)])
def test_mean_update_is_the_gradient(head_on_cpu, monkeypatch, div_mode, signs):
    from niti_amd import ti_torch
    monkeypatch.setattr(ti_torch, "DIV_MODE", div_mode)
    assert ti_torch.GRAD_ROUND_METHOD is ti_torch.PstoShift and ti_torch.GRAD_BITWIDTH == 5
    dw, unit = grid(signs)
    head = head_on_cpu(torch.ones((3, dw.shape[1]), dtype=torch.float64), dw)
    head.forward((torch.ones((3, dw.shape[1]), dtype=torch.int8), -5), target=torch.zeros(3, dtype=torch.int64))
    head.backward()
    assert 2.0 ** int(head.grad_exp) == unit
    sign = torch.sign(dw)
    err = (head.grad.double() * sign).mean(1) - (dw * sign).mean(1) / unit
    print(err.tolist())
    assert float(err[:-1].abs().max()) <= TOLERANCE
    assert torch.equal(head.weight, -head.grad)


def test_mean_error_is_the_gradient(head_on_cpu, monkeypatch):
    """The same of the error for the layers below, with PstoShift chosen for it: 7 bits, units four times as fine."""
    from niti_amd import ti_torch
    monkeypatch.setattr(ti_torch, "ERROR_ROUND_METHOD", ti_torch.PstoShift)
    monkeypatch.setattr(ti_torch, "DIV_MODE", "trunc")
    da, unit = grid(True)
    head = head_on_cpu(da, torch.ones((4, da.shape[1]), dtype=torch.float64))
    head.forward((torch.ones(da.shape, dtype=torch.int8), -5), target=torch.zeros(len(da), dtype=torch.int64))
    err, exp = head.backward()
    assert 2.0 ** int(exp) == unit / 4
    sign = torch.sign(da)
    bias = (err.double() * sign).mean(1) - (da * sign).mean(1) / (unit / 4)
    assert float(bias[:-1].abs().max()) <= TOLERANCE


def test_what_bfloat16_would_give():
    """The other side: integers made of bfloat16 numbers, rounded by the same oracle, lie far above their values."""
    dw, unit = grid(False)
    from niti_amd import ti_vocab
    mean = {}
    for dtype in (torch.bfloat16, torch.float32):
        x, e = ti_vocab._fixed_point(dw.to(dtype))
        y, shift = po.grad_calc(x, 5)
        assert 2.0 ** (int(e) + shift) == unit
        mean[dtype] = y.double().mean(1) - dw.mean(1) / unit
    assert float(mean[torch.float32][:-1].abs().max()) <= TOLERANCE
    assert bool((mean[torch.bfloat16][:7] > torch.tensor([0.05, 0.1, 0.2, 0.4, 0.4, 0.15, 0.3])).all())


@pytest.mark.parametrize("shape", [(0, 12), (0, 3, 12), (3, 0, 12)])
def test_no_rows(head_on_cpu, shape):
    """A batch of none is a step like any other: nothing is learnt, the error has the input's shape."""
    head = head_on_cpu(torch.zeros(shape, dtype=torch.float64), torch.zeros((5, 12), dtype=torch.float64))
    loss = head.forward((torch.empty(shape, dtype=torch.int8), -5), target=torch.empty(shape[:-1], dtype=torch.int64))
    assert loss.shape == shape[:-1]
    err, exp = head.backward()
    assert err.shape == shape and err.dtype == torch.int8 and exp.dtype == torch.int32 and exp.shape == (1,)
    assert bool((head.weight == 0).all())
    with pytest.raises(RuntimeError, match="forward"):
        head.backward()
