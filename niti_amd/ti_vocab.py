"""A classifier over many classes together with its loss, as a layer: what TiLinear(last_layer=True) and TiLoss are for ten classes, for
tens of thousands.

TiLinear rounds its logits to int8 and TiLoss its gradient (p < 1/256 becomes 0 or a random bit), and both lie in memory.  Here the
int32 sums become probabilities where they are made (ops.vocab_loss, ops.vocab_distill), the gradients come back as real numbers
(ops.vocab_backward), and the layer brings them into the integer form that the layers below and the update expect: the error as
int8 with an exponent (ERROR_ROUND_METHOD), the weights' gradient rounded to GRAD_BITWIDTH bits (GRAD_ROUND_METHOD) and subtracted."""
from __future__ import annotations

import torch

from . import ops, ti_torch


def _power(n):
    """2^n of an int32 tensor, -126 <= n <= 127, from its bits: ``ldexp`` goes through ``pow``, which need not be exact on a GPU."""
    return ((n.clamp(-126, 127) + 127) << 23).view(torch.float32)


def _fixed_point(x):
    """(int32 tensor, exponent): x = int32 2^exponent, the largest magnitude just below 2^24, the exponent a 1-element int32 device tensor.
    x is float32 from float32 sums: PstoShift takes the low half of the bits that it drops for its random number, so these have to be
    the sum's own.  Eight significant bits in front of zeros (bfloat16) would round almost every fraction up.
    A gradient with NaN in it (a target outside the classes; the loss says so) becomes zero: nothing is learnt from it."""
    m = torch.nan_to_num(x.abs().amax(), nan=0.0, posinf=0.0)
    e = torch.frexp(m)[1]
    half = (24 - e) // 2
    y = torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0) * torch.where(m > 0, _power(half), 0.0) * _power(24 - e - half)
    return y.to(torch.int32), (e - 24).reshape(1).to(torch.int32)


class TiVocabHead(ti_torch.UpdateWeight):
    """forward((act int8 [..., in_features], exponent), target=..., teacher=(top logits, classes)) -> loss per row, float32;
    backward(grad) -> (int8 error, exponent), weights updated.

    ``target`` alone: softmax cross entropy.  ``teacher`` alone: distillation at ``temperature``.  Both: ``alpha`` of the first and
    1 - ``alpha`` of the second.  ``ignore_index``: targets that do not count."""

    def __init__(self, in_features, classes, ignore_index=-100):
        super().__init__()
        self._init_weight(torch.Size([classes, in_features]))
        self.ignore_index = ignore_index
        self._parts = None

    def forward(self, input, target=None, teacher=None, temperature=1.0, alpha=0.5):
        if target is None and teacher is None:
            raise RuntimeError("TiVocabHead: a target or a teacher expected")
        act, exp_in = input
        d = self.__dict__
        d["act_in"] = act
        d["act_in_exp"] = exp = ti_torch._exp_tensor(exp_in, act.device)
        parts, loss = [], None
        if target is not None:
            loss, d["lse"], state = ops.vocab_loss(act, self.weight, exp, self._wexp(), target, self.ignore_index)
            parts.append((1.0 if teacher is None else alpha, state))
        if teacher is not None:
            soft, lse, state = ops.vocab_distill(act, self.weight, exp, self._wexp(), teacher[0], teacher[1], temperature)
            parts.append((1.0 if target is None else 1.0 - alpha, state))
            if target is None:
                loss, d["lse"] = soft, lse
            else:
                loss = alpha * loss + (1.0 - alpha) * soft
        d["_parts"] = parts
        return loss

    def backward(self, grad=None):
        """``grad``: weight of each row's loss, or one for all (float32); None: the mean over the rows."""
        d = self.__dict__
        if d["_parts"] is None:
            raise RuntimeError("TiVocabHead: backward without a forward call")
        act, exp, w_exp = d["act_in"], d["act_in_exp"], self._wexp()
        if grad is None:
            grad = torch.full((1,), 1.0 / max(1, act[..., 0].numel()), dtype=torch.float32, device=act.device)
        da = dw = None
        for share, state in d["_parts"]:
            a, w = ops.vocab_backward(act, self.weight, exp, w_exp, state, grad if share == 1.0 else grad * share, torch.float32)
            da, dw = (a, w) if da is None else (da + a, dw + w)
        d["_parts"] = None
        if not self.weight.is_contiguous():
            self.weight = self.weight.contiguous()
        dev = act.device
        # the update, as UpdateWeight.weight_update does it, from fixed point
        g, g_exp = _fixed_point(dw)
        method = ti_torch._method_name(ti_torch.GRAD_ROUND_METHOD)
        self.grad_exp = torch.empty(1, dtype=torch.int32, device=dev)
        self.grad, self.grad_shift = ops.grad_update(
            g, self.weight, ops.absmax_i32(g), ti_torch.GRAD_BITWIDTH, method, ti_torch.DIV_MODE, ti_torch.BW_MODE,
            ti_torch._rand_bits_like(g) if method == "sto" else None, want_grad=self.keep_grad, exp_a=g_exp, exp_out=self.grad_exp)
        if da.numel() == 0:      # no rows
            y, exp_out = torch.empty(da.shape, dtype=torch.int8, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
        else:
            err, err_exp = _fixed_point(da)
            y, _, exp_out = ti_torch._requant(err, ti_torch.BITWIDTH, ti_torch.ERROR_ROUND_METHOD, exp_a=err_exp, want_exp=True)
        self.err_exp = exp_out
        return y, exp_out

    def top_logits(self, input, k, rows=1024):
        """The k largest logits of every row, largest first, and their classes: ([..., k] float32, [..., k] int64), what ``teacher`` of
        another head's forward takes.  ``rows``: so many rows' logits are in memory at a time."""
        act, exp_in = input
        scale = _power(ti_torch._exp_tensor(exp_in, act.device) + self._wexp())
        flat = act.reshape(-1, act.shape[-1])
        found = [torch.topk(ops.gemm(flat[i:i + rows].contiguous(), self.weight, trans_b=True), k) for i in range(0, flat.shape[0], rows)]
        lead = act.shape[:-1] + (k,)
        values = torch.cat([f.values for f in found]).float() * scale if found else flat.new_zeros((0, k), dtype=torch.float32)
        classes = torch.cat([f.indices for f in found]) if found else flat.new_zeros((0, k), dtype=torch.int64)
        return values.reshape(lead), classes.reshape(lead)
