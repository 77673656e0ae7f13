"""Losses over many classes in 64 bits, elementary torch operations on any device: what niti_amd.ops.vocab_loss, vocab_distill and
vocab_backward compute, by the formulas, with the sums that bound their rounding errors."""
import torch


def softmax_parts(act, w, exp_a, exp_w, temperature=1.0):
    """(logits / T, log sum exp of them, softmax), act [N,F] and w [V,F] int8."""
    z = (act.double() @ w.double().t()) * (2.0 ** (exp_a + exp_w)) / temperature
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    s = e.sum(1, keepdim=True)
    return z, (m + torch.log(s)).squeeze(1), e / s


def target_weights(classes, target=None, ignore_index=-100, top_val=None, top_idx=None, temperature=1.0):
    """q [N,V] and whether a row is undefined: the target's one, or the teacher's softmax over a row's used places."""
    if top_idx is None:
        top_idx = torch.where(target == ignore_index, -1, target.long())[:, None]
        undefined = ((target != ignore_index) & ((target < 0) | (target >= classes)))
        top_val = torch.zeros(top_idx.shape, device=top_idx.device)
    else:
        top_idx = top_idx.long()
        undefined = (top_idx >= classes).any(1)
    used = (top_idx >= 0) & (top_idx < classes)
    v = torch.where(used, top_val.double() / temperature, -torch.inf)
    best = v.max(1, keepdim=True).values
    e = torch.where(v == -torch.inf, 0.0, torch.exp(v - torch.where(best == -torch.inf, 0.0, best)))
    norm = e.sum(1, keepdim=True)
    place = torch.where(norm == 0, 0.0, e / norm)
    q = torch.zeros((top_idx.shape[0], classes), dtype=torch.float64, device=top_idx.device)
    q.scatter_add_(1, torch.where(used, top_idx, 0), torch.where(used, place, 0.0))
    # a place keeps a term of its own in the entropy, also where two of them name one class
    entropy = torch.where(place > 0, place * torch.log(torch.where(place > 0, place, 1.0)), place * 0).sum(1)
    undefined = undefined | torch.isnan(norm).squeeze(1)
    return q, entropy, undefined


def forward(act, w, exp_a, exp_w, temperature=1.0, **targets):
    """(loss, lse) of every row."""
    z, lse, _ = softmax_parts(act, w, exp_a, exp_w, temperature)
    q, entropy, undefined = target_weights(w.shape[0], temperature=temperature, **targets)
    q = torch.where(undefined[:, None], 0.0, q)
    loss = temperature ** 2 * (entropy + (q * (lse[:, None] - z)).sum(1))
    return torch.where(undefined, torch.nan, loss), lse


def logit_gradient(act, w, exp_a, exp_w, temperature=1.0, **targets):
    """d loss / d z for the logits z in front of the temperature, [N,V]."""
    _, _, p = softmax_parts(act, w, exp_a, exp_w, temperature)
    q, _, undefined = target_weights(w.shape[0], temperature=temperature, **targets)
    g = temperature * (p * (q.sum(1, keepdim=True) > 0) - q)
    return torch.where(undefined[:, None], torch.nan, g)


def backward(act, w, exp_a, exp_w, weight=None, temperature=1.0, **targets):
    """(d_act, d_w, bound_act, bound_w): gradients of sum(weight * loss), and the same sums over magnitudes, which relative
    errors of the terms are taken of."""
    g = logit_gradient(act, w, exp_a, exp_w, temperature, **targets)
    g = g * (torch.ones(act.shape[0], device=act.device) if weight is None else weight.reshape(-1).expand(act.shape[0])).double()[:, None]
    a, b = act.double(), w.double()
    return ((g @ b) * 2.0 ** exp_w, (g.t() @ a) * 2.0 ** exp_a,
            (g.abs() @ b.abs()) * 2.0 ** exp_w, (g.abs().t() @ a.abs()) * 2.0 ** exp_a)
