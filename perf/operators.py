"""Timing cases of the losses over a large vocabulary: a classifier of many classes with its loss, the logits kept nowhere.

Operands are the package's: int8 activations [rows, features] and int8 weights [classes, features], each with an exponent (a
1-element int32 tensor); a logit is z = (a . w) 2^(ea + ew).  Kinds of case (``"kind"``):

``entropy``  softmax cross entropy against one class per row (-100: the row does not count)
``distill``  cross entropy against a teacher's softmax at a temperature T, of which only the top logits are known: per row K
             (value, class) pairs, class -1 where a list is shorter; loss T^2 KL(teacher || softmax(z / T))

``"grads"``: False, the loss and the logarithm of the softmax's denominator of every row (scoring, evaluation); True, a training
step: the loss, and the gradients of sum(weight_n loss_n) with respect to activations and weights, rounded to bfloat16."""
import math

import torch

own = False
DEVICE = "cuda"
IGNORED = -100
TEACHER = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
INDEX = {"int64": torch.int64, "int32": torch.int32}


def listed():
    return [
        # one sample scored against the classes of a small image classifier: the shortest call, launch latency and host cost
        {"name": "entropy_score_one", "kind": "entropy", "grads": False, "rows": 1, "features": 512, "classes": 1000},
        # sixteen sequences whose next token is scored in serving: one pass over the weights
        {"name": "entropy_score_16", "kind": "entropy", "grads": False, "rows": 16, "features": 4096, "classes": 32000},
        # evaluation of a held-out text, odd number of rows and classes
        {"name": "entropy_score_text", "kind": "entropy", "grads": False, "rows": 4099, "features": 2048, "classes": 65537},
        # the benchmark's batch of images on its fully connected width, over ten thousand labels
        {"name": "entropy_train_batch", "kind": "entropy", "grads": True, "rows": 128, "features": 1024, "classes": 10000},
        # a micro-batch of a few rows on a wide layer: what is written is the weight gradient
        {"name": "entropy_train_few", "kind": "entropy", "grads": True, "rows": 31, "features": 4096, "classes": 32000},
        # nothing a multiple of anything, rows cut out of a wider tensor
        {"name": "entropy_train_odd", "kind": "entropy", "grads": True, "rows": 1003, "features": 997, "classes": 20011, "index": "int32", "strided": True},
        # an ordinary training step over tokens
        {"name": "entropy_train_tokens", "kind": "entropy", "grads": True, "rows": 4096, "features": 2048, "classes": 32768},
        # the largest layer
        {"name": "entropy_train_large", "kind": "entropy", "grads": True, "rows": 8192, "features": 4096, "classes": 131072},
        # a small classifier that learns from another one's five best answers
        {"name": "distill_train_small", "kind": "distill", "grads": True, "rows": 16, "features": 512, "classes": 1000, "top": 5, "temperature": 4.0},
        # the package's default batch on its fully connected width
        {"name": "distill_train_batch", "kind": "distill", "grads": True, "rows": 256, "features": 1024, "classes": 10000, "top": 16, "temperature": 2.0,
         "teacher": "bfloat16"},
        # how far a student is from its teacher on a held-out text, odd sizes
        {"name": "distill_score_odd", "kind": "distill", "grads": False, "rows": 2047, "features": 1544, "classes": 30011, "top": 33, "temperature": 1.0,
         "teacher": "float16", "index": "int32"},
        # a training step over tokens with long lists
        {"name": "distill_train_tokens", "kind": "distill", "grads": True, "rows": 8192, "features": 2048, "classes": 65536, "top": 64, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    """Uniform over the logarithm, any whole number."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    features = _log(rng, 64, 4096)
    if rng.random() < 0.6:      # most layers' widths are whole multiples of something
        features = max(64, features // 64 * 64)
    case = {"kind": rng.choice(["entropy", "distill"]), "grads": rng.random() < 0.65, "rows": _log(rng, 1, 8192), "features": features,
            "classes": _log(rng, 100, 131072), "index": rng.choice(sorted(INDEX)), "strided": rng.random() < 0.25}
    if case["kind"] == "distill":
        case.update(top=_log(rng, 1, 64), temperature=rng.choice([1.0, 2.0, 4.0]), teacher=rng.choice(sorted(TEACHER)))
    return case


def _inputs(case, seed):
    """Activations and weights as quantisers leave them (most values far from the ends of int8), logits a few units wide, the
    class to be learnt ahead of the others by more on some rows than on others, up to about even odds; some rows do not count,
    some lists are short."""
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    n, f, v = case["rows"], case["features"], case["classes"]
    index = INDEX[case.get("index", "int64")]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=DEVICE)

    w = (30.0 * normal(v, f)).round_().clamp_(-127, 127).to(torch.int8)
    learnt = (v * uniform(n) ** 2).long().clamp_(max=v - 1)       # frequent and rare classes
    lead = (math.log(v) + 3.0) / 2.5 * uniform(n, 1) / math.sqrt(f)
    act = (30.0 * normal(n, f) + lead * w[learnt].float()).round().clamp_(-127, 127).to(torch.int8)
    if case.get("strided"):
        wide = torch.zeros((n, f + 24), dtype=torch.int8, device=DEVICE)
        wide[:, 8:8 + f] = act
        act = wide[:, 8:8 + f]
    e = round(math.log2(2.5 / (900.0 * math.sqrt(f))))
    s = {"act": act, "w": w,
         "ea": torch.full((1,), -5, dtype=torch.int32, device=DEVICE), "ew": torch.full((1,), e + 5, dtype=torch.int32, device=DEVICE)}
    if case["kind"] == "entropy":
        target = learnt.clone()
        target[uniform(n) < 0.05] = IGNORED
        s["target"] = target.to(index)
    else:
        k = min(case["top"], v)
        step = 1 + (uniform(n, k) * (v // k)).long().clamp_(max=v // k - 1)
        step[:, 0] = 0
        top_idx = (learnt[:, None] + step.cumsum(1)) % v           # distinct: the steps add up to less than v
        top_val = 10.0 + normal(n, 1) - (0.4 * uniform(n, k)).cumsum(1)
        length = torch.where(uniform(n) < 0.15, (uniform(n) * (k + 1)).long(), k)
        top_idx[torch.arange(k, device=DEVICE)[None, :] >= length[:, None]] = -1
        s["top_val"] = top_val.to(TEACHER[case.get("teacher", "float32")])
        s["top_idx"] = top_idx.to(index)
        s["temperature"] = float(case["temperature"])
    # the weight of each row's loss: the mean over the rows, some samples counting for less
    s["weight"] = torch.where(uniform(n) < 0.25, 0.5, 1.0) / n
    return s


def prepare(case, seed):
    return dict(_inputs(case, seed), kind=case["kind"], grads=bool(case["grads"]))


def _run_own(s):
    from niti_amd import ops
    if s["kind"] == "entropy":
        loss, lse, state = ops.vocab_loss(s["act"], s["w"], s["ea"], s["ew"], s["target"], ignore_index=IGNORED)
    else:
        loss, lse, state = ops.vocab_distill(s["act"], s["w"], s["ea"], s["ew"], s["top_val"], s["top_idx"], temperature=s["temperature"])
    if not s["grads"]:
        return loss, lse
    d_act, d_w = ops.vocab_backward(s["act"], s["w"], s["ea"], s["ew"], state, s["weight"])
    return loss, d_act, d_w


def _run_plain(s):
    a, w = s["act"].float(), s["w"].float()
    temperature = s.get("temperature", 1.0)
    z = (a @ w.t()) * (torch.exp2((s["ea"] + s["ew"]).float()) / temperature)
    m = z.amax(1, keepdim=True)
    z -= m
    p = torch.exp(z)
    denom = p.sum(1, keepdim=True)
    log_denom = torch.log(denom)
    lse = (log_denom + m).squeeze(1)
    if s["kind"] == "entropy":
        idx = s["target"].long()[:, None]
        used = idx != IGNORED
        t = used.float()
        entropy = torch.zeros_like(lse)
    else:
        idx = s["top_idx"].long()
        used = idx >= 0
        top = torch.where(used, s["top_val"].float() / temperature, -torch.inf)
        top = torch.where(used, top - top.amax(1, keepdim=True), -torch.inf)
        t = torch.exp(top)
        norm = t.sum(1, keepdim=True)
        t = torch.where(norm > 0, t / norm, 0.0)
        entropy = torch.where(t > 0, t * torch.log(t), 0.0).sum(1)
    at = torch.where(used, idx, 0)
    loss = temperature ** 2 * (entropy + (t * (log_denom - z.gather(1, at))).sum(1))
    if not s["grads"]:
        return loss, lse
    g = p / denom * used.any(1, keepdim=True)
    g.scatter_add_(1, at, -t)
    g *= temperature * s["weight"][:, None]
    d_act = (g @ w) * torch.exp2(s["ew"].float())
    d_w = (g.t() @ a) * torch.exp2(s["ea"].float())
    return loss, d_act.to(torch.bfloat16), d_w.to(torch.bfloat16)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    n, f, v = case["rows"], case["features"], case["classes"]
    flops, moved = 2.0 * n * f * v, float(n * f + v * f + 8 * n)
    moved += n * INDEX[case.get("index", "int64")].itemsize if case["kind"] == "entropy" else \
        n * case["top"] * (INDEX[case.get("index", "int64")].itemsize + TEACHER[case.get("teacher", "float32")].itemsize)
    if case["grads"]:       # the logits, and a product for each of the two gradients
        flops *= 3.0
        moved += 2.0 * (n * f + v * f)
    return {"bytes": moved, "flops": flops}


def exact(case, seed):
    """From the definition in 64 bits: the loss of each row by its log-probabilities, the gradients by differentiating their sum."""
    s = _inputs(case, seed)
    a = torch.ldexp(s["act"].double(), s["ea"]).requires_grad_(case["grads"])
    w = torch.ldexp(s["w"].double(), s["ew"]).requires_grad_(case["grads"])
    temperature = case.get("temperature", 1.0)
    losses, lses, pieces = [], [], 1024         # rows at a time: the logits of all of them in 64 bits are not wanted at once
    for i in range(0, case["rows"], pieces):
        z = torch.matmul(a[i:i + pieces], w.t()) / temperature
        lse = torch.logsumexp(z, 1)
        logp = z - lse[:, None]
        if case["kind"] == "entropy":
            target = s["target"][i:i + pieces].long()
            counted = target != IGNORED
            loss = -logp[torch.arange(len(target), device=DEVICE), target.clamp(min=0)] * counted
        else:
            idx = s["top_idx"][i:i + pieces].long()
            teacher = torch.zeros_like(z)
            value = s["top_val"][i:i + pieces].double().div(temperature).exp() * (idx >= 0)
            value = value / value.sum(1, keepdim=True).clamp(min=1e-300)
            teacher.scatter_add_(1, idx.clamp(min=0), value)
            loss = temperature ** 2 * (torch.xlogy(teacher, teacher) - teacher * logp).sum(1)
        losses.append(loss.detach())
        lses.append(lse.detach())
        if case["grads"]:
            (loss * s["weight"][i:i + pieces].double()).sum().backward()
        del z, logp, loss, lse
    if not case["grads"]:
        return torch.cat(losses), torch.cat(lses)
    return torch.cat(losses), a.grad, w.grad
