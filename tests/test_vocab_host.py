"""Losses over many classes without a GPU: the oracle's gradients against differences of its loss, and what the C ABI refuses."""
import ctypes as C

import pytest
import torch

from oracle import vocab_oracle as vo


def _inputs(n=5, f=12, v=17):
    g = torch.Generator().manual_seed(3)
    act = torch.randint(-128, 128, (n, f), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (v, f), generator=g, dtype=torch.int8)
    target = torch.randint(0, v, (n,), generator=g)
    target[2] = -100
    idx = torch.randint(0, v, (n, 4), generator=g)
    idx[0, 1] = idx[0, 0]
    idx[1, 2:] = -1
    idx[3] = -1
    idx[4] = torch.tensor([1, 5, 9, 16])
    val = torch.randn((n, 4), generator=g)
    weight = torch.randn(n, generator=g)
    return act, w, {"target": target}, {"top_val": val, "top_idx": idx}, weight


@pytest.mark.parametrize("kind,temperature", [("entropy", 1.0), ("distill", 1.0), ("distill", 3.0)])
def test_oracle_gradients_against_differences(kind, temperature):
    """Real-valued activations and weights in the same formulas; central differences of 2^-14 in 64 bits: truncation h^2 / 6 times third
    derivatives of a few units, rounding 2^-52 / h: both below 2^-20."""
    act, w, entropy, distill, weight = _inputs()
    targets = entropy if kind == "entropy" else distill
    a, b = act.double() / 64, w.double() / 64          # |logits| <= 50 or so
    da, dw, _, _ = vo.backward(a, b, 0, 0, weight, temperature, **targets)

    def total(x, y):
        return float((vo.forward(x, y, 0, 0, temperature, **targets)[0] * weight.double()).sum())

    h = 2.0 ** -14
    for x, d in ((a, da), (b, dw)):
        for r in range(x.shape[0]):
            for c in range(0, x.shape[1], 5):
                keep = float(x[r, c])
                x[r, c] = keep + h
                up = total(a, b)
                x[r, c] = keep - h
                down = total(a, b)
                x[r, c] = keep
                assert abs((up - down) / (2 * h) - float(d[r, c])) <= 2.0 ** -20 * (1 + abs(float(d[r, c])))


def test_oracle_agrees_with_torch():
    act, w, entropy, distill, _ = _inputs()
    z = act.double() @ w.double().t() * 2.0 ** -10
    loss, lse = vo.forward(act, w, -6, -4, **entropy)
    want = torch.nn.functional.cross_entropy(z, entropy["target"], reduction="none")
    assert torch.allclose(loss, want, rtol=1e-12, atol=1e-12) and torch.allclose(lse, torch.logsumexp(z, 1), rtol=1e-12)
    t = 2.5
    loss, _ = vo.forward(act, w, -6, -4, t, **distill)
    row = distill["top_idx"][4]
    q = torch.softmax(distill["top_val"][4].double() / t, 0)
    want = t * t * (q * (torch.log(q) - torch.log_softmax(z[4] / t, 0)[row])).sum()
    assert abs(float(loss[4] - want)) < 1e-12 and float(loss[3]) == 0.0


def test_refusals_without_a_gpu():
    from niti_amd import _lib
    lib = _lib.lib()
    buf = (C.c_char * 65536)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 16
    n = None

    def entropy(a=p, pa=64, w=p, pw=64, ea=p, ew=p, rows=4, feats=64, classes=9, t=p, tb=8, loss=p, lse=p, state=p, ws=p, wb=65536):
        return lib.niti_vocab_entropy_i8(a, pa, w, pw, ea, ew, rows, feats, classes, t, tb, -100, loss, lse, state, ws, wb, n)

    for name in ("a", "w", "ea", "ew", "t", "loss", "lse", "state"):
        assert entropy(**{name: n}) == 1 and b"null" in lib.niti_last_error(), name
    for name in ("rows", "feats", "classes"):
        assert entropy(**{name: 0}) == 1 and entropy(**{name: -3}) == 1
    assert entropy(pa=63) == 1 and b"hold no" in lib.niti_last_error()
    assert entropy(pw=-64) == 1
    assert entropy(tb=2) == 1 and entropy(state=p + 4) == 1
    assert entropy(feats=65537, pa=70000, pw=70000) == 2 and b"65536" in lib.niti_last_error()
    assert entropy(pa=1 << 22) == 2
    assert entropy(ws=n) == 3 and entropy(wb=16) == 3 and b"workspace" in lib.niti_last_error()

    def distill(v=p, vt=0, i=p, ib=8, top=3, t=2.0, ws=n):
        return lib.niti_vocab_distill_i8(p, 64, p, 64, p, p, 4, 64, 9, v, vt, i, ib, top, t, p, p, p, ws, 0, n)

    assert distill(v=n) == 1 and distill(i=n) == 1 and distill(vt=3) == 1 and distill(top=0) == 1 and distill(ib=1) == 1
    assert distill(t=0.0) == 1 and distill(t=float("inf")) == 1 and b"temperature" in lib.niti_last_error()
    assert distill(top=1025) == 2
    assert distill() == 3

    def backward(state=p, weight=p, weights=4, da=p, dw=p, t=1.0, ws=n, top=1):
        return lib.niti_vocab_backward_i8(p, 64, p, 64, p, p, 4, 64, 9, top, t, state, weight, weights, da, dw, ws, 0, n)

    assert backward(state=n) == 1 and backward(da=n) == 1 and backward(dw=n) == 1
    assert backward(weights=3) == 1 and b"weights" in lib.niti_last_error()
    assert backward(da=p + 2) == 1 and backward(dw=p + 8) == 1 and backward(t=-1.0) == 1 and backward(top=0) == 1
    assert backward() == 3
    assert backward(weight=n, weights=0) == 3


def test_workspace_and_state_sizes():
    from niti_amd import _lib
    lib = _lib.lib()
    assert [lib.niti_vocab_state_words(k) for k in (0, 1, 2, 3, 1024)] == [0, 8, 8, 12, 2052]
    even = lib.niti_vocab_forward_workspace(256, 64, 512, 64, 10, 64, 1000)
    odd = lib.niti_vocab_forward_workspace(256, 64, 513, 65, 10, 64, 1000)
    assert 0 < even and odd >= even + 64 * 1000                  # a copy of the weights
    # the gradient's piece is bounded whatever the classes: two million of them need no 60 GB
    assert lib.niti_vocab_backward_workspace(256, 1024, 512, 1024, 8192, 1024, 2000000) < 2 << 30
    assert lib.niti_vocab_backward_workspace(256, 64, 512, 64, 0, 64, 10) == 0


def test_float32_gradients_refusals_and_workspace():
    from niti_amd import _lib
    lib = _lib.lib()
    buf = (C.c_char * 65536)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 16

    def backward(state=p, weight=p, weights=4, da=p, dw=p, t=1.0, ws=None, top=1):
        return lib.niti_vocab_backward_i8_f32(p, 64, p, 64, p, p, 4, 64, 9, top, t, state, weight, weights, da, dw, ws, 0, None)

    assert backward(state=None) == 1 and backward(da=None) == 1 and backward(dw=None) == 1 and backward(weights=3) == 1
    assert backward(da=p + 4) == 1 and backward(dw=p + 8) == 1 and backward(t=-1.0) == 1 and backward(top=0) == 1
    assert backward() == 3
    # the sums of both gradients pass through it
    size = (256, 64, 512, 64, 10, 64, 1000)
    assert lib.niti_vocab_backward_f32_workspace(*size) >= lib.niti_vocab_backward_workspace(*size) > 0
    assert lib.niti_vocab_backward_f32_workspace(*size) >= 4 * 64 * (10 + 1000)
    assert lib.niti_vocab_backward_f32_workspace(256, 64, 512, 64, 0, 64, 10) == 0
