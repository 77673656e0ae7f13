"""Losses over many classes (ops.vocab_loss, ops.vocab_distill, ops.vocab_backward) against the formulas in 64 bits.

Tolerances, from the kernels' number formats:
  loss, lse   A row's denominator is a sum of float32 terms: a term is 2^x with |relative error| <= 2^-23 (the exponential) plus
              |x| 2^-23 ln 2 (rounding of x, whose weight 2^x makes it count for at most 2^-23 of the denominator's share), and no
              more than 64 additions of 2^-24 each lie between a term and the joined sums, which are doubles.  Relative error of the denominator below
              80 * 2^-24 < 2^-17, hence of its logarithm 2^-17 absolute, times T^2 in a distillation's loss; the result itself is rounded
              to float32, and the softmax of a teacher's values taken in float32 adds 2^-20 of the loss's terms.
  gradients   p - q as float16 (2^-11), row weight times activation as float16 (2^-11), the denominator's 2^-17 and the exponential's: each
              term of a sum is within 2^-9.9 of its value; n additions in float32 add n 2^-24; the result is rounded to bfloat16 (2^-8).  The sums
              over magnitudes come from the oracle.  What float16 cannot hold below 2^-39 is far under these."""
import pytest
import torch

from oracle import vocab_oracle as vo

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return torch.device("cuda:0")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def make(dev, n, f, v, seed=0, spread=3.0):
    g = _gen(dev, 1000 + seed)
    act = torch.randint(-128, 128, (n, f), generator=g, device=dev, dtype=torch.int8)
    w = torch.randint(-128, 128, (v, f), generator=g, device=dev, dtype=torch.int8)
    e = round(float(torch.log2(torch.tensor(spread / (5400.0 * f ** 0.5)))))
    return act, w, -7, e + 7


def make_target(dev, n, v, seed=0, dtype=torch.int64, none=True):
    g = _gen(dev, 2000 + seed)
    t = torch.randint(0, v, (n,), generator=g, device=dev)
    if none and n > 2:
        t[n // 2] = -100
    t[-1] = v - 1
    return t.to(dtype)


def make_teacher(dev, n, v, k, seed=0, value=torch.float32, index=torch.int64):
    g = _gen(dev, 3000 + seed)
    idx = torch.randint(0, v, (n, k), generator=g, device=dev)        # classes named twice among them
    val = (3.0 * torch.randn((n, k), generator=g, device=dev)).to(value)
    length = torch.randint(0, k + 1, (n,), generator=g, device=dev)
    length[::3] = k
    idx[torch.arange(k, device=dev)[None] >= length[:, None]] = -1
    return val, idx.to(index)


def exp_of(e, dev):
    return torch.full((1,), e, dtype=torch.int32, device=dev)


def call(kind, act, w, ea, ew, t, **targets):
    from niti_amd import ops
    a, b = exp_of(ea, act.device), exp_of(ew, act.device)
    if kind == "entropy":
        return ops.vocab_loss(act, w, a, b, targets["target"], targets.get("ignore_index", -100))
    return ops.vocab_distill(act, w, a, b, targets["top_val"], targets["top_idx"], t)


def check_forward(got, want, t, teacher_terms=0.0):
    loss, lse = got[:2]
    el, es = want
    assert loss.dtype == lse.dtype == torch.float32
    assert torch.equal(torch.isnan(loss), torch.isnan(el))
    fine = ~torch.isnan(el)
    tol = t * t * 2.0 ** -17 + 2.0 ** -22 * el.abs() + t * t * 2.0 ** -20 * teacher_terms
    assert bool(((loss.double() - el).abs() <= tol)[fine].all()), float(((loss.double() - el).abs() / tol)[fine].max())
    assert bool(((lse.double() - es).abs() <= 2.0 ** -17 + 2.0 ** -22 * es.abs()).all())


def check_gradients(got, want, n, v):
    for x, e, bound, terms in zip(got, want[:2], want[2:], (v, n)):
        assert x.dtype == torch.bfloat16 and x.shape == e.shape
        assert torch.equal(torch.isnan(x), torch.isnan(e))
        tol = 2.0 ** -8 * e.abs() + (2.0 ** -9.9 + terms * 2.0 ** -24) * bound + 2.0 ** -38 * bound.max()
        err = (x.double() - e).abs()
        assert bool((err <= tol).logical_or(torch.isnan(e)).all()), float((err / tol).nan_to_num(0.0).max())


def run(kind, dev, n, f, v, t=1.0, k=1, seed=0, weight=None, act=None, value=torch.float32, index=torch.int64):
    from niti_amd import ops
    a, w, ea, ew = make(dev, n, f, v, seed)
    a = a if act is None else act
    if kind == "entropy":
        targets = {"target": make_target(dev, n, v, seed, index)}
    else:
        targets = dict(zip(("top_val", "top_idx"), make_teacher(dev, n, v, k, seed, value, index)))
    got = call(kind, a, w, ea, ew, t, **targets)
    terms = 0.0 if kind == "entropy" else (targets["top_val"].double().abs().nan_to_num(0.0).max() / t + 20.0)
    check_forward(got, vo.forward(a, w, ea, ew, t, **targets), t, terms)
    grads = ops.vocab_backward(a, w, exp_of(ea, dev), exp_of(ew, dev), got[2], weight)
    check_gradients(grads, vo.backward(a, w, ea, ew, weight, t, **targets), n, v)
    return got, grads


# few rows (a kernel of its own), the tiles' edges, reductions that end inside a stage or a 16-byte piece
@pytest.mark.parametrize("n,f,v", [
    (1, 1, 1), (1, 1, 2), (1, 16, 1000), (2, 17, 7), (1, 512, 1000), (3, 100, 255), (16, 64, 257), (31, 129, 1000), (32, 128, 256), (33, 128, 256),
    (33, 127, 511), (64, 256, 512), (65, 65, 65), (127, 333, 1021), (128, 1024, 1000), (255, 48, 4100), (256, 256, 256), (257, 257, 257), (300, 1000, 777),
    (1, 4096, 5000), (700, 16, 33), (1024, 32, 5), (2049, 80, 600)])
def test_entropy(dev, n, f, v):
    print("entropy", n, f, v, flush=True)
    run("entropy", dev, n, f, v, seed=n + f + v)


@pytest.mark.parametrize("n,f,v,k,t,value,index", [
    (1, 1, 1, 1, 1.0, torch.float32, torch.int64), (1, 512, 1000, 5, 4.0, torch.float32, torch.int64), (5, 33, 40, 64, 2.0, torch.bfloat16, torch.int32),
    (16, 512, 1000, 8, 4.0, torch.float16, torch.int64), (32, 100, 300, 3, 0.5, torch.float32, torch.int32), (33, 64, 257, 17, 1.0, torch.bfloat16, torch.int64),
    (100, 96, 2000, 33, 2.0, torch.float16, torch.int32), (256, 128, 999, 16, 2.0, torch.bfloat16, torch.int64), (258, 500, 3000, 100, 8.0, torch.float32, torch.int64),
    (3, 64, 5000, 1024, 1.0, torch.float32, torch.int64), (40, 48, 9, 1024, 3.0, torch.float32, torch.int32)])
def test_distill(dev, n, f, v, k, t, value, index):
    print("distill", n, f, v, k, t, flush=True)
    run("distill", dev, n, f, v, t, k, seed=n + f + v + k, value=value, index=index)


@pytest.mark.parametrize("kind", ["entropy", "distill"])
def test_several_pieces_of_the_classes(dev, kind):
    """So many rows that the gradient is made in two and more pieces, the last one of a single class; partial sums of d_act are carried on."""
    for n, v in ((16500, 4097), (16500, 8999)):
        print("pieces", kind, n, v, flush=True)
        run(kind, dev, n, 48, v, t=2.0 if kind == "distill" else 1.0, k=3, seed=v)


@pytest.mark.parametrize("n,f,v", [(20000, 64, 300), (40, 64, 70000), (33, 2000, 100)])
def test_long_reductions_are_cut(dev, n, f, v):
    print("cut", n, f, v, flush=True)
    run("entropy", dev, n, f, v, seed=n)


# few tiles of long reductions: features and classes that end inside a stage, fewer stages than wavefronts and no multiple of them
@pytest.mark.parametrize("n", [1, 17, 32, 33, 65])
@pytest.mark.parametrize("f,v", [(512, 64), (528, 1000), (1041, 333), (1100, 4100), (1552, 65), (2304, 721), (4100, 1500)])
def test_few_tiles_of_long_reductions(dev, n, f, v):
    print("long", n, f, v, flush=True)
    run("entropy", dev, n, f, v, seed=n + f)
    run("distill", dev, n, f, v, t=2.0, k=5, seed=n + v, weight=torch.rand(n, device=dev))


@pytest.mark.parametrize("n", [20, 300])
def test_row_weights(dev, n):
    g = _gen(dev, n)
    each = torch.randn(n, generator=g, device=dev) * 10.0 ** torch.randint(-6, 3, (n,), generator=g, device=dev)
    each[3] = 0.0
    for weight in (each, torch.zeros(n, device=dev), torch.full((1,), -0.37, device=dev), torch.tensor(1e-20, device=dev), torch.full((n,), 3e30, device=dev)):
        print("weights", n, tuple(weight.shape), flush=True)
        run("entropy", dev, n, 80, 400, weight=weight)
        run("distill", dev, n, 80, 400, t=2.0, k=7, weight=weight)


def test_strides_and_alignment(dev):
    """Rows cut out of a wider tensor, at any byte; more leading dimensions than one; the same values give the same bits."""
    from niti_amd import ops
    n, f, v = 42, 96, 500
    act, w, ea, ew = make(dev, n, f, v)
    t = make_target(dev, n, v)
    e = (exp_of(ea, dev), exp_of(ew, dev))
    base = ops.vocab_loss(act, w, *e, t)
    grads = ops.vocab_backward(act, w, *e, base[2])
    for off, pitch in ((0, 96), (1, 97), (16, 128), (8, 120), (3, 1000)):
        wide = torch.randint(-128, 128, (n, pitch + 16), device=dev, dtype=torch.int8)
        a = wide[:, off:off + f]
        a.copy_(act)
        tall = torch.randint(-128, 128, (v, pitch + 16), device=dev, dtype=torch.int8)
        b = tall[:, off:off + f]
        b.copy_(w)
        for x, y in ((a, w), (act, b), (a, b)):
            got = ops.vocab_loss(x, y, *e, t)
            assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
            for p, q in zip(ops.vocab_backward(x, y, *e, got[2]), grads):
                assert p.is_contiguous() and torch.equal(p, q)
    got = ops.vocab_loss(act.view(6, 7, f), w, *e, t.view(6, 7))
    assert got[0].shape == (6, 7) and torch.equal(got[0].view(-1), base[0])
    da, dw = ops.vocab_backward(act.view(6, 7, f), w, *e, got[2], torch.ones(6, 7, device=dev))
    assert da.shape == (6, 7, f) and torch.equal(da.view(n, f), grads[0]) and torch.equal(dw, grads[1])


@pytest.mark.parametrize("n", [5, 70])
def test_rows_without_targets_and_outside_of_the_classes(dev, n):
    from niti_amd import ops
    f, v = 64, 300
    act, w, ea, ew = make(dev, n, f, v)
    e = (exp_of(ea, dev), exp_of(ew, dev))
    none = torch.full((n,), -7, dtype=torch.int64, device=dev)
    loss, lse, state = ops.vocab_loss(act, w, *e, none, ignore_index=-7)
    assert bool((loss == 0).all()) and bool(torch.isfinite(lse).all())
    da, dw = ops.vocab_backward(act, w, *e, state)
    assert bool((da == 0).all()) and bool((dw == 0).all())
    # an ignored class may be one of the classes
    t = make_target(dev, n, v, none=False)
    t[1] = 4
    got = call("entropy", act, w, ea, ew, 1.0, target=t, ignore_index=4)
    check_forward(got, vo.forward(act, w, ea, ew, target=t, ignore_index=4), 1.0)
    assert float(got[0][1]) == 0.0
    check_gradients(ops.vocab_backward(act, w, *e, got[2]), vo.backward(act, w, ea, ew, target=t, ignore_index=4), n, v)
    for wrong in (v, -1, 2 ** 31 - 1, -(2 ** 31)):
        t = make_target(dev, n, v, none=False)
        t[2] = wrong
        loss, _, state = ops.vocab_loss(act, w, *e, t)
        assert bool(torch.isnan(loss[2])) and int(torch.isnan(loss).sum()) == 1
        da, dw = ops.vocab_backward(act, w, *e, state)
        assert bool(torch.isnan(da[2]).all()) and int(torch.isnan(da).any(1).sum()) == 1 and bool(torch.isnan(dw).all())
    t = torch.full((n,), 2 ** 40 + 5, dtype=torch.int64, device=dev)          # not class 5
    assert bool(torch.isnan(ops.vocab_loss(act, w, *e, t)[0]).all())


def test_teacher_values_that_are_not_finite(dev):
    """-inf is a place of weight zero, also where all of a row's are; the type's lowest value is a value; +inf and NaN make the row NaN; an unused
    place's value does not matter."""
    from niti_amd import ops
    n, f, v, k = 9, 64, 300, 4
    act, w, ea, ew = make(dev, n, f, v)
    e = (exp_of(ea, dev), exp_of(ew, dev))
    for value in (torch.float32, torch.bfloat16, torch.float16):
        val, idx = make_teacher(dev, n, v, k, value=value)
        idx = torch.randint(0, v, (n, k), device=dev)
        val[0, 1:] = -torch.inf
        val[1] = -torch.inf
        val[2] = torch.finfo(value).min
        val[3, 0] = torch.finfo(value).min
        val[4, 1] = torch.nan
        val[5, 2] = torch.inf
        idx[6, 1], val[6, 1] = -1, torch.nan
        idx[7, 2], val[7, 2] = -5, torch.inf
        idx[8, 3] = v
        got = ops.vocab_distill(act, w, *e, val, idx)
        want = vo.forward(act, w, ea, ew, top_val=val, top_idx=idx)
        assert torch.isnan(got[0]).tolist() == [i in (4, 5, 8) for i in range(n)]
        assert float(got[0][1]) == 0.0
        check_forward(got, want, 1.0, 30.0)
        da, dw = ops.vocab_backward(act, w, *e, got[2])
        assert bool((da[1] == 0).all()) and torch.isnan(da).any(1).tolist() == [i in (4, 5, 8) for i in range(n)]
        ok = torch.tensor([i not in (4, 5, 8) for i in range(n)], device=dev)
        a, x, y = act[ok], val[ok], idx[ok]
        got = ops.vocab_distill(a, w, *e, x, y)
        check_gradients(ops.vocab_backward(a, w, *e, got[2]), vo.backward(a, w, ea, ew, top_val=x, top_idx=y), a.shape[0], v)


def test_extreme_logits(dev):
    """Logits far apart (a softmax of one class), all equal, and exponents that leave float32's range."""
    from niti_amd import ops
    n, f, v = 40, 64, 300
    act, w, _, _ = make(dev, n, f, v)
    t = make_target(dev, n, v, none=False)
    for ea, ew in ((0, 0), (-60, -60), (30, 30)):
        got = call("entropy", act, w, ea, ew, 1.0, target=t)
        el, es = vo.forward(act, w, ea, ew, target=t)
        assert bool(((got[0].double() - el).abs() <= 2.0 ** -17 + 2.0 ** -22 * el.abs()).all())
        assert bool(((got[1].double() - es).abs() <= 2.0 ** -17 + 2.0 ** -22 * es.abs()).all())
        # a logit of 2^20 and more is a float32 number whose last bit counts in the exponential: gradients at the moderate ones only
        if ea + ew <= 0:
            g = ops.vocab_backward(act, w, exp_of(ea, dev), exp_of(ew, dev), got[2])
            assert bool(torch.isfinite(g[0]).all()) and bool(torch.isfinite(g[1]).all())
            check_gradients(g, vo.backward(act, w, ea, ew, target=t), n, v)
    top = (act.float() @ w.float().t()).argmax(1)
    loss, _, state = call("entropy", act, w, 100, 100, 1.0, target=top)       # 2^200: the largest logit's row is sure of itself
    assert bool((loss == 0).all())
    da, dw = ops.vocab_backward(act, w, exp_of(100, dev), exp_of(100, dev), state)
    assert bool((da == 0).all()) and bool((dw == 0).all())
    one = torch.zeros_like(w)
    got = call("entropy", act, one, -3, -3, 1.0, target=t)
    assert bool(((got[0] - torch.log(torch.tensor(float(v)))).abs() < 1e-5).all())


def test_largest_feature_count(dev):
    """65536 features of -128: a logit's sum is 2^30, and nothing wraps."""
    n, f, v = 2, 65536, 5
    act = torch.full((n, f), -128, dtype=torch.int8, device=dev)
    w = torch.full((v, f), -128, dtype=torch.int8, device=dev)
    w[1], w[2] = 127, 0
    act[1] = 127
    t = torch.tensor([1, 0], device=dev)
    got = call("entropy", act, w, -14, -14, 1.0, target=t)
    check_forward(got, vo.forward(act, w, -14, -14, target=t), 1.0)


def test_no_rows(dev):
    from niti_amd import ops
    act, w, ea, ew = make(dev, 1, 32, 50)
    e = (exp_of(ea, dev), exp_of(ew, dev))
    loss, lse, state = ops.vocab_loss(act[:0], w, *e, torch.empty(0, dtype=torch.int64, device=dev))
    assert loss.shape == lse.shape == (0,)
    da, dw = ops.vocab_backward(act[:0], w, *e, state)
    assert da.shape == (0, 32) and dw.shape == (50, 32) and bool((dw == 0).all())
    loss, _, state = ops.vocab_distill(act[:0].view(0, 3, 32), w, *e, torch.empty((0, 3, 4), device=dev), torch.empty((0, 3, 4), dtype=torch.int32, device=dev))
    assert loss.shape == (0, 3)


def test_gradient_against_differences(dev):
    """Central differences of the loss itself, one int8 value 64 steps up and down: h = 64 2^-9 = 2^-3 of a real value.  Values are at most
    60 2^-9 < 2^-3, so a row's logits move by at most 2^-6; the third derivative of a row's loss along a logit is at most 1, hence the
    truncation h^2 / 6 (2^-3)^3 < 2^-17 for each of the n rows (twice that at T = 2 with its T^2).  Losses are within T^2 2^-17, a
    difference over 2 h = 2^-2 within n T^2 2^-14.  The gradient itself is a bfloat16 number of terms within 2^-9.9."""
    from niti_amd import ops
    n, f, v = 12, 32, 60
    act, w, _, _ = make(dev, n, f, v)
    act, w = act.clamp(-60, 60), w.clamp(-60, 60)
    ea, ew = -9, -9
    t = make_target(dev, n, v)
    val, idx = make_teacher(dev, n, v, 5)
    for kind, targets, temp in (("entropy", {"target": t}, 1.0), ("distill", {"top_val": val, "top_idx": idx}, 2.0)):
        _, _, state = call(kind, act, w, ea, ew, temp, **targets)
        da, dw = ops.vocab_backward(act, w, exp_of(ea, dev), exp_of(ew, dev), state)
        for which in range(6):
            for x, d, r in ((act, da, which), (w, dw, int(t[which % 3]))):
                c = (which * 5) % f
                up, down = x.clone(), x.clone()
                up[r, c] += 64
                down[r, c] -= 64
                pair = [call(kind, *((y, w) if x is act else (act, y)), ea, ew, temp, **targets)[0].double() for y in (up, down)]
                slope = float((pair[0] - pair[1]).sum()) * 4.0
                rows = 1 if x is act else n
                tol = rows * temp ** 2 * (2.0 ** -14 + 2.0 ** -16) + 2.0 ** -8 * abs(slope) + 2.0 ** -9.9 * rows * temp * 2.0 ** -2
                assert abs(slope - float(d[r, c])) <= tol


def test_repeated_calls_and_streams_give_the_same_bits(dev):
    from niti_amd import ops
    for n, f, v in ((8, 256, 4000), (300, 200, 3000), (20000, 32, 300)):
        act, w, ea, ew = make(dev, n, f, v)
        e = (exp_of(ea, dev), exp_of(ew, dev))
        val, idx = make_teacher(dev, n, v, 9)

        def both():
            loss, lse, state = ops.vocab_distill(act, w, *e, val, idx, 2.0)
            return (loss, lse) + ops.vocab_backward(act, w, *e, state)

        base = both()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = both()
        torch.cuda.current_stream().wait_stream(side)
        for x, y, z in zip(base, other, both()):
            assert torch.equal(x, y) and torch.equal(x, z)


def test_in_a_graph(dev):
    """Captured once, replayed on new data between eager calls."""
    from niti_amd import ops
    n, f, v = 100, 128, 2000
    act, w, ea, ew = make(dev, n, f, v)
    e = (exp_of(ea, dev), exp_of(ew, dev))
    t = make_target(dev, n, v)
    weight = torch.rand(n, device=dev)

    def step():
        loss, lse, state = ops.vocab_loss(act, w, *e, t)
        return (loss, lse) + ops.vocab_backward(act, w, *e, state, weight)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        a, b, _, _ = make(dev, n, f, v, seed + 5)
        act.copy_(a)
        w.copy_(b)
        t.copy_(make_target(dev, n, v, seed + 5))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, step()):
            assert torch.equal(x, y)


def test_long_offsets(dev):
    """A weight matrix of more than 2^31 bytes, and a result of more than 2^32: rows behind the boundaries count as the others do."""
    from niti_amd import ops
    n, f, v = 3, 16384, 140000
    g = _gen(dev, 4)
    act = torch.randint(-20, 21, (n, f), generator=g, device=dev, dtype=torch.int8)
    w = torch.empty((v, f), dtype=torch.int8, device=dev)
    for i in range(0, v, 20000):
        w[i:i + 20000] = torch.randint(-20, 21, (min(20000, v - i), f), generator=g, device=dev, dtype=torch.int8)
    t = torch.tensor([0, 131071, v - 1], device=dev)
    e = (exp_of(-8, dev), exp_of(-6, dev))
    loss, lse, state = ops.vocab_loss(act, w, *e, t)
    z = torch.cat([act.double() @ w[i:i + 20000].double().t() for i in range(0, v, 20000)], 1) * 2.0 ** -14
    want = torch.logsumexp(z, 1)
    assert bool(((lse.double() - want).abs() <= 2.0 ** -17 + 2.0 ** -22 * want).all())
    assert bool(((loss.double() - (want - z.gather(1, t[:, None])[:, 0])).abs() <= 2.0 ** -16).all())
    da, dw = ops.vocab_backward(act, w, *e, state)
    p = torch.exp(z - want[:, None])
    p[torch.arange(n, device=dev), t] -= 1.0
    for i in (0, 65536, 131071, 131072, v - 1):
        x = (p[:, i:i + 1].t() @ act.double())[0] * 2.0 ** -8
        bound = (p[:, i:i + 1].abs().t() @ act.double().abs())[0] * 2.0 ** -8
        assert bool(((dw[i].double() - x).abs() <= 2.0 ** -8 * x.abs() + 2.0 ** -9.9 * bound + 2.0 ** -38).all())
    x, bound = torch.zeros((n, f), dtype=torch.float64, device=dev), torch.zeros((n, f), dtype=torch.float64, device=dev)
    for i in range(0, v, 20000):
        x += p[:, i:i + 20000] @ w[i:i + 20000].double() * 2.0 ** -6
        bound += p[:, i:i + 20000].abs() @ w[i:i + 20000].double().abs() * 2.0 ** -6
    assert bool(((da.double() - x).abs() <= 2.0 ** -8 * x.abs() + (2.0 ** -9.9 + v * 2.0 ** -24) * bound).all())


def test_refusals(dev):
    from niti_amd import _lib, ops
    act, w, ea, ew = make(dev, 6, 64, 50)
    e = (exp_of(ea, dev), exp_of(ew, dev))
    t = make_target(dev, 6, 50)
    val, idx = make_teacher(dev, 6, 50, 3)
    _, _, state = ops.vocab_loss(act, w, *e, t)
    _, _, listed = ops.vocab_distill(act, w, *e, val, idx)

    def refused(f, *a, match=None, **k):
        with pytest.raises((RuntimeError, _lib.NitiError), match=match):
            f(*a, **k)

    refused(ops.vocab_loss, act.cpu(), w, *e, t, match="GPU")
    refused(ops.vocab_loss, act.float(), w, *e, t, match="int8")
    refused(ops.vocab_loss, act, w.short(), *e, t, match="int8")
    refused(ops.vocab_loss, act[:, :32], w, *e, t, match="features")
    refused(ops.vocab_loss, act[0], w, *e, t[0], match="features")
    refused(ops.vocab_loss, act, w[:0], *e, t, match="class")
    refused(ops.vocab_loss, act.t().contiguous().t(), w, *e, t, match="contiguous")
    refused(ops.vocab_loss, act[:1].expand(6, 64), w, *e, t, match="overlap")
    refused(ops.vocab_loss, act, w, *e, t[:5], match="target")
    refused(ops.vocab_loss, act, w, *e, t.float(), match="int64 or int32")
    refused(ops.vocab_loss, act, w, e[0].float(), e[1], t, match="exponent")
    refused(ops.vocab_loss, act, w, None, e[1], t, match="exponent")
    refused(ops.vocab_distill, act, w, *e, val[:, :2].contiguous(), idx, match="places")
    refused(ops.vocab_distill, act, w, *e, val.double(), idx, match="float32")
    refused(ops.vocab_distill, act, w, *e, val[:, :0], idx[:, :0], match="places")
    refused(ops.vocab_distill, act, w, *e, val, idx, 0.0, match="temperature")
    refused(ops.vocab_distill, act, w, *e, val, idx, float("nan"), match="temperature")
    refused(ops.vocab_distill, act, w, *e, val, idx, -1.0, match="temperature")
    refused(ops.vocab_distill, act, w, *e, val[:, :1].expand(6, 1025).contiguous(), idx[:, :1].expand(6, 1025).contiguous(), match="1024")
    refused(ops.vocab_backward, act[:5], w, *e, state, match="state")
    listed.top = 1
    refused(ops.vocab_backward, act, w, *e, listed, match="state")
    refused(ops.vocab_backward, act, w, *e, state, torch.ones(5, device=dev), match="grad")
    refused(ops.vocab_backward, act, w, *e, state, torch.ones(6, device=dev).double(), match="grad")
    refused(ops.vocab_backward, act, w, *e, state, torch.ones(6), match="GPU")
    wide = torch.zeros((2, 65552), dtype=torch.int8, device=dev)
    refused(ops.vocab_loss, wide, wide, *e, t[:2], match="features")
