"""What a call of the losses over many classes takes, without a GPU: memory, limits."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from niti_amd import _lib
    return _lib.lib()


@pytest.mark.parametrize("rows,features", [(20000, 64), (65536, 1024), (1000000, 64), (1000000, 1024), (4000000, 256)])
@pytest.mark.parametrize("classes", [5000, 32000, 300000])
def test_the_backward_workspace_of_many_rows(lib, rows, features, classes):
    """A row's 8 KiB of the gradient, 2 bytes per feature of the activations' copy and 4 of the sums, beside a piece's weights: 256 MiB of their
    copy, 512 of their float32 sums, which a long reduction leaves in several parts whatever the result's type."""
    size = (256, features, 512, features, rows, features, classes)
    row = 8192 + 6 * features
    short, wide = lib.niti_vocab_backward_workspace(*size), lib.niti_vocab_backward_f32_workspace(*size)
    assert rows * 2 * (3000 + features) <= short <= wide <= rows * row + (769 << 20)


def test_calls_beyond_a_grid_are_refused(lib):
    """By the check of the arguments, not by a launch that fails when others have run: NITI_ERR_UNSUPPORTED."""
    buf = (C.c_char * 4096)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 16

    def forward(rows, features, classes):
        return lib.niti_vocab_entropy_i8(p, features, p, features, p, p, rows, features, classes, p, 8, -100, p, p, p, p, 1 << 60, None)

    def backward(rows, features, classes):
        return lib.niti_vocab_backward_i8(p, features, p, features, p, p, rows, features, classes, 1, 1.0, p, None, 0, p, p, p, 1 << 60, None)

    for call in (forward, backward):
        assert call(1 << 26, 64, 100) == 2 and b"rows" in lib.niti_last_error()
        assert call(0x7fffffff, 64, 100) == 2
    assert backward(1 << 25, 1024, 100) == 2 and b"workgroups" in lib.niti_last_error()
    # 2^30 tiles of 256 work-items: a 32-bit number of workgroups, none of work-items
    assert forward(1 << 20, 64, 1 << 24) == 2 and b"workgroups" in lib.niti_last_error()


def _plan(lib, rows, features, classes):
    plan = (C.c_int * 6)()
    assert lib.niti_vocab_plan(rows, features, classes, plan) == 0
    return list(plan)


def test_the_sizes_of_the_gpu_tests_reach_every_kernel(lib):
    """The rules that choose a tile are refitted now and then: none may lose its test by it."""
    from vocab_sizes import SIZES, TILES
    plans = [((kind, n, f, v, k), _plan(lib, n, f, v)) for kind, n, f, v, k in SIZES]
    for kind in ("entropy", "distill"):
        seen = [p for (what, *_), p in plans if what == kind]
        of_logits = set(TILES) - {"short"}       # a tile of the sums alone
        assert {TILES[p[2]] for p in seen} >= {"large", "middle", "short", "small_apart"}, kind
        assert {TILES[p[0]] for p in seen} >= {"large", "middle", "small", "quad"} and {TILES[p[1]] for p in seen} >= {"large", "middle", "small", "quad"}, kind
    assert {TILES[p[0]] for _, p in plans} == of_logits == {TILES[p[1]] for _, p in plans}
    assert {TILES[p[2]] for _, p in plans} == set(TILES)
    large = TILES.index("large")
    tiles = [-(-v // 256) * -(-n // 256) for (_, n, _, v, _), p in plans if p[0] == large]
    assert min(tiles) > 256 and max(tiles) > 4 * 256                                                      # in turn, and more than twice
    assert any(p[2] == large and p[3] < v for (_, _, _, v, _), p in plans)                                # sums over several pieces
    assert any(p[2] == large and p[4] > 1 for _, p in plans) and any(p[5] > 1 for _, p in plans)          # cut reductions
    for name, most in (("large", 0), ("middle", 32), ("quad", 32), ("small_apart", 32), ("few_apart", 128)):   # longer lists than the tile writes
        assert any(p[1] == TILES.index(name) and k > most for (kind, _, _, _, k), p in plans if kind == "distill"), name


def test_plan_refusals(lib):
    plan = (C.c_int * 6)()
    for wrong in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (-1, 1, 1)):
        assert lib.niti_vocab_plan(*wrong, plan) == 1
    assert lib.niti_vocab_plan(1, 1, 1, None) == 1
