"""What a call of the losses over many classes takes, without a GPU: memory, limits."""
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
