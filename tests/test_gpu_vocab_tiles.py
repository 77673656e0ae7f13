"""Every tile of the losses over many classes against the oracle, at the tolerances of test_gpu_vocab.py."""
import pytest
import torch

from test_gpu_vocab import run
from vocab_sizes import SIZES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return torch.device("cuda:0")


@pytest.mark.parametrize("kind,n,f,v,k", SIZES)
def test_every_tile(dev, kind, n, f, v, k):
    print("tile", kind, n, f, v, k, flush=True)
    run(kind, dev, n, f, v, t=1.0 if kind == "entropy" else 2.0, k=k, seed=n + k, weight=torch.rand(n, device=dev))
    torch.cuda.empty_cache()
