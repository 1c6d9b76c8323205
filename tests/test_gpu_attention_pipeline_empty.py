"""The token pipeline without tokens: no rows, no sequences, sequences of length 0."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pipe():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd.pipeline import TokenPipeline
    from spmm_amd.q4 import Q4Format
    g = torch.Generator().manual_seed(0)
    w = [Q4Format(torch.randint(0, 256, (n * 32, 64), generator=g, dtype=torch.uint8).cuda(), torch.ones(n * 32, 1).cuda()) for n in (4, 2, 2)]
    return TokenPipeline(*w, 4, 2, pages=8)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def test_nothing(pipe):
    none = torch.zeros(0, 128).cuda()
    table = torch.zeros(0, 3, dtype=torch.int32).cuda()
    assert pipe.prompt(none, ints(0), table, ints()).shape == (0, 128)
    assert pipe.step(none, table, ints()).shape == (0, 128)
    assert pipe.prompt(none, ints(0, 0), ints(1, 2, 3)[None], ints(0)).shape == (0, 128)
    assert (pipe.k_pages == 0).all() and (pipe.v_pages == 0).all()


def test_empty_sequences(pipe):
    x = torch.randn(3, 128, generator=torch.Generator().manual_seed(1)).cuda()
    assert (pipe.prompt(x, ints(0, 0), ints(1, 2, 3)[None], ints(0)) == 0).all()
    assert (pipe.step(x, torch.zeros(3, 2, dtype=torch.int32).cuda(), ints(0, 0, 0)) == 0).all()
    assert (pipe.k_pages == 0).all() and (pipe.v_pages == 0).all()
