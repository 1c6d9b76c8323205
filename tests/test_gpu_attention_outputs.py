"""Which rows of which outputs a call over packed sequences writes: of each tensor that the call allocates every row is
defined, of each that is given only the sequences' own rows are touched."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
NAMES = ("dq", "dk", "dv")


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import attention
    return attention


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def poison():
    """What the allocator hands out next holds NaN."""
    held = [torch.full((n,), math.nan, device="cuda") for n in (64, 256, 1024, 4096, 1 << 14, 1 << 16, 1 << 18) for _ in range(8)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("cuts", [(0, 100, 150), (0,), (0, 0)], ids=str)
@pytest.mark.parametrize("given", [g for n in range(4) for g in itertools.combinations(NAMES, n)], ids=str)
def test_gradients_some_given(A, cuts, given):
    n, rest = cuts[-1], 60
    q, k, v, do = rnd(1, n + rest, 4, 32), rnd(2, n + rest, 2, 32), rnd(3, n + rest, 2, 32), rnd(4, n + rest, 4, 32)
    cu = torch.tensor(cuts, dtype=torch.int32).cuda()
    out, lse = A.window_attention(q, k, v, 20, 2, cu_q=cu)
    ref = A.window_attention_backward(do, q, k, v, out, lse, 20, 2, cu_q=cu)
    mine = {name: torch.full_like(t, 7.0) for name, t in zip(NAMES, (q, k, v)) if name in given}
    poison()
    got = A.window_attention_backward(do, q, k, v, out, lse, 20, 2, cu_q=cu, **mine)
    for name, x, r in zip(NAMES, got, ref):
        assert torch.equal(x[:n], r[:n]) and (x[n:] == (7 if name in given else 0)).all(), name
        assert name not in given or x is mine[name]


@pytest.mark.parametrize("cuts", [(0, 100, 150), (0,), (0, 0)], ids=str)
@pytest.mark.parametrize("given", [g for n in range(3) for g in itertools.combinations(("out", "lse"), n)], ids=str)
def test_forward_some_given(A, cuts, given):
    n, rest = cuts[-1], 60
    q, k, v = rnd(1, n + rest, 4, 32), rnd(2, n + rest, 2, 32), rnd(3, n + rest, 2, 32)
    cu = torch.tensor(cuts, dtype=torch.int32).cuda()
    ref, rl = A.window_attention(q, k, v, 20, 2, cu_q=cu)
    mine = {name: torch.full_like(t, 7.0) for name, t in (("out", ref), ("lse", rl)) if name in given}
    poison()
    out, lse = A.window_attention(q, k, v, 20, 2, cu_q=cu, **mine)
    assert torch.equal(out[:n], ref[:n]) and torch.equal(lse[:n], rl[:n])
    assert (out[n:] == (7 if "out" in given else 0)).all() and (lse[n:] == (7 if "lse" in given else -math.inf)).all()
