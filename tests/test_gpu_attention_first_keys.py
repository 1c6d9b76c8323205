"""Gradients of the first keys of a packed batch on either side of the rule that splits their queries into parts: which side a
batch is on is read from the workspace, so a rule that moves empties no case without a word."""
import ctypes as C
import itertools

import pytest
import torch

import attention_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import attention
    return attention


def rnd(seed, *shape, dtype):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# (lengths, rows behind the last, split): one long sequence among short ones has a mean below a block's queries
CASES = [([860] + [4] * 9, 0, False), ([4] * 5 + [860] + [4] * 4, 0, False), ([1500] + [3] * 12, 7, False), ([860, 4], 0, True),
         ([4, 1500, 0, 70], 0, True)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}-{max(c[0])}-{c[2]}")
def test_long_among_short(A, case, dtype):
    lens, rest, split = case
    h, hk, d, window, sinks, n = 4, 2, 64, 40, 4, sum(lens)
    desc = A._Desc(0, A._DTYPES[dtype], h, hk, d, window, sinks, d ** -0.5, len(lens), n + rest, n + rest, 1, 0)
    need = C.c_size_t()
    assert A.lib.spmm_attn_window_work(desc, 1, need) == 0
    plain = A._Desc(0, A._DTYPES[dtype], h, hk, d, window, 0, d ** -0.5, len(lens), n + rest, n + rest, 1, 0)
    least = C.c_size_t()
    assert A.lib.spmm_attn_window_work(plain, 1, least) == 0           # without first keys there are no parts
    assert (need.value > least.value) == split
    q, do = (rnd(i, n + rest, h, d, dtype=dtype) for i in (1, 4))
    k, v = (rnd(i, n + rest, hk, d, dtype=dtype) for i in (2, 3))
    cu = torch.tensor([0] + list(itertools.accumulate(lens)), dtype=torch.int32).cuda()
    out, lse = A.window_attention(q, k, v, window, sinks, cu_q=cu)
    got = A.window_attention_backward(do, q, k, v, out, lse, window, sinks, cu_q=cu)
    at = 0
    for m in lens:
        s = slice(at, at + m)
        r = O.attention(q[s], k[s], v[s], window, sinks)
        O.check("out", out[s], r["out"], r["tol_out"])
        g = O.gradients(r, do[s])
        for name, x in zip(("dq", "dk", "dv"), got):
            O.check(name, x[s], g[name], g["tol_" + name])
        at += m
    assert all((x[at:] == 0).all() for x in (out,) + got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_large_scores_in_16_bits(A, dtype):
    """Scores far beyond the exponential's range, of both signs, with gradients."""
    q, k = (rnd(i, 90, 2, 64, dtype=dtype) * 40 for i in (1, 2))
    v, do = (rnd(i, 90, 2, 64, dtype=dtype) for i in (3, 4))
    out, lse = A.window_attention(q[None], k[None], v[None], 33, 1)
    r = O.attention(q, k, v, 33, 1)
    O.check("out", out[0], r["out"], r["tol_out"])
    O.check("lse", lse[0], r["lse"], r["tol_lse"])
    g = O.gradients(r, do)
    for name, x in zip(("dq", "dk", "dv"), A.window_attention_backward(do[None], q[None], k[None], v[None], out, lse, 33, 1)):
        O.check(name, x[0], g[name], g["tol_" + name])
