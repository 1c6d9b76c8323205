"""A value that is not finite, at a place that is seen, makes its column of the result so, whatever the score there and wherever
the borders of tiles, waves and parts fall; other columns and lse are as without it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TYPES = [BF16, F16, F32]


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import attention
    return attention


def rnd(seed, *shape, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def is_value(x, value):
    return (x.isnan() if math.isnan(value) else x == value).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("nats", [20, 130])
@pytest.mark.parametrize("shape", [(700, 2, 1, 64), (1100, 32, 8, 128), (300, 2, 2, 96)], ids=str)
def test_window(A, dtype, nats, shape):
    """The key's score lies far below the others': its weight is too small for float16, or for float32."""
    n, h, hk, d = shape
    q, k, v = rnd(1, n, h, d, dtype=dtype), rnd(2, n, hk, d, dtype=dtype), rnd(3, n, hk, d, dtype=dtype)
    q[..., 0] = 4.0                                          # the score gets 4 k[0] / sqrt(d)
    q, k, v = (t[None].cuda() for t in (q, k, v))
    for where, value in ((0, math.inf), (37, -math.inf), (130, math.nan), (n - 70, math.inf)):
        kk, vv = k.clone(), v.clone()
        kk[:, where, :, 0] = -nats * d ** 0.5 / 4
        ref, rl = A.window_attention(q, kk, vv)
        vv[:, where, :, 3] = value
        out, lse = A.window_attention(q, kk, vv)
        assert is_value(out[0, where:, :, 3], value), (where, value)
        assert torch.equal(out[0, :where], ref[0, :where]) and torch.equal(lse, rl)
        rest = [c for c in range(d) if c != 3]
        assert torch.equal(out[..., rest], ref[..., rest])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_window_both_signs_and_first_keys(A, dtype):
    """Under a window with first keys: each query by what it sees, both signs together give NaN."""
    n, window, sinks = 600, 90, 5
    q, k, v = (rnd(i, n, 2, 64, dtype=dtype) for i in (1, 2, 3))
    q[..., 0] = 4.0
    k[3, :, 0] = k[200, :, 0] = k[220, :, 0] = -400.0
    v[3, :, 7], v[200, :, 7], v[220, :, 8] = math.inf, -math.inf, -math.inf
    out, lse = (x[0].cpu() for x in A.window_attention(*(t[None].cuda() for t in (q, k, v)), window, sinks))
    i = torch.arange(n)
    assert out[i < 3][..., 7].isfinite().all() and lse.isfinite().all()
    both = (i >= 200) & (i < 290)
    assert out[both][..., 7].isnan().all() and (out[(i >= 3) & ~both][..., 7] == math.inf).all()
    low = (i >= 220) & (i < 310)
    assert (out[low][..., 8] == -math.inf).all() and out[~low][..., 8].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("nats", [20, 130])
@pytest.mark.parametrize("length", [40, 250, 5000])
def test_paged(A, dtype, nats, length):
    h, hk, d, page = 4, 2, 64, 16
    pages = -(-length // page)
    k, v = (rnd(i, pages, page, hk, d, dtype=dtype) for i in (1, 2))
    q = rnd(3, 1, h, d, dtype=dtype)
    q[..., 0] = 4.0
    table = torch.arange(pages, dtype=torch.int32)[None].cuda()
    lengths = torch.tensor([length], dtype=torch.int32).cuda()
    for where, value in ((0, math.inf), (length // 2, -math.inf), (length - 1, math.inf), (length // 3, math.nan)):
        kk, vv = k.clone(), v.clone()
        kk[where // page, where % page, :, 0] = -nats * d ** 0.5 / 4
        args = (q.cuda(), kk.cuda())
        ref, rl = A.paged_attention(*args, vv.cuda(), table, lengths)
        vv[where // page, where % page, :, 3] = value
        out, lse = A.paged_attention(*args, vv.cuda(), table, lengths)
        assert is_value(out[..., 3], value), (where, value)
        rest = [c for c in range(d) if c != 3]
        assert torch.equal(lse, rl) and torch.isfinite(out[..., rest]).all()
        # what the 16-bit remainders of the other weights add is the same, in the same order
        assert torch.equal(out[..., rest], ref[..., rest])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_paged_scores_that_rise(A, dtype):
    """The value that is infinite comes first and the scores rise by hundreds of powers of two after it, in the same wave and
    in others: what is rescaled stays infinite."""
    length, page, d = 400, 16, 64
    k, v = (rnd(i, 25, page, 1, d, dtype=dtype) for i in (1, 2))
    k[..., 0] = torch.arange(400).reshape(25, page, 1).float().mul(4).to(dtype)
    q = torch.zeros(1, 2, d, dtype=dtype)
    q[..., 0] = 4.0
    v[0, 5, 0, 9] = math.inf
    table = torch.arange(25, dtype=torch.int32)[None].cuda()
    for n in (100, 250, 400):
        out, lse = A.paged_attention(q.cuda(), k.cuda(), v.cuda(), table, torch.tensor([n], dtype=torch.int32).cuda())
        assert (out[..., 9] == math.inf).all() and torch.isfinite(out[..., :9]).all() and torch.isfinite(lse).all()
