"""Attention in float16 where one key, as a first key often does, has a score far above all others and a value near 0: the result
is then made of thousands of weights that lie below float16's normal numbers next to it.

The kernels round weights to the type as multiples of themselves: spmm_attn_window as 2^7 times what they are next to the largest
so far, and once; spmm_attn_paged as 2^15 times, in two parts.  With u = 2^-11 a weight w (the largest being 1) is off by
at most u w + 2^-32, or u^2 w + 2^-40 (half of float16's smallest number, 2^-25, over the multiple).  These are taken to add up
here: the keys are alike.  A result is rounded once more (u), or to a multiple of 2^-24.  In 32 bits, e = 2^-24: a weight is off by
2 (d + 12) e times its score's magnitude on either side, a sum of n by n e (its terms alike).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U, E32 = 2.0 ** -11, 2.0 ** -24
N, H, HK, D = 20000, 4, 2, 64


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import attention
    return attention


def make(nats, where):
    """Every query's score with key `where` is `nats`, with the others 0 but for a hundredth; values there 0, elsewhere about 1."""
    g = torch.Generator().manual_seed(1)
    q, k = torch.zeros(40, H, D), torch.randn(N, HK, D, generator=g) * 0.01
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[where, :, 0] = nats
    v = 1 + 0.25 * torch.randn(N, HK, D, generator=g)
    v[where] = 0.0
    return q.half(), k.half(), v.half()


def expected(q, k, v, off, relative):
    q, k, v = q.double(), k.double().repeat_interleave(H // HK, 1), v.double().repeat_interleave(H // HK, 1)
    out, tol, lse = [], [], []
    for h in range(H):
        s = q[:, h] @ k[:, h].t() / math.sqrt(D)
        seen = torch.arange(N)[None] <= torch.arange(len(q))[:, None] + N - len(q)
        s = torch.where(seen, s, -math.inf)
        top = s.amax(1, keepdim=True)
        w = torch.exp(s - top)
        total = w.sum(1, keepdim=True)
        o = w @ v[:, h] / total
        arithmetic = 4 * (D + 12) * E32 * top.abs() + 2 * N * E32
        out.append(o)
        tol.append((U + relative + arithmetic) * o.abs() + off * seen.double() @ v[:, h].abs() / total + 2.0 ** -25)
        lse.append(torch.logsumexp(s, 1))
    return torch.stack(out, 1), torch.stack(tol, 1), torch.stack(lse, 1)


CASES = [(nats, where) for nats in (9.0, 13.5, 15.5, 17.6) for where in (0, 7777, N - 100)]


@pytest.mark.parametrize("nats,where", CASES)
def test_window(A, nats, where):
    q, k, v = make(nats, where)
    out, lse = A.window_attention(q[None].cuda(), k[None].cuda(), v[None].cuda())
    want, tol, wl = expected(q, k, v, 2.0 ** -32, U)
    assert ((out[0].cpu().double() - want).abs() <= tol).all()
    assert ((lse[0].cpu().double() - wl).abs() <= 4 * (D + 12) * E32 * nats + N * E32).all()


@pytest.mark.parametrize("nats,where", CASES)
def test_paged(A, nats, where):
    q, k, v = make(nats, where)
    page = 16
    pages = lambda t: t.reshape(N // page, page, HK, D).cuda()
    table = torch.arange(N // page, dtype=torch.int32)[None].cuda()
    out, lse = A.paged_attention(q[-1:].cuda(), pages(k), pages(v), table, torch.tensor([N], dtype=torch.int32).cuda())
    want, tol, wl = expected(q[-1:], k, v, 2.0 ** -40, U * U)
    assert ((out.cpu().double() - want).abs() <= tol).all()
    assert ((lse.cpu().double() - wl).abs() <= 4 * (D + 12) * E32 * nats + N * E32).all()


@pytest.mark.parametrize("nats", [13.5, 15.5, 17.0])
def test_paged_in_one_part(A, nats):
    """So many sequences that none is cut: a wave that has the first key has a quarter of all the others."""
    q, k, v = make(nats, 0)
    n, page, batch = 2000, 16, 1100
    pages = lambda t: t[:n].reshape(n // page, page, HK, D).cuda()
    table = torch.arange(n // page, dtype=torch.int32)[None].cuda().expand(batch, n // page)
    out, lse = A.paged_attention(q[:1].expand(batch, H, D).cuda(), pages(k), pages(v), table, torch.full((batch,), n, dtype=torch.int32).cuda())
    s = (q[0].double()[:, None] * k[:n].double().repeat_interleave(H // HK, 1).transpose(0, 1)).sum(-1) / math.sqrt(D)       # [H, n]
    w = torch.softmax(s, 1)
    vv = v[:n].double().repeat_interleave(H // HK, 1).transpose(0, 1)                                                        # [H, n, D]
    want = (w[..., None] * vv).sum(1)
    tol = (U + U * U + 4 * (D + 12) * E32 * nats + 2 * n * E32) * want.abs() + 2.0 ** -40 * vv.abs().sum(1) + 2.0 ** -25
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_first_keys_of_a_window(A):
    """Under a window, the first key dominating: 3000 tokens, each of a thousand far below it."""
    n, window = 3000, 1000
    g = torch.Generator().manual_seed(2)
    q, k = torch.zeros(n, H, D), torch.zeros(n, HK, D)
    q[..., 0] = 8.0
    k[0, :, 0] = 16.0
    v = 1 + 0.25 * torch.randn(n, HK, D, generator=g)
    v[0] = 0.0
    q, k, v = q.half(), k.half(), v.half()
    out, _ = A.window_attention(q[None].cuda(), k[None].cuda(), v[None].cuda(), window, 1)
    vv = v.double().repeat_interleave(H // HK, 1)
    c = torch.cat((torch.zeros(1, H, D, dtype=torch.float64), vv.cumsum(0)))
    i = torch.arange(n)
    lo = (i - window + 1).clamp(min=1)
    e = math.exp(-16.0)
    total = 1 + e * (i - lo + 1).clamp(min=0)[:, None, None]
    want = e * (c[i + 1] - c[lo]) / total
    tol = (2 * U + 4 * (D + 12) * E32 * 16 + 2 * n * E32) * want.abs() + 2.0 ** -32 * window * 2 + 2.0 ** -25
    assert ((out[0].cpu().double() - want).abs() <= tol)[1:].all()
