"""Gradients of window attention in float16 where they are small, large, or of many keys, against float64.

The kernels round P and dS to the element type for dv and dk, and dS into two parts for dq.  Float16 has normal numbers down
to 2^-14 only, so both are brought into its range by powers of two that are taken out of the 32-bit sums again: P by
2^12, dS by a factor for every sum that keeps the largest |dS| met so far in it at 2^7 or more.  With u = 2^-11 an entry is then
off by at most

    P:   u P + 2^-37                          (half of the smallest number, 2^-25, over 2^12)
    dS:  u |dS| + 2^-32 max |dS|              (2^-25 over 2^7; the maximum over the entries of the sum)
         and u^2 |dS| + 2^-32 max |dS| in two parts,

and a result is rounded once more (u).  Roundings of different entries are independent, and the largest of each is squared
here, of which the expected square is at most a third; so the root of the sum of these squares bounds the error of a whole
gradient in the norm, with thousands of elements in each.  The 32-bit arithmetic is counted the same way, e = 2^-24: a
weight is off by 2 (d + 12) e times its score's magnitudes and (sqrt(keys) + 40) e for what its row is divided by, dP - D by
(d + 2) e of its magnitudes, a sum over n entries by sqrt(n) e of the sum of their magnitudes.  In dq, D = <dout, out> is off by
what out is, whose elements are rounded and the sum of rounded weights.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U, E32 = 2.0 ** -11, 2.0 ** -24


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import attention
    return attention


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def bounds(q, k, v, do, window, sinks, scale):
    """Gradients in float64 of [rows, heads, d] inputs and the norms that their errors may have."""
    nq, h, d = q.shape
    nk, hk = k.shape[:2]
    p0 = torch.arange(nq, device="cuda")[:, None] + nk - nq
    j0 = torch.arange(nk, device="cuda")[None, :]
    seen = (j0 <= p0) & ((p0 - j0 < window) | (j0 < sinks) if window else torch.ones_like(j0 <= p0))
    inf = torch.tensor(float("inf"), dtype=torch.float64, device="cuda")
    want = {n: torch.zeros(t.shape, dtype=torch.float64, device="cuda") for n, t in (("dq", q), ("dk", k), ("dv", v))}
    var = {n: torch.zeros_like(t) for n, t in want.items()}         # squares of the largest errors
    on, small, mm = seen.double(), 2.0 ** -32, torch.matmul
    for head in range(h):
        g = head // (h // hk)
        qq, kk, vv, dd = (t.cuda().double().contiguous() for t in (q[:, head], k[:, g], v[:, g], do[:, head]))
        s = torch.where(seen, scale * mm(qq, kk.t().contiguous()), -inf)
        p = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
        dp = mm(dd, vv.t().contiguous())
        ds = p * (dp - (p * dp).sum(1, keepdim=True))
        pt, dst, out = p.t().contiguous(), ds.t().contiguous(), mm(p, vv)
        want["dq"][:, head] = scale * mm(ds, kk)
        want["dk"][:, g] += scale * mm(dst, qq)
        want["dv"][:, g] += mm(pt, dd)
        rel = 2 * (d + 12) * E32 * abs(scale) * mm(qq.abs(), kk.abs().t().contiguous()) + (nk ** 0.5 + 40) * E32
        err = rel * ds.abs() + (d + 2) * E32 * p * (mm(dd.abs(), vv.abs().t().contiguous()) + (dd * out).abs().sum(1, keepdim=True))
        off = (dd ** 2 * ((U * out) ** 2 + mm((U * p + rel * p + 2.0 ** -25 * on) ** 2, vv ** 2))).sum(1, keepdim=True)
        two = U * U * ds.abs() + small * ds.abs().amax(1, keepdim=True) * on + err
        one = (U * ds.abs() + small * ds.abs().amax(0, keepdim=True) * on + err).t().contiguous()
        var["dq"][:, head] += scale ** 2 * (mm(two ** 2, kk ** 2) + off * mm(p, kk) ** 2 + nk * E32 ** 2 * mm(ds.abs(), kk.abs()) ** 2)
        var["dk"][:, g] += scale ** 2 * (mm(one ** 2, qq ** 2) + nq * E32 ** 2 * mm(dst.abs(), qq.abs()) ** 2)
        var["dv"][:, g] += mm(((U + rel) * p + 2.0 ** -37 * on).t().contiguous() ** 2, dd ** 2) + nq * E32 ** 2 * mm(pt, dd.abs()) ** 2
    # a result that is rounded, to a multiple of 2^-24 if it is that small
    return want, {n: (var[n] + (U * w + 2.0 ** -25) ** 2).sum().sqrt().item() for n, w in want.items()}


# (queries, keys, heads, key heads, width, window, sinks, scale, factor of dout)
CASES = [
    (3000, 3000, 4, 1, 64, 2048, 0, 0.125, 1e-3), (3000, 3000, 4, 1, 64, 2048, 0, 0.125, 1e-4),
    (2500, 2500, 16, 16, 128, 0, 0, 0.08, 1e-3), (600, 5000, 2, 1, 80, 4000, 4, 0.1, 1e-3),
    (64, 50000, 2, 1, 64, 0, 0, 0.125, 1.0), (64, 50000, 2, 2, 128, 0, 0, 0.08, 1.0),
    (3000, 3000, 2, 1, 64, 1500, 4, 0.125, 1e-2),                   # the first keys' sums in parts
    (500, 500, 2, 2, 64, 4, 0, 0.01, 2.0 ** 13), (1500, 1500, 16, 16, 128, 4, 0, 0.01, 2.0 ** 13),     # dS beyond 65504
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_gradients_keep_their_bits(A, case):
    nq, nk, h, hk, d, window, sinks, scale, size = case
    q, k, v, do = rnd(1, nq, h, d).half(), rnd(2, nk, hk, d).half(), rnd(3, nk, hk, d).half(), (size * rnd(4, nq, h, d)).half()
    args = [t[None].cuda() for t in (q, k, v)]
    out, lse = A.window_attention(*args, window, sinks, scale)
    got = A.window_attention_backward(do[None].cuda(), *args, out, lse, window, sinks, scale)
    want, norms = bounds(q, k, v, do, window, sinks, scale)
    print()
    errors = {n: (x[0].double() - want[n]).norm().item() for n, x in zip(("dq", "dk", "dv"), got)}
    for n, e in errors.items():
        print(f"{n}: error {e:.3g}, bound {norms[n]:.3g}, norm {want[n].norm().item():.3g}")
    assert all(e <= norms[n] for n, e in errors.items())


def test_growing_gradients(A):
    """The factor follows what it meets: dout grows by 2^20 along the sequence, and falls again."""
    n, h, hk, d = 900, 2, 1, 64
    size = torch.exp2(20 - 20 * (torch.arange(n) / (n / 2) - 1).abs() - 14)[:, None, None]
    q, k, v, do = rnd(1, n, h, d).half(), rnd(2, n, hk, d).half(), rnd(3, n, hk, d).half(), (size * rnd(4, n, h, d)).half()
    args = [t[None].cuda() for t in (q, k, v)]
    for window in (0, 100):
        out, lse = A.window_attention(*args, window, 0)
        got = A.window_attention_backward(do[None].cuda(), *args, out, lse, window, 0)
        want, norms = bounds(q, k, v, do, window, 0, d ** -0.5)
        for name, x in zip(("dq", "dk", "dv"), got):
            assert (x[0].double() - want[name]).norm().item() <= norms[name], name


def test_zero_gradients(A):
    q, k, v = (rnd(i, 1, 300, 2, 64).half().cuda() for i in (1, 2, 3))
    out, lse = A.window_attention(q, k, v, 50, 2)
    for g in A.window_attention_backward(torch.zeros_like(q), q, k, v, out, lse, 50, 2):
        assert (g == 0).all()
