"""Attention over pages at the longest lengths: 2^30 - 1 positions a sequence, of pages that all sequences share and whose rows
are one row (strides of 0), so the result is known: the value itself, and lse = score + log(positions)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,kv_heads,length", [(1, 1, 2 ** 30 - 1), (64, 1, 2 ** 30 - 1), (3, 2, 2 ** 29 + 5)], ids=str)
def test_longest(batch, kv_heads, length):
    from spmm_amd import attention as A
    page, d = 2 ** 20, 16
    g = torch.Generator().manual_seed(1)
    k = torch.randn(1, 1, kv_heads, d, generator=g).half().cuda()
    v = torch.tensor([1.0, -2.0, 0.5, 4.0] * (kv_heads * d // 4)).reshape(1, 1, kv_heads, d).half().cuda()
    q = torch.randn(batch, kv_heads, d, generator=g).half().cuda()
    table = torch.zeros(1, 1024, dtype=torch.int32).cuda().expand(batch, 1024)
    lengths = torch.full((batch,), length, dtype=torch.int32).cuda()
    out, lse = A.paged_attention(q, k.expand(1, page, kv_heads, d), v.expand(1, page, kv_heads, d), table, lengths)
    torch.cuda.synchronize()
    # Every weight is 1 and every value a power of two, so a wave's sums, of 2^24 keys at most, are exact; four waves and 256
    # parts are joined with a rounding each.
    tol = (4 + 256) * 2.0 ** -24
    want = v.double().expand(batch, 1, kv_heads, d)[:, 0]
    assert ((out.double() - want).abs() <= want.abs() * (2.0 ** -11 + tol) + 2.0 ** -24).all()
    s = (q.double() * k[:, 0].double()).sum(-1) / math.sqrt(d)
    assert ((lse.double() - s - math.log(length)).abs() <= tol + 2.0 ** -24 * (64 + 20 * s.abs())).all()
