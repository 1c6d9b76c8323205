"""Packed calls whose offsets hold no sequence: every row lies behind the last one."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import attention
    return attention


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def test_c_calls_without_sequences(A):
    q, k, v = rnd(1, 50, 4, 32), rnd(2, 70, 2, 32), rnd(3, 70, 2, 32)
    out, lse = torch.full_like(q, 7.0), torch.full((50, 4), 7.0).cuda()
    cu = torch.zeros(1, dtype=torch.int32).cuda()
    d = A._Desc(0, A.F32, 4, 2, 32, 20, 2, 0.2, 0, 50, 70, 1, 0)
    rows = lambda t: A._Rows(t.data_ptr(), 0, *t.stride()[:2])
    stream = torch.cuda.current_stream().cuda_stream
    assert A.lib.spmm_attn_window(d, rows(q), rows(k), rows(v), cu.data_ptr(), cu.data_ptr(), rows(out), lse.data_ptr(), stream) == 0
    assert (out == 0).all() and (lse == -math.inf).all()
    need = A.C.c_size_t()
    assert A.lib.spmm_attn_window_work(d, 1, need) == 0
    work = torch.empty(need.value, dtype=torch.uint8).cuda()
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    assert A.lib.spmm_attn_window_grad(d, rows(q), rows(q), rows(k), rows(v), rows(out), lse.data_ptr(), cu.data_ptr(), cu.data_ptr(),
                                       *map(rows, grads), work.data_ptr(), need.value, stream) == 0
    assert all((g == 0).all() for g in grads)
    d.zero_rest = 0
    out.fill_(7.0)
    assert A.lib.spmm_attn_window(d, rows(q), rows(k), rows(v), cu.data_ptr(), cu.data_ptr(), rows(out), lse.data_ptr(), stream) == 0
    assert (out == 7).all()


def test_keys_without_queries(A):
    """No query rows at all: the keys' gradients are still written."""
    k, cu = rnd(2, 70, 2, 32), torch.zeros(1, dtype=torch.int32).cuda()
    q = torch.zeros(0, 4, 32).cuda()
    out, lse = A.window_attention(q, k, k, 20, 2, cu_q=cu, cu_k=cu)
    dq, dk, dv = A.window_attention_backward(out, q, k, k, out, lse, 20, 2, cu_q=cu, cu_k=cu)
    assert out.shape == dq.shape == (0, 4, 32) and (dk == 0).all() and (dv == 0).all()


@pytest.mark.parametrize("window", [0, 20])
def test_many_rows(A, window):
    """More rows than a part of the first keys' queries, in every block shape."""
    q, k, cu = rnd(1, 3000, 16, 64), rnd(2, 3000, 16, 64), torch.zeros(1, dtype=torch.int32).cuda()
    out, lse = A.window_attention(q, k, k, window, 4, cu_q=cu)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert all((g == 0).all() for g in A.window_attention_backward(q, q, k, k, out, lse, window, 4, cu_q=cu))
