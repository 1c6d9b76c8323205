"""stream=0 is the null stream, and what a call allocates belongs to it like that of a call on the current one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import attention, q4
    return attention, q4


def calls(A, Q):
    q, k, v = (torch.randn(1, 500, 4, 64, generator=torch.Generator().manual_seed(i)).cuda() for i in (1, 2, 3))
    out, lse = A.window_attention(q, k, v, 40, 2)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.full((1,), 500, dtype=torch.int32).cuda()
    f = Q.Q4Format(torch.zeros(4096, 64, dtype=torch.uint8).cuda(), torch.ones(4096, 1).cuda())
    x = torch.randn(16, 128).cuda()
    return [
        lambda **kw: A.window_attention(q, k, v, 40, 2, **kw),
        lambda **kw: A.window_attention_backward(q, q, k, v, out, lse, 40, 2, **kw),
        lambda **kw: A.paged_attention(q[0, :1], k, v, table, lengths, **kw),
        lambda **kw: (f.matvec(x, **kw),),
        lambda **kw: (Q.Q4Format(torch.zeros(4096, 64, dtype=torch.uint8).cuda(), torch.ones(4096, 1).cuda(), **kw)._layout,),
    ]


def owner(t):
    """The stream that the allocator keeps a tensor's memory for."""
    for seg in torch.cuda.memory_snapshot():
        if seg["address"] <= t.data_ptr() < seg["address"] + seg["total_size"]:
            return seg["stream"]


def test_allocations_belong_to_it(mods):
    side = torch.cuda.Stream()
    for call in calls(*mods):
        want = [t.clone() for t in call()]
        torch.cuda.synchronize()
        res = call(stream=0)
        assert all(torch.equal(a, b) for a, b in zip(res, want))
        assert all(owner(t) == 0 for t in res)
        res = call(stream=side.cuda_stream)
        assert all(owner(t) == side.cuda_stream for t in res)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_in_the_context_of_another_stream(mods):
    """The handle says where the work goes, whatever the current stream; rows that the call fills by itself too."""
    A = mods[0]
    side = torch.cuda.Stream()
    q, k, v = (torch.randn(300, 4, 64, generator=torch.Generator().manual_seed(i)).cuda() for i in (1, 2, 3))
    cu = torch.tensor([0, 200], dtype=torch.int32).cuda()
    want, wl = A.window_attention(q, k, v, 40, 2, cu_q=cu)
    grads = A.window_attention_backward(q, q, k, v, want, wl, 40, 2, cu_q=cu)
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(side):
            given, gdq = torch.full_like(wl, 7.0), torch.full_like(q, 7.0)
        side.synchronize()
        with torch.cuda.stream(side):
            out, _ = A.window_attention(q, k, v, 40, 2, cu_q=cu, lse=given, stream=0)
            dq, dk, dv = A.window_attention_backward(q, q, k, v, want, wl, 40, 2, cu_q=cu, dq=gdq, stream=0)
        torch.cuda.default_stream().synchronize()
        assert torch.equal(out, want) and torch.equal(dk, grads[1]) and torch.equal(dv, grads[2]) and torch.equal(dq[:200], grads[0][:200])


def test_what_is_no_handle(mods):
    A = mods[0]
    q = torch.randn(1, 20, 2, 16).cuda()
    for bad in (True, 1.5, "0"):
        with pytest.raises(TypeError, match="stream"):
            A.window_attention(q, q, q, stream=bad)
