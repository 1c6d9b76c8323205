"""No operator returns a result that has lost its gradient without a word: with gradients on, tensors that require
one are refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import attention, q4
    return attention, q4


def calls(A, Q):
    q, k, v = (torch.randn(1, 20, 2, 16, generator=torch.Generator().manual_seed(i)).cuda() for i in (1, 2, 3))
    table, lengths = torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.full((1,), 20, dtype=torch.int32).cuda()
    f = Q.Q4Format(torch.zeros(8, 64, dtype=torch.uint8).cuda(), torch.ones(8, 1).cuda())
    pages = torch.zeros(2, 20, 2, 16).cuda()
    return [
        (A.window_attention, [q, k, v], (0, 1, 2)),
        (A.paged_attention, [q[0, :1], k, v, table, lengths], (0, 1, 2)),
        (A.cache_append, [k[0, :1], v[0, :1], pages, pages.clone(), table, lengths], (0, 1, 2, 3)),
        (f.matvec, [torch.randn(3, 128).cuda()], (0,)),
    ]


def test_tensors_that_require_gradients(mods):
    for call, args, which in calls(*mods):
        call(*args)
        for i in which:
            x = [t.clone().requires_grad_(j == i and t.is_floating_point()) for j, t in enumerate(args)]
            with pytest.raises(ValueError, match="requires a gradient"):
                call(*x)
            with torch.no_grad():
                call(*x)
            call(*[t.detach() for t in x])


def test_scales_that_require_gradients(mods):
    Q = mods[1]
    with pytest.raises(ValueError, match="requires a gradient"):
        Q.Q4Format(torch.zeros(8, 64, dtype=torch.uint8).cuda(), torch.ones(8, 1).cuda().requires_grad_())


def test_second_derivatives(mods):
    """A backward pass that is to be differentiated runs with gradients on."""
    A = mods[0]
    q, k, v = (torch.randn(1, 20, 2, 16, generator=torch.Generator().manual_seed(i)).cuda() for i in (1, 2, 3))
    out, lse = A.window_attention(q, k, v)
    A.window_attention_backward(q, q, k, v, out, lse)
    for i in range(4):
        x = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, q, k, v))]
        with pytest.raises(ValueError, match="requires a gradient"):
            A.window_attention_backward(*x, out, lse)
        with torch.no_grad():
            A.window_attention_backward(*x, out, lse)


def test_an_autograd_function_around_them(mods):
    """How a training program ties them to autograd: forward and backward of a Function run with gradients off."""
    A = mods[0]

    class Attention(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v):
            out, lse = A.window_attention(q, k, v, 10, 1)
            ctx.save_for_backward(q, k, v, out, lse)
            return out

        @staticmethod
        def backward(ctx, dout):
            return A.window_attention_backward(dout.contiguous(), *ctx.saved_tensors, 10, 1)

    q, k, v = (torch.randn(1, 40, 2, 16, generator=torch.Generator().manual_seed(i)).cuda().requires_grad_() for i in (1, 2, 3))
    out = Attention.apply(q, k, v)
    w = torch.randn(1, 40, 2, 16, generator=torch.Generator().manual_seed(4)).cuda()
    got = torch.autograd.grad((out * w).sum(), (q, k, v))
    with torch.no_grad():
        o, l = A.window_attention(q, k, v, 10, 1)
        want = A.window_attention_backward(w, q, k, v, o, l, 10, 1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
