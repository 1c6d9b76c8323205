"""A 4-bit format, what it is made from and a token pipeline may be dropped while work on another stream still reads them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Q():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import q4
    return q4


def weights(seed, rows=4096, cols=4096, group=64):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8).cuda(),
            torch.rand(rows, cols // group, generator=g).cuda(), torch.randint(0, 16, (rows, cols // group), generator=g, dtype=torch.uint8).cuda())


def busy(stream):
    """Some milliseconds of work, so that what follows is not done when the call returns."""
    with torch.cuda.stream(stream):
        x = torch.ones(4096, 4096, device="cuda")
        for _ in range(20):
            x = x @ x * 2.0 ** -12
    return x


@pytest.mark.parametrize("explicit", [True, False])
def test_format_dropped(Q, explicit):
    x = torch.randn(3, 4096, generator=torch.Generator().manual_seed(1)).cuda()
    f = Q.Q4Format(*weights(2), group=64)
    want = f.matvec(x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    held, at = busy(side), f._layout.data_ptr()
    if explicit:
        y = f.matvec(x, stream=side.cuda_stream)
    else:
        with torch.cuda.stream(side):
            y = f.matvec(x)
    size = f._layout.numel()
    del f
    other = torch.zeros(size, dtype=torch.uint8, device="cuda")
    assert other.data_ptr() != at                          # its memory is still in use
    side.synchronize()
    assert torch.equal(y, want)


def test_arguments_dropped(Q):
    x = torch.randn(3, 4096, generator=torch.Generator().manual_seed(1)).cuda()
    w = weights(2)
    want = Q.Q4Format(*w, group=64).matvec(x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    held, at = busy(side), {t.data_ptr() for t in w}
    f = Q.Q4Format(*w, group=64, stream=side.cuda_stream)
    shapes = [(t.shape, t.dtype) for t in w]
    del w
    others = [torch.zeros(s, dtype=d, device="cuda") for s, d in shapes]
    assert not at & {t.data_ptr() for t in others}
    y = f.matvec(x, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(y, want)
    f.matvec(x, stream=0)
    torch.cuda.synchronize()


def test_pipeline_dropped(Q):
    """Its pages as well."""
    from spmm_amd.pipeline import TokenPipeline
    make = lambda: TokenPipeline(*(Q.Q4Format(*weights(i, rows=n * 64, cols=512), group=64) for i, n in ((1, 8), (2, 2), (3, 2))),
                                 heads=8, kv_heads=2, pages=3000)
    table = torch.arange(64, dtype=torch.int32).cuda()[None].contiguous()
    lengths, cu = torch.tensor([1000], dtype=torch.int32).cuda(), torch.tensor([0, 1000], dtype=torch.int32).cuda()
    x = torch.randn(1000, 512, generator=torch.Generator().manual_seed(4)).cuda()
    more = lengths + 1

    def run(p):
        p.prompt(x, cu, table, lengths)
        return p.step(x[:1], table, more)
    want = run(make())
    p, side = make(), torch.cuda.Stream()
    torch.cuda.synchronize()
    held, at, shape = busy(side), {p.k_pages.data_ptr(), p.v_pages.data_ptr()}, p.k_pages.shape
    with torch.cuda.stream(side):
        y = run(p)
    del p
    others = [torch.zeros(shape, device="cuda") for _ in range(2)]
    assert not at & {t.data_ptr() for t in others}
    side.synchronize()
    assert torch.equal(y, want)


def test_captured_on_its_own_stream(Q):
    """A graph captures on a stream of its own: the layout is looked after there, and the replays are right."""
    x = torch.zeros(3, 4096).cuda()
    f = Q.Q4Format(*weights(2), group=64)
    f.matvec(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = f.matvec(x)
    for i in range(3):
        x.copy_(torch.randn(3, 4096, generator=torch.Generator().manual_seed(i)))
        want = f.matvec(x)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    del f
    torch.cuda.synchronize()
    assert torch.zeros(8, device="cuda").sum() == 0
