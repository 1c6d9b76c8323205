"""Products with 4-bit weights on the GPU against float64 (attention_oracle.q4_weights gives the weights and the bound's
magnitudes: the kernel sums (16 + q) x and (16 + zero) x of a group in float32 and takes their difference)."""
import math

import pytest
import torch

import attention_oracle as O

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def Q():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import q4
    return q4


def make(Q, rows, cols, group, zeros, dtype, seed=3):
    g = torch.Generator().manual_seed(seed)
    packed = torch.randint(0, 256, (rows, (cols + 1) // 2), generator=g, dtype=torch.uint8).cuda()
    groups = -(-cols // group)
    scales = (torch.randn(rows, groups, generator=g) * 0.1).to(dtype).cuda()
    z = torch.randint(0, 16, (rows, groups), generator=g, dtype=torch.uint8).cuda() if zeros else None
    return packed, scales, z


def check(x, y, packed, scales, zeros, cols, group):
    w, mag = O.q4_weights(packed, scales, zeros, cols, group)
    xd = x.cpu().double().reshape(-1, cols)
    want = xd @ w.t()
    # a group's sums in order, the groups' sums in order, the waves' sums in order; x is exact
    tol = O.half_step(y.dtype) * want.abs() + (max(group, 128) + cols / 128 + 32) * O.E32 * (xd.abs() @ mag.t())
    O.check("y", y.reshape(-1, y.shape[-1]), want, tol)


CASES = [(1, 1, 32, False, 1), (16, 128, 32, True, 1), (17, 129, 64, False, 2), (512, 512, 32, False, 1),
         (100, 1000, 128, True, 5), (333, 257, 256, False, 16), (64, 4096, 128, True, 3), (2048, 640, 384, True, 17),
         (31, 95, 64, True, 40), (4096, 128, 128, False, 4), (48, 8191, 1024, True, 1)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_matvec(Q, case, dtype):
    rows, cols, group, zeros, tokens = case
    packed, scales, z = make(Q, rows, cols, group, zeros, dtype)
    f = Q.Q4Format(packed, scales, z, cols=cols, group=group)
    x = torch.randn(tokens, cols, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    y = f.matvec(x)
    check(x, y, packed, scales, z, cols, group)
    if tokens == 1:
        assert torch.equal(f.matvec(x[0]), y[0])
    assert torch.equal(f.matvec(x), y)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_nibble_and_position(Q, dtype):
    """Unit vectors pick single weights: each is exact, whatever its place in a tile."""
    rows, cols = 16, 256
    packed, scales, z = make(Q, rows, cols, 64, True, dtype, seed=8)
    scales.fill_(0.5)
    f = Q.Q4Format(packed, scales, z, cols=cols, group=64)
    w, _ = O.q4_weights(packed, scales, z, cols, 64)
    y = f.matvec(torch.eye(cols, dtype=dtype).cuda())
    assert torch.equal(y.cpu().double(), w.t())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides_and_alignment(Q, dtype):
    rows, cols, group = 50, 200, 32
    packed, scales, z = make(Q, rows, cols, group, True, dtype)
    wp = torch.zeros(rows, 117, dtype=torch.uint8).cuda()
    wp[:, 3:103] = packed
    ws = torch.zeros(rows, 11, dtype=dtype).cuda()
    ws[:, 1:8] = scales
    wz = torch.zeros(rows, 9, dtype=torch.uint8).cuda()
    wz[:, 1:8] = z
    f = Q.Q4Format(wp[:, 3:103], ws[:, 1:8], wz[:, 1:8], cols=cols, group=group)
    x = torch.randn(6, 211, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()[:, 5:205]
    out = torch.zeros(6, 57, dtype=dtype).cuda()
    y = f.matvec(x, out=out[:, 3:53])
    check(x, y, packed, scales, z, cols, group)
    assert (out[:, :3] == 0).all() and (out[:, 53:] == 0).all()
    assert torch.equal(f.matvec(x.contiguous()), y)
    assert torch.equal(f.matvec(x[:1].expand(4, cols)), y[:1].expand(4, rows))


def test_float32_parts_are_exact(Q):
    """32-bit vectors over the whole range of exponents: the three parts sum to the value, so a unit weight returns it."""
    cols = 128
    packed = torch.full((1, 64), 0x99, dtype=torch.uint8).cuda()          # q - 8 = 1
    f = Q.Q4Format(packed, torch.ones(1, 1).cuda(), cols=cols)
    g = torch.Generator().manual_seed(2)
    vals = torch.randn(40, generator=g) * torch.exp2(torch.randint(-90, 100, (40,), generator=g).float())
    x = torch.zeros(40, cols)
    x[torch.arange(40), torch.arange(40) * 3] = vals
    y = f.matvec(x.cuda())[:, 0].cpu()
    # 25 x - 24 x in float32
    assert ((y.double() - vals.double()).abs() <= 49 * 3 * O.E32 * vals.double().abs()).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_not_finite_stays_in_its_vector(Q, dtype, value):
    packed, scales, z = make(Q, 40, 300, 32, False, dtype)
    f = Q.Q4Format(packed, scales, z, cols=300, group=32)
    x = torch.randn(7, 300, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    ref = f.matvec(x)
    x[3, 77] = value
    y = f.matvec(x)
    keep = torch.arange(7) != 3
    assert torch.equal(y[keep], ref[keep]) and not torch.isfinite(y[3]).any()


def test_empty(Q):
    f = Q.Q4Format(torch.zeros(5, 0, dtype=torch.uint8).cuda(), torch.zeros(5, 0).cuda())
    assert (f.matvec(torch.zeros(2, 0).cuda()) == 0).all()
    f = Q.Q4Format(torch.zeros(0, 4, dtype=torch.uint8).cuda(), torch.zeros(0, 1).cuda())
    assert f.matvec(torch.zeros(2, 8).cuda()).shape == (2, 0)
    f = Q.Q4Format(torch.zeros(3, 4, dtype=torch.uint8).cuda(), torch.zeros(3, 1).cuda())
    assert f.matvec(torch.zeros(0, 8).cuda()).shape == (0, 3)


def test_graph_and_stream(Q):
    packed, scales, z = make(Q, 300, 512, 64, True, torch.float16)
    f = Q.Q4Format(packed, scales, z, group=64)
    x = torch.zeros(3, 512, dtype=torch.float16).cuda()
    f.matvec(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = f.matvec(x)
    s = torch.cuda.Stream()
    for i in range(4):
        x.copy_(torch.randn(3, 512, generator=torch.Generator().manual_seed(i)).half())
        want = f.matvec(x)
        y.zero_()
        g.replay()
        s.wait_stream(torch.cuda.current_stream())
        other = f.matvec(x, stream=s.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(other, want)
