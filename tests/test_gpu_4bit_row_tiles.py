"""4-bit products whose blocks take one, two or four tiles of 16 rows, with a last block that is not full, against float64."""
import pytest
import torch

import attention_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Q():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import q4
    return q4


# (rows, columns, group, zero points, vectors): 512 tiles of rows and 2048 are where blocks of two and of four begin
CASES = [(rows, cols, group, zeros, tokens) for rows in (8176, 8193, 32752, 32769, 40025)
         for cols, group, zeros, tokens in ((200, 32, True, 1), (333, 64, False, 3), (129, 128, True, 5), (700, 256, False, 17))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rows(Q, case, dtype):
    rows, cols, group, zeros, tokens = case
    g = torch.Generator().manual_seed(rows + cols)
    packed = torch.randint(0, 256, (rows, (cols + 1) // 2), generator=g, dtype=torch.uint8)
    groups = -(-cols // group)
    scales = (torch.randn(rows, groups, generator=g) * 0.1).to(dtype)
    z = torch.randint(0, 16, (rows, groups), generator=g, dtype=torch.uint8) if zeros else None
    x = torch.randn(tokens, cols, generator=g).to(dtype)
    f = Q.Q4Format(packed.cuda(), scales.cuda(), z.cuda() if zeros else None, cols=cols, group=group)
    y = f.matvec(x.cuda())
    w, mag = O.q4_weights(packed, scales, z, cols, group)
    want = x.double() @ w.t()
    # a group's sums in order, the groups' sums in order, the waves' sums in order; x is exact
    tol = O.half_step(dtype) * want.abs() + (max(group, 128) + cols / 128 + 32) * O.E32 * (x.double().abs() @ mag.t())
    O.check("y", y, want, tol)
    assert torch.equal(f.matvec(x.cuda()), y)
