"""The block norms' gradients of weight and scale over millions of rows: partial sums
in fp32 are of 256 rows at most, so that what rounding leaves of a gradient does not
grow with the rows.

All rows are the same (views without memory of their own) and all terms of a sum are
equal; adding them one by one in fp32 would be off by up to `rows` half steps."""
import pytest
import torch

from uttt_amd.norm import norm_after_block, norm_before_block

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def near(got, want, name):
    # 8 roundings of a term; 256 additions of a partial sum and 32 of a workgroup's,
    # the sum of them in 64 bits and its rounding
    off = ((got.double() - want).abs() / want.abs()).max().item()
    assert off <= (8 + 256 + 32 + 2) * U, f"{name}: {off / U:.1f} half steps"


def values(N):
    v = torch.tensor([0.1, 0.3, 0.7, 1.1, 1.3, 1.7], device="cuda")
    return v[torch.arange(N, device="cuda") % 6]


# with one, one, four, four and sixteen or more rows of a workgroup at a time
@pytest.mark.parametrize("rows,N", [(1 << 21, 513), (1500000, 1536), (3000000, 768), (1 << 23, 200), (1 << 25, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_after(rows, N, dtype):
    """x of ones and no eps: x / rms(x) is 1, so that both gradients are sums of dy."""
    x = torch.ones(N, device="cuda", dtype=dtype).expand(rows, N)
    w, s = (torch.ones(N, device="cuda", requires_grad=True) for _ in range(2))
    dy = values(N).to(dtype)
    y = norm_after_block(x, w, scale=s, eps=0.0)
    for name, g in zip(("weight", "scale"), torch.autograd.grad(y, (w, s), dy.expand(rows, N))):
        near(g, rows * dy.double(), name)


@pytest.mark.parametrize("rows,N", [(1 << 21, 513), (3000000, 768)])
def test_before(rows, N):
    """A sum of ones likewise, half of it from x: dw is a sum of dy, and ds, of the sum's
    own gradient alone, one of half of that."""
    x = torch.full((N,), 0.5, device="cuda").expand(rows, N)
    w, s = (torch.ones(N, device="cuda", requires_grad=True) for _ in range(2))
    dy = values(N)
    y, total = norm_before_block(x, x, w, scale=s, eps=0.0)
    near(torch.autograd.grad(y, w, dy.expand(rows, N), retain_graph=True)[0], rows * dy.double(), "weight")
    near(torch.autograd.grad(total, s, dy.expand(rows, N))[0], rows * 0.5 * dy.double(), "scale")
