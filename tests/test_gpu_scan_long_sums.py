"""Gradients that are sums over all tokens (A, D, dt_bias), of long sequences that
are one run: partial sums in fp32 are of 256 tokens at most, so that what rounding
leaves of the sums does not grow with the length.

Rates of zero keep a state as it is: a first state (B of 0) stays 1 and its adjoint 1,
so that the gradient of its rate is the sum of the steps; a second state (B of 1) has
the adjoint 1 and no C, so that a step's gradient is x.  All terms of a sum are equal
and exact; adding them one by one in fp32 would be off by up to T U of the sum."""
import pytest
import torch

from uttt_amd.state_space import selective_scan

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


def sums(B, T, D, G, N, dtype, values, cu=None):
    """Gradients of A's first column, of D and of dt_bias, and their exact values."""
    seqs = B if cu is None else len(cu) - 1
    step = torch.tensor([values[d % len(values)] for d in range(D)], device="cuda")
    v = step.to(dtype)
    x, dt = v.expand(B, T, D), step.expand(B, T, D)
    A = torch.zeros(D, N, device="cuda", requires_grad=True)
    skip = torch.zeros(D, device="cuda", requires_grad=True)
    bias = torch.zeros(D, device="cuda", requires_grad=True)
    Bm = torch.zeros(B, T, G, N, dtype=dtype, device="cuda")
    Bm[..., 1] = 1
    C = torch.zeros_like(Bm)
    h0 = torch.zeros(seqs, D, N, device="cuda")
    h0[..., 0] = 1
    offsets = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    y, h = selective_scan(x, dt, A, Bm, C, D=skip, dt_bias=bias, initial_state=h0, output_final_state=True,
                          cu_seqlens=offsets)
    got = torch.autograd.grad([y, h], [A, skip, bias], [torch.ones_like(y), torch.ones_like(h)])
    tokens = B * T if cu is None else cu[-1] - cu[0]
    return (got[0][:, 0], got[1], got[2]), (tokens * step.double(), tokens * v.double(), tokens * v.double())


def near(got, want, names=("A", "D", "dt_bias")):
    for n, g, w in zip(names, got, want):
        # 256 additions of a partial sum, the sums of the partial sums and their
        # rounding to fp32: 256 + 16 half steps
        off = ((g.double() - w).abs() / w.abs()).max().item()
        assert off <= (256 + 16) * U, f"{n}: {off / U:.1f} half steps"


VALUES = [0.1, 0.3, 0.7, 1.1, 1.3, 1.7]


@pytest.mark.parametrize("N", [2, 8, 16, 24, 40])
@pytest.mark.parametrize("T", [256, 272, 5000, 16384])
def test_whole_sequences(N, T):
    """So many groups that a sequence is one run whatever its length."""
    near(*sums(16, T, 96, 96, N, F32, VALUES))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_runs_of_a_split_sequence(dtype):
    near(*sums(4, 20000, 64, 64, 4, dtype, VALUES))


def test_packed():
    """Long runs, short ones, empty ones and tokens of no sequence."""
    cu = [40, 30000, 30000, 30001, 30300, 61000]
    near(*sums(1, 61100, 128, 128, 16, BF16, VALUES, cu))


def test_channels_of_one_group():
    """Several channels of a thread's sums in a workgroup, the last one's partly empty."""
    near(*sums(150, 2100, 300, 5, 16, F32, VALUES))
