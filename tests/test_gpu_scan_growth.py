"""States that grow (rates above zero, or steps below it): where a run's growth
passes fp32's range, states and adjoints of zero stay zero and small ones become
what the recurrence makes of them, as token by token."""
import pytest
import torch

from state_space_cases import BF16, F32, call, check, check_scan, scan_exact, scan_inputs

pytestmark = pytest.mark.gpu

FRONT, GROWTH, BEHIND = 96, 120, 40   # tokens; runs of 16 at these sizes


def growing(sign, dtype=F32, B=2, N=5, D=6, G=1, seed=0):
    """A first part as usual; a step of -2000 that leaves no state, in 64 bits neither;
    growth by e^{3 to 8} a token without inputs, e^{48} to e^{128} a run and e^{360}
    and more in all; a last part as usual, without gradients."""
    T = FRONT + GROWTH + BEHIND
    a, soft, (dy, dhT) = scan_inputs(B=B, T=T, D=D, N=N, G=G, dtype=dtype, dt_dtype=F32, gate=True, bias=False, soft=False,
                                     state=True, seed=seed)
    gen = torch.Generator().manual_seed(seed)
    a["A"] = sign * (0.5 + 0.5 * torch.rand(D, N, generator=gen)).cuda()
    dt = 0.02 + 0.02 * torch.rand(B, T, D, generator=gen)
    dt[:, FRONT] = -2000.0
    dt[:, FRONT + 1:FRONT + GROWTH] = 6.0 + 2.0 * torch.rand(B, GROWTH - 1, D, generator=gen)
    a["dt"] = (sign * dt).cuda()
    a["x"] = a["x"].clone()
    a["x"][:, FRONT:FRONT + GROWTH] = 0
    dy[:, FRONT:] = 0
    return a, soft, (dy, torch.zeros_like(dhT))


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dtype,N", [(F32, 5), (BF16, 16), (BF16, 40)])
def test_zeros_stay_zero(sign, dtype, N):
    """No state enters the growth and no adjoint comes back into it."""
    check_scan(*growing(sign, dtype, N=N, seed=N))


def test_zeros_stay_zero_in_packed_sequences():
    a, soft, (dy, dhT) = growing(1.0, BF16, B=1, N=8, D=12, G=2)
    T = a["x"].shape[1]
    more = {n: t if t is None or n in ("A", "D") else torch.cat([t, t[:, :70], t], 1) for n, t in a.items()
            if n != "initial_state"}
    cu = [0, T, T + 70, 2 * T + 70]
    more["initial_state"] = a["initial_state"].expand(3, -1, -1).contiguous()
    grads = torch.cat([dy, dy[:, :70], dy], 1), dhT.expand(3, -1, -1).contiguous()
    check_scan(more, soft, grads, cu=cu)


def test_without_an_initial_state():
    """Zeros before the first input, the most ordinary kind, and no final state's gradient."""
    a, soft, (dy, _) = growing(1.0)
    keep = slice(FRONT + 1, None)
    a = {n: t if t is None or t.dim() < 3 or n == "initial_state" else t[:, keep] for n, t in a.items()}
    a["initial_state"] = None
    val, err = scan_exact(a, soft)
    y, h = call(a, soft)
    check(y, val["y"], err["y"], "y")
    check(h, val["state"], err["state"], "state")


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_small_values_grow_and_large_ones_decay(sign):
    """1e-30 by e^112 in one run and back in another, or 1e30 by e^-112 and back: in
    range at each token, in both directions, though the runs' factors are not."""
    B, T, D, N = 1, 96, 4, 3
    a, soft, (dy, dhT) = scan_inputs(B=B, T=T, D=D, N=N, gate=False, bias=False, soft=False, skip=False, seed=1)
    gen = torch.Generator().manual_seed(3)
    a["A"] = (0.9 + 0.1 * torch.rand(D, N, generator=gen)).cuda()
    dt = torch.zeros(B, T, D)
    dt[:, 16:32] = sign * 7.0      # to e^{+-112}
    dt[:, 48:64] = -sign * 7.0     # and back
    a["dt"] = dt.cuda()
    a["x"] = torch.zeros_like(a["x"])
    a["initial_state"] = a["initial_state"].sign() * (1e-30 if sign > 0 else 1e30)
    # adjoints that stay in range on the same way back
    dy = torch.zeros_like(dy)
    dhT = dhT.sign() * (1e-22 if sign < 0 else 1e20)
    check_scan(a, soft, (dy, dhT))
