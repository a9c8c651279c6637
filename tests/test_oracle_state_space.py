"""The 64-bit state space oracle: its scan's formulas against torch's autograd
through the recurrence and against differences, its bounds against the same
formulas carried out in fp32, the convolution against torch's, and planted
mistakes."""
import pytest
import torch

from oracle import state_space as O

F64 = torch.float64


def inputs(T=9, D=6, N=3, G=2, gate=True, seed=0, dtype=F64):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=dtype)  # noqa: E731
    return dict(x=r(T, D), dt=0.5 * r(T, D), A=-torch.exp(r(D, N)), B=r(T, G, N), C=r(T, G, N), D=r(D),
                z=r(T, D) if gate else None, bias=r(D) - 1, h0=r(D, N)), r(T, D), r(D, N)


def recurrence(x, dt, A, B, C, D, z, bias, h0, soft):
    step = dt + bias
    step = torch.nn.functional.softplus(step, threshold=1e9) if soft else step
    group, h, out = torch.arange(x.shape[1]) // (x.shape[1] // B.shape[1]), h0, []
    for t in range(x.shape[0]):
        h = h * torch.exp(step[t, :, None] * A) + (step[t] * x[t])[:, None] * B[t, group]
        y = (h * C[t, group]).sum(-1) + D * x[t]
        out.append(y if z is None else y * torch.nn.functional.silu(z[t]))
    return torch.stack(out), h


@pytest.mark.parametrize("soft", [False, True])
@pytest.mark.parametrize("gate", [False, True])
def test_formulas_are_autograds(soft, gate):
    a, dy, dhT = inputs(gate=gate)
    leaf = {n: None if t is None else t.clone().requires_grad_() for n, t in a.items()}
    y, h = recurrence(**leaf, soft=soft)
    val, _ = O.scan_sequence(**a, softplus=soft, dy=dy, dhT=dhT)
    assert torch.allclose(val["y"], y, rtol=1e-12, atol=1e-12) and torch.allclose(val["state"], h, rtol=1e-12, atol=1e-12)
    names = [n for n in a if a[n] is not None]
    for n, want in zip(names, torch.autograd.grad([y, h], [leaf[n] for n in names], [dy, dhT])):
        assert torch.allclose(val["d_" + n], want, rtol=1e-10, atol=1e-10), n


@pytest.mark.parametrize("name", ["x", "dt", "A", "B", "C", "D", "z", "bias", "h0"])
def test_formulas_are_differences(name):
    a, dy, dhT = inputs(T=4, D=4, N=2)
    gen = torch.Generator().manual_seed(1)
    way = torch.randn(a[name].shape, generator=gen, dtype=F64)

    def loss(s):
        val, _ = O.scan_sequence(**dict(a, **{name: a[name] + s * way}), softplus=True)
        return (val["y"] * dy).sum() + (val["state"] * dhT).sum()

    val, _ = O.scan_sequence(**a, softplus=True, dy=dy, dhT=dhT)
    want = (loss(1e-5) - loss(-1e-5)) / 2e-5
    assert abs((val["d_" + name] * way).sum() - want) < 1e-7 * (1 + abs(want))


@pytest.mark.parametrize("soft", [False, True])
def test_bounds_hold_for_fp32_and_are_not_idle(soft):
    """The same formulas in fp32 stay within the bounds, by no more than a factor
    of 200 on any result (majorants of sums whose terms cancel), of 2000 where 40
    tokens' errors are added up as if they had one sign."""
    a, dy, dhT = inputs(T=40, D=8, N=6, dtype=torch.float32)
    if not soft:   # steps below zero grow past fp32's range
        a.update(dt=a["dt"].abs(), bias=a["bias"].abs())
    low, _ = O.scan_sequence(**a, softplus=soft, dy=dy, dhT=dhT)
    up = lambda t: t.double()  # noqa: E731
    val, err = O.scan_sequence(**{n: up(t) for n, t in a.items()}, softplus=soft, dy=up(dy), dhT=up(dhT))
    for n in val:
        off = (low[n].double() - val[n]).abs()
        assert (off <= 1.5 * err[n] + 2 * O.U * val[n].abs()).all(), n
        assert (off / err[n]).max() > (1 / 2000 if n in ("d_A", "d_D", "d_bias") else 1 / 200), n


def test_a_planted_mistake_is_outside_the_bounds():
    """A decay taken a token late, a gate's slope without its second term, a step's
    slope left out."""
    a, dy, dhT = inputs(T=12)
    val, err = O.scan_sequence(**a, softplus=True, dy=dy, dhT=dhT)
    late, _ = O.scan_sequence(**dict(a, dt=a["dt"].roll(1, 0)), softplus=True, dy=dy, dhT=dhT)
    assert ((late["y"] - val["y"]).abs() > 100 * err["y"]).any()
    s = torch.sigmoid(a["z"])
    assert ((val["d_z"] / (s * (1 + a["z"] * (1 - s))) * s - val["d_z"]).abs() > 100 * err["d_z"]).any()
    raw = a["dt"] + a["bias"]
    assert ((val["d_dt"] / torch.sigmoid(raw) - val["d_dt"]).abs() > 100 * err["d_dt"]).any()


def test_packed_is_each_sequence_alone():
    a, dy, dhT = inputs(T=12)
    one = lambda n: a[n][None]  # noqa: E731
    cu = [2, 5, 5, 11]
    h0 = torch.stack([a["h0"], 2 * a["h0"], -a["h0"]])
    val, _ = O.selective_scan(one("x"), one("dt"), a["A"], one("B"), one("C"), a["D"], one("z"), a["bias"], True, h0,
                              dy[None], torch.stack([dhT] * 3), cu)
    assert (val["y"][0, :2] == 0).all() and (val["y"][0, 11:] == 0).all() and (val["d_x"][0, 11:] == 0).all()
    assert torch.equal(val["state"][1], h0[1]) and torch.equal(val["d_h0"][1], dhT)
    part, _ = O.scan_sequence(a["x"][5:11], a["dt"][5:11], a["A"], a["B"][5:11], a["C"][5:11], a["D"], a["z"][5:11],
                              a["bias"], True, h0[2], dy[5:11], dhT)
    assert torch.equal(val["y"][0, 5:11], part["y"]) and torch.equal(val["d_B"][0, 5:11], part["d_B"])


@pytest.mark.parametrize("W", [2, 4, 7])
def test_convolution_is_torchs(W):
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=F64)  # noqa: E731
    x, w, b = r(2, 9, 5), r(5, W), r(5)
    y, state = O.causal_conv(x, w, b)
    padded = torch.nn.functional.pad(x.transpose(1, 2), (W - 1, 0))
    want = torch.nn.functional.conv1d(padded, w[:, None], b, groups=5).transpose(1, 2)
    assert torch.allclose(y, want, rtol=1e-12, atol=1e-12)
    assert torch.equal(state, padded.transpose(1, 2)[:, -(W - 1):])
    # in two halves, the second from the first one's state
    first, mid = O.causal_conv(x[:, :4], w, b, silu=True)
    second, end = O.causal_conv(x[:, 4:], w, b, silu=True, initial_state=mid)
    assert torch.allclose(torch.cat([first, second], 1), O.causal_conv(x, w, b, silu=True)[0], rtol=1e-12, atol=1e-12)
    assert torch.equal(end, state)


def test_norms():
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=F64)  # noqa: E731
    x, res, w, s = r(3, 8), r(3, 8), r(8), r(8)
    y, total = O.norm_before_block(x, res, w, s, eps=0.0)
    assert torch.allclose((y / w).square().mean(-1), torch.ones(3, dtype=F64)) and torch.equal(total, res + s * x)
    assert torch.allclose(O.norm_after_block(x, w, scale=s, residual=res) - res, s * w * O.norm_after_block(x))
