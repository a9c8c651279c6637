"""Infinities and NaN in the gated delta rule: what a token brings in reaches it
and later tokens of its sequence, as in the recurrence, and no earlier one.  The
earlier tokens' results are the bits of a call with ordinary values there."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
NAMES = ("q", "k", "v", "g", "beta")
# heads, widths and batch that take 16, 32 and 64 columns a workgroup, both key
# heads shared and not, all the kernels' feature steps
SHAPES = [(1, 1, 2, 64, 64), (1, 2, 2, 96, 72), (32, 2, 4, 128, 64), (65, 2, 4, 64, 64), (64, 1, 4, 256, 136),
          (1, 1, 1, 192, 192)]


def make(B, Hk, Hv, Dk, Dv, T, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(BF16)  # noqa: E731
    return dict(q=unit(r(B, T, Hk, Dk)), k=unit(r(B, T, Hk, Dk)), v=r(B, T, Hv, Dv).to(BF16),
                g=-0.1 * r(B, T, Hv).abs(), beta=torch.sigmoid(r(B, T, Hv))), 0.3 * r(B, Hv, Dk, Dv)


def run(x, h0, cu=None):
    from uttt_amd.delta import gated_delta_rule
    return gated_delta_rule(*(x[n] for n in NAMES), initial_state=h0, output_final_state=True, cu_seqlens=cu)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("name", NAMES)
def test_earlier_tokens_keep_their_outputs(shape, name, value):
    B, Hk, Hv, Dk, Dv = shape
    if name == "g" and value == -math.inf:
        return   # a state forgotten altogether: an ordinary value
    x, h0 = make(*shape, 200)
    want, _ = run(x, h0)
    for at in (0, 1, 15, 37, 63, 64, 100, 127, 199):
        bad = {n: t.clone() for n, t in x.items()}
        bad[name][-1, at, -1].view(-1)[-1] = value   # the last row, head and feature alone
        o, S = run(bad, h0)
        assert torch.equal(o[:-1], want[:-1]) and torch.isfinite(S[:-1]).all(), (at, "other rows")
        assert torch.equal(o[-1, :at], want[-1, :at]), (at, "earlier tokens")
        heads = slice(Hv - 1, Hv) if name in ("v", "g", "beta") else slice(Hv - Hv // Hk, Hv)
        assert torch.equal(o[-1, :, :heads.start], want[-1, :, :heads.start]), (at, "other heads")
        if name == "q":   # outputs of its own token alone
            assert not torch.isfinite(o[-1, at, heads]).any()
            assert torch.equal(o[-1, at + 1:], want[-1, at + 1:]) and torch.isfinite(S).all()
        elif name == "v":   # its own column alone
            assert not torch.isfinite(o[-1, at:, -1, -1]).any() and not torch.isfinite(S[-1, -1, :, -1]).any()
            assert torch.equal(o[-1, :, -1, :-1], want[-1, :, -1, :-1]) and torch.isfinite(S[-1, -1, :, :-1]).all()
        else:
            assert not torch.isfinite(o[-1, at:, heads]).any(), at
            assert not torch.isfinite(S[-1, heads]).any(), at


@pytest.mark.parametrize("shape", SHAPES)
def test_states_of_one_column(shape):
    """An initial state's column that is not finite stays by itself."""
    x, h0 = make(*shape, 130)
    want, wS = run(x, h0)
    bad = h0.clone()
    bad[-1, -1, 3, 1] = math.nan
    o, S = run(x, bad)
    rest = torch.arange(shape[4], device="cuda") != 1
    assert torch.equal(o[-1, :, -1][:, rest], want[-1, :, -1][:, rest])
    assert torch.equal(S[-1, -1][:, rest], wS[-1, -1][:, rest])
    assert not torch.isfinite(o[-1, :, -1, 1]).any() and not torch.isfinite(S[-1, -1, :, 1]).any()


def test_a_padded_batch_with_garbage_behind_its_tokens():
    """Rows of 70 and 130 real tokens of 200, whatever lies behind them."""
    x, h0 = make(2, 2, 2, 64, 64, 200)
    want, _ = run(x, h0)
    for n in NAMES:
        x[n][0, 70:] = math.nan
        x[n][1, 130:] = math.inf
    o, _ = run(x, h0)
    assert torch.equal(o[0, :70], want[0, :70]) and torch.equal(o[1, :130], want[1, :130])


def test_packed_sequences_keep_to_themselves():
    x, _ = make(1, 2, 2, 64, 64, 200)
    _, h0 = make(3, 2, 2, 64, 64, 1)
    cu = torch.tensor([0, 70, 130, 200], device="cuda")
    want, wS = run(x, h0, cu)
    bad = {n: t.clone() for n, t in x.items()}
    bad["k"][0, 100] = math.nan
    o, S = run(bad, h0, cu)
    for s in (slice(0, 100), slice(130, 200)):
        assert torch.equal(o[:, s], want[:, s])
    assert torch.equal(S[[0, 2]], wS[[0, 2]]) and not torch.isfinite(o[:, 100:130]).any()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("at", [1, 40, 63, 64, 127, 129])
def test_gradients_before_values_that_are_not_finite(shape, at):
    """v of a token and all behind it not finite, and no gradient given to their
    outputs, as for padding that a loss leaves out: the gradients of the tokens
    before it, and of the initial state, are those of a call without them."""
    x, h0 = make(*shape, 200)
    do = torch.randn(x["v"].shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(BF16)
    do[:, at:] = 0
    bad = dict(x, v=x["v"].clone())
    bad["v"][:, at:] = math.nan
    bad["v"][:, -1] = math.inf

    def grads(y):
        leaf = [y[n].clone().requires_grad_() for n in NAMES] + [h0.clone().requires_grad_()]
        o, _ = run(dict(zip(NAMES, leaf)), leaf[-1])
        return torch.autograd.grad(o, leaf, do)

    for n, a, b in zip(NAMES + ("h0",), grads(bad), grads(x)):
        same = torch.equal(a, b) if n == "h0" else torch.equal(a[:, :at], b[:, :at])
        assert same, n
