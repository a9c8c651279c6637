"""The gated delta rule on the GPU against the 64-bit recurrence.

Tolerances, relative in the 2-norm.  bf16's half step is H = 2^-8.  An fp32
operand of a product goes in as two bf16 values, which leave out at most H^2 =
2^-16 of it, and of which the product of the two small parts, H^2 again, is
left out; a value passes through up to four such operands in a row (S, R, T,
U), a gradient through as many again on its way back.
  states, their gradients, dg and dbeta as fp32     8 H^2
  o, dv, dg and dbeta as bf16 (fp16)     the result's rounding, and that
  dq         D (once rounded), then the result      2 H
  dk         D or M, then the result                2 H
dg and dbeta are sums over Dk x Dv terms that may cancel: the terms' order is
that of |S0| |dS'|, so theirs is relative to the larger of the result and that.
"""
import math

import pytest
import torch

from oracle import delta as oracle

pytestmark = pytest.mark.gpu
H = 2.0 ** -8
Q = 8 * H * H
TOL = dict(o=H + Q, state=Q, dv=H + Q, dq=2 * H + Q, dk=2 * H + Q, dg=Q, dbeta=Q, dh0=Q)
BF16 = torch.bfloat16


def close(name, ours, ref, what=None, more=0.0):
    ours, ref = ours.detach().double().cpu(), ref.detach().double()
    assert ours.shape == ref.shape, (what, name, ours.shape, ref.shape)
    assert torch.isfinite(ours).all(), f"{what} {name}: not finite"
    off, norm = (ours - ref).norm().item(), ref.norm().item()
    allowed = TOL[name] * norm + more
    assert off <= allowed + 1e-30, f"{what} {name}: {off:.3e} of {norm:.3e} > {allowed:.3e}"


def inputs(B, T, n, Hk, Hv, Dk, Dv, seed=0, gates=torch.float32, rate=0.1, beta_at=0.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(BF16)  # noqa: E731
    x = dict(q=unit(r(B, T, Hk, Dk) + 0.2), k=unit(r(B, T, Hk, Dk) + 0.2), v=r(B, T, Hv, Dv).to(BF16),
             g=(-rate * torch.nn.functional.softplus(r(B, T, Hv))).to(gates),
             beta=torch.sigmoid(r(B, T, Hv) + beta_at).to(gates), h0=0.3 * r(n, Hv, Dk, Dv))
    return x, r(B, T, Hv, Dv).to(BF16), 0.3 * r(n, Hv, Dk, Dv)


def check(x, do, dht, cu=None, cu_dtype=torch.int32, h0=True, scale=None, grads=True, what=None,
          move=lambda name, t: t.cuda()):
    """Forward and backward against the recurrence; returns what the framework gave."""
    from uttt_amd.delta import gated_delta_rule
    names = [n for n in ("q", "k", "v", "g", "beta", "h0") if h0 or n != "h0"]
    ref = {n: x[n].double().requires_grad_(grads) for n in names}
    s = x["q"].shape[-1] ** -0.5 if scale is None else scale
    ro, rs = oracle.gated_delta_rule(ref["q"], ref["k"], ref["v"], ref["g"], ref["beta"], s,
                                     ref.get("h0"), cu)
    ours = {n: move(n, x[n]).requires_grad_(grads) for n in names}
    cut = None if cu is None else torch.tensor(cu, dtype=cu_dtype, device="cuda")
    o, S = gated_delta_rule(ours["q"], ours["k"], ours["v"], ours["g"], ours["beta"], scale=scale,
                            initial_state=ours.get("h0"), output_final_state=True, cu_seqlens=cut)
    assert o.dtype == BF16 and S.dtype == torch.float32
    got = dict(o=o, state=S)
    close("o", o, ro, what)
    close("state", S, rs, what)
    if grads:
        some = 0.0 * sum(t.nan_to_num(neginf=0.0).sum() for t in ref.values())   # a graph where there are no tokens too
        ro, rs = ro + some, rs + some
        rg = torch.autograd.grad([ro, rs], [ref[n] for n in names], [do.double(), dht.double()])
        og = torch.autograd.grad([o, S], [ours[n] for n in names], [do.cuda(), dht.cuda()])
        for n, a, b in zip(names, og, rg):
            assert a.dtype == x[n].dtype
            more = 0.0
            if n in ("g", "beta"):   # the rounding to its type, and terms of |S0| |dS'|
                more = (torch.finfo(x[n].dtype).eps / 2 * b.norm() +
                        Q * (rs.detach().norm() + x["h0"].double().norm()) *
                        (dht.double().norm() + rg[-1].norm() * h0)).item()
            close("d" + n, a, b, what, more)
            got["d" + n] = a
    return got


@pytest.mark.parametrize("T", [1, 2, 15, 63, 64, 65, 127, 128, 193])
def test_lengths(T):
    check(*inputs(2, T, 2, 1, 2, 64, 64, seed=T), what=T)


@pytest.mark.parametrize("Hk,Hv,Dk,Dv", [(1, 1, 8, 8), (1, 1, 16, 200), (2, 2, 40, 72), (1, 3, 96, 96),
                                         (2, 4, 104, 136), (1, 2, 128, 128), (3, 3, 160, 64),
                                         (1, 1, 192, 192), (1, 2, 200, 24), (1, 1, 256, 256)])
def test_widths_and_heads(Hk, Hv, Dk, Dv):
    check(*inputs(1, 150, 1, Hk, Hv, Dk, Dv, seed=Dk, gates=BF16), what=(Hk, Hv, Dk, Dv))


@pytest.mark.parametrize("Dk", [64, 96, 128, 192, 256])
def test_many_heads_take_wide_columns(Dk):
    """Enough heads for 32 columns a wave."""
    check(*inputs(64, 70, 64, 4, 4, Dk, 40, seed=1), what=Dk)


@pytest.mark.parametrize("Dk", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("B,Dv", [(32, 64), (65, 64), (64, 136)])
def test_column_widths(Dk, B, Dv):
    """Enough heads for 32 and for 64 columns a workgroup, a last block of which
    has few; two value heads to a key head."""
    check(*inputs(B, 70, B, 2, 4, Dk, Dv, seed=Dk + B), what=(Dk, B, Dv))


@pytest.mark.parametrize("cu", [[0, 200], [0, 1, 1, 65, 130, 200], [0, 0, 0, 200], [0, 64, 128, 192, 200],
                                [0, 200, 200], [7, 70, 135], [0, 63], [100, 100], [0, 3, 5, 190]])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_packed(cu, dtype):
    """Empty sequences, ends inside and at chunks, tokens before and behind the
    sequences: zeros there, whatever lies in them."""
    x, do, dht = inputs(1, 200, len(cu) - 1, 1, 2, 64, 72, seed=len(cu))
    outside = torch.ones(200, dtype=torch.bool)
    for s, e in zip(cu[:-1], cu[1:]):
        outside[s:e] = False
    got = check(x, do, dht, cu, dtype, what=cu)
    dirty = {n: t.clone() for n, t in x.items()}
    for n in ("q", "k", "v", "g", "beta"):
        dirty[n][:, outside] = math.nan
    from uttt_amd.delta import gated_delta_rule
    leaf = {n: t.cuda().requires_grad_() for n, t in dirty.items()}
    o, S = gated_delta_rule(leaf["q"], leaf["k"], leaf["v"], leaf["g"], leaf["beta"],
                            initial_state=leaf["h0"], output_final_state=True,
                            cu_seqlens=torch.tensor(cu, dtype=dtype, device="cuda"))
    names = list(leaf)
    dod = do.clone()
    dod[:, outside] = math.nan
    grads = torch.autograd.grad([o, S], [leaf[n] for n in names], [dod.cuda(), dht.cuda()])
    for n, t in dict(o=o, state=S, **{"d" + n: t for n, t in zip(names, grads)}).items():
        assert torch.equal(t, got[n]), n
        if n not in ("state", "dh0"):
            assert (t[:, outside] == 0).all(), n


def test_offsets_that_do_not_ascend_stay_inside():
    """Offsets past the tokens or descending are clamped: no access outside."""
    from uttt_amd.delta import gated_delta_rule
    x, _, _ = inputs(1, 100, 4, 1, 1, 64, 64)
    x = {n: t.cuda() for n, t in x.items()}
    call = lambda cu: gated_delta_rule(  # noqa: E731
        x["q"], x["k"], x["v"], x["g"], x["beta"], initial_state=x["h0"], output_final_state=True,
        cu_seqlens=torch.tensor(cu, device="cuda"))
    for bad, good in (([-5, 30, 20, 90, 1000], [0, 30, 30, 90, 100]), ([0, 500, 3, 4, 5], [0, 100, 100, 100, 100])):
        for a, b in zip(call(bad), call(good)):
            assert torch.equal(a, b)


def test_many_sequences_fill_several_rounds_of_the_table():
    n = 2100
    cu = [0] + [min(i, 300) if i % 7 else min(i - 1, 300) for i in range(1, n + 1)]
    cu = [max(cu[:i + 1]) for i in range(n + 1)]
    x, do, dht = inputs(1, cu[-1], n, 1, 1, 8, 8)
    check(x, do, dht, cu, what="many")


@pytest.mark.parametrize("n", [255, 256, 257])
def test_sequences_ranked_by_length(n):
    """Up to 256 sequences are taken up longest first, each with its own states."""
    gen = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 4, (n,), generator=gen)
    lens[n // 2], lens[n - 1] = 200, 131
    cu = [0] + lens.cumsum(0).tolist()
    x, do, dht = inputs(1, cu[-1], n, 1, 2, 16, 24)
    check(x, do, dht, cu, what=n)


def test_decays():
    """No decay, a strong one everywhere, single tokens that forget everything
    (-inf, also twice in a row and first in a chunk), none at all between."""
    for rate in (0.0, 1e-3, 5.0, 60.0):
        check(*inputs(1, 130, 1, 1, 2, 64, 64, rate=rate), what=rate)
    x, do, dht = inputs(1, 200, 1, 1, 2, 64, 64, rate=0.05)
    for t in (0, 10, 11, 64, 100, 191):
        x["g"][:, t, 0] = -math.inf
    x["g"][:, 150, 1] = -1000.0
    got = check(x, do, dht, what="resets")
    assert torch.isfinite(got["dg"]).all()


def test_repeated_keys_and_full_writes():
    """beta = 1 and 2 (reflections) on keys that repeat: the inverse of I + A is
    far from I."""
    x, do, dht = inputs(1, 140, 1, 1, 1, 64, 64, rate=0.01)
    x["k"][:, 1::2] = x["k"][:, 0::2]
    x["beta"][:] = 1.0
    check(x, do, dht, what="repeated")
    x["k"][:] = x["k"][:, :1]
    check(x, do, dht, what="one key")
    x, do, dht = inputs(1, 140, 1, 1, 1, 64, 64, rate=0.01)
    x["beta"][:] = 2.0
    check(x, do, dht, what="reflections")


def test_writes_of_strength_zero():
    x, do, dht = inputs(1, 100, 1, 1, 1, 64, 64)
    x["beta"][:] = 0.0
    check(x, do, dht, what="beta 0")


def test_scale_and_no_initial_state():
    check(*inputs(2, 100, 2, 1, 2, 64, 64), h0=False, scale=0.7)


@pytest.mark.parametrize("gates", [torch.float32, BF16, torch.float16])
def test_gate_types(gates):
    check(*inputs(1, 100, 1, 2, 2, 64, 64, gates=gates), what=gates)


def test_views():
    """Parts of one fused projection, head-major storage, shared (expanded)
    batch rows, and rows that are not 16-byte aligned (copied)."""
    x, do, dht = inputs(2, 90, 2, 2, 2, 64, 64)

    def fused(name, t):
        if name not in "qkv":
            return t.cuda()
        big = torch.full((2, 90, 3, 2, 64), math.nan, dtype=BF16, device="cuda")
        big[:, :, 1] = t.cuda()
        return big[:, :, 1]

    check(x, do, dht, move=fused, what="fused")
    check(x, do, dht, move=lambda n, t: t.cuda().transpose(1, 2).contiguous().transpose(1, 2)
          if n in "qkv" else t.cuda(), what="head-major")

    def odd(name, t):
        if name not in "qkv":
            return t.cuda()
        big = torch.zeros(2, 90, 2, 67, dtype=BF16, device="cuda")
        big[..., 3:] = t.cuda()
        return big[..., 3:]

    check(x, do, dht, move=odd, what="unaligned")
    one = {n: t[:1].expand(2, *t.shape[1:]).contiguous() for n, t in x.items()}
    check(one, do, dht, move=lambda n, t: t[:1].cuda().expand(2, -1, -1, -1) if n in "qk" else t.cuda(),
          what="expanded")


def test_gradient_of_an_expanded_input_sums():
    from uttt_amd.delta import gated_delta_rule
    x, do, _ = inputs(2, 70, 2, 1, 1, 64, 64)
    x = {n: t.cuda() for n, t in x.items()}
    q = x["q"][:1].clone().requires_grad_()
    o, _ = gated_delta_rule(q.expand(2, -1, -1, -1), x["k"], x["v"], x["g"], x["beta"])
    (dq,) = torch.autograd.grad(o, q, do.cuda())
    q2 = x["q"][:1].expand(2, -1, -1, -1).contiguous().requires_grad_()
    o2, _ = gated_delta_rule(q2, x["k"], x["v"], x["g"], x["beta"])
    (dq2,) = torch.autograd.grad(o2, q2, do.cuda())
    assert torch.equal(dq, dq2.sum(0, keepdim=True))


def test_gradient_of_one_output_alone():
    from uttt_amd.delta import gated_delta_rule
    x, do, dht = inputs(1, 100, 1, 1, 1, 64, 64)
    leaf = {n: t.cuda().requires_grad_() for n, t in x.items()}
    args = [leaf[n] for n in ("q", "k", "v", "g", "beta")]
    run = lambda: gated_delta_rule(*args, initial_state=leaf["h0"], output_final_state=True)  # noqa: E731
    zero_o, zero_s = torch.zeros_like(do).cuda(), torch.zeros_like(dht).cuda()
    for pick, full in (((0, do), (do, None)), ((1, dht), (None, dht))):
        out = run()
        a = torch.autograd.grad(out[pick[0]], list(leaf.values()), pick[1].cuda())
        out = run()
        b = torch.autograd.grad(out, list(leaf.values()),
                                [zero_o if full[0] is None else do.cuda(),
                                 zero_s if full[1] is None else dht.cuda()])
        for s, t in zip(a, b):
            assert torch.equal(s, t)
    o, none = gated_delta_rule(*args)
    assert none is None and o.requires_grad
    v = x["v"].cuda().requires_grad_()   # one leaf alone
    o, _ = gated_delta_rule(x["q"].cuda(), x["k"].cuda(), v, x["g"].cuda(), x["beta"].cuda())
    assert torch.autograd.grad(o, v, do.cuda())[0].shape == v.shape


def test_gradients_against_differences():
    """Central differences of a loss on the fp32 states, which are exact to 4
    H^2: two losses over steps of e carry 8 H^2 |loss| / 2e.  The difference's
    own higher orders are what the 64-bit recurrence's difference is off its
    gradient by.  The gradients themselves are off by their tolerance."""
    from uttt_amd.delta import gated_delta_rule
    x, _, dht = inputs(1, 100, 1, 1, 1, 64, 64)
    names = ("q", "k", "v", "g", "beta", "h0")
    args = lambda y: [y[n] for n in names]  # noqa: E731

    def ours(y):
        y = {n: t.cuda() for n, t in y.items()}
        S = gated_delta_rule(*args(y)[:5], initial_state=y["h0"], output_final_state=True)[1]
        return (S.double() * dht.cuda().double()).sum().cpu()

    def exact(y):
        y = {n: t.double() for n, t in y.items()}
        return (oracle.gated_delta_rule(*args(y)[:5], 0.125, y["h0"])[1] * dht.double()).sum()

    leaf = {n: t.clone().requires_grad_(n != "q") for n, t in x.items()}
    grads = dict(zip(names[1:], torch.autograd.grad(ours(leaf), args(leaf)[1:])))
    ref = dict(zip(names[1:], torch.autograd.grad(exact(leaf), args(leaf)[1:])))
    for name, e in (("g", 0.05), ("beta", 0.05), ("h0", 1.0)):
        d = torch.sign(ref[name])
        moved = lambda f, s: f({**x, name: x[name] + s * e * d}).item()  # noqa: E731
        hi, lo = moved(ours, 1), moved(ours, -1)
        want = (hi - lo) / (2 * e)
        own = (moved(exact, 1) - moved(exact, -1)) / (2 * e) - (ref[name].double() * d).sum().item()
        have = (grads[name].double() * d).sum().item()
        noise = 8 * H * H * max(abs(hi), abs(lo)) / (2 * e)
        off = TOL["d" + name] * grads[name].double().norm().item() * d.double().norm().item()
        assert abs(have + own - want) <= noise + off, (name, have, own, want, noise, off)


def test_twice_the_same_bits():
    x, do, dht = inputs(2, 300, 2, 2, 4, 128, 128, gates=BF16)
    a, b = check(x, do, dht), check(x, do, dht)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_no_tokens():
    from uttt_amd.delta import gated_delta_rule
    x, _, _ = inputs(2, 0, 2, 1, 1, 64, 64)
    leaf = {n: t.cuda().requires_grad_() for n, t in x.items()}
    o, S = gated_delta_rule(*(leaf[n] for n in ("q", "k", "v", "g", "beta")), initial_state=leaf["h0"],
                            output_final_state=True)
    assert o.shape == (2, 0, 1, 64) and torch.equal(S, leaf["h0"])
    (dh,) = torch.autograd.grad(S, leaf["h0"], torch.ones_like(S))
    assert (dh == 1).all()


def test_other_stream_and_interleaved_calls():
    """Two calls in flight on two streams, each with its own workspace."""
    from uttt_amd.delta import gated_delta_rule
    a, b = ({n: t.cuda() for n, t in inputs(1, 500, 1, 2, 2, 64, 64, seed=s)[0].items()} for s in (1, 2))
    run = lambda x: gated_delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"],  # noqa: E731
                                     initial_state=x["h0"], output_final_state=True)
    want = [run(a), run(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, x in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append(run(x))
    torch.cuda.synchronize()
    for w, h in zip(want, got):
        assert torch.equal(w[0], h[0]) and torch.equal(w[1], h[1])


# ------------------------------------------------------------- single tokens --
def step_reference(x, state, idx):
    """Rows in order, each against its slot."""
    o = torch.zeros(x["v"].shape, dtype=torch.float64)
    state = state.double().clone()
    for b, i in enumerate(idx):
        if 0 <= i < state.shape[0]:
            o[b], state[i] = oracle.recurrence(*(x[n][b].double() for n in ("q", "k", "v", "g", "beta")),
                                               state[i], x["q"].shape[-1] ** -0.5)
    return o, state


@pytest.mark.parametrize("dtype", [torch.float32, BF16, torch.float16])
@pytest.mark.parametrize("B,T,Hk,Hv,Dk,Dv", [(1, 1, 1, 1, 64, 64), (3, 1, 1, 2, 40, 72), (2, 4, 2, 2, 96, 192),
                                             (5, 1, 1, 1, 1, 4), (70, 2, 2, 4, 128, 128), (2, 1, 1, 3, 250, 20),
                                             (64, 1, 4, 8, 200, 64), (40, 3, 1, 16, 64, 64)])
def test_step(dtype, B, T, Hk, Hv, Dk, Dv):
    """fp32 throughout, outputs rounded once: its half step, and the order of
    sums over Dk (2^-24 each, sqrt(Dk) of them on average, 16 allowed for)."""
    from uttt_amd.delta import gated_delta_step
    x, _, _ = inputs(B, T, 1, Hk, Hv, Dk, Dv, seed=B + Dk)
    x = {n: t.to(dtype) if n in "qkv" else t for n, t in x.items()}
    gen = torch.Generator().manual_seed(9)
    state = 0.3 * torch.randn(B + 3, Hv, Dk, Dv, generator=gen)
    idx = torch.randperm(B + 3, generator=gen)[:B].tolist()
    if B > 2:
        idx[1], idx[-1] = -1, B + 3    # padding, and an index of no slot
    ro, rs = step_reference(x, state, idx)
    ours = state.cuda()
    y = {n: t.cuda() for n, t in x.items()}
    o = gated_delta_step(y["q"], y["k"], y["v"], y["g"], y["beta"], ours,
                         state_indices=torch.tensor(idx, device="cuda"))
    assert o.dtype == dtype
    tol = torch.finfo(dtype).eps / 2 + 16 * 2.0 ** -24
    assert (o.double().cpu() - ro).norm() <= tol * ro.norm()
    assert (ours.double().cpu() - rs).norm() <= 16 * 2.0 ** -24 * rs.norm()
    untouched = [i for i in range(B + 3) if i not in idx]
    assert torch.equal(ours.cpu()[untouched], state[untouched])
    for b, i in enumerate(idx):
        if not 0 <= i < B + 3:
            assert (o[b] == 0).all()


@pytest.mark.parametrize("Dk,Dv", [(40, 64), (100, 132), (128, 128), (256, 68)])
def test_step_of_many_rows(Dk, Dv):
    """Enough workgroups for 64 columns each, a last block of which has few."""
    test_step(BF16, 33, 2, 1, 2, Dk, Dv)


@pytest.mark.parametrize("width", [(64, 64), (128, 128)])
def test_step_rows_of_one_slot_follow_one_another(width):
    from uttt_amd.delta import gated_delta_step
    for B, idx in ((6, [2, 0, 2, -1, 2, 1]), (300, [(7 * i) % 11 for i in range(300)])):
        x, _, _ = inputs(B, 1, 1, 1, 2, *width, seed=B)
        state = torch.randn(11, 2, *width, generator=torch.Generator().manual_seed(3))
        ro, rs = step_reference(x, state, idx)
        ours = state.cuda()
        y = {n: t.cuda() for n, t in x.items()}
        o = gated_delta_step(y["q"], y["k"], y["v"], y["g"], y["beta"], ours,
                             state_indices=torch.tensor(idx, dtype=torch.int32, device="cuda"))
        assert (o.double().cpu() - ro).norm() <= (H + 30 * 2.0 ** -24) * ro.norm()
        assert (ours.double().cpu() - rs).norm() <= 30 * 2.0 ** -24 * rs.norm()


def test_step_on_a_layers_slice_of_a_pool():
    from uttt_amd.delta import gated_delta_step
    x, _, _ = inputs(4, 1, 1, 1, 2, 64, 64)
    y = {n: t.cuda() for n, t in x.items()}
    pool = torch.randn(6, 3, 2, 64, 64, device="cuda")
    before, alone = pool.clone(), pool[:, 1].contiguous()
    args = (y["q"], y["k"], y["v"], y["g"], y["beta"])
    a = gated_delta_step(*args, pool[:, 1])
    b = gated_delta_step(*args, alone)
    assert torch.equal(a, b) and torch.equal(pool[:, 1], alone)
    assert torch.equal(pool[:, 0], before[:, 0]) and torch.equal(pool[:, 2], before[:, 2])
    assert torch.equal(pool[4:], before[4:])


def test_prompt_then_tokens_is_the_whole_sequence():
    """The states that the chunked pass leaves carry on token by token."""
    from uttt_amd.delta import gated_delta_rule, gated_delta_step
    x, _, _ = inputs(2, 140, 2, 2, 4, 64, 72, rate=0.02)
    ro, rs = oracle.gated_delta_rule(*(x[n].double() for n in ("q", "k", "v", "g", "beta")), 64 ** -0.5,
                                     x["h0"].double())
    y = {n: t.cuda() for n, t in x.items()}
    part = lambda s: [y[n][:, s] for n in ("q", "k", "v", "g", "beta")]  # noqa: E731
    o, S = gated_delta_rule(*part(slice(0, 133)), initial_state=y["h0"], output_final_state=True)
    outs = [o] + [gated_delta_step(*part(slice(t, t + 1)), S) for t in range(133, 140)]
    close("o", torch.cat(outs, 1), ro)
    close("state", S, rs)


def test_step_in_a_graph():
    """Captured once, replayed on new tokens, between eager calls."""
    from uttt_amd.delta import gated_delta_step
    x, _, _ = inputs(8, 6, 1, 1, 2, 64, 64)
    y = {n: t.cuda() for n, t in x.items()}
    state = torch.randn(8, 2, 64, 64, device="cuda")
    eager, graphed = state.clone(), state.clone()
    fixed = {n: y[n][:, :1].clone() for n in ("q", "k", "v", "g", "beta")}
    idx = torch.randperm(8, device="cuda")
    warm = state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gated_delta_step(*fixed.values(), warm, state_indices=idx)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gated_delta_step(*fixed.values(), graphed, state_indices=idx)
    for t in range(6):
        for n in fixed:
            fixed[n].copy_(y[n][:, t:t + 1])
        graph.replay()
        want = gated_delta_step(*(y[n][:, t:t + 1] for n in fixed), eager, state_indices=idx)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(graphed, eager), t


def test_rule_in_a_graph():
    """Forward captured with packed offsets that change between replays."""
    from uttt_amd.delta import gated_delta_rule
    x, _, _ = inputs(1, 200, 2, 1, 2, 64, 64)
    y = {n: t.cuda() for n, t in x.items()}
    cu = torch.tensor([0, 90, 200], device="cuda")
    run = lambda: gated_delta_rule(y["q"], y["k"], y["v"], y["g"], y["beta"],  # noqa: E731
                                   initial_state=y["h0"], output_final_state=True, cu_seqlens=cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, S = run()
    for i, ends in enumerate(([0, 90, 200], [5, 70, 140], [0, 0, 200], [0, 128, 200])):
        cu.copy_(torch.tensor(ends))
        y["v"].mul_(-1.0 if i % 2 else 1.0)
        graph.replay()
        wo, wS = run()
        torch.cuda.synchronize()
        assert torch.equal(o, wo) and torch.equal(S, wS), ends


def test_backward_in_a_graph():
    """Forward and backward captured together, replayed on new values."""
    from uttt_amd.delta import gated_delta_rule
    x, do, _ = inputs(1, 130, 1, 1, 2, 64, 64)
    names = ("q", "k", "v", "g", "beta")
    fixed = {n: x[n].cuda().requires_grad_() for n in names}
    grad = do.cuda()

    def run(t):
        o, _ = gated_delta_rule(*(t[n] for n in names))
        return torch.autograd.grad(o, [t[n] for n in names], grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(fixed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(fixed)
    for i in range(3):
        with torch.no_grad():
            fixed["v"].mul_(-0.5)
        graph.replay()
        want = run({n: t.detach().clone().requires_grad_() for n, t in fixed.items()})
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


def test_packed_without_tokens():
    """The states pass through, forwards and backwards."""
    x, do, dht = inputs(1, 0, 3, 1, 2, 64, 64)
    got = check(x, do, dht, cu=[0, 0, 0, 0])
    assert torch.equal(got["state"].detach().cpu(), x["h0"]) and torch.equal(got["dh0"].cpu(), dht)


def test_step_without_rows_or_tokens():
    from uttt_amd.delta import gated_delta_step
    for B, T in ((0, 1), (2, 0)):
        state = torch.randn(3, 2, 16, 16, device="cuda")
        before = state.clone()
        r = lambda *s: torch.randn(*s, device="cuda", dtype=BF16)  # noqa: E731
        o = gated_delta_step(r(B, T, 1, 16), r(B, T, 1, 16), r(B, T, 2, 16), r(B, T, 2), r(B, T, 2), state)
        assert o.shape == (B, T, 2, 16) and torch.equal(state, before)


def test_tokens_far_apart():
    """Rows 2^23 elements apart and more: past a chunk's 31-bit offsets."""
    def far(name, t):
        if name not in ("q", "k", "v"):
            return t.cuda()
        room = torch.zeros(t.shape[1], 2 ** 23 + 8, dtype=t.dtype, device="cuda")
        view = room[:, :t[0, 0].numel()].view(1, t.shape[1], *t.shape[2:])
        view.copy_(t)
        return view.detach()

    check(*inputs(1, 66, 1, 1, 2, 64, 64, seed=3), move=far)


def test_offsets_past_32_bits():
    """q, k, v, outputs and gradients of more than 2^31 elements: the tokens at
    the end, and at the start, give the bits of calls that have only them."""
    from uttt_amd.delta import gated_delta_rule
    T, Hh, D = 2 ** 21 + 192, 16, 64
    cut = T - 384

    def make(*s):
        gen = torch.Generator(device="cuda").manual_seed(len(s))
        return torch.randn(1, T, Hh, *s, device="cuda", dtype=BF16, generator=gen)

    q, k, v, do = make(D), make(D).mul_(0.1), make(D), make(D)
    g, beta = -make().abs().float().mul_(0.1), torch.sigmoid(make().float())
    leaf = [t.requires_grad_() for t in (q, k, v, g, beta)]
    o, S = gated_delta_rule(*leaf, output_final_state=True)
    grads = torch.autograd.grad(o, leaf, do)
    with torch.no_grad():
        start, S1 = gated_delta_rule(*(t[:, :cut] for t in leaf), output_final_state=True)
        assert torch.equal(start[:, :256], o[:, :256])
        del start
    few = [t[:, cut:].detach().clone().requires_grad_() for t in leaf]
    o2, S2 = gated_delta_rule(*few, initial_state=S1, output_final_state=True)
    assert torch.equal(o[:, cut:], o2) and torch.equal(S, S2)
    for n, a, b in zip(("q", "k", "v", "g", "beta"), grads, torch.autograd.grad(o2, few, do[:, cut:])):
        assert torch.equal(a[:, cut:], b), n


def test_step_in_a_slot_past_32_bits():
    from uttt_amd.delta import gated_delta_step
    slots = 2 ** 31 // (16 * 128 * 128) + 2
    state = torch.zeros(slots, 16, 128, 128, device="cuda")
    r = lambda *s: torch.randn(*s, device="cuda", dtype=BF16)  # noqa: E731
    x = r(2, 1, 8, 128), r(2, 1, 8, 128).mul_(0.1), r(2, 1, 16, 128), -r(2, 1, 16).abs(), r(2, 1, 16).abs()
    own = torch.randn(2, 16, 128, 128, device="cuda")
    state[slots - 1], state[0] = own[0], own[1]
    o = gated_delta_step(*x, state, state_indices=torch.tensor([slots - 1, 0], device="cuda"))
    assert torch.equal(o, gated_delta_step(*x, own))
    assert torch.equal(state[slots - 1], own[0]) and torch.equal(state[0], own[1])
    assert not state[1:-1].any()


def test_addresses_between_pieces_and_strides_of_one():
    """Contiguous tensors that start 2 bytes behind a multiple of 16, and axes of
    one with strides of no use."""
    def behind(name, t):
        if name not in ("q", "k", "v"):
            return t.cuda()
        room = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:] = t.flatten().cuda()
        return room[1:].view(t.shape).detach()

    def odd(name, t):
        if name not in ("q", "k", "v"):
            return t.cuda()
        room = torch.zeros(t.numel() + 16, dtype=t.dtype, device="cuda")
        room[:t.numel()] = t.flatten().cuda()
        return room.as_strided(t.shape, (13, 7, *t.stride()[2:])).detach()

    check(*inputs(1, 70, 1, 1, 2, 64, 64, seed=4), move=behind)
    check(*inputs(1, 1, 1, 2, 2, 64, 64, seed=5), move=odd)
