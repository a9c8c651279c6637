"""The fp32 results of the gated delta rule are exact to fp32's order: states and
their gradients against the 64-bit recurrence, per case in the 2-norm, within N =
16 * 2^-24.

A chunk's part of the state passes through at most Dk / 32 + 1 accumulations of
K S0, R, 12 of U = T R, 6 of K^T U and the decay, some 30 roundings of at most
2^-24 that add up as their square root, 5.5; T and its norm (up to 2 for these
keys) carry U's to at most 11 of them, decays and earlier chunks come in as they
are.  16 are allowed.  A product with an operand cut to two bf16 values, 2^-16 of
it left out, is off by 20 N."""
import pytest
import torch

from delta_cases import BF16, CASES, F32, by_sequence, groups_of_heads, make, name_of, offsets, reference

pytestmark = pytest.mark.gpu
N = 16 * 2.0 ** -24
EXACT = [dict(c, gates=F32) for c in CASES]


@pytest.mark.parametrize("c", EXACT, ids=name_of)
def test_states_and_their_gradients(c):
    """The gradient's chain has Q^T dO, P^T dO and K dS' beside T^T dU and K^T dR: as
    many roundings again."""
    from uttt_amd.delta import gated_delta_rule
    x, do, dht = make(c)
    y = {n: t.cuda() for n, t in x.items()}
    cu = None if c["B"] else torch.tensor(offsets(c), dtype=torch.int32, device="cuda")
    args = [y[n] for n in ("q", "k", "v", "g", "beta")]
    S = gated_delta_rule(*args, initial_state=y["h0"], output_final_state=True, cu_seqlens=cu)[1]
    y["h0"].requires_grad_()   # with what a backward reads
    o, S2 = gated_delta_rule(*args, initial_state=y["h0"], output_final_state=True, cu_seqlens=cu)
    assert torch.equal(S2, S)
    (dh0,) = torch.autograd.grad([o, S2], y["h0"], [do.cuda(), dht.cuda()])
    for heads in groups_of_heads(c):
        ref = reference(c, x, do, dht, heads, "cuda")[1]
        for name, got, want in (("state", S, ref["S"][:, -1]), ("dh0", dh0, ref["dh0"])):
            off, norm = (got[:, heads].double() - want).norm().item(), want.norm().item()
            assert off <= N * norm, (name, heads.tolist(), off / norm)


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("c", EXACT, ids=name_of)
def test_gradients_of_fp32_gates(c, types):
    """dg and dbeta of a head: N of the norms of the products that they are sums of
    (tests/delta_cases.py), as their factors are off by N, and 2^-24 of themselves
    for every one of the 64 + 16 additions in a row at most, 9 as their square root.
    Where one of the two gates is fp32, its gradient is; the other's is rounded."""
    from uttt_amd.delta import gated_delta_rule
    x, do, dht = make(c)
    x["g"], x["beta"] = x["g"].to(types[0]), x["beta"].to(types[1])
    leaf = {n: t.cuda().requires_grad_(n in ("g", "beta")) for n, t in x.items()}
    cu = None if c["B"] else torch.tensor(offsets(c), dtype=torch.int32, device="cuda")
    out = gated_delta_rule(*(leaf[n] for n in ("q", "k", "v", "g", "beta")), initial_state=leaf["h0"],
                           output_final_state=True, cu_seqlens=cu)
    grads = torch.autograd.grad(out, [leaf["g"], leaf["beta"]], [do.cuda(), dht.cuda()])
    for heads in groups_of_heads(c):
        ref = reference(c, x, do, dht, heads, "cuda")[1]
        for name, got, dtype in zip(("g", "beta"), grads, types):
            mine = torch.nn.utils.rnn.pad_sequence(by_sequence(c, got[:, :, heads]), batch_first=True).double()
            off, norm = (mine - ref["d" + name]).norm(dim=1), ref["d" + name].norm(dim=1)
            n = c["Dk"] * c["Dv"] if name == "g" else c["Dv"]
            bound = (torch.finfo(dtype).eps / 2 + 9 * 2.0 ** -24 + N) * norm + 4 * N * ref["size_" + name].norm(dim=1) / n ** 0.5
            assert got.dtype == dtype and (off <= bound).all(), (name, (off / bound).max().item())


@pytest.mark.parametrize("c", CASES, ids=name_of)
def test_bf16_results_are_rounded_once(c):
    """o, dq, dk and dv are the 64-bit results rounded to bf16 but where those lie
    next to a border: values off by Q = 8 H^2 of their size end up on its other side
    in 2 Q / H = 16 H of the cases, as a step is H or 2 H of the value.  An operand
    rounded to bf16 on the way moves a third of the values."""
    from uttt_amd.delta import gated_delta_rule
    names = ("q", "k", "v", "g", "beta", "h0")
    x, do, dht = make(c)
    leaf = {n: t.cuda().requires_grad_() for n, t in x.items()}
    cu = None if c["B"] else torch.tensor(offsets(c), dtype=torch.int32, device="cuda")
    o, S = gated_delta_rule(*(leaf[n] for n in names[:5]), initial_state=leaf["h0"], output_final_state=True, cu_seqlens=cu)
    ours = dict(zip(("dq", "dk", "dv"), torch.autograd.grad([o, S], [leaf[n] for n in names[:3]], [do.cuda(), dht.cuda()])),
                o=o.detach())
    pad = lambda t: torch.nn.utils.rnn.pad_sequence(by_sequence(c, t), batch_first=True)  # noqa: E731
    per = c["Hv"] // c["Hk"]
    moved = dict.fromkeys(ours, 0)
    for heads in groups_of_heads(c):
        a, ref = reference(c, x, do, dht, heads, "cuda")
        real = ref["size_g"] > 0
        want = {n: ref[n].unflatten(2, (-1, per)).sum(3) for n in ("dq", "dk")}
        want.update(dv=ref["dv"], o=(a["q"][..., None] * ref["S"][:, 1:]).sum(-2) * c["Dk"] ** -0.5 * real[..., None])
        for n, w in want.items():
            mine = pad(ours[n][:, :, heads[::per] // per if n in ("dq", "dk") else heads])
            moved[n] += (mine != w.to(BF16)).sum().item()
    for n, m in moved.items():
        assert m <= 16 * 2.0 ** -8 * ours[n].numel(), (n, m / ours[n].numel())
