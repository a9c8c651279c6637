"""The gated delta rule sequence by sequence and head by head against the 64-bit
recurrence: three chunks and more with 16, 32 and 64 columns a workgroup, whole
batches and packed sequences, shared key heads, last column blocks of a few.

Bounds per sequence and head, in the 2-norm: those of tests/delta_cases.py for dg
and dbeta; of the others the rounding of the result (bf16's half step H), the
fp32 operands in two bf16 values (Q), and for dq and dk that D and M are rounded
to bf16 once, whose errors add up as the terms of D K do, to H of it."""
import pytest
import torch

from delta_cases import BF16, CASES, F32, H, Q, allowed, by_sequence, groups_of_heads, make, name_of, offsets, reference

pytestmark = pytest.mark.gpu
NAMES = ("q", "k", "v", "g", "beta", "h0")


@pytest.mark.parametrize("c", CASES, ids=name_of)
def test_every_head(c):
    from uttt_amd.delta import gated_delta_rule
    x, do, dht = make(c)
    leaf = {n: t.cuda().requires_grad_() for n, t in x.items()}
    cu = None if c["B"] else torch.tensor(offsets(c), dtype=torch.int32, device="cuda")
    o, S = gated_delta_rule(*(leaf[n] for n in NAMES[:5]), initial_state=leaf["h0"], output_final_state=True,
                            cu_seqlens=cu)
    ours = dict(zip(("d" + n for n in NAMES), torch.autograd.grad([o, S], [leaf[n] for n in NAMES],
                                                                 [do.cuda(), dht.cuda()])), o=o.detach(), S=S.detach())
    for n, t in ours.items():
        assert torch.isfinite(t).all(), n
    pad = lambda t: torch.nn.utils.rnn.pad_sequence(by_sequence(c, t), batch_first=True).double()  # noqa: E731
    per = c["Hv"] // c["Hk"]
    for heads in groups_of_heads(c):
        a, ref = reference(c, x, do, dht, heads, "cuda")
        khead = heads[::per] // per
        want = {n: ref[n].unflatten(2, (-1, per)).sum(3) for n in ("dq", "dk")}
        # S_t for t from 1 on: what token t - 1 leaves
        want.update(o=(a["q"][..., None] * ref["S"][:, 1:]).sum(-2) * c["Dk"] ** -0.5, S=ref["S"][:, -1],
                    **{n: ref[n] for n in ("dv", "dg", "dbeta", "dh0")})
        for n, w in want.items():
            if n in ("S", "dh0"):
                off, bound = (ours[n][:, heads].double() - w).flatten(2).norm(dim=2), Q * w.flatten(2).norm(dim=2)
            else:
                mine = pad(ours[n][:, :, khead if n in ("dq", "dk") else heads])
                if n == "o":   # behind a sequence's end the recurrence goes on reading its state
                    for i, length in enumerate(c["lens"] if not c["B"] else ()):
                        w[i, length:] = 0
                d = (mine - w).transpose(1, 2).flatten(2)
                off = d.norm(dim=2)
                bound = allowed(c, ref, n[1:]) if n in ("dg", "dbeta") else (
                    (H + Q if n in ("o", "dv") else 2 * H) * w.transpose(1, 2).flatten(2).norm(dim=2))
            ratio = (off / bound.clamp_min(1e-30)).max().item()
            assert (off <= bound + 1e-30).all(), (n, ratio, heads.tolist())
        del a, ref, want
