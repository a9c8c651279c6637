"""The bounds of tests/delta_cases.py on the CPU: they hold the gradients' own
terms apart.  The mistakes are planted in the oracle's values."""
import pytest
import torch

from delta_cases import CASES, allowed, by_sequence, groups_of_heads, make, name_of, offsets, reference, scan_tiles, shape
from oracle import delta as oracle

C = 64


def test_gradients_of_the_oracle():
    """Against autograd through the recurrence."""
    c = dict(B=2, lens=[70], Hk=1, Hv=2, Dk=8, Dv=16)
    x, do, dht = make(c)
    a, got = reference(c, x, do, dht, torch.arange(2))
    leaf = [x[n].double().requires_grad_() for n in ("q", "k", "v", "g", "beta", "h0")]
    o, S = oracle.gated_delta_rule(*leaf[:5], 8 ** -0.5, leaf[5])
    want = torch.autograd.grad([o, S], leaf, [do.double(), dht.double()])
    got["dq"], got["dk"] = got["dq"].sum(2, keepdim=True), got["dk"].sum(2, keepdim=True)
    for n, w in zip(("dq", "dk", "dv", "dg", "dbeta", "dh0"), want):
        assert torch.allclose(got[n], w, rtol=1e-11, atol=1e-12), n
    assert torch.allclose(got["S"][:, -1], S.detach(), rtol=1e-12, atol=1e-13)


@pytest.mark.parametrize("c", CASES, ids=name_of)
def test_cases_take_their_column_widths(c):
    T, n, packed = shape(c)
    assert scan_tiles(T, n, c["Hv"], c["Dk"], c["Dv"], packed) == c["tiles"]
    assert scan_tiles(T, n, c["Hv"], c["Dk"], c["Dv"], packed, True) == c.get("back", c["tiles"])
    assert max(c["lens"]) > 2 * C   # three chunks or more
    if packed:
        assert offsets(c)[-1] + c["behind"] == T and len(by_sequence(c, torch.zeros(1, T))) == n


def terms(c, a, got):
    """The chunked form's terms of dg and dbeta (formulas in csrc/delta_bwd.hip)."""
    scale = c["Dk"] ** -0.5
    dg = {n: torch.zeros_like(a["g"]) for n in ("pairs", "q", "k", "ahead", "state")}
    db = {n: torch.zeros_like(a["g"]) for n in ("v", "state", "pairs")}
    T = a["g"].shape[1]
    for s in range(0, T, C):
        e = min(s + C, T)
        q, k, v, u, du, do = (t[:, s:e].transpose(1, 2) for t in (a["q"], a["k"], a["v"], got["u"], got["du"], a["do"]))
        g, b = a["g"][:, s:e].transpose(1, 2), a["beta"][:, s:e].transpose(1, 2)
        S0, dS = got["S"][:, s], got["dS"][:, e]
        G = g.cumsum(-1)
        E = torch.exp((G[..., :, None] - G[..., None, :])).tril()
        kk, qk = k @ k.transpose(-1, -2), q @ k.transpose(-1, -2)
        D = scale * E * (do @ u.transpose(-1, -2))
        m = -E.tril(-1) * (du @ u.transpose(-1, -2))
        X = D * qk + b[..., None] * m * kk
        before = torch.ones(e - s, e - s, dtype=torch.float64).triu(1)       # j < t
        Z = X @ before
        i_t = torch.ones(e - s, e - s, dtype=torch.float64).tril()            # i >= t
        gam = torch.exp(G)
        kS = (k * (du @ S0.transpose(-1, -2))).sum(-1)
        here = lambda d, n, t: d[n][:, s:e].copy_(t.transpose(1, 2))  # noqa: E731
        here(dg, "pairs", (Z * i_t).sum(-2))
        here(dg, "q", (scale * gam * (q * (do @ S0.transpose(-1, -2))).sum(-1)) @ i_t)
        here(dg, "k", -(b * gam * kS) @ i_t)
        here(dg, "ahead", (torch.exp(G[..., -1:] - G) * (k * (u @ dS.transpose(-1, -2))).sum(-1)) @ before)
        here(dg, "state", (gam[..., -1:] * (S0 * dS).sum((-2, -1))[..., None]).expand_as(G))
        here(db, "v", (du * v).sum(-1))
        here(db, "state", -gam * kS)
        here(db, "pairs", (m * kk).sum(-1))
    return dg, db


@pytest.mark.parametrize("c", CASES, ids=name_of)
def test_bounds_hold_the_terms_apart(c):
    """One term of dg or dbeta, one head or one chunk left out is out of bounds in
    every case, for a few of its heads."""
    x, do, dht = make(c)
    heads = groups_of_heads(c, 1 << 24)[0]
    a, got = reference(c, x, do, dht, heads)
    a["do"] = torch.nn.utils.rnn.pad_sequence(by_sequence(c, do[:, :, heads]), batch_first=True).double()
    longest = max(range(len(c["lens"])), key=lambda i: c["lens"][i]) if not c["B"] else 0
    for name, parts in zip(("g", "beta"), terms(c, a, got)):
        ref, bound = got["d" + name], allowed(c, got, name)
        for n in parts:   # behind a sequence's end
            parts[n] = parts[n] * (got["size_g"] > 0)
        assert torch.allclose(sum(parts.values()), ref, rtol=1e-9, atol=1e-9 * ref.abs().max().item()), name
        over = lambda off: off.norm(dim=1) > bound  # noqa: E731
        for n, part in parts.items():
            assert over(part)[longest].all(), (name, n)
        assert over(ref)[longest].all()   # a head that gets nothing
        for s in range(0, c["lens"][longest], C):
            part = torch.zeros_like(ref)
            part[:, s:s + C] = ref[:, s:s + C]
            if min(C, c["lens"][longest] - s) >= 16:
                assert over(part)[longest].all(), (name, "chunk", s)
