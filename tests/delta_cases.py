"""Cases and bounds for the gradients of the gated delta rule, head by head.

Bounds, relative in the 2-norm over one sequence's tokens of one head, with H =
2^-8 bf16's half step and Q = 8 H^2 what fp32 operands taken as two bf16 values
leave out along the way (tests/test_gpu_delta.py).  dg is <S, dS> and dbeta is
du.(v - S^T k), sums over Dk Dv and Dv products of two factors that are off by Q
of their own size; the factors' errors do not follow the other factor, so of
n products' sizes the error adds up as sqrt(n) of them: the product of the
2-norms over sqrt(n), of which 4 are allowed (four deviations of such a sum for
one token, and the norm is over many)."""
import torch

from oracle import delta as oracle

H = 2.0 ** -8
Q = 8 * H * H
BF16, F32 = torch.bfloat16, torch.float32

# lens: one number of tokens and rows B, or packed sequences of a token axis that
# starts with `front` and ends with `behind` tokens of none; tiles: the 16-column
# tiles a scan's workgroup takes (back: in the backward, where it takes others),
# which a change of that choice has to keep here
CASES = [
    dict(B=2, lens=[330], Hk=1, Hv=2, Dk=64, Dv=64, tiles=1),
    dict(B=1, lens=[200], Hk=2, Hv=2, Dk=192, Dv=72, tiles=1),
    dict(B=48, lens=[200], Hk=2, Hv=2, Dk=40, Dv=40, tiles=2),
    dict(B=32, lens=[260], Hk=1, Hv=2, Dk=96, Dv=72, tiles=2),
    dict(B=16, lens=[200], Hk=2, Hv=2, Dk=128, Dv=136, tiles=2, gates=BF16),
    dict(B=4, lens=[200], Hk=8, Hv=8, Dk=256, Dv=136, tiles=2),
    dict(B=24, lens=[330], Hk=4, Hv=8, Dk=64, Dv=40, tiles=4),
    dict(B=32, lens=[200], Hk=2, Hv=4, Dk=96, Dv=72, tiles=4, gates=BF16),
    dict(B=32, lens=[200], Hk=4, Hv=4, Dk=128, Dv=72, tiles=4),
    dict(B=16, lens=[200], Hk=2, Hv=4, Dk=192, Dv=136, tiles=4, back=2),
    dict(B=8, lens=[270], Hk=4, Hv=8, Dk=256, Dv=136, tiles=2),
    dict(B=0, lens=[300, 1, 0, 129, 250], front=7, behind=13, Hk=8, Hv=16, Dk=64, Dv=64, tiles=1),
    dict(B=0, lens=[64, 200, 0, 65, 40], front=20, behind=11, Hk=32, Hv=128, Dk=40, Dv=40, tiles=2),
    dict(B=0, lens=[271, 1, 128], front=0, behind=0, Hk=48, Hv=48, Dk=64, Dv=136, tiles=2),
    dict(B=0, lens=[330, 3, 0, 64, 65, 100, 10, 100], front=28, behind=0, Hk=32, Hv=96, Dk=96, Dv=72, tiles=4),
    dict(B=0, lens=[200, 0, 0, 17, 63, 80, 1, 20], front=0, behind=19, Hk=24, Hv=48, Dk=128, Dv=136, tiles=4),
]


def name_of(c):
    rows = f"{c['B']}x{c['lens'][0]}" if c["B"] else f"{len(c['lens'])}packed"
    return f"{rows}-{c['Hk']}-{c['Hv']}-{c['Dk']}x{c['Dv']}-{c['tiles']}"


def scan_tiles(T, nseq, Hv, Dk, Dv, packed, backward=False, stored=True):
    """The choice of csrc/delta.h."""
    total, cps = T // 64 + nseq, (T + 63) // 64
    mean = -(-total // nseq)
    cost = {}
    for tiles, tenths in ((1, 20), (2, 28), (4, 40 if stored else 43)):
        if tiles == 4 and Dk > (128 if backward else 192):
            continue
        blocks = -(-Dv // (16 * tiles))
        if packed:
            cost[tiles] = max(min(3 * mean, total), total * Hv * blocks // 256) * tenths
        else:
            cost[tiles] = -(-nseq * Hv * blocks // 256) * cps * tenths
    return min(cost, key=lambda t: (cost[t], t))


def shape(c):
    """tokens, sequences, packed"""
    if c["B"]:
        return c["lens"][0], c["B"], False
    return c["front"] + sum(c["lens"]) + c["behind"], len(c["lens"]), True


def make(c, seed=0):
    T, n, packed = shape(c)
    B, gen = max(c["B"], 1), torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(BF16)  # noqa: E731
    gates = c.get("gates", F32)
    x = dict(q=unit(r(B, T, c["Hk"], c["Dk"]) + 0.2), k=unit(r(B, T, c["Hk"], c["Dk"]) + 0.2),
             v=r(B, T, c["Hv"], c["Dv"]).to(BF16), g=(-0.1 * torch.nn.functional.softplus(r(B, T, c["Hv"]))).to(gates),
             beta=torch.sigmoid(r(B, T, c["Hv"])).to(gates), h0=0.3 * r(n, c["Hv"], c["Dk"], c["Dv"]))
    return x, r(B, T, c["Hv"], c["Dv"]).to(BF16), 0.3 * r(n, c["Hv"], c["Dk"], c["Dv"])


def offsets(c):
    cu = [c["front"]]
    for n in c["lens"]:
        cu.append(cu[-1] + n)
    return cu


def by_sequence(c, t):
    """[B, T, ..] as a list of sequences' [length, ..]."""
    if c["B"]:
        return list(t)
    cu = offsets(c)
    return [t[0, s:e] for s, e in zip(cu[:-1], cu[1:])]


def reference(c, x, do, dht, heads, device="cpu"):
    """oracle.gradients of the value heads `heads`, sequences padded behind their
    end by tokens that change nothing and get zeros."""
    pad = lambda t: torch.nn.utils.rnn.pad_sequence(by_sequence(c, t), batch_first=True).double().to(device)  # noqa: E731
    group = torch.arange(c["Hv"]) // (c["Hv"] // c["Hk"])
    a = {n: pad(x[n][:, :, group[heads]] if n in "qk" else x[n][:, :, heads]) for n in ("q", "k", "v", "g", "beta")}
    got = oracle.gradients(a["q"], a["k"], a["v"], a["g"], a["beta"], x["h0"][:, heads].double().to(device),
                           pad(do[:, :, heads]), dht[:, heads].double().to(device), c["Dk"] ** -0.5)
    if not c["B"]:
        real = torch.arange(max(c["lens"]), device=device) < torch.tensor(c["lens"], device=device)[:, None]
        for n in ("dq", "dk", "dv", "dg", "dbeta", "size_g", "size_beta"):
            got[n] = got[n] * real.view(*real.shape, *(1,) * (got[n].dim() - 2))
    return a, got


def groups_of_heads(c, most=1 << 27):
    """Value heads a few at a time (whole groups of a key head), for the states of every token."""
    T = max(c["lens"]) + 1
    per = c["Hv"] // c["Hk"]
    n = max(1, most // (T * shape(c)[1] * c["Dk"] * c["Dv"] * per)) * per
    return [torch.arange(s, min(s + n, c["Hv"])) for s in range(0, c["Hv"], n)]


def allowed(c, got, name):
    """[N, heads]: what dg or dbeta may be off in the 2-norm over a sequence."""
    ref, size = got["d" + name].norm(dim=1), got["size_" + name].norm(dim=1)
    n = c["Dk"] * c["Dv"] if name == "g" else c["Dv"]
    rounding = torch.finfo(c.get("gates", F32)).eps / 2
    return (rounding + Q) * ref + 4 * Q * size / n ** 0.5
