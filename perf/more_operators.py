"""The state space memory layer's operators as measurable cases: the short
causal convolution, the selective state space scan, both by whole prompts and by
single tokens, and the norms before and after a block.

A case is one pass through one operator at one set of sizes:

  conv   uttt_amd.state_space.causal_conv over whole or packed sequences:
         outputs and the inputs that the next tokens need; with train=True also
         the gradients of the inputs, weights, bias and initial state for given
         gradients of both outputs
  cstep  uttt_amd.state_space.causal_conv_step: a few tokens per sequence
         against a pool's states, updated in place
  scan   uttt_amd.state_space.selective_scan over whole or packed sequences:
         outputs and the state after each sequence; with train=True also the
         gradients of every input
  step   uttt_amd.state_space.selective_scan_step against a pool's states
  after  uttt_amd.norm.norm_after_block: a block's outputs normed, gated, scaled
         and added to the residual; with train=True its backward too
  before uttt_amd.norm.norm_before_block: the last block's outputs scaled and
         added to the residual, and the next block's norm of the sum; with
         train=True its backward too

Widths are the framework's (768: its 124M models; 1536: twice that and the 760M
model's) and odd ones; token counts run from one token over a chunk of 4096 to
batches of packed prompts.  `run` is the plain torch form where `own` is false
and the framework's call where it is true; `exact` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp16": torch.float16}
F32 = torch.float32
BLOCK = 64   # tokens whose states the plain scan holds at a time
EPS = 1e-5


def listed():
    return [
        # prefill of packed prompts of very different lengths in front of a scan, state out
        dict(name="conv_packed", op="conv", lens="5000,1,2311,64,700,0,2,333,129,3000,17,1025", B=0,
             D=1536, W=4, bias=True, act=True, dtype="bf16", wtype="fp32", train=False),
        # a training step's layer: 16 sequences of 2048 tokens
        dict(name="conv_train", op="conv", lens="2048", B=16, D=1536, W=4, bias=True, act=True,
             dtype="bf16", wtype="fp32", train=True),
        # generation for one user: one token of one sequence
        dict(name="cstep_one", op="cstep", B=1, T=1, D=1536, W=4, slots=1, pad=0, dtype="bf16"),
        # generation at serving load: 250 sequences in a pool of 288 slots, padded to 256 rows
        dict(name="cstep_batch", op="cstep", B=256, T=1, D=1536, W=4, slots=288, pad=6, dtype="bf16"),
        # the shortest prompt that matters: a question of some words, one sequence
        dict(name="scan_short", op="scan", lens="77", B=1, D=1536, N=16, G=1, gate=True, soft=True,
             dtype="bf16", dtdtype="bf16", train=False),
        # serving prefill: packed prompts of very different lengths
        dict(name="scan_packed", op="scan", lens="5000,1,2311,64,700,0,4096,333,129,3000,17,1025",
             B=0, D=1536, N=16, G=1, gate=True, soft=True, dtype="bf16", dtdtype="bf16", train=False),
        # a training step's layer: 16 sequences of 2048 tokens
        dict(name="scan_train", op="scan", lens="2048", B=16, D=1536, N=16, G=1, gate=True, soft=True,
             dtype="bf16", dtdtype="bf16", train=True),
        # training on packed documents, ragged, all in 32 bits: an odd width, two groups of B and C,
        # steps used as given, no gate
        dict(name="scan_train_packed", op="scan", lens="1531,77,900,1,640,1203", B=0, D=390, N=24, G=2,
             gate=False, soft=False, dtype="fp32", dtdtype="fp32", train=True),
        # one token of one sequence
        dict(name="step_one", op="step", B=1, T=1, D=1536, N=16, G=1, slots=1, pad=0, dtype="bf16"),
        # 250 sequences in a pool of 288 slots, padded to 256 rows
        dict(name="step_batch", op="step", B=256, T=1, D=1536, N=16, G=1, slots=288, pad=6,
             dtype="bf16"),
        # a training step's norm per head of 192 with the heads' gate, a slice of the projection
        dict(name="after_train", op="after", rows=32768, H=8, N=192, gate=True, residual=False,
             scale=False, dtype="bf16", rtype="bf16", train=True),
        # a training step's norm of the residual stream kept in 32 bits, the block's scale learned
        dict(name="before_train", op="before", rows=32768, N=768, scale=True, dtype="bf16",
             rtype="fp32", train=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lens(rng, total):
    """Whole sequences of one length, or packed ones."""
    if rng.random() < 0.5:
        B = rng.randint(1, 6)
        return dict(B=B, lens=str(max(1, min(total // B, 5000))))
    cuts = sorted(rng.randint(0, total) for _ in range(rng.randint(1, 9)))
    lens = [min(b - a, 5000) for a, b in zip([0] + cuts, cuts + [total])]
    return dict(B=0, lens=",".join(map(str, lens)))


def draw(rng):
    op = rng.choice(["conv", "cstep", "scan", "scan", "scan", "step", "after", "before"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.5
    if op == "conv":
        D = rng.choice([_spread(rng, 1, 2000), 8 * rng.randint(1, 240), 768])
        most = int(16 * 2048 * 1536 / D / (2 if dtype == "fp32" else 1))
        return dict(op=op, **_lens(rng, _spread(rng, 1, min(24000, most))), D=D,
                    W=rng.choice([2, 3, 4, 4, 4, 8]), bias=rng.random() < 0.7, act=rng.random() < 0.7,
                    dtype=dtype, wtype=rng.choice(["fp32", dtype]), train=train)
    if op == "scan":
        G = rng.choice([1, 1, 1, 2, 4])
        D = G * rng.choice([_spread(rng, 1, 500), 64 * rng.randint(1, 12), 384])
        N = rng.choice([1, 4, 7, 8, 16, 16, 16, 24, 32, 64])
        wide = 4 * (-(-N // 4))
        most = int(16 * 2048 * 1536 * 16 / (D * wide) / (2 if dtype == "fp32" else 1))
        return dict(op=op, **_lens(rng, _spread(rng, 1, min(16000, most))), D=D, N=N, G=G,
                    gate=rng.random() < 0.6, soft=rng.random() < 0.6, dtype=dtype,
                    dtdtype=rng.choice(["fp32", dtype]), train=train)
    if op in ("cstep", "step"):
        B, G = _spread(rng, 1, 256), rng.choice([1, 1, 2])
        case = dict(op=op, B=B, T=rng.choice([1, 1, 1, 2, 5]), D=G * rng.choice([384, 768, _spread(rng, 1, 768)]),
                    slots=B + rng.randint(0, 32), pad=rng.randint(0, B // 4), dtype=dtype)
        return dict(case, W=rng.choice([2, 3, 4, 4, 8])) if op == "cstep" else dict(
            case, N=rng.choice([1, 7, 8, 16, 16, 32]), G=G)
    H = 1 if op == "before" else rng.choice([1, 4, 8, 12])
    N = rng.choice([rng.randint(1, 300), _spread(rng, 64, 8192), 8 * rng.randint(8, 200)])
    most = 32768 * 768 // (H * N) // (2 if dtype == "fp32" else 1)
    case = dict(op=op, rows=_spread(rng, 1, max(1, min(65536, most))), N=N, scale=rng.random() < 0.5,
                dtype=dtype, rtype=rng.choice(["fp32", dtype]), train=train)
    return case if op == "before" else dict(case, H=H, gate=rng.random() < 0.7,
                                            residual=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs --
def _ints(text):
    return [int(n) for n in text.split(",")]


def _shape(case):
    """(batch, tokens on the token axis, sequences)"""
    lens = _ints(case["lens"])
    return (case["B"], lens[0], case["B"]) if case["B"] else (1, sum(lens), len(lens))


def _offsets(case):
    if case["B"]:
        return None
    lens = _ints(case["lens"])
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def _slots(case, gen):
    idx = torch.randperm(case["slots"], generator=gen, device="cuda")[:case["B"]].to(torch.int32)
    if case["pad"]:
        idx[case["B"] - case["pad"]:] = -1   # rows behind the last sequence of a padded batch
    return idx


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dt = case["op"], TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    s = dict(case=case)
    if op in ("conv", "cstep"):
        D, W = case["D"], case["W"]
        s["w"] = randn(D, W) / W ** 0.5
        s["b"] = 0.3 * randn(D)
        if op == "cstep":
            s["x"] = randn(case["B"], case["T"], D).to(dt)
            s["state"] = randn(case["slots"], W - 1, D).to(dt)
            s["idx"] = _slots(case, gen)
            return s
        B, T, n = _shape(case)
        wt = TYPES[case["wtype"]]
        s["x"] = randn(B, T, 2, D).to(dt)[:, :, 0]   # half of a fused projection
        s["w"], s["b"] = s["w"].to(wt), s["b"].to(wt) if case["bias"] else None
        s["h0"] = randn(n, W - 1, D).to(dt)
        s["cu"] = _offsets(case)
        if case["train"]:
            s["dy"], s["dht"] = randn(B, T, D).to(dt), randn(n, W - 1, D).to(dt)
            s["names"] = [m for m in ("x", "w", "b", "h0") if s[m] is not None]
    elif op in ("scan", "step"):
        D, N, G = case["D"], case["N"], case["G"]
        B, T, n = _shape(case) if op == "scan" else (case["B"], case["T"], case["slots"])
        soft = case.get("soft", True)
        # decays from nearly none a token to all but gone after some
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=F32) * torch.exp(0.3 * randn(D, N))
        rate = torch.exp(torch.empty(D, device="cuda").uniform_(math.log(1e-3), math.log(0.1), generator=gen))
        s["dtb"] = torch.log(torch.expm1(rate)) if soft else None
        raw = 0.5 * randn(B, T, D)
        dtt = TYPES[case.get("dtdtype", case["dtype"])]
        s["dt"] = (raw if soft else rate * torch.exp(raw)).to(dtt)
        xz = randn(B, T, 2, D)
        s["x"] = torch.nn.functional.silu(xz[:, :, 0]).to(dt)
        s["z"] = xz.to(dt)[:, :, 1] if case.get("gate", True) else None
        bc = randn(B, T, 2, G, N).to(dt)   # slices of one projection
        s["B"], s["C"] = bc[:, :, 0], bc[:, :, 1]
        s["D"] = 1 + 0.2 * randn(D)
        s["h0"] = 0.3 * randn(n, D, N)
        s["soft"] = soft
        if op == "step":
            s["idx"] = _slots(case, gen)
            return s
        s["cu"] = _offsets(case)
        if case["train"]:
            s["dy"], s["dht"] = randn(B, T, D).to(dt), 0.3 * randn(n, D, N)
            s["names"] = [m for m in ("x", "dt", "A", "B", "C", "D", "z", "dtb", "h0") if s[m] is not None]
    else:
        N, rows, rt = case["N"], case["rows"], TYPES[case["rtype"]]
        shape = (rows, N) if op == "before" else (rows, case["H"], N)
        s["x"] = (2.0 * randn(*shape) + 0.3).to(dt)
        s["w"] = 1 + 0.2 * randn(N)
        s["s"] = 0.1 * randn(N) if case["scale"] else None
        s["r"] = randn(*shape).to(rt) if op == "before" or case["residual"] else None
        s["z"] = None
        if op == "after" and case["gate"]:
            s["z"] = randn(rows, 2, *shape[1:]).to(dt)[:, 1]   # half of a fused projection
        if case["train"]:
            s["dy"] = randn(*shape).to(dt if op == "before" or s["r"] is None else rt)
            s["dh"] = randn(*shape).to(rt)
            s["names"] = [m for m in ("x", "w", "z", "r", "s") if s[m] is not None]
    for m in s.get("names", ()):
        s[m].requires_grad_()
    return s


# ------------------------------------------------------------- plain forms --
def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x)))


def _places(case, cu):
    """Packed rows: their sequence and their place in it."""
    lens = _ints(case["lens"])
    pos = torch.arange(sum(lens), device="cuda")
    seq = torch.searchsorted(cu[1:].long(), pos, right=True)
    return seq, pos - cu.long()[seq], max(lens)


def _rows(case, cu):
    """Functions from [B, T, ...] to a batch of padded sequences and back."""
    if case["B"]:
        return (lambda t: t), (lambda t: t), torch.full((case["B"],), _ints(case["lens"])[0], device="cuda")
    seq, place, longest = _places(case, cu)
    n = cu.numel() - 1

    def out(t):
        return torch.zeros((n, longest) + t.shape[2:], dtype=t.dtype, device="cuda").index_put((seq, place), t[0])

    return out, (lambda t: t[seq, place][None]), (cu[1:] - cu[:-1]).long()


def _run_conv_plain(s):
    case = s["case"]
    W, dt = case["W"], s["x"].dtype
    pack, unpack, lens = _rows(case, s["cu"])
    full = torch.cat([s["h0"].float(), pack(s["x"].float())], 1)
    w, n = s["w"].float(), full.shape[1] - W + 1
    pre = sum(full[:, k:k + n] * w[:, k] for k in range(W))
    if s["b"] is not None:
        pre = pre + s["b"].float()
    y = unpack(_silu(pre) if case["act"] else pre).to(dt)
    at = lens[:, None] + torch.arange(W - 1, device="cuda")
    state = torch.gather(full, 1, at[..., None].expand(-1, -1, full.shape[2])).to(dt)
    if not case["train"]:
        return dict(y=y, state=state)
    grads = torch.autograd.grad([y, state], [s[m] for m in s["names"]], [s["dy"], s["dht"]])
    return dict(y=y.detach(), state=state.detach(), **{"d_" + m: t for m, t in zip(s["names"], grads)})


def _run_cstep_plain(s):
    case = s["case"]
    keep = s["idx"] >= 0
    rows, W, T = s["idx"][keep].long(), case["W"], case["T"]
    full = torch.cat([s["state"][rows], s["x"][keep]], 1)
    x = full.float()
    pre = sum(x[:, k:k + T] * s["w"][:, k] for k in range(W)) + s["b"]
    y = torch.zeros_like(s["x"])
    y[keep] = _silu(pre).to(y.dtype)
    s["state"][rows] = full[:, T:]
    return dict(y=y, state=s["state"])


def _per_channel(t, D):
    """[n, L, G, N] -> [n, L, D, N]: each group's values for its channels."""
    G = t.shape[2]
    return t[:, :, :, None].expand(-1, -1, -1, D // G, -1).reshape(*t.shape[:2], D, t.shape[3])


def _scan_forward(u, dt, A, Bm, Cm, h, keep):
    """y of [n, L, D], the last state, and all states by blocks where kept."""
    D, ys, states = A.shape[0], [], []
    for t0 in range(0, u.shape[1], BLOCK):
        blk = slice(t0, t0 + BLOCK)
        a = torch.exp(dt[:, blk, :, None] * A)
        ub = u[:, blk, :, None] * _per_channel(Bm[:, blk], D)
        hs = []
        for t in range(a.shape[1]):
            h = ub[:, t] + a[:, t] * h
            hs.append(h)
        hs = torch.stack(hs, 1)
        ys.append((hs * _per_channel(Cm[:, blk], D)).sum(-1))
        if keep:
            states.append(hs)
    return torch.cat(ys, 1) if ys else u, h, states


def _scan_backward(u, dt, A, Bm, Cm, h0, states, dy, carry):
    """Gradients of u, dt, A, B, C and h0 for gradients dy of y, carry of the last state."""
    (n, L, D), G, N = u.shape, Bm.shape[2], A.shape[1]
    du, ddt, dB, dC = [], [], [], []
    dA = torch.zeros_like(A)

    def by_group(t):
        return t.reshape(n, -1, G, D // G, N).sum(3)

    for i in reversed(range(len(states))):
        blk = slice(i * BLOCK, (i + 1) * BLOCK)
        hs = states[i]
        before = torch.cat([(states[i - 1][:, -1] if i else h0)[:, None], hs[:, :-1]], 1)
        a = torch.exp(dt[:, blk, :, None] * A)
        g = dy[:, blk, :, None] * _per_channel(Cm[:, blk], D)
        for t in reversed(range(a.shape[1])):
            g[:, t] += carry
            carry = a[:, t] * g[:, t]
        dC.append(by_group(dy[:, blk, :, None] * hs))
        dB.append(by_group(u[:, blk, :, None] * g))
        du.append((g * _per_channel(Bm[:, blk], D)).sum(-1))
        w = g * a * before
        ddt.append((w * A).sum(-1))
        dA += (w * dt[:, blk, :, None]).sum((0, 1))
    if not states:
        return u, dt, dA, Bm, Cm, carry
    return *(torch.cat(t[::-1], 1) for t in (du, ddt)), dA, *(torch.cat(t[::-1], 1) for t in (dB, dC)), carry


@torch.no_grad()
def _run_scan_plain(s):
    case, train = s["case"], s["case"]["train"]
    pack, unpack, _ = _rows(case, s["cu"])
    f = {m: None if s[m] is None else s[m].detach().float() for m in ("x", "dt", "A", "B", "C", "D", "z", "dtb", "h0")}
    raw = f["dt"] if f["dtb"] is None else f["dt"] + f["dtb"]
    dt = pack(_softplus(raw) if s["soft"] else raw)   # no step at all behind a sequence's end
    x, Bm, Cm, A = pack(f["x"]), pack(f["B"]), pack(f["C"]), f["A"]
    u = dt * x
    core, state, states = _scan_forward(u, dt, A, Bm, Cm, f["h0"], train)
    core = unpack(core + f["D"] * x)
    y = core if f["z"] is None else core * _silu(f["z"])
    out = dict(y=y.to(s["x"].dtype), state=state)
    if not train:
        return out
    dy = s["dy"].float()
    g = {}
    if f["z"] is not None:
        sig = 1 / (1 + torch.exp(-f["z"]))
        g["z"] = dy * core * sig * (1 + f["z"] * (1 - sig))
        dy = dy * f["z"] * sig
    du, ddt, g["A"], dB, dC, g["h0"] = _scan_backward(u, dt, A, Bm, Cm, f["h0"], states, pack(dy), s["dht"])
    g["x"] = unpack(du * dt) + f["D"] * dy
    g["D"] = (dy * f["x"]).sum((0, 1))
    g["dt"] = unpack(ddt + du * x)
    if s["soft"]:
        g["dt"] = g["dt"] / (1 + torch.exp(-raw))
    if f["dtb"] is not None:
        g["dtb"] = g["dt"].sum((0, 1))
    g["B"], g["C"] = unpack(dB), unpack(dC)
    return dict(out, **{"d_" + m: g[m].to(s[m].dtype) for m in s["names"]})


def _run_step_plain(s):
    case = s["case"]
    keep = s["idx"] >= 0
    rows, D = s["idx"][keep].long(), case["D"]
    h, out = s["h0"][rows], []
    x, z = s["x"][keep].float(), s["z"][keep].float()
    dt = _softplus(s["dt"][keep].float() + s["dtb"])
    Bm, Cm = (_per_channel(s[m][keep].float(), D) for m in ("B", "C"))
    for t in range(case["T"]):
        h = torch.exp(dt[:, t, :, None] * s["A"]) * h + (dt[:, t] * x[:, t])[..., None] * Bm[:, t]
        out.append(((h * Cm[:, t]).sum(-1) + s["D"] * x[:, t]) * _silu(z[:, t]))
    s["h0"][rows] = h
    y = torch.zeros_like(s["x"])
    y[keep] = torch.stack(out, 1).to(y.dtype)
    return dict(y=y, state=s["h0"])


def _run_norm_plain(s):
    case, f = s["case"], {m: None if s[m] is None else s[m].float() for m in ("x", "w", "s", "r", "z")}
    x = f["x"]
    if case["op"] == "before":
        h = f["r"] + (x if f["s"] is None else x * f["s"])
        y = (h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * f["w"]).to(s["x"].dtype)
        out = dict(y=y, h=h.to(s["r"].dtype))
    else:
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * f["w"]
        if f["z"] is not None:
            y = y * _silu(f["z"])
        if f["s"] is not None:
            y = y * f["s"]
        if f["r"] is not None:
            y = y + f["r"]
        out = dict(y=y.to(s["x"].dtype if s["r"] is None else s["r"].dtype))
    if not case["train"]:
        return out
    grads = torch.autograd.grad(list(out.values()), [s[m] for m in s["names"]],
                                [s["dy"], s["dh"]][:len(out)])
    return {**{m: t.detach() for m, t in out.items()}, **{"d_" + m: t for m, t in zip(s["names"], grads)}}


# ----------------------------------------------------- the framework's calls --
def _run_own(s):
    from uttt_amd import norm, state_space
    case = s["case"]
    op = case["op"]
    if op == "cstep":
        y = state_space.causal_conv_step(s["x"], s["w"], s["state"], s["b"], activation="silu",
                                         state_indices=s["idx"])
        return dict(y=y, state=s["state"])
    if op == "step":
        y = state_space.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["h0"], D=s["D"],
                                            gate=s["z"], dt_bias=s["dtb"], dt_softplus=True,
                                            state_indices=s["idx"])
        return dict(y=y, state=s["h0"])
    if op == "conv":
        out = state_space.causal_conv(s["x"], s["w"], s["b"], activation="silu" if case["act"] else None,
                                      initial_state=s["h0"], output_final_state=True, cu_seqlens=s["cu"])
        out = dict(zip(("y", "state"), out))
    elif op == "scan":
        out = state_space.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], gate=s["z"],
                                         dt_bias=s["dtb"], dt_softplus=s["soft"], initial_state=s["h0"],
                                         output_final_state=True, cu_seqlens=s["cu"])
        out = dict(zip(("y", "state"), out))
    elif op == "before":
        out = dict(zip(("y", "h"), norm.norm_before_block(s["x"], s["r"], s["w"], scale=s["s"], eps=EPS)))
    else:
        out = dict(y=norm.norm_after_block(s["x"], s["w"], gate=s["z"], residual=s["r"], scale=s["s"], eps=EPS))
    if not case["train"]:
        return out
    given = [s["dy"]] + ([] if len(out) == 1 else [s["dh"] if op == "before" else s["dht"]])
    grads = torch.autograd.grad(list(out.values()), [s[m] for m in s["names"]], given)
    return {**{m: t.detach() for m, t in out.items()}, **{"d_" + m: t for m, t in zip(s["names"], grads)}}


def run(state):
    if own:
        return _run_own(state)
    plain = dict(conv=_run_conv_plain, cstep=_run_cstep_plain, scan=_run_scan_plain, step=_run_step_plain)
    return plain.get(state["case"]["op"], _run_norm_plain)(state)


def work(case):
    """Every input read once, every output written once.  Operations: 2 W a
    channel of a convolution, 6 a state of a scan (its decay's product and
    exponential, its update and its output; three times that with its gradients)
    and some for each element."""
    op, size = case["op"], TYPES[case["dtype"]].itemsize
    if op in ("conv", "cstep"):
        D, W = case["D"], case["W"]
        if op == "cstep":
            rows = case["B"] - case["pad"]
            n = rows * case["T"] * D
            return dict(bytes=2 * n * size + 2 * rows * (W - 1) * D * size + 4 * D * (W + 1),
                        flops=n * (2 * W + 4))
        B, T, seqs = _shape(case)
        n, ends = B * T * D, seqs * (W - 1) * D * size
        par = (W + bool(case["bias"])) * D * TYPES[case["wtype"]].itemsize
        by, fl = 2 * n * size + 2 * ends + par, n * (2 * W + (4 if case["act"] else 0))
        if case["train"]:   # x and dy read, dx written
            by, fl = by + 3 * n * size + 2 * ends + 2 * par, 3 * fl
        return dict(bytes=by, flops=fl)
    if op in ("scan", "step"):
        D, N, G = case["D"], case["N"], case["G"]
        par = 4 * D * (N + 2)
        if op == "step":
            rows = case["B"] - case["pad"]
            tok = rows * case["T"]
            return dict(bytes=rows * D * N * 8 + tok * (4 * D + 2 * G * N) * size + par, flops=6 * tok * D * N)
        B, T, seqs = _shape(case)
        row = (D * (2 if case["gate"] else 1) + 2 * G * N) * size + D * TYPES[case["dtdtype"]].itemsize
        by, fl = B * T * (row + D * size) + 2 * seqs * D * N * 4 + par, 6 * B * T * D * N
        if case["train"]:
            by += B * T * (2 * row + D * size) + 2 * seqs * D * N * 4 + 2 * par
            fl *= 3
        return dict(bytes=by, flops=fl)
    n, rt = case["rows"] * case.get("H", 1) * case["N"], TYPES[case["rtype"]].itemsize
    par = case["N"] * 4 * (2 if case["scale"] else 1)
    if op == "before":   # x and the residual in, the norm and the sum out; their gradients in, two out
        by = 2 * n * (size + rt) + par
        return dict(bytes=by + (3 * n * (size + rt) + 2 * par if case["train"] else 0),
                    flops=n * (24 if case["train"] else 8))
    ins, z = n * size, n * size if case["gate"] else 0
    r, y = n * rt if case["residual"] else 0, n * (rt if case["residual"] else size)
    by = ins + z + r + y + par
    if case["train"]:
        by += 2 * (ins + z) + y + r + 2 * par
    return dict(bytes=by, flops=n * (36 if case["train"] else 12))


# -------------------------------------------------- the definition, 64 bits --
def _exact_conv(case, s):
    W = case["W"]
    leaf = {m: s[m].detach().double() for m in ("x", "w", "b", "h0") if s[m] is not None}
    if case["train"]:
        leaf = {m: t.requires_grad_() for m, t in leaf.items()}
    x = leaf["x"]
    seqs = list(x) if case["B"] else list(torch.split(x[0], _ints(case["lens"])))
    ys, ends = [], []
    for h0, part in zip(leaf["h0"], seqs):
        full = torch.cat([h0, part])
        ends.append(full[full.shape[0] - (W - 1):])
        if part.shape[0]:
            pre = torch.matmul(full.unfold(0, W, 1)[..., None, :], leaf["w"][..., None])[..., 0, 0]
            pre = pre + leaf["b"] if "b" in leaf else pre
            ys.append(pre * torch.sigmoid(pre) if case["act"] else pre)
    y = torch.stack(ys) if case["B"] else torch.cat(ys or [x[0]])[None]
    out = dict(y=y, state=torch.stack(ends))
    if not case["train"]:
        return out
    grads = torch.autograd.grad(list(out.values()), [leaf[m] for m in s["names"]],
                                [s["dy"].double(), s["dht"].double()], allow_unused=True)
    grads = [torch.zeros_like(leaf[m]) if t is None else t for m, t in zip(s["names"], grads)]
    return {**{m: t.detach() for m, t in out.items()}, **{"d_" + m: t for m, t in zip(s["names"], grads)}}


def _exact_scan(case, s):
    """Token by token over all sequences at once, the longer ones first."""
    B, T, n = _shape(case)
    lens = [T] * n if case["B"] else _ints(case["lens"])
    D, N, G = case["D"], case["N"], case["G"]
    held = sum(lens) * D * N * 8 * (5 if case["train"] else 0)
    if max(lens) * (5 if case["train"] else 1) > 40000 or held > 100e9:
        return None
    leaf = {m: s[m].detach().double() for m in ("x", "dt", "A", "B", "C", "D", "z", "dtb", "h0") if s[m] is not None}
    if case["train"]:
        leaf = {m: t.requires_grad_() for m, t in leaf.items()}
    first = [0] * n if case["B"] else [sum(lens[:i]) for i in range(n)]
    order = sorted(range(n), key=lambda i: -lens[i])
    step = leaf["dt"] + leaf["dtb"] if "dtb" in leaf else leaf["dt"]
    if s["soft"]:
        step = torch.logaddexp(step, torch.zeros((), dtype=step.dtype, device="cuda"))
    flat = lambda t: t.reshape(B * T, *t.shape[2:])  # noqa: E731
    step, x, Bm, Cm = flat(step), flat(leaf["x"]), flat(leaf["B"]), flat(leaf["C"])
    start = torch.tensor([i * T if case["B"] else first[i] for i in order], device="cuda")
    h, ends, ys = leaf["h0"][torch.tensor(order, device="cuda")], [], []
    tokens = []
    for t in range(max(lens) if lens else 0):
        live = sum(lens[i] > t for i in order)
        if live < h.shape[0]:
            ends.append(h[live:])
            h = h[:live]
        at = start[:live] + t
        dtt = step[at]
        B_t, C_t = (m[at].repeat_interleave(D // G, 1) for m in (Bm, Cm))
        h = h * (dtt[..., None] * leaf["A"]).exp() + B_t * (dtt * x[at])[..., None]
        ys.append(torch.matmul(h[..., None, :], C_t[..., None])[..., 0, 0])
        tokens.append(at)
    ends.append(h)
    back = torch.empty(n, dtype=torch.long, device="cuda")
    back[torch.tensor(order, device="cuda")] = torch.arange(n, device="cuda")
    state = torch.cat(ends[::-1])[back]
    y = x * 0
    if ys:
        where = torch.argsort(torch.cat(tokens))
        y = torch.cat(ys)[where] + leaf["D"] * x
    y = y.reshape(B, T, D)
    if "z" in leaf:
        y = y * leaf["z"] * torch.sigmoid(leaf["z"])
    out = dict(y=y, state=state)
    if not case["train"]:
        return out
    grads = torch.autograd.grad([y, state], [leaf[m] for m in s["names"]],
                                [s["dy"].double(), s["dht"].double()], allow_unused=True)
    grads = [torch.zeros_like(leaf[m]) if t is None else t for m, t in zip(s["names"], grads)]
    return dict(y=y.detach(), state=state.detach(), **{"d_" + m: t for m, t in zip(s["names"], grads)})


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "conv":
        return _exact_conv(case, s)
    if op == "scan":
        return _exact_scan(case, s)
    if op == "cstep":
        y, state = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda"), s["state"].double()
        used = [(b, i) for b, i in enumerate(s["idx"].tolist()) if i >= 0]
        if used:
            b, i = (torch.tensor(t, device="cuda") for t in zip(*used))
            win = state[i]
            for t in range(case["T"]):
                win = torch.cat([win, s["x"][b, t:t + 1].double()], 1)
                pre = torch.matmul(s["w"].double()[:, None], win.permute(0, 2, 1)[..., None])[..., 0, 0] + s["b"].double()
                y[b, t] = pre * torch.sigmoid(pre)
                win = win[:, 1:]
            state[i] = win
        return dict(y=y, state=state)
    if op == "step":
        y, state = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda"), s["h0"].double()
        group = torch.arange(case["D"], device="cuda") // (case["D"] // case["G"])
        used = [(b, i) for b, i in enumerate(s["idx"].tolist()) if i >= 0]
        if used:
            b, i = (torch.tensor(t, device="cuda") for t in zip(*used))
            h = state[i]
            for t in range(case["T"]):
                x, z, raw = (s[m][b, t].double() for m in ("x", "z", "dt"))
                dt = torch.nn.functional.softplus(raw + s["dtb"].double(), threshold=200.0)
                B_t, C_t = (s[m][b, t].double()[:, group] for m in ("B", "C"))
                h = (dt[..., None] * s["A"].double()).exp() * h + B_t * (dt * x)[..., None]
                core = torch.matmul(h[..., None, :], C_t[..., None])[..., 0, 0] + s["D"].double() * x
                y[b, t] = core * z * torch.sigmoid(z)
            state[i] = h
        return dict(y=y, state=state)
    leaf = {m: s[m].detach().double().requires_grad_() for m in ("x", "w", "s", "r", "z") if s[m] is not None}
    x = leaf["x"]
    if op == "before":
        h = leaf["r"] + x * leaf.get("s", 1.0)
        out = dict(y=h * (h.pow(2).sum(-1, keepdim=True) / case["N"] + EPS).pow(-0.5) * leaf["w"], h=h)
    else:
        y = x * (x.pow(2).sum(-1, keepdim=True) / case["N"] + EPS).pow(-0.5) * leaf["w"] * leaf.get("s", 1.0)
        if "z" in leaf:
            y = y * leaf["z"] * torch.sigmoid(leaf["z"])
        out = dict(y=y + leaf.get("r", 0.0))
    if not case["train"]:
        return {m: t.detach() for m, t in out.items()}
    grads = torch.autograd.grad(list(out.values()), [leaf[m] for m in s["names"]],
                                [s["dy"].double(), s["dh"].double()][:len(out)])
    return {**{m: t.detach() for m, t in out.items()}, **{"d_" + m: t for m, t in zip(s["names"], grads)}}
