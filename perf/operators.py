"""The gated delta rule, layer norm and the rotary embedding over several
position axes, as measurable cases.

A case is one pass through one operator at one set of sizes:

  delta   uttt_amd.delta.gated_delta_rule over whole prompts or packed
          sequences: outputs and the state after each sequence; with
          train=True also the gradients of q, k, v, g, beta and the initial
          state for given gradients of both outputs
  step    uttt_amd.delta.gated_delta_step: a few tokens per sequence against
          states kept in place in a pool, one slot per sequence
  norm    uttt_amd.norm.layer_norm; with train=True its backward too
  rotary  uttt_amd.positions.rotary_axes on a view of a fused projection;
          with train=True its backward too

Head widths are the framework's (192: the 124M models' four heads; 96: its
CPU configuration) and the generic 64 and 128; token counts run from one token
over a chunk of 4096 to batches of packed prompts.  `run` is the plain torch
form where `own` is false and the framework's call where it is true; `exact`
is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16
TYPES = {"bf16": BF16, "fp32": F32, "fp16": F16}
CHUNK = 64


def listed():
    return [
        # the shortest prompt that matters: a question of some words, one sequence
        dict(name="delta_short", op="delta", lens="77", B=1, Hk=4, Hv=4, Dk=64, Dv=64,
             gates="fp32", train=False),
        # one chunk of 4096 tokens of a 124M-width layer (four heads of 192), state in and out
        dict(name="delta_chunk", op="delta", lens="4096", B=1, Hk=4, Hv=4, Dk=192, Dv=192,
             gates="fp32", train=False),
        # serving prefill: packed prompts of very different lengths, two value heads per key head
        dict(name="delta_packed", op="delta", lens="5000,1,2311,64,700,0,4096,333,129,3000,17,1025",
             B=0, Hk=8, Hv=16, Dk=128, Dv=128, gates="fp32", train=False),
        # a training step's layer: 16 sequences of 2048 tokens, 12 heads (hidden size 1536)
        dict(name="delta_train", op="delta", lens="2048", B=16, Hk=12, Hv=12, Dk=128, Dv=128,
             gates="bf16", train=True),
        # training on packed documents, ragged, shared key heads, value width unlike key width
        dict(name="delta_train_packed", op="delta", lens="1531,77,900,1,640,1203", B=0, Hk=2, Hv=4,
             Dk=96, Dv=192, gates="bf16", train=True),
        # generation for one user: one token of one sequence
        dict(name="step_one", op="step", B=1, T=1, Hk=4, Hv=4, Dk=192, Dv=192, slots=1, pad=0,
             dtype="bf16"),
        # generation at serving load: 250 sequences in a pool of 288 slots, padded to 256 rows
        dict(name="step_batch", op="step", B=256, T=1, Hk=8, Hv=16, Dk=128, Dv=128, slots=288,
             pad=6, dtype="bf16"),
        # layer norm of a decode step: a few rows of 768
        dict(name="norm_few", op="norm", rows=8, N=768, dtype="bf16", wtype="bf16", train=False),
        # a training step's layer norm over 65 536 tokens of 768
        dict(name="norm_train", op="norm", rows=65536, N=768, dtype="bf16", wtype="fp32",
             train=True),
        # a width that no vector divides, all in 32 bits
        dict(name="norm_odd", op="norm", rows=4099, N=1537, dtype="fp32", wtype="fp32", train=True),
        # image tokens of eight views of 16 x 32 patches: view, row and column positions
        dict(name="rotary_views", op="rotary", B=1, L=4096, H=12, D=64, sections="8,12,12",
             dtype="bf16", interleaved=False, train=False),
        # video training: time, row and column; part of the features unrotated; pairs side by side
        dict(name="rotary_train", op="rotary", B=3, L=8191, H=12, D=128, sections="16,16,16",
             dtype="bf16", interleaved=True, train=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["delta", "delta", "delta", "step", "norm", "rotary"])
    if op == "delta":
        train = rng.random() < 0.5
        Hk = rng.choice([1, 2, 4, 6, 8])
        Hv = Hk * rng.choice([1, 1, 2, 3])
        Dk, Dv = rng.choice([40, 64, 96, 128, 192]), rng.choice([64, 72, 128, 192])
        # at most the largest listed case's tokens x heads x widths
        most = int(16 * 2048 * 12 * 128 * 128 / (Hv * Dk * Dv) / (4 if train else 2))
        total = _spread(rng, 3, min(24000, most))
        case = dict(op="delta", Hk=Hk, Hv=Hv, Dk=Dk, Dv=Dv, gates="bf16" if train else
                    rng.choice(["fp32", "bf16"]), train=train)
        if rng.random() < 0.5:
            B = rng.randint(1, 4)
            return dict(case, B=B, lens=str(max(1, min(total // B, 6000))))
        cuts = sorted(rng.randint(0, total) for _ in range(rng.randint(1, 9)))
        lens = [b - a for a, b in zip([0] + cuts, cuts + [total])]
        return dict(case, B=0, lens=",".join(str(min(n, 6000)) for n in lens))
    if op == "step":
        Hk = rng.choice([1, 2, 4, 8])
        B = _spread(rng, 1, 256)
        return dict(op="step", B=B, T=rng.choice([1, 1, 1, 2, 5]), Hk=Hk,
                    Hv=Hk * rng.choice([1, 2]), Dk=rng.choice([40, 64, 96, 128]),
                    Dv=rng.choice([64, 72, 128]), slots=B + rng.randint(0, 32),
                    pad=rng.randint(0, B // 4), dtype=rng.choice(["bf16", "bf16", "fp32", "fp16"]))
    if op == "norm":
        N = rng.choice([rng.randint(1, 300), _spread(rng, 64, 16384), 8 * rng.randint(8, 700)])
        return dict(op="norm", rows=_spread(rng, 1, min(65536, 65536 * 768 // N)), N=N,
                    dtype=rng.choice(["bf16", "fp32", "fp16"]),
                    wtype=rng.choice(["fp32", "bf16", "none"]), train=rng.random() < 0.6)
    s = [rng.randint(1, 16) for _ in range(rng.choice([1, 2, 3, 3, 4]))]
    return dict(op="rotary", B=rng.randint(1, 3), L=_spread(rng, 1, 8000), H=rng.choice([1, 4, 12]),
                D=2 * sum(s) + rng.choice([0, 0, 2, 16, 33]), sections=",".join(map(str, s)),
                dtype=rng.choice(["bf16", "fp32", "fp16"]), interleaved=rng.random() < 0.5,
                train=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs --
def _ints(text):
    return [int(n) for n in text.split(",")]


def _delta_shape(case):
    """(batch, tokens on the token axis, sequences)"""
    lens = _ints(case["lens"])
    return (case["B"], lens[0], case["B"]) if case["B"] else (1, sum(lens), len(lens))


def _gates(gen, shape, dtype):
    """Log decays from nearly one to strong forgetting, write strengths in (0, 1)."""
    rate = torch.exp(torch.empty(shape[-1], device="cuda").uniform_(-6.0, 0.0, generator=gen))
    g = -rate * torch.nn.functional.softplus(torch.randn(shape, device="cuda", generator=gen))
    beta = torch.sigmoid(torch.randn(shape, device="cuda", generator=gen))
    return g.to(dtype), beta.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    def unit(*shape):
        x = randn(*shape) + 0.3
        return x / x.norm(dim=-1, keepdim=True)

    s = dict(case=case)
    if case["op"] == "delta":
        B, T, n = _delta_shape(case)
        Hk, Hv, Dk, Dv = case["Hk"], case["Hv"], case["Dk"], case["Dv"]
        s["q"], s["k"] = unit(B, T, Hk, Dk).to(BF16), unit(B, T, Hk, Dk).to(BF16)
        s["v"] = randn(B, T, Hv, Dv).to(BF16)
        s["g"], s["beta"] = _gates(gen, (B, T, Hv), TYPES[case["gates"]])
        s["h0"] = 0.3 * randn(n, Hv, Dk, Dv)
        s["cu"] = None
        if not case["B"]:
            lens = _ints(case["lens"])
            s["cu"] = torch.tensor([sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32,
                                   device="cuda")
        if case["train"]:
            s["do"] = randn(B, T, Hv, Dv).to(BF16)
            s["dht"] = 0.3 * randn(n, Hv, Dk, Dv)
            for name in ("q", "k", "v", "g", "beta", "h0"):
                s[name].requires_grad_()
    elif case["op"] == "step":
        B, T, Hk, Hv, Dk, Dv = (case[x] for x in ("B", "T", "Hk", "Hv", "Dk", "Dv"))
        dt = TYPES[case["dtype"]]
        s["q"], s["k"] = unit(B, T, Hk, Dk).to(dt), unit(B, T, Hk, Dk).to(dt)
        s["v"] = randn(B, T, Hv, Dv).to(dt)
        s["g"], s["beta"] = _gates(gen, (B, T, Hv), F32)
        s["state"] = 0.3 * randn(case["slots"], Hv, Dk, Dv)
        idx = torch.randperm(case["slots"], generator=gen, device="cuda")[:B].to(torch.int32)
        if case["pad"]:
            idx[B - case["pad"]:] = -1   # rows behind the last sequence of a padded batch
        s["idx"] = idx
    elif case["op"] == "norm":
        s["x"] = (2.0 * randn(case["rows"], case["N"]) + 0.5).to(TYPES[case["dtype"]])
        s["w"] = s["b"] = None
        if case["wtype"] != "none":
            s["w"] = (1 + 0.2 * randn(case["N"])).to(TYPES[case["wtype"]])
            s["b"] = (0.2 * randn(case["N"])).to(TYPES[case["wtype"]])
        if case["train"]:
            s["dy"] = randn(case["rows"], case["N"]).to(TYPES[case["dtype"]])
            s["leaves"] = [t.requires_grad_() for t in (s["x"], s["w"], s["b"]) if t is not None]
    else:
        B, L, H, D = case["B"], case["L"], case["H"], case["D"]
        sections = _ints(case["sections"])
        # q of a fused q | k | v projection
        s["x"] = randn(B, L, 3, H, D).to(TYPES[case["dtype"]])[:, :, 0]
        s["sections"] = sections
        # a token's position on each axis; the first axis far along (a long video)
        pos = torch.randint(0, 64, (B, L, len(sections)), device="cuda", generator=gen)
        pos[..., 0] += 100_000
        s["pos"] = pos.to(torch.int32)
        R = sum(sections)
        s["freq"] = (10000.0 ** (-torch.arange(R, device="cuda", dtype=torch.float64) / R)).float()
        if case["train"]:
            s["x"].requires_grad_()
            s["dy"] = randn(B, L, H, D).to(TYPES[case["dtype"]])
    return s


# ------------------------------------------------------------- plain forms --
def _inverse(A):
    """(I + A)^-1 of strictly lower triangular [..., C, C], C a power of two:
    diagonal blocks of 1, then pairs of blocks joined."""
    C = A.shape[-1]
    T = torch.ones(A.shape[:-2] + (C, 1, 1), dtype=A.dtype, device=A.device)
    size = 1
    while size < C:
        n = C // (2 * size)
        D = A.reshape(A.shape[:-2] + (n, 2 * size, n, 2 * size))
        D = D.diagonal(dim1=-4, dim2=-2).movedim(-1, -3)      # diagonal blocks [.., n, 2s, 2s]
        A21 = D[..., size:, :size]
        T11, T22 = T[..., 0::2, :, :], T[..., 1::2, :, :]
        T21 = -(T22 @ (A21 @ T11))
        T = torch.cat([torch.cat([T11, torch.zeros_like(T11)], -1),
                       torch.cat([T21, T22], -1)], -2)
        size *= 2
    return T[..., 0, :, :]


def _delta_plain(q, k, v, g, beta, h0, scale):
    """Chunked form in fp32 of [N, H, L, .] with L a multiple of the chunk."""
    N, H, Lx, Dk = q.shape
    n = Lx // CHUNK
    cut = lambda x: x.reshape(N, H, n, CHUNK, *x.shape[3:])  # noqa: E731
    q, k, v, g, beta = cut(q), cut(k), cut(v), cut(g), cut(beta)[..., None]
    G = g.cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = (G[..., :, None] - G[..., None, :]).masked_fill(~lower, -math.inf).exp()
    kt = k.transpose(-1, -2)
    A = (beta * (k @ kt) * decay).masked_fill(~lower.tril(-1), 0.0)
    Ti = _inverse(A)
    P = scale * (q @ kt) * decay
    gam = G.exp()[..., None]
    U0, W = Ti @ (beta * v), Ti @ (beta * gam * k)
    last = G[..., -1:]
    kd = (k * (last - G).exp()[..., None]).transpose(-1, -2)
    qg, end = scale * gam * q, last.exp()[..., None]
    S, out = h0, []
    for c in range(n):
        U = U0[:, :, c] - W[:, :, c] @ S
        out.append(qg[:, :, c] @ S + P[:, :, c] @ U)
        S = end[:, :, c] * S + kd[:, :, c] @ U
    o = torch.stack(out, 2) if n else v
    return o.reshape(N, H, Lx, v.shape[-1]), S


def _rows_of(case, cu):
    """Packed rows -> (sequence, place): gather indices into a padded batch and back."""
    lens = _ints(case["lens"])
    T = sum(lens)
    pos = torch.arange(T, device="cuda")
    seq = torch.searchsorted(cu[1:].long(), pos, right=True)
    return seq, pos - cu.long()[seq], max(lens)


def _run_delta_plain(s):
    case = s["case"]
    Hk, Hv = case["Hk"], case["Hv"]
    x = [s[n].float() for n in ("q", "k", "v", "g", "beta")]
    x[0], x[1] = (t.repeat_interleave(Hv // Hk, 2) for t in x[:2])
    if case["B"]:
        Lx = _ints(case["lens"])[0]
        full = -(-Lx // CHUNK) * CHUNK
        x = [torch.nn.functional.pad(t.transpose(1, 2), (0, 0) * (t.dim() - 3) + (0, full - Lx))
             for t in x]
        o, S = _delta_plain(*x, s["h0"], case["Dk"] ** -0.5)
        o = o[:, :, :Lx].transpose(1, 2).to(BF16)
    else:
        seq, place, longest = _rows_of(case, s["cu"])
        n, full = s["cu"].numel() - 1, -(-longest // CHUNK) * CHUNK
        pad = [torch.zeros((n, full) + t.shape[2:], device="cuda").index_put((seq, place), t[0])
               for t in x]
        o, S = _delta_plain(*(t.transpose(1, 2) for t in pad), s["h0"], case["Dk"] ** -0.5)
        o = o.transpose(1, 2)[seq, place][None].to(BF16)
    if not case["train"]:
        return dict(o=o, state=S)
    names = ("q", "k", "v", "g", "beta", "h0")
    grads = torch.autograd.grad([o, S], [s[n] for n in names], [s["do"], s["dht"]])
    return dict(o=o.detach(), state=S.detach(), **{"d" + n: t for n, t in zip(names, grads)})


def _run_step_plain(s):
    case = s["case"]
    r = case["Hv"] // case["Hk"]
    q, k = (s[n].float().repeat_interleave(r, 2) for n in ("q", "k"))
    v, alpha, beta = s["v"].float(), s["g"].exp(), s["beta"]
    keep = s["idx"] >= 0
    rows = s["idx"][keep].long()
    S, out = s["state"][rows], []
    q, k, v, alpha, beta = (t[keep] for t in (q, k, v, alpha, beta))
    for t in range(case["T"]):
        S = S * alpha[:, t, :, None, None]
        u = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, :, None] * S).sum(-2))
        S = S + k[:, t, :, :, None] * u[:, :, None, :]
        out.append((q[:, t, :, :, None] * S).sum(-2) * case["Dk"] ** -0.5)
    s["state"][rows] = S
    o = torch.zeros(s["v"].shape, device="cuda")
    o[keep] = torch.stack(out, 1)
    return dict(o=o.to(s["v"].dtype), state=s["state"])


def _run_norm_plain(s):
    x = s["x"].detach().float()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    xh = c * rstd
    w = None if s["w"] is None else s["w"].detach().float()
    y = (xh if w is None else xh * w + s["b"].detach().float()).to(s["x"].dtype)
    if not s["case"]["train"]:
        return dict(y=y)
    dy = s["dy"].float()
    wdy = dy if w is None else dy * w
    dx = rstd * (wdy - wdy.mean(-1, keepdim=True) - xh * (wdy * xh).mean(-1, keepdim=True))
    out = dict(y=y, dx=dx.to(s["x"].dtype))
    if w is not None:
        out.update(dw=(dy * xh).sum(0).to(s["w"].dtype), db=dy.sum(0).to(s["b"].dtype))
    return out


def _rotate_plain(x, cos, sin, R, interleaved):
    x = x.float()
    a, b = (x[..., 0:2 * R:2], x[..., 1:2 * R:2]) if interleaved else (x[..., :R], x[..., R:2 * R])
    u, w = a * cos - b * sin, a * sin + b * cos
    rot = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([rot, x[..., 2 * R:]], -1)


def _run_rotary_plain(s):
    case = s["case"]
    R = sum(s["sections"])
    axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device="cuda"),
                                   torch.tensor(s["sections"], device="cuda"), output_size=R)
    angle = s["pos"][..., axis].double() * s["freq"].double()
    cos, sin = (f(angle).float()[:, :, None] for f in (torch.cos, torch.sin))
    dt = s["x"].dtype
    y = _rotate_plain(s["x"].detach(), cos, sin, R, case["interleaved"]).to(dt)
    if not case["train"]:
        return dict(y=y)
    return dict(y=y, dx=_rotate_plain(s["dy"], cos, -sin, R, case["interleaved"]).to(dt))


# ----------------------------------------------------- the framework's calls --
def _run_own(s):
    case = s["case"]
    if case["op"] == "delta":
        from uttt_amd.delta import gated_delta_rule
        o, S = gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_state=s["h0"],
                                output_final_state=True, cu_seqlens=s["cu"])
        if not case["train"]:
            return dict(o=o, state=S)
        names = ("q", "k", "v", "g", "beta", "h0")
        grads = torch.autograd.grad([o, S], [s[n] for n in names], [s["do"], s["dht"]])
        return dict(o=o.detach(), state=S.detach(), **{"d" + n: t for n, t in zip(names, grads)})
    if case["op"] == "step":
        from uttt_amd.delta import gated_delta_step
        o = gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"],
                             state_indices=s["idx"])
        return dict(o=o, state=s["state"])
    if case["op"] == "norm":
        from uttt_amd.norm import layer_norm
        y = layer_norm(s["x"], s["w"], s["b"])
        if not case["train"]:
            return dict(y=y)
        grads = torch.autograd.grad(y, s["leaves"], s["dy"])
        return dict(y=y.detach(), **dict(zip(("dx", "dw", "db"), grads)))
    from uttt_amd.positions import rotary_axes
    y = rotary_axes(s["x"], s["pos"], s["freq"], s["sections"], interleaved=case["interleaved"])
    if not case["train"]:
        return dict(y=y)
    return dict(y=y.detach(), dx=torch.autograd.grad(y, s["x"], s["dy"])[0])


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "delta":
        return _run_delta_plain(state)
    if op == "step":
        return _run_step_plain(state)
    return _run_norm_plain(state) if op == "norm" else _run_rotary_plain(state)


def work(case):
    """Every input read once, every output written once; the flops of the
    recurrence (read, correct, write: 6 Dk Dv per token and head; its adjoint
    twice that)."""
    op = case["op"]
    if op == "delta":
        B, T, n = _delta_shape(case)
        Hk, Hv, Dk, Dv = case["Hk"], case["Hv"], case["Dk"], case["Dv"]
        gate = 4 if case["gates"] == "fp32" else 2
        rows = B * T * (2 * (2 * Hk * Dk + Hv * Dv) + 2 * gate * Hv)   # q, k, v, g, beta
        state = n * Hv * Dk * Dv * 4
        by, fl = rows + B * T * Hv * Dv * 2 + 2 * state, 6 * B * T * Hv * Dk * Dv
        if case["train"]:   # do and the inputs again, every gradient
            by += 2 * rows + B * T * Hv * Dv * 2 + 2 * state
            fl *= 3
        return dict(bytes=by, flops=fl)
    if op == "step":
        rows = case["B"] - case["pad"]
        tok = rows * case["T"]
        size = TYPES[case["dtype"]].itemsize
        hv = case["Hv"] * case["Dv"]
        by = rows * hv * case["Dk"] * 8 + tok * (2 * case["Hk"] * case["Dk"] + 2 * hv) * size
        return dict(bytes=by + tok * case["Hv"] * 8, flops=6 * tok * hv * case["Dk"])
    size = TYPES[case["dtype"]].itemsize
    if op == "norm":
        n = case["rows"] * case["N"]
        w = 0 if case["wtype"] == "none" else case["N"] * TYPES[case["wtype"]].itemsize
        if case["train"]:
            return dict(bytes=5 * n * size + 5 * w, flops=20 * n)
        return dict(bytes=2 * n * size + 2 * w, flops=8 * n)
    n = case["B"] * case["L"] * case["H"] * case["D"]
    passes = 2 if case["train"] else 1
    by = 2 * n * size + case["B"] * case["L"] * len(_ints(case["sections"])) * 4
    return dict(bytes=passes * by, flops=passes * 3 * n)


# -------------------------------------------------- the definition, 64 bits --
def _delta_exact(case, s):
    """Token by token: S = exp(g) S; S += k (beta (v - S^T k))^T; o = S^T q.
    Key heads are independent: as many at a time as their states fit in."""
    B, T, n = _delta_shape(case)
    lens = [T] * n if case["B"] else _ints(case["lens"])
    longest, r = max(lens), case["Hv"] // case["Hk"]
    kept = n * r * case["Dk"] * case["Dv"] * 8 * (3 * longest if case["train"] else 3)
    at_once = max(1, int(60e9 // kept))
    parts = -(-case["Hk"] // at_once)
    if longest * (4 if case["train"] else 1) * parts > 60000 or kept > 120e9:
        return None
    got = [_delta_exact_heads(case, s, lens, slice(h, h + at_once), slice(h * r, (h + at_once) * r))
           for h in range(0, case["Hk"], at_once)]
    axis = {"state": 1, "dh0": 1}
    return {m: torch.cat([p[m] for p in got], axis.get(m, 2)) for m in got[0]}


def _delta_exact_heads(case, s, lens, kheads, vheads):
    names = ("q", "k", "v", "g", "beta")
    leaf = {m: s[m].detach()[:, :, kheads if m in "qk" else vheads].double() for m in names}
    leaf["h0"] = s["h0"].detach()[:, vheads].double()
    if case["train"]:
        for t in leaf.values():
            t.requires_grad_()
    # one row per sequence, behind its end tokens that change nothing
    rows = {m: (list(leaf[m]) if case["B"] else list(torch.split(leaf[m][0], lens))) for m in names}
    rows = {m: torch.nn.utils.rnn.pad_sequence(x, batch_first=True) for m, x in rows.items()}
    v, g, beta = rows["v"], rows["g"], rows["beta"]
    r = case["Hv"] // case["Hk"]
    group = torch.arange(v.shape[2], device="cuda") // r
    q, k = rows["q"][:, :, group], rows["k"][:, :, group]
    S, out = leaf["h0"], []
    for t in range(max(lens)):
        S = torch.exp(g[:, t])[..., None, None] * S
        err = v[:, t] - torch.matmul(k[:, t][..., None, :], S)[..., 0, :]
        S = S + k[:, t][..., None] * (beta[:, t][..., None] * err)[..., None, :]
        out.append(torch.matmul(q[:, t][..., None, :], S)[..., 0, :])
    o = torch.stack(out, 1) / math.sqrt(case["Dk"])
    o = o if case["B"] else torch.cat([o[i, :m] for i, m in enumerate(lens)])[None]
    if not case["train"]:
        return dict(o=o, state=S)
    keys = names + ("h0",)
    do, dht = s["do"][:, :, vheads].double(), s["dht"][:, vheads].double()
    grads = torch.autograd.grad([o, S], [leaf[m] for m in keys], [do, dht])
    return dict(o=o.detach(), state=S.detach(), **{"d" + m: t for m, t in zip(keys, grads)})


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "delta":
        return _delta_exact(case, s)
    if op == "step":
        S, o = s["state"].double(), torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda")
        head = torch.arange(case["Hv"], device="cuda") // (case["Hv"] // case["Hk"])
        used = [(b, i) for b, i in enumerate(s["idx"].tolist()) if i >= 0]
        if used:
            b, i = (torch.tensor(x, device="cuda") for x in zip(*used))
            M = S[i]
            for t in range(case["T"]):
                q, k, v = (s[m][b, t].double() for m in ("q", "k", "v"))
                M = torch.exp(s["g"][b, t].double())[..., None, None] * M
                err = v - torch.matmul(k[:, head][..., None, :], M)[..., 0, :]
                M = M + k[:, head][..., None] * (s["beta"][b, t].double()[..., None] * err)[..., None, :]
                o[b, t] = torch.matmul(q[:, head][..., None, :], M)[..., 0, :] / math.sqrt(case["Dk"])
            S[i] = M
        return dict(o=o, state=S)
    if op == "norm":
        x = s["x"].detach().double().requires_grad_()
        w, b = (None if t is None else t.detach().double().requires_grad_() for t in (s["w"], s["b"]))
        y = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + 1e-5)
        y = y if w is None else y * w + b
        if not case["train"]:
            return dict(y=y)
        grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], s["dy"].double())
        return dict(y=y, **dict(zip(("dx", "dw", "db"), grads)))
    # the rotation as a product of complex numbers
    R, start, turns = sum(s["sections"]), 0, []
    for a, m in enumerate(s["sections"]):
        turns.append(s["pos"][..., a:a + 1].double() * s["freq"][start:start + m].double())
        start += m
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.cat(turns, -1))[:, :, None]

    def turned(x, z):
        x = x.detach().double()
        y = x.clone()
        if case["interleaved"]:
            w = torch.view_as_complex(x[..., :2 * R].unflatten(-1, (R, 2)).contiguous()) * z
            y[..., 0:2 * R:2], y[..., 1:2 * R:2] = w.real, w.imag
        else:
            w = torch.complex(x[..., :R].contiguous(), x[..., R:2 * R].contiguous()) * z
            y[..., :R], y[..., R:2 * R] = w.real, w.imag
        return y

    y = turned(s["x"], z)
    return dict(y=y, dx=turned(s["dy"], z.conj())) if case["train"] else dict(y=y)
