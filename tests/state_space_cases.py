"""Inputs of the state space layer's tests, and how near their results have to be.

A result may be off by what fp32 arithmetic leaves of it (bounds next to the
64-bit formulas: oracle/state_space.py; to the first order, of which 1.5 times
are allowed for the higher ones) and by one rounding to its type, half a step."""
import torch

from oracle import state_space as O

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TINY = {BF16: 2.0 ** -133, F16: 2.0 ** -24, F32: 2.0 ** -126}   # a denormal may be flushed or rounded


def check(got, want, bound, name=""):
    """Elementwise, with both on the CPU."""
    got, t = got.detach().cpu(), got.dtype
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    off = (got.double() - want).abs()
    most = 1.5 * bound + torch.finfo(t).eps / 2 * (want.abs() + 1.5 * bound) + TINY[t]
    worst = (off / most).max().item() if off.numel() else 0.0
    assert worst <= 1, f"{name}: {worst:.3g} times the tolerance"


def scan_inputs(B=1, T=1, D=1, N=1, G=1, dtype=F32, dt_dtype=None, gate=True, skip=True, bias=True, soft=True, state=True,
                seqs=None, seed=0):
    """Tensors on the GPU as a layer makes them: x and the gate halves of one
    projection, B and C slices of another; rates from slow to fast."""
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    n = B if seqs is None else seqs
    step = torch.exp(-6 + 4 * torch.rand(D, generator=gen))
    raw = 0.5 * r(B, T, D)
    xz, bc = r(B, T, 2, D).to(dtype).cuda(), r(B, T, 2, G, N).to(dtype).cuda()
    if not soft:
        raw = step * torch.exp(raw)
    elif not bias:
        raw = raw + torch.log(torch.expm1(step))
    a = dict(x=xz[:, :, 0], dt=raw.to(dt_dtype or dtype).cuda(),
             A=(-torch.arange(1.0, N + 1) * torch.exp(0.3 * r(D, N))).cuda(), B=bc[:, :, 0], C=bc[:, :, 1])
    a["D"] = (1 + 0.2 * r(D)).cuda() if skip else None
    a["gate"] = xz[:, :, 1] if gate else None
    a["dt_bias"] = None if not bias else (torch.log(torch.expm1(step)) if soft else 0.1 * step).cuda()
    a["initial_state"] = 0.3 * r(n, D, N).cuda() if state else None
    grads = r(B, T, D).to(dtype).cuda(), 0.3 * r(n, D, N).cuda()
    return a, soft, grads


def up(t):
    return None if t is None else t.detach().double().cpu()


def scan_exact(a, soft, grads=None, cu=None):
    dy, dhT = (None, None) if grads is None else map(up, grads)
    return O.selective_scan(up(a["x"]), up(a["dt"]), up(a["A"]), up(a["B"]), up(a["C"]), up(a["D"]), up(a["gate"]),
                            up(a["dt_bias"]), soft, up(a["initial_state"]), dy, dhT, cu)


def call(a, soft, cu=None, **kw):
    from uttt_amd.state_space import selective_scan
    a = dict(a, **kw)
    return selective_scan(*(a[n] for n in ("x", "dt", "A", "B", "C")), D=a["D"], gate=a["gate"], dt_bias=a["dt_bias"],
                          dt_softplus=soft, initial_state=a["initial_state"], output_final_state=True,
                          cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda"))


NAMES = dict(x="d_x", dt="d_dt", A="d_A", B="d_B", C="d_C", D="d_D", gate="d_z", dt_bias="d_bias", initial_state="d_h0")


def check_scan(a, soft, grads, cu=None, backward=True):
    """Outputs, states and gradients against the formulas; outputs without
    gradients have to be the same bits."""
    with torch.no_grad():
        y0, h0 = call(a, soft, cu)
    val, err = scan_exact(a, soft, grads if backward else None, cu)
    check(y0, val["y"], err["y"], "y")
    check(h0, val["state"], err["state"], "state")
    if not backward:
        return
    a = {n: None if t is None else t.detach().requires_grad_() for n, t in a.items()}
    y, h = call(a, soft, cu)
    assert torch.equal(y, y0) and torch.equal(h, h0)
    names = [n for n in NAMES if a[n] is not None]
    got = torch.autograd.grad([y, h], [a[n] for n in names], list(grads))
    for n, g in zip(names, got):
        assert g.dtype == a[n].dtype, n
        check(g, val[NAMES[n]], err[NAMES[n]], NAMES[n])
    return dict(zip(names, got))


# ------------------------------------------------------------- convolution --
def conv_bounds(x, w, b, h0, silu, dy, dstate, cu):
    """Values and bounds of the convolution and its gradients.  With U half an ulp,
    a sum of n products is off by (n + 1) U of their sizes, a sigmoid by 24 U and
    by U of its argument (which holds for both of the kernels' forms), a product of
    silu's slope, whose own slope is at most 1/2, accordingly."""
    leaf = [t if t is None else t.clone().requires_grad_() for t in (x, w, b, h0)]
    y, state = O.causal_conv(leaf[0], leaf[1], leaf[2], silu, leaf[3], cu)
    names = [n for n, t in zip(("x", "w", "b", "h0"), leaf) if t is not None]
    got = torch.autograd.grad([y, state], [t for t in leaf if t is not None], [dy, dstate])
    val = dict(zip(names, got), y=y.detach(), state=state.detach())
    # p, its slope and their errors per token
    p, _ = O.causal_conv(x, w, b, False, h0, cu)
    ab = lambda t: None if t is None else t.abs()  # noqa: E731
    size, _ = O.causal_conv(x.abs(), w.abs(), ab(b), False, ab(h0), cu)
    W, U = w.shape[1], O.U
    e_p = (W + 1) * U * size
    sig = torch.sigmoid(p)
    e_y = 1.1 * e_p + (26 + p.abs()) * U * (p * sig).abs() if silu else e_p
    slope = (sig * (1 + p * (1 - sig))).abs() if silu else torch.ones_like(p)
    dp = dy.abs() * slope
    e_dp = dy.abs() * (0.5 * e_p + (30 + 2 * p.abs()) * U) if silu else torch.zeros_like(p)
    # the majorants go the way of the gradients: through a convolution with |w|
    lx, lw, lh = x.abs().requires_grad_(), w.abs().requires_grad_(), None if h0 is None else h0.abs().requires_grad_()
    lb = None if b is None else torch.zeros_like(b).requires_grad_()
    q, st = O.causal_conv(lx, lw, lb, False, lh, cu)
    through = [t for t in (lx, lw, lb, lh) if t is not None]
    mag = dict(zip(names, torch.autograd.grad([q, st], through, [dp, dstate.abs()], retain_graph=True)))
    off = dict(zip(names, torch.autograd.grad(q, through, e_dp, allow_unused=True)))
    tokens = x.shape[0] * x.shape[1]
    err = dict(y=e_y, state=torch.zeros_like(state))
    for n in names:
        terms = W + 2 if n in ("x", "h0") else min(tokens, 32) + 10
        err[n] = (0 if off[n] is None else off[n]) + terms * U * mag[n]
    return val, {n: t.detach() for n, t in err.items()}
