"""The norms before and after a block on the GPU against 64 bits.

Bounds, to the first order, with U = 2^-24 (1.5 times of them are allowed,
and half a step of the result's type).  A row's sum of N squares is off by (N / 4
+ 16) U of itself at most (a lane adds its elements in a row: never more than a
quarter of N where a row has lanes of its own, and trees above), so 1 / rms by
half of that and 4 U, called r.  n = v / rms is then off by r + 2 U of itself (v by
2 U of its terms' sizes where it is a sum), a gate's silu and slope as in the
convolution's bounds, each product by U.  The backward's sum over m n is off by
(N / 4 + 16) U of its terms' sizes and what its factors are off by; sums over
rows by (rows + 16) U of their terms' sizes and their terms' errors."""
import pytest
import torch

from oracle import state_space as O
from state_space_cases import BF16, F16, F32, check, up

pytestmark = pytest.mark.gpu
U = O.U


def make(shape, dtype=BF16, rtype=F32, weight=F32, scale=F32, gate=True, residual=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    N = shape[-1]
    a = dict(x=(2 * r(*shape) + 0.3).to(dtype).cuda())
    a["weight"] = None if weight is None else (1 + 0.2 * r(N)).to(weight).cuda()
    a["scale"] = None if scale is None else scale if isinstance(scale, float) else (0.5 * r(N)).to(scale).cuda()
    a["gate"] = r(*shape).to(dtype).cuda() if gate else None
    a["residual"] = r(*shape).to(rtype).cuda() if residual else None
    return a, r(*shape), r(*shape)


def off_rstd(v, e_v, eps):
    """1 / rms and its error, absolute."""
    N = v.shape[-1]
    rstd = 1 / O.rms(v, eps)
    sq = v.square().sum(-1, keepdim=True)
    rel = (N / 4 + 16) * U / 2 + (v.abs() * e_v).sum(-1, keepdim=True) / (sq + N * eps) + 4 * U
    return rstd, rstd * rel


def after_bounds(a, dy, eps):
    x, w, s, z, r = (up(a[n]) if isinstance(a[n], torch.Tensor) else a[n] for n in ("x", "weight", "scale", "gate", "residual"))
    N = x.shape[-1]
    one = torch.ones(N, dtype=x.dtype)
    w, sc = one if w is None else w, one if s is None else s * one
    rstd, e_r = off_rstd(x, torch.zeros_like(x), eps)
    n, e_n = x * rstd, x.abs() * e_r + U * (x * rstd).abs()
    if z is None:
        f, e_f, df, e_df = torch.ones_like(x), torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    else:
        q = torch.sigmoid(z)
        f, df = z * q, q * (1 + z * (1 - q))
        e_f, e_df = (26 + z.abs()) * U * f.abs(), (30 + 2 * z.abs()) * U * (1 + z.abs()) * q
    y = n * w * f * sc
    e_y = (e_n * (w * f * sc).abs() + e_f * (n * w * sc).abs() + 4 * U * y.abs())
    if r is not None:
        y, e_y = y + r, e_y + U * (y.abs() + r.abs())
    val, err = dict(y=y), dict(y=e_y)
    o, m = dy * sc, dy * sc * w * f
    e_m = e_f * (o * w).abs() + 3 * U * m.abs()
    c = (m * n).mean(-1, keepdim=True)
    e_c = ((N / 4 + 16) * U * (m * n).abs() + e_m * n.abs() + e_n * m.abs()).mean(-1, keepdim=True) + U * c.abs()
    val["x"] = rstd * (m - n * c)
    err["x"] = e_r * (m - n * c).abs() + rstd * (e_m + e_n * c.abs() + n.abs() * e_c + 3 * U * (m.abs() + (n * c).abs()))
    rows = x.numel() // N
    flat = lambda t: t.reshape(-1, N)  # noqa: E731
    total = lambda t, e: (flat(t).sum(0), flat(e).sum(0) + (rows + 16) * U * flat(t).abs().sum(0))  # noqa: E731
    e_nf = e_n * f.abs() + e_f * n.abs() + 3 * U * (n * f).abs()
    val["weight"], err["weight"] = total(o * n * f, o.abs() * e_nf)
    val["scale"], err["scale"] = total(dy * n * f * w, (dy * w).abs() * e_nf)
    val["gate"], err["gate"] = o * n * w * df, (o * w).abs() * (e_n * df.abs() + n.abs() * e_df) + 4 * U * (o * n * w * df).abs()
    val["residual"], err["residual"] = dy, torch.zeros_like(dy)
    return val, err


def before_bounds(a, dy, dt, eps):
    x, w, s, r = (up(a[n]) if isinstance(a[n], torch.Tensor) else a[n] for n in ("x", "weight", "scale", "residual"))
    N = x.shape[-1]
    one = torch.ones(N, dtype=x.dtype)
    w, sc = one if w is None else w, one if s is None else s * one
    t = r + x * sc
    e_t = 2 * U * (r.abs() + (x * sc).abs())
    rstd, e_r = off_rstd(t, e_t, eps)
    n = t * rstd
    e_n = t.abs() * e_r + e_t * rstd + U * n.abs()
    val, err = dict(y=n * w, total=t), dict(y=e_n * w.abs() + 2 * U * (n * w).abs(), total=e_t)
    m = dy * w
    c = (m * n).mean(-1, keepdim=True)
    e_c = ((N / 4 + 16) * U * (m * n).abs() + U * (m * n).abs() + e_n * m.abs()).mean(-1, keepdim=True) + U * c.abs()
    g = rstd * (m - n * c)
    e_g = e_r * (m - n * c).abs() + rstd * (U * m.abs() + e_n * c.abs() + n.abs() * e_c + 3 * U * (m.abs() + (n * c).abs()))
    d, e_d = dt + g, e_g + U * (dt.abs() + g.abs())
    rows = x.numel() // N
    flat = lambda v: v.reshape(-1, N)  # noqa: E731
    total = lambda v, e: (flat(v).sum(0), flat(e).sum(0) + (rows + 16) * U * flat(v).abs().sum(0))  # noqa: E731
    val["residual"], err["residual"] = d, e_d
    val["x"], err["x"] = sc * d, sc.abs() * e_d + U * (sc * d).abs()
    val["weight"], err["weight"] = total(dy * n, dy.abs() * e_n)
    val["scale"], err["scale"] = total(x * d, x.abs() * e_d)
    return val, err


def run_after(a, eps=1e-5):
    from uttt_amd.norm import norm_after_block
    return norm_after_block(a["x"], a["weight"], gate=a["gate"], residual=a["residual"], scale=a["scale"], eps=eps)


def run_before(a, eps=1e-5):
    from uttt_amd.norm import norm_before_block
    return norm_before_block(a["x"], a["residual"], a["weight"], scale=a["scale"], eps=eps)


def leaves(a):
    return {n: t.detach().requires_grad_() if isinstance(t, torch.Tensor) else t for n, t in a.items()}


def check_after(a, dy, eps=1e-5):
    with torch.no_grad():
        y0 = run_after(a, eps)
    dy = dy.to(y0.dtype)
    val, err = after_bounds(a, dy.double(), eps)
    check(y0, val["y"], err["y"], "y")
    leaf = leaves(a)
    y = run_after(leaf, eps)
    assert torch.equal(y, y0) and y.dtype == (a["x"] if a["residual"] is None else a["residual"]).dtype
    names = [n for n in leaf if isinstance(leaf[n], torch.Tensor)]
    got = torch.autograd.grad(y, [leaf[n] for n in names], dy.cuda())
    for n, g in zip(names, got):
        assert g.dtype == leaf[n].dtype
        check(g, val[n], err[n], n)
    return [y0, *got]


def check_before(a, dy, dt, eps=1e-5):
    a = {n: t for n, t in a.items() if n != "gate"}
    with torch.no_grad():
        y0, t0 = run_before(a, eps)
    dy, dt = dy.to(y0.dtype), dt.to(t0.dtype)
    val, err = before_bounds(a, dy.double(), dt.double(), eps)
    check(y0, val["y"], err["y"], "y")
    check(t0, val["total"], err["total"], "total")
    leaf = leaves(a)
    y, t = run_before(leaf, eps)
    assert torch.equal(y, y0) and torch.equal(t, t0) and t.dtype == a["residual"].dtype and y.dtype == a["x"].dtype
    names = [n for n in leaf if isinstance(leaf[n], torch.Tensor)]
    got = torch.autograd.grad([y, t], [leaf[n] for n in names], [dy.cuda(), dt.cuda()])
    for n, g in zip(names, got):
        assert g.dtype == leaf[n].dtype
        check(g, val[n], err[n], n)
    return [y0, t0, *got]


WIDTHS = [1, 2, 7, 8, 16, 24, 63, 64, 65, 96, 128, 129, 192, 200, 256, 264, 300, 512, 513, 768, 1000, 1024, 1032, 1537, 2048,
          2056, 2049, 4096, 4104, 6000, 8191, 8192]


@pytest.mark.parametrize("N", WIDTHS)
@pytest.mark.parametrize("dtype,rtype", [(BF16, F32), (F32, F32), (BF16, BF16), (F32, BF16), (F16, F32)])
def test_widths(N, dtype, rtype):
    rows = 5 if N > 300 else 37
    a, dy, dt = make((rows, N), dtype, rtype, seed=N)
    check_after(a, dy)
    check_before(a, dy, dt)


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("scale", [None, 0.7, F32, BF16])
@pytest.mark.parametrize("weight", [None, F32, F16])
def test_options(gate, residual, scale, weight):
    a, dy, dt = make((3, 11, 40), BF16, F32, weight, scale, gate, residual)
    check_after(a, dy, eps=1e-3)
    if residual:
        check_before(a, dy, dt, eps=1e-3)


@pytest.mark.parametrize("rows", [1, 2, 31, 33, 100, 6143, 6145, 20000])
def test_rows(rows):
    a, dy, dt = make((rows, 24), BF16, F32, seed=rows)
    check_after(a, dy)
    check_before(a, dy, dt)


@pytest.mark.parametrize("shape", [(7,), (1, 7), (4, 3, 2, 16), (2, 1, 5, 96), (0, 8), (3, 0, 8)])
def test_shapes(shape):
    a, dy, dt = make(shape, F32, F32)
    check_after(a, dy)
    check_before(a, dy, dt)


def test_rows_of_zeros_and_of_nothing_finite():
    """A row of zeros is normed by eps alone; a row that is not finite stays so alone."""
    a, dy, dt = make((6, 96), BF16, F32)
    a["x"][2] = 0
    check_after(a, dy)
    y = run_after(a)
    bad = a["x"].clone()
    bad[4, 5] = float("nan")
    got = run_after(dict(a, x=bad))
    assert torch.equal(got[[0, 1, 2, 3, 5]], y[[0, 1, 2, 3, 5]]) and got[4].isnan().all()


def test_views():
    """Heads of a fused projection, other strides and addresses: the bits of copies."""
    gen = torch.Generator().manual_seed(0)
    proj = torch.randn(4, 9, 3, 5, 64, generator=gen).to(BF16).cuda()
    a, dy, dt = make((4, 9, 5, 64), BF16, BF16)
    a.update(x=proj[:, :, 0], gate=proj[:, :, 2], residual=proj[:, :, 1])
    copied = {n: t.contiguous() if isinstance(t, torch.Tensor) else t for n, t in a.items()}
    for s, t in zip(check_after(a, dy), check_after(copied, dy)):
        assert torch.equal(s, t)
    for s, t in zip(check_before(a, dy, dt), check_before(copied, dy, dt)):
        assert torch.equal(s, t)
    for change in (lambda t: torch.nn.functional.pad(t, (3, 2))[..., 3:-2], lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                   lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)):
        moved = {n: change(t) if isinstance(t, torch.Tensor) and t.dim() > 1 else t for n, t in a.items()}
        check_after(moved, change(dy))
        check_before(moved, change(dy), change(dt))
    e = dict(a, residual=proj[:1, :1, 1].expand(4, 9, 5, 64))
    assert torch.equal(run_before(e)[1], run_before(dict(a, residual=e["residual"].contiguous()))[1])


def test_the_same_bits_twice_and_one_gradient_alone():
    a, dy, dt = make((3000, 192), BF16, F32)
    for s, t in zip(check_after(a, dy), check_after(a, dy)):
        assert torch.equal(s, t)
    b = {n: t for n, t in a.items() if n != "gate"}
    leaf = leaves(b)
    wanted = list(leaf.values())
    y, t = run_before(leaf)
    zero = torch.zeros_like
    dy, dt = dy.to(y.dtype).cuda(), dt.to(t.dtype).cuda()
    for i, (gy, gt) in enumerate(((dy, zero(dt)), (zero(dy), dt))):
        y, t = run_before(leaf)
        full = torch.autograd.grad([y, t], wanted, [gy, gt])
        out = run_before(leaf)
        alone = torch.autograd.grad(out[i], wanted, (gy, gt)[i], allow_unused=True)
        for p, q in zip(full, alone):
            assert torch.equal(p, zero(p) if q is None else q)


def test_in_a_graph_and_on_another_stream():
    a, dy, dt = make((200, 96), BF16, F32)
    leaf = leaves(a)
    wanted = list(leaf.values())
    gy, gt = dy.cuda(), dt.cuda()

    def run():
        y = run_after(leaf)
        z, t = run_before(leaf)
        return [y.detach(), z.detach(), t.detach(), *torch.autograd.grad([y, z, t], wanted, [gy, gy.to(z.dtype), gt])]

    want = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    del got, want
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(3):
        with torch.no_grad():
            leaf["x"].copy_(torch.randn(200, 96, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, run()):
            assert torch.equal(p, q), i
        torch.cuda.synchronize()
