"""Layer norm on the GPU against 64 bits.

Tolerances per element.  A result is rounded once, to half a step of its type
(h = eps / 2).  In fp32 a normalised value (x - mean) rstd carries a few
roundings of its own size and the rounding of the mean, 2^-24 of |mean|, which
the subtraction keeps: 16 * 2^-24 (|value| + rstd |mean|) and the same of the
products' sizes.  Sums over R rows in fp32 are off by 2^-24 of the sum of their
terms' sizes for each of the log2(R) + R / 4096 additions in a row, 64 allowed."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def reference(x, w, b, eps, dy):
    x, dy = x.double(), dy.double()
    w = None if w is None else w.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    h = (x - mean) * rstd
    y = h if w is None else h * w
    y = y if b is None else y + b.double()
    d = dy if w is None else dy * w
    m0, m1 = d.mean(-1, keepdim=True), (d * h).mean(-1, keepdim=True)
    dx = rstd * (d - m0 - h * m1)
    err_h = 16 * U * (h.abs() + rstd * mean.abs() + 1)
    ww = 1.0 if w is None else w.abs()
    err = dict(y=err_h * ww + (0 if b is None else 4 * U * b.double().abs()),
               dx=rstd * (16 * U * (d.abs() + d.abs().mean(-1, keepdim=True)) +
                          2 * err_h * (d * h).abs().mean(-1, keepdim=True) +
                          (h.abs() + 1) * (err_h * d.abs()).mean(-1, keepdim=True)) + 16 * U * dx.abs(),
               dw=(64 * U * (dy * h).abs() + err_h * dy.abs()).sum(0), db=64 * U * dy.abs().sum(0))
    return dict(y=y, dx=dx, dw=(dy * h).sum(0), db=dy.sum(0)), err


def check(x, w, b, dy, eps=1e-5, move=lambda t: t.cuda(), flat=True):
    from uttt_amd.norm import layer_norm
    N = x.shape[-1]
    ref, err = reference(x.reshape(-1, N), w, b, eps, dy.reshape(-1, N))
    xs = move(x).requires_grad_()
    ws, bs = (None if t is None else t.cuda().requires_grad_() for t in (w, b))
    y = layer_norm(xs, ws, bs, eps)
    assert y.shape == x.shape and y.dtype == x.dtype
    leaves = dict(dx=xs, dw=ws, db=bs)
    leaves = {n: t for n, t in leaves.items() if t is not None}
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), move(dy))), y=y.detach())
    with torch.no_grad():
        assert torch.equal(layer_norm(xs, ws, bs, eps), got["y"])
    for n, t in got.items():
        assert t.dtype == (x.dtype if n in ("y", "dx") else leaves[n].dtype)
        r = ref[n].reshape(t.shape)
        allowed = torch.finfo(t.dtype).eps / 2 * (r.abs() + err[n].reshape(t.shape)) + err[n].reshape(t.shape)
        tiny = torch.finfo(t.dtype).smallest_normal * torch.finfo(t.dtype).eps
        off = (t.double().cpu() - r).abs()
        assert (off <= allowed + tiny).all(), (n, (off - allowed).max().item(), N)
    return got


def make(rows, N, dtype, wtype, seed=0, mean=0.5):
    gen = torch.Generator().manual_seed(seed)
    x = (2 * torch.randn(rows, N, generator=gen) + mean).to(dtype)
    w, b = (None, None) if wtype is None else (
        (1 + 0.3 * torch.randn(N, generator=gen)).to(wtype), (0.3 * torch.randn(N, generator=gen)).to(wtype))
    return x, w, b, torch.randn(rows, N, generator=gen).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N", [1, 2, 7, 8, 63, 64, 65, 128, 136, 200, 257, 512, 513, 768, 1000, 1024, 1537, 2048,
                               2056, 4096, 5000, 6001, 8192, 8193, 16384, 16392, 20001])
def test_widths(dtype, N):
    check(*make(9, N, dtype, F32 if N % 2 else dtype, seed=N))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 15, 16, 17, 255, 1023, 4099, 20000])
@pytest.mark.parametrize("N", [24, 96, 200, 136 * 8])
def test_rows(rows, N):
    if rows * N > 5_000_000:
        rows = 5_000_000 // N
    check(*make(rows, N, BF16, F32, seed=rows))


@pytest.mark.parametrize("wtype", [None, BF16, F16, F32])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_types(dtype, wtype):
    check(*make(33, 384, dtype, wtype))
    check(*make(33, 385, dtype, wtype))


def test_weight_or_bias_alone():
    x, w, b, dy = make(20, 96, BF16, F32)
    check(x, w, None, dy)
    check(x, None, b, dy)


def test_a_large_mean_and_constant_rows():
    """The variance is taken about the mean, and of a constant row is 0."""
    check(*make(40, 768, F32, F32, mean=1e4))
    x, w, b, dy = make(4, 512, F32, F32)
    x[1] = 3.0
    x[2] = 0.0
    check(x, w, b, dy)


def test_non_finite_rows_stay_by_themselves():
    from uttt_amd.norm import layer_norm
    x, w, b, _ = make(6, 100, F32, F32)
    clean = layer_norm(x.cuda(), w.cuda(), b.cuda())
    x[1, 3], x[4, 0] = math.nan, math.inf
    y = layer_norm(x.cuda(), w.cuda(), b.cuda())
    for i in range(6):
        assert torch.isnan(y[i]).all() if i in (1, 4) else torch.equal(y[i], clean[i])


def test_views():
    """Evenly spaced rows in place, others through a copy; the gradient's rows too."""
    x, w, b, dy = make(30, 256, BF16, BF16)

    def part(t):
        big = torch.full((t.shape[0], 3, 256), math.nan, dtype=t.dtype, device="cuda")
        big[:, 1] = t.cuda()
        return big[:, 1]

    def unaligned(t):
        big = torch.zeros(t.shape[0], 261, dtype=t.dtype, device="cuda")
        big[:, 3:259] = t.cuda()
        return big[:, 3:259]

    want = check(x, w, b, dy)
    for move in (part, unaligned, lambda t: t.cuda().t().contiguous().t()):
        got = check(x, w, b, dy, move=move)
        assert torch.equal(got["y"], want["y"]) or move is unaligned
    x3, dy3 = x.view(5, 6, 256), dy.view(5, 6, 256)
    check(x3, w, b, dy3)
    check(x3, w, b, dy3, move=lambda t: t.cuda().transpose(0, 1).contiguous().transpose(0, 1))


def test_broadcast_gradient_and_input():
    from uttt_amd.norm import layer_norm
    x, w, b, _ = make(30, 64, F32, F32)
    leaf = [t.cuda().requires_grad_() for t in (x, w, b)]
    ones = torch.autograd.grad(layer_norm(*leaf), leaf, torch.ones(30, 64, device="cuda"))
    summed = torch.autograd.grad(layer_norm(*leaf).sum(), leaf)   # an expanded scalar
    row = torch.autograd.grad(layer_norm(*leaf), leaf, torch.ones(64, device="cuda").expand(30, 64))
    for s, t, u in zip(ones, summed, row):
        assert torch.equal(s, t) and torch.equal(s, u)
    one = x[:1].cuda().requires_grad_()
    (g,) = torch.autograd.grad(layer_norm(one.expand(5, 64)).square().sum(), one)
    many = x[:1].cuda().expand(5, 64).contiguous().requires_grad_()
    (g2,) = torch.autograd.grad(layer_norm(many).square().sum(), many)
    assert torch.equal(g, g2.sum(0, keepdim=True))


def test_no_rows_and_one_leaf():
    from uttt_amd.norm import layer_norm
    w, b = (torch.ones(16, device="cuda", requires_grad=True) for _ in range(2))
    x = torch.zeros(0, 3, 16, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert y.shape == x.shape and dx.shape == x.shape and (dw == 0).all() and (db == 0).all()
    x = torch.randn(7, 16, device="cuda")
    full = [t.clone().requires_grad_() for t in (x, w.detach(), b.detach())]
    want = torch.autograd.grad(layer_norm(*full), full, torch.ones_like(x))
    for i in range(3):
        args = [t.detach().clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        (got,) = torch.autograd.grad(layer_norm(*args), args[i], torch.ones_like(x))
        assert torch.equal(got, want[i])


def test_gradient_against_differences():
    """Central differences in fp32 over a step e: the loss of 640 terms of order
    1 is good to 2^-24 * 640, its difference to that over e; the third order is
    e^2 of the gradient's scale."""
    from uttt_amd.norm import layer_norm
    x, w, b, dy = (t.cuda() for t in make(10, 64, F32, F32))
    loss = lambda x, w, b: (layer_norm(x, w, b).double() * dy.double()).sum()  # noqa: E731
    leaf = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(loss(*leaf), leaf)
    e = 1e-2
    for i, g in enumerate(grads):
        d = torch.randn(g.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(i))
        hi, lo = (loss(*(t + s * e * d if j == i else t for j, t in enumerate((x, w, b)))) for s in (1, -1))
        want = ((hi - lo) / (2 * e)).item()
        have = (g.double() * d.double()).sum().item()
        scale = (g.double().abs() * d.double().abs()).sum().item()
        assert abs(have - want) <= U * 640 / e + 10 * e * e * scale, (i, have, want)


def test_twice_the_same_bits_and_in_a_graph():
    from uttt_amd.norm import layer_norm
    x, w, b, dy = (t.cuda() for t in make(5000, 320, BF16, F32))
    leaf = [t.requires_grad_() for t in (x, w, b)]

    def run(leaf):
        y = layer_norm(*leaf)
        return [y.detach(), *torch.autograd.grad(y, leaf, dy)]

    for s, t in zip(run(leaf), run(leaf)):
        assert torch.equal(s, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(leaf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(leaf)
    for _ in range(3):
        with torch.no_grad():
            x.mul_(-0.7)
        graph.replay()
        want = run([t.detach().clone().requires_grad_() for t in (x, w, b)])
        torch.cuda.synchronize()
        for s, t in zip(got, want):
            assert torch.equal(s, t)


@pytest.mark.parametrize("N", [1024, 1025])
def test_offsets_past_32_bits(N):
    """The last rows of more than 2^31 elements give the bits of a call that has
    only them."""
    from uttt_amd.norm import layer_norm
    rows, few = 2 ** 31 // 1024 + 5, 7
    x = torch.randn(few, N, device="cuda", dtype=BF16).repeat(rows // few + 1, 1)[:rows].requires_grad_()
    w = torch.randn(N, device="cuda")
    y = layer_norm(x, w)
    dy = torch.randn(few, N, device="cuda", dtype=BF16).repeat(rows // few + 1, 1)[:rows]
    dx, = torch.autograd.grad(y, x, dy)
    end = x[-few:].detach().clone().requires_grad_()
    y2 = layer_norm(end, w)
    assert torch.equal(y[-few:], y2)
    assert torch.equal(dx[-few:], torch.autograd.grad(y2, end, dy[-few:])[0])
