"""The rotary embedding over several axes on the GPU against complex products
in 64 bits.  Tolerance per element: the result's half step, and in fp32 the
angle's reduction to half turns (2^-24 pi), sine and cosine (2 * 2^-24) and
three operations, 8 * 2^-24 of the pair's length in all."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def turned(x, pos, freq, sections, interleaved, back=False):
    x, R = x.double(), sum(sections)
    axis = [a for a, m in enumerate(sections) for _ in range(m)]
    angle = pos.double()[..., axis] * freq.double()
    z = torch.polar(torch.ones_like(angle), -angle if back else angle)
    z = z.expand(x.shape[0], x.shape[1], R)[:, :, None]
    y, size = x.clone(), torch.zeros_like(x)
    a, b = (slice(0, 2 * R, 2), slice(1, 2 * R, 2)) if interleaved else (slice(0, R), slice(R, 2 * R))
    w = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * z
    y[..., a], y[..., b] = w.real, w.imag
    size[..., a] = size[..., b] = w.abs()
    return y, size


def check(x, pos, freq, sections, interleaved, dy=None, move=lambda t: t.cuda()):
    from uttt_amd.positions import rotary_axes
    xs = move(x).requires_grad_()
    y = rotary_axes(xs, pos.cuda(), freq.cuda(), sections, interleaved=interleaved)
    dy = torch.randn(x.shape, generator=torch.Generator().manual_seed(5)).to(x.dtype) if dy is None else dy
    (dx,) = torch.autograd.grad(y, xs, move(dy))
    for got, (ref, size) in ((y, turned(x, pos, freq, sections, interleaved)),
                             (dx, turned(dy, pos, freq, sections, interleaved, True))):
        assert got.dtype == x.dtype and got.shape == x.shape
        inner = 8 * 2.0 ** -24 * size
        allowed = torch.finfo(x.dtype).eps / 2 * (ref.abs() + inner) + inner
        tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
        off = (got.detach().double().cpu() - ref).abs()
        assert (off <= allowed + tiny).all(), (off - allowed).max().item()
    return y.detach()


def make(B, L, H, D, sections, dtype, pos_type=torch.int32, seed=0, far=1000):
    from uttt_amd.positions import axis_frequencies
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, H, D, generator=gen).to(dtype)
    pos = torch.randint(-far, far, (B, L, len(sections)), generator=gen).to(pos_type)
    return x, pos, axis_frequencies(sections)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("sections,D", [([8, 12, 12], 64), ([16, 16, 16], 128), ([1], 2), ([3], 7), ([2, 3], 10),
                                        ([4, 4], 16), ([8], 16), ([8, 8], 48), ([2, 2], 9), ([5, 0, 6], 24),
                                        ([1] * 8, 16), ([12, 20, 32], 128), ([4], 12), ([700, 700], 2800)])
def test_sections(sections, D, dtype, interleaved):
    check(*make(2, 37, 3, D, sections, dtype), sections, interleaved)


@pytest.mark.parametrize("B,L,H", [(1, 1, 1), (1, 1, 40), (3, 129, 1), (2, 1000, 12), (1, 4099, 4)])
def test_tokens_and_heads(B, L, H):
    check(*make(B, L, H, 64, [8, 12, 12], BF16), [8, 12, 12], False)


@pytest.mark.parametrize("pos_type", [torch.int32, torch.int64])
def test_far_positions(pos_type):
    check(*make(1, 200, 2, 64, [16, 16], F32, pos_type, far=2_000_000_000), [16, 16], False)


def test_positions_shared_by_the_batch_and_strided():
    sections = [8, 8]
    x, pos, freq = make(3, 50, 2, 32, sections, F32)
    shared = pos[0]
    got = check(x, shared, freq, sections, True)
    from uttt_amd.positions import rotary_axes
    full = shared.expand(3, 50, 2).contiguous()
    assert torch.equal(got, rotary_axes(x.cuda(), full.cuda(), freq.cuda(), sections, interleaved=True))
    axes_first = full.cuda().permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(got, rotary_axes(x.cuda(), axes_first, freq.cuda(), sections, interleaved=True))


@pytest.mark.parametrize("interleaved", [False, True])
def test_views(interleaved):
    x, pos, freq = make(2, 40, 3, 64, [16, 8], BF16)

    def fused(t):
        big = torch.full((2, 40, 3, 3, 64), float("nan"), dtype=t.dtype, device="cuda")
        big[:, :, 2] = t.cuda()
        return big[:, :, 2]

    def unaligned(t):
        big = torch.zeros(2, 40, 3, 67, dtype=t.dtype, device="cuda")
        big[..., 1:65] = t.cuda()
        return big[..., 1:65]

    want = check(x, pos, freq, [16, 8], interleaved)
    for move in (fused, unaligned, lambda t: t.cuda().transpose(1, 2).contiguous().transpose(1, 2),
                 lambda t: t.cuda().permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)):
        assert torch.equal(check(x, pos, freq, [16, 8], interleaved, move=move), want)


def test_expanded_heads_and_gradient():
    from uttt_amd.positions import rotary_axes
    x, pos, freq = make(1, 30, 1, 32, [16], F32)
    one = x.cuda().requires_grad_()
    y = rotary_axes(one.expand(1, 30, 4, 32), pos.cuda(), freq.cuda(), [16])
    (g,) = torch.autograd.grad(y.sum(), one)   # an expanded scalar gradient
    many = x.cuda().expand(1, 30, 4, 32).contiguous().requires_grad_()
    y2 = rotary_axes(many, pos.cuda(), freq.cuda(), [16])
    (g2,) = torch.autograd.grad(y2, many, torch.ones_like(y2))
    assert torch.equal(y, y2) and torch.equal(g, g2.sum(2, keepdim=True))


def test_there_and_back_and_axes_apart():
    """One axis alone turns its own section only; equal positions on all axes
    are one position."""
    from uttt_amd.positions import axis_frequencies, rotary_axes
    sections = [4, 12, 16]
    x, pos, freq = (t.cuda() for t in make(1, 20, 2, 64, sections, F32))
    zero = pos.clone()
    zero[..., 1:] = 0
    y = rotary_axes(x, zero, freq, sections)
    for keep in (slice(4, 32), slice(36, 64)):
        assert torch.equal(y[..., keep], x[..., keep])
    same = pos[..., :1].expand(1, 20, 3)
    assert torch.equal(rotary_axes(x, same, freq, sections), rotary_axes(x, pos[..., :1], freq, [32]))
    per = axis_frequencies(sections, per_axis=True)
    assert per.shape == (32,) and per[0] == per[4] == per[16] == 1.0


def test_empty_and_in_a_graph():
    from uttt_amd.positions import rotary_axes
    x, pos, freq = (t.cuda() for t in make(2, 300, 4, 64, [16, 16], BF16))
    for a, b in ((x[:0], pos[:0]), (x[:, :0], pos[:, :0]), (x[:, :, :0], pos)):
        assert rotary_axes(a, b, freq, [16, 16]).shape == a.shape
    run = lambda: rotary_axes(x, pos, freq, [16, 16])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    for i in range(3):
        pos.add_(7)
        x.mul_(-0.5)
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("sections,D", [([20, 20, 20], 120), ([14, 13, 14], 100), ([2, 2], 12), ([5], 11)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_piece_widths(sections, D, interleaved):
    """Pairs and features that divide into 8-byte pieces, into single ones, and
    a last piece of half the features."""
    for dtype in (BF16, F32):
        check(*make(2, 37, 5, D, sections, dtype), sections, interleaved)


def test_offsets_past_32_bits():
    from uttt_amd.positions import axis_frequencies, rotary_axes
    L, H, D = 2 ** 21 + 3, 16, 64
    x = torch.randn(1, L, H, D, device="cuda", dtype=BF16)
    pos = torch.arange(L, device="cuda")[:, None]
    freq = axis_frequencies([32], device="cuda")
    y = rotary_axes(x, pos, freq, [32])
    assert torch.equal(y[:, -100:], rotary_axes(x[:, -100:], pos[-100:], freq, [32]))
    assert torch.equal(y[:, :100], rotary_axes(x[:, :100], pos[:100], freq, [32]))
