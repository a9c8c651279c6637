"""The short causal convolution on the GPU against 64 bits (tolerances:
tests/state_space_cases.py)."""
import pytest
import torch

from oracle import state_space as O
from state_space_cases import BF16, F16, F32, check, conv_bounds, up

pytestmark = pytest.mark.gpu


def inputs(B=1, T=1, D=1, W=4, dtype=F32, wdtype=F32, bias=True, state=True, seqs=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    n = B if seqs is None else seqs
    x = r(B, T, 2, D).to(dtype).cuda()[:, :, 0]
    w, b = (r(D, W) / W ** 0.5).to(wdtype).cuda(), (0.3 * r(D)).to(wdtype).cuda() if bias else None
    h0 = r(n, W - 1, D).to(dtype).cuda() if state else None
    return [x, w, b, h0], (r(B, T, D).to(dtype).cuda(), r(n, W - 1, D).to(dtype).cuda())


def call(x, w, b, h0, silu, cu=None):
    from uttt_amd.state_space import causal_conv
    return causal_conv(x, w, b, activation="silu" if silu else None, initial_state=h0, output_final_state=True,
                       cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda"))


def check_conv(a, grads, silu, cu=None):
    with torch.no_grad():
        y0, s0 = call(*a, silu, cu)
    val, err = conv_bounds(*map(up, a), silu, *map(up, grads), cu)
    check(y0, val["y"], err["y"], "y")
    assert torch.equal(s0.double().cpu(), val["state"])
    leaf = [None if t is None else t.detach().requires_grad_() for t in a]
    y, s = call(*leaf, silu, cu)
    assert torch.equal(y, y0) and torch.equal(s, s0)
    names = [n for n, t in zip(("x", "w", "b", "h0"), leaf) if t is not None]
    got = torch.autograd.grad([y, s], [t for t in leaf if t is not None], list(grads))
    for n, g, t in zip(names, got, [t for t in leaf if t is not None]):
        assert g.dtype == t.dtype
        check(g, val[n], err[n], n)
    return [y0, s0, *got]


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 7, 8, 9, 16, 31, 32, 33, 35, 36, 63, 64, 65, 100, 260])
@pytest.mark.parametrize("silu", [False, True])
def test_lengths(T, silu):
    check_conv(*inputs(B=2, T=T, D=20, dtype=BF16, seed=T), silu)


@pytest.mark.parametrize("W", range(2, 9))
@pytest.mark.parametrize("T", [1, 6, 45])
@pytest.mark.parametrize("D", [8, 13])
def test_widths(W, T, D):
    check_conv(*inputs(B=3, T=T, D=D, W=W, seed=W), True)


@pytest.mark.parametrize("D", [1, 2, 3, 4, 31, 64, 100, 127, 129, 260, 1536])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16), (F32, BF16)])
def test_channels_and_types(D, dtype, wdtype):
    check_conv(*inputs(B=1, T=40, D=D, dtype=dtype, wdtype=wdtype, bias=D % 2 == 0, state=D % 3 != 0, seed=D), True)


@pytest.mark.parametrize("lens,front,behind", [
    ([1], 0, 0), ([0], 3, 2), ([0, 0, 5, 0], 0, 0), ([17, 64, 0, 1, 130, 2, 3], 0, 0), ([70, 3, 0], 5, 40),
    ([1] * 40, 0, 1), ([2] * 20, 1, 0), ([200, 1, 65], 64, 64), ([0, 0], 0, 0), ([0], 0, 0)])
@pytest.mark.parametrize("D,W", [(64, 4), (33, 8)])
def test_packed(lens, front, behind, D, W):
    """No sequence sees another's inputs; tokens of no sequence get zeros; states of
    sequences shorter than the window keep part of what was there before."""
    cu = [front + sum(lens[:i]) for i in range(len(lens) + 1)]
    a, grads = inputs(T=cu[-1] + behind, D=D, W=W, dtype=BF16, seqs=len(lens), seed=W)
    y, _, dx, *_ = check_conv(a, grads, True, cu)
    loose = [t for t in range(cu[-1] + behind) if t < front or t >= cu[-1]]
    assert (y[:, loose] == 0).all() and (dx[:, loose] == 0).all()


def test_large():
    """The longer runs of large calls."""
    from uttt_amd.state_space import causal_conv
    a, _ = inputs(B=3, T=3000, D=1536, dtype=BF16, seed=1)
    y, s = call(*a, True)
    for b in (0, 2):
        want, state = O.causal_conv(up(a[0][b:b + 1, :, :96]), up(a[1][:96]), up(a[2][:96]), True, up(a[3][b:b + 1, :, :96]))
        size, _ = O.causal_conv(up(a[0][b:b + 1, :, :96]).abs(), up(a[1][:96]).abs(), up(a[2][:96]).abs(), False,
                                up(a[3][b:b + 1, :, :96]).abs())
        check(y[b:b + 1, :, :96], want, 40 * O.U * size, "y")
        assert torch.equal(s[b:b + 1, :, :96].double().cpu(), state)
    alone = causal_conv(a[0][1:2, 100:], a[1], a[2], activation="silu", initial_state=a[0][1:2, 97:100].contiguous())[0]
    assert torch.equal(alone, y[1:2, 100:])


def test_views():
    a, grads = inputs(B=2, T=45, D=36, dtype=BF16)
    want = check_conv(a, grads, True)

    def wide(t, front):
        big = t.new_zeros(*t.shape[:-1], t.shape[-1] + 5)
        big[..., front:front + t.shape[-1]] = t
        return big[..., front:front + t.shape[-1]]

    for change in (lambda t: wide(t, 1), lambda t: wide(t, 4), lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                   lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)):
        b = [t if t is None or t.dim() < 2 else change(t) for t in a]
        for x, y in zip(check_conv(b, tuple(map(change, grads)), True), want):
            assert torch.equal(x, y)
    assert torch.equal(call(a[0][:1].expand(2, -1, -1), *a[1:3], None, True)[0][1], call(a[0][:1], *a[1:3], None, True)[0][0])


def test_values_that_are_not_finite():
    cu = [4, 60, 95]
    a, grads = inputs(T=120, D=40, dtype=BF16, seqs=2, seed=5)
    clean = check_conv(a, grads, True, cu)
    x = a[0].clone()
    x[0, :4] = x[0, 95:] = float("nan")
    dy = grads[0].clone()
    dy[0, :4] = dy[0, 95:] = float("inf")
    leaf = [t.detach().requires_grad_() for t in [x] + a[1:]]
    y, s = call(*leaf, True, cu)
    got = torch.autograd.grad([y, s], leaf, [dy, grads[1]])
    for p, q in zip([y, s, *got], clean):
        assert torch.equal(p, q)
    x = a[0].clone()
    x[0, 58, 7] = float("inf")      # near the first sequence's end: its state, not the second
    y, s = call(x, *a[1:], True, cu)
    assert torch.equal(y[:, :58], clean[0][:, :58]) and torch.equal(y[:, 60:], clean[0][:, 60:])
    assert torch.equal(s[1], clean[1][1]) and s[0, 1, 7] == float("inf")


def test_no_tokens():
    a, grads = inputs(B=2, T=0, D=10)
    y, s, dx, dw, db, dh0 = check_conv(a, grads, True)
    assert torch.equal(s, a[3]) and torch.equal(dh0, grads[1]) and (dw == 0).all() and (db == 0).all()


def test_one_gradient_alone_and_the_same_bits():
    a, grads = inputs(B=2, T=300, D=68, dtype=BF16)
    leaf = [t.detach().requires_grad_() for t in a]
    zero = torch.zeros_like
    for g in ((grads[0], zero(grads[1])), (zero(grads[0]), grads[1])):
        one = grads[0] is g[0]
        full = torch.autograd.grad(call(*leaf, True), leaf, list(g))
        alone = torch.autograd.grad(call(*leaf, True)[0 if one else 1], leaf, g[0 if one else 1], allow_unused=True)
        for s, t in zip(full, alone):
            assert torch.equal(s, zero(s) if t is None else t)
    want = torch.autograd.grad(call(*leaf, True)[0], leaf[2], grads[0])[0]
    leaf[1].requires_grad_(False)
    assert torch.equal(torch.autograd.grad(call(*leaf, True)[0], leaf[2], grads[0])[0], want)


def test_backward_in_a_graph():
    a, grads = inputs(T=150, D=40, dtype=BF16, seqs=2)
    cu = torch.tensor([0, 70, 140], device="cuda")
    leaf = [t.detach().requires_grad_() for t in a]
    from uttt_amd.state_space import causal_conv

    def run():
        y, s = causal_conv(*leaf[:3], activation="silu", initial_state=leaf[3], output_final_state=True, cu_seqlens=cu)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], leaf, list(grads))]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(3):
        with torch.no_grad():
            leaf[0].copy_(torch.randn(leaf[0].shape, device="cuda"))
        cu.copy_(torch.tensor([[0, 70, 140], [3, 3, 150], [10, 20, 30]][i], device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, run()):
            assert torch.equal(x, y), i
        torch.cuda.synchronize()


# --------------------------------------------------------------- by tokens --
def step(x, w, b, state, idx=None, silu=True):
    from uttt_amd.state_space import causal_conv_step
    return causal_conv_step(x, w, state, b, activation="silu" if silu else None, state_indices=idx)


@pytest.mark.parametrize("D,W", [(1, 2), (5, 3), (64, 4), (257, 4), (300, 8)])
@pytest.mark.parametrize("T", [1, 2, 9])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_step_is_the_convolution(D, W, T, dtype):
    """Outputs within the bounds, states exactly."""
    a, grads = inputs(B=4, T=T, D=D, W=W, dtype=dtype, bias=T != 2, seed=D)
    val, err = conv_bounds(*map(up, a), True, *map(up, grads), None)
    state = a[3].clone()
    check(step(*a[:3], state), val["y"], err["y"], "y")
    assert torch.equal(state.double().cpu(), val["state"])


def test_step_rows_of_a_pool():
    a, _ = inputs(B=7, T=2, D=70, dtype=BF16, seed=1)
    pool = torch.randn(6, 2, 3, 70, device="cuda").to(BF16)
    before = pool.clone()
    for dtype in (torch.int32, torch.int64):
        pool.copy_(before)
        idx = torch.tensor([4, -1, 0, 4, 9, 2, 4], dtype=dtype, device="cuda")
        y = step(*a[:3], pool[:, 1], idx)
        ref, want = before.clone(), torch.zeros_like(y)
        for row, slot in enumerate(idx.tolist()):
            if 0 <= slot < 6:
                s = ref[slot:slot + 1, 1].clone()
                want[row] = step(a[0][row:row + 1], *a[1:3], s)[0]
                ref[slot, 1] = s[0]
        assert torch.equal(y, want) and torch.equal(pool, ref)


def test_step_without_rows_or_tokens():
    a, _ = inputs(B=3, T=1, D=8)
    state = a[3].clone()
    assert step(a[0][:, :0], *a[1:3], state).shape == (3, 0, 8) and torch.equal(state, a[3])
    assert step(a[0][:0], *a[1:3], state).shape == (0, 1, 8) and torch.equal(state, a[3])


def test_step_in_a_graph():
    a, _ = inputs(B=3, T=1, D=70, dtype=BF16)
    state = torch.randn(5, 3, 70, device="cuda").to(BF16)
    eager, idx = state.clone(), torch.tensor([3, 0, -1], dtype=torch.int32, device="cuda")
    step(*a[:3], state.clone(), idx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*a[:3], state, idx)
    for i in range(4):
        a[0].copy_(torch.randn(a[0].shape, device="cuda"))
        idx.copy_(torch.tensor([[3, 0, -1], [1, 1, 1], [4, 2, 0], [-1, 7, 3]][i], device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = step(*a[:3], eager, idx)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, eager), i
