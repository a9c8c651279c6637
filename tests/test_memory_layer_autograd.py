"""What autograd may do with the memory layer's operators beyond one backward
pass, without a GPU: the kernels' fake implementations carry the shapes."""
import pytest
import torch
from torch.autograd import forward_ad

from uttt_amd import delta, norm, positions

BF16, F32 = torch.bfloat16, torch.float32


def leaf(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="meta", requires_grad=True)


def rule_leaves(T=10):
    return [leaf(2, T, 1, 64), leaf(2, T, 1, 64), leaf(2, T, 2, 32), leaf(2, T, 2, dtype=F32), leaf(2, T, 2, dtype=F32)]


@pytest.mark.parametrize("linear", [True, False])
@pytest.mark.parametrize("one", [None, 0, 1, 2, 3, 4, 5])
def test_second_order_of_the_rule_is_refused(monkeypatch, linear, one):
    """A penalty on its gradients would be lost in silence: with a gradient of
    its outputs that is constant and one that is not, for any leaf alone."""
    monkeypatch.setattr(delta, "_fwd", delta._fwd_fake)
    monkeypatch.setattr(delta, "_bwd", delta._bwd_fake)
    leaves = rule_leaves() + [leaf(2, 2, 64, 32, dtype=F32)]
    if one is not None:
        leaves = [t.requires_grad_(i == one) for i, t in enumerate(leaves)]
    o, S = delta.gated_delta_rule(*leaves[:5], initial_state=leaves[5], output_final_state=True)
    loss = o.float().sum() + S.sum() if linear else o.float().square().sum() + S.square().sum()
    wanted = [t for t in leaves if t.requires_grad]
    once = torch.autograd.grad(loss, wanted, retain_graph=True)
    assert not any(g.requires_grad for g in once)
    grads = torch.autograd.grad(loss, wanted, create_graph=True)
    assert [g.shape for g in grads] == [t.shape for t in wanted]
    for g in grads:
        for t in wanted:
            with pytest.raises(RuntimeError, match="gradients of its gradients"):
                torch.autograd.grad(loss + g.float().square().sum(), t, retain_graph=True)


@pytest.mark.parametrize("linear", [True, False])
@pytest.mark.parametrize("one", [None, 0, 1, 2])
def test_second_order_of_layer_norm_is_refused(monkeypatch, linear, one):
    monkeypatch.setattr(norm, "_fwd", norm._fwd_fake)
    monkeypatch.setattr(norm, "_bwd", norm._bwd_fake)
    leaves = [leaf(4, 16), leaf(16, dtype=F32), leaf(16)]
    if one is not None:
        leaves = [t.requires_grad_(i == one) for i, t in enumerate(leaves)]
    y = norm.layer_norm(*leaves).float()
    loss = y.sum() if linear else y.square().sum()
    wanted = [t for t in leaves if t.requires_grad]
    once = torch.autograd.grad(loss, wanted, retain_graph=True)
    assert not any(g.requires_grad for g in once)
    grads = torch.autograd.grad(loss, wanted, create_graph=True)
    assert [g.shape for g in grads] == [t.shape for t in wanted]
    for g in grads:
        for t in wanted:
            with pytest.raises(RuntimeError, match="gradients of its gradients"):
                torch.autograd.grad(loss + g.float().square().sum(), t, retain_graph=True)


def turn_in_torch(x, positions, inv_freq, sections, interleaved, inverse):
    """The rotary kernel's product, for tensors on the CPU."""
    R = sum(sections)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    angle = (positions[..., axis] * inv_freq)[:, :, None] * (-1 if inverse else 1)
    a, b = (x[..., 0:2 * R:2], x[..., 1:2 * R:2]) if interleaved else (x[..., :R], x[..., R:2 * R])
    u, w = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    return torch.cat([torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1),
                      x[..., 2 * R:]], -1).detach()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_is_differentiable_any_number_of_times(monkeypatch, interleaved):
    """Linear in x: its gradient's gradient is the turn itself, here with the
    kernel's product in torch.  Up to third order, against differences."""
    monkeypatch.setattr(positions, "_turn", turn_in_torch)
    monkeypatch.setattr(positions.L, "require_device", lambda *t: None)
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 2, 10, generator=gen, dtype=F32).requires_grad_()
    pos = torch.randint(-9, 9, (2, 3, 2), generator=gen)
    f = lambda t: positions.rotary_axes(t, pos, torch.tensor([1.0, 0.3, 0.1]), [1, 2], interleaved=interleaved)  # noqa: E731
    w = torch.randn(x.shape, generator=gen)
    # y.y is |x|^2, so that its gradient is 2 x and that of |gradient|^2 8 x
    (g,) = torch.autograd.grad(f(x).square().sum(), x, create_graph=True)
    assert torch.allclose(g, 2 * x, atol=1e-5)
    (gg,) = torch.autograd.grad(g.square().sum(), x, create_graph=True)
    assert torch.allclose(gg, 8 * x, atol=1e-4)
    (ggg,) = torch.autograd.grad(gg.square().sum(), x)
    assert torch.allclose(ggg, 128 * x, atol=1e-3)
    # a loss linear in y: the gradient does not depend on x, but on what it is given
    v = w.clone().requires_grad_()
    (g,) = torch.autograd.grad(f(x), x, v, create_graph=True)
    (gv,) = torch.autograd.grad(g, v, w)
    assert torch.allclose(gv, f(w), atol=1e-5)
    (g,) = torch.autograd.grad((f(x) * w).sum(), x, create_graph=True)
    assert torch.allclose(f(g.detach()), w, atol=1e-5)


def test_rotary_refuses_frequencies_that_require_gradients():
    """None would reach them."""
    x, pos = leaf(1, 3, 2, 8), torch.empty(1, 3, 1, dtype=torch.int32, device="meta")
    freq = leaf(4, dtype=F32)
    with pytest.raises(AssertionError, match="inv_freq"):
        positions.rotary_axes(x, pos, freq, [4])
    with pytest.raises(AssertionError, match="inv_freq"):
        positions.rotary_axes(x.detach(), pos, freq, [4])


def test_rotary_takes_such_frequencies_where_gradients_are_off(monkeypatch):
    monkeypatch.setattr(positions, "_turn", positions._turn_fake)
    x, pos = leaf(1, 3, 2, 8), torch.empty(1, 3, 1, dtype=torch.int32, device="meta")
    with torch.no_grad():
        assert positions.rotary_axes(x, pos, leaf(4, dtype=F32), [4]).shape == x.shape


def step_inputs(slots=3, device="meta"):
    e = lambda *s, dtype=BF16: torch.empty(*s, dtype=dtype, device=device)  # noqa: E731
    return [e(2, 1, 1, 64), e(2, 1, 1, 64), e(2, 1, 2, 32), e(2, 1, 2, dtype=F32), e(2, 1, 2, dtype=F32)], e(
        slots, 2, 64, 32, dtype=F32)


@pytest.fixture
def launched(monkeypatch):
    """The step up to its launch, on meta tensors."""
    calls = []
    monkeypatch.setattr(delta.L, "call_on", lambda t, name, *args: calls.append((name, args)))
    monkeypatch.setattr(delta.L, "stream_of", lambda t: 0)
    return calls


def test_the_step_says_that_it_changes_the_state(launched):
    """A state that another op has saved for its backward raises there, as after
    any torch operation in place; through a view of a pool too."""
    x, state = step_inputs()
    state.requires_grad_()
    loss = state.square().sum()
    with torch.no_grad():
        delta.gated_delta_step(*x, state)
    assert len(launched) == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    pool = torch.empty(3, 4, 2, 64, 32, device="meta")
    before = pool._version
    delta.gated_delta_step(*x, pool[:, 1])
    assert pool._version == before + 1
    before = [t._version for t in x]
    delta.gated_delta_step(*x, pool[:, 1])
    assert [t._version for t in x] == before


def test_the_step_takes_states_of_inference_mode(launched):
    x, state = step_inputs()
    with torch.inference_mode():
        own = torch.empty_like(state)
        delta.gated_delta_step(*x, own)
        delta.gated_delta_step(*x, state)
    delta.gated_delta_step(*x, own)   # which nothing can save for a backward
    assert len(launched) == 3


@pytest.mark.parametrize("which", range(6))
def test_the_step_refuses_forward_gradients(launched, which):
    """Their tangents would be lost in silence."""
    x, state = step_inputs()
    args = x + [state]
    with forward_ad.dual_level():
        delta.gated_delta_step(*args)   # none of them has one
        args[which] = forward_ad.make_dual(args[which], torch.empty_like(args[which]))
        with pytest.raises(AssertionError, match="no gradient"):
            delta.gated_delta_step(*args)
    assert len(launched) == 1


def test_the_others_refuse_forward_gradients(monkeypatch):
    monkeypatch.setattr(delta, "_infer", delta._infer_fake)
    monkeypatch.setattr(norm, "_infer", norm._infer_fake)
    monkeypatch.setattr(positions, "_turn", positions._turn_fake)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t.detach(), torch.empty_like(t))  # noqa: E731
        q, k, v, g, beta = rule_leaves()
        for call in (lambda: delta.gated_delta_rule(dual(q), k.detach(), v.detach(), g.detach(), beta.detach()),
                     lambda: norm.layer_norm(dual(leaf(4, 16))),
                     lambda: positions.rotary_axes(dual(leaf(1, 2, 1, 8)), torch.empty(2, 1, dtype=torch.int32, device="meta"),
                                                   torch.empty(4, device="meta"), [4])):
            with pytest.raises(NotImplementedError):
                call()
