"""Second-order gradients of the memory layer's operators and the step's version
count with the kernels themselves (the rules: tests/test_memory_layer_autograd.py)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def rule_inputs(T=70):
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    unit = lambda t: (t / t.norm(dim=-1, keepdim=True)).to(BF16)  # noqa: E731
    return [unit(r(1, T, 1, 64)), unit(r(1, T, 1, 64)), r(1, T, 2, 64).to(BF16), -0.1 * r(1, T, 2).abs(),
            torch.sigmoid(r(1, T, 2))]


def test_rotary_twice():
    """|x|^2 through a turn: its gradient is 2 x, and of |gradient|^2 8 x; each turn
    is off by 8 * 2^-24 of a pair's length, and a gradient of a gradient has four."""
    from uttt_amd.positions import axis_frequencies, rotary_axes
    x = torch.randn(2, 50, 3, 32, device="cuda").requires_grad_()
    pos = torch.randint(-1000, 1000, (2, 50, 2), device="cuda")
    y = rotary_axes(x, pos, axis_frequencies([8, 8], device="cuda"), [8, 8])
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    (gg,) = torch.autograd.grad(g.square().sum(), x)
    length = (x[..., :16].square() + x[..., 16:].square()).sqrt().repeat(1, 1, 1, 2)
    assert ((g - 2 * x).abs() <= 2 * 2 * 8 * 2.0 ** -24 * length).all()
    assert ((gg - 8 * x).abs() <= 8 * 4 * 8 * 2.0 ** -24 * length).all()


def test_gradients_under_create_graph_are_the_same_and_refuse_more():
    from uttt_amd.delta import gated_delta_rule
    from uttt_amd.norm import layer_norm
    leaves = [t.requires_grad_() for t in rule_inputs()]
    h0 = torch.randn(1, 2, 64, 64, device="cuda", requires_grad=True)
    x, w, b = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((40, 96), (96,), (96,)))
    rule = lambda: sum(t.float().sum() for t in gated_delta_rule(*leaves, initial_state=h0, output_final_state=True))  # noqa: E731
    for loss, wanted in ((rule, leaves + [h0]), (lambda: layer_norm(x, w, b).sum(), [x, w, b])):
        once = torch.autograd.grad(loss(), wanted)
        total = loss()
        grads = torch.autograd.grad(total, wanted, create_graph=True)
        for s, t in zip(once, grads):
            assert torch.equal(s, t)
        with pytest.raises(RuntimeError, match="gradients of its gradients"):
            torch.autograd.grad(total + sum(g.float().square().sum() for g in grads), wanted)


def test_a_state_saved_before_the_step():
    from uttt_amd.delta import gated_delta_step
    x = rule_inputs(1)
    state = torch.randn(1, 2, 64, 64, device="cuda", requires_grad=True)
    loss = state.square().sum()
    with torch.no_grad():
        gated_delta_step(*x, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_the_states_of_a_rule_step_on_before_its_backward():
    """An initial state that carries on elsewhere in place: the rule's backward does
    not read it again."""
    from uttt_amd.delta import gated_delta_rule, gated_delta_step
    x = rule_inputs()
    leaf = torch.randn(1, 2, 64, 64, device="cuda", requires_grad=True)
    want = torch.autograd.grad(gated_delta_rule(*x, initial_state=leaf * 1.0)[0].float().sum(), leaf)[0]
    state = leaf * 1.0
    o, _ = gated_delta_rule(*x, initial_state=state)
    with torch.no_grad():
        gated_delta_step(*(t[:, :1] for t in x), state.detach())
    assert torch.equal(torch.autograd.grad(o.float().sum(), leaf)[0], want)
