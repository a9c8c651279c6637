"""What autograd may do with the memory layer's operators beyond one backward
pass, without a GPU: the kernels' fake implementations carry the shapes."""
import pytest
import torch

from uttt_amd import delta, norm

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
