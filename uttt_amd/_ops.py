"""torch.library registrations of this package's C-ABI calls (namespace
`uttt_hip`), each with a fake implementation that gives its outputs' shapes
and dtypes, so that torch.compile traces the drop-in ops into its graph
instead of breaking the graph at every kernel call.

`traced_op(name, fake)` registers a function as torch.ops.uttt_hip.<name>
and returns a wrapper that calls the registered op while torch.compile
traces, and the function itself otherwise (eager calls skip the dispatcher,
and count a change of the arguments that they write to themselves, so that
autograd refuses a backward that saved one of them before).
"""
from __future__ import annotations

import ctypes
import functools
import inspect

import torch
from torch._C._functorch import is_dead_tensor_wrapper
from torch._functorch.utils import unwrap_dead_wrappers
from torch.autograd import forward_ad


def traced_op(name, fake, mutates_args=()):
    def deco(fn):
        op = torch.library.custom_op(f"uttt_hip::{name}", fn, mutates_args=mutates_args)
        op.register_fake(fake)
        names = list(inspect.signature(fn).parameters)
        written = [names.index(n) for n in mutates_args]

        @functools.wraps(fn)
        def call(*args, **kwargs):
            if torch.compiler.is_compiling():
                return op(*args, **kwargs)
            out = fn(*args, **kwargs)
            for i in written:
                t = args[i] if i < len(args) else kwargs[names[i]]
                if not t.is_inference():   # those have no count, and nothing saves them
                    torch.autograd.graph.increment_version(t)
            return out

        call.op = op
        return call

    return deco


class _NoGraph:
    """The ctx of a forward whose graph nobody keeps."""

    def save_for_backward(self, *tensors):
        pass

    def mark_non_differentiable(self, *tensors):
        pass


def run_function(fn, *args, graph=True):
    """fn.apply(*args) of a torch.autograd.Function, or its forward alone where
    nothing could see the difference: gradients are off (or the caller knows
    that no input requires one: graph=False) and neither torch.compile, jit
    tracing, a functorch transform nor a forward-mode level is active (under
    which apply records, refuses or transforms the call).
    A forward that hands an input through returns it as it is, where apply
    returns an alias: its caller makes one (permute_with_expert_mask).
    apply costs 5 to 8 us of host time per call; a routed read without
    gradients, three of them, is paced by its host time (88 us against 61 on
    the GPU for 16 384 tokens of 192 over 48 experts)."""
    if (graph and torch.is_grad_enabled() or torch.compiler.is_compiling()
            or torch._C._are_functorch_transforms_active()
            or torch._C._get_tracing_state() is not None or forward_ad._current_level >= 0):
        return fn.apply(*args)
    try:
        return fn.forward(_NoGraph(), *args)
    except RuntimeError:
        # a tensor that outlived its functorch transform is a shell without an
        # address around the real one, which apply hands on
        if not any(isinstance(a, torch.Tensor) and is_dead_tensor_wrapper(a) for a in args):
            raise
    return fn.forward(_NoGraph(), *unwrap_dead_wrappers(args))


class _FirstOrder(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, n, *tensors):
        ctx.what = what
        return tensors[:n]

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.what}: gradients of its gradients are not built")


def first_order_only(what, grads, *inputs):
    """A backward's `grads`, through which no gradient passes: under
    create_graph=True they hang on `inputs` (what they are computed from, the
    given gradients included) by a node that raises, so that a loss made of them
    raises too and loses no term in silence.  (torch's once_differentiable lets
    gradients through without a graph where the given ones require none, as
    those of any loss linear in the outputs.)"""
    if not torch.is_grad_enabled():
        return grads
    return _FirstOrder.apply(what, len(grads), *grads, *(t for t in inputs if t is not None))


def no_gradient(what, *tensors):
    """Refuses tensors through which a gradient would have to flow, backward or
    forward, in a call that changes its states in place."""
    tensors = [t for t in tensors if t is not None]
    assert not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)) and not (
        forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)), (
        f"{what}: no gradient flows through a state that is updated in place")


@functools.lru_cache(maxsize=256)
def _int64s(*values):
    """Host integers as the C ABI takes them (read during a call, never written)."""
    return (ctypes.c_int64 * len(values))(*values)


def strides_of(t, axes):
    """Element strides of t's first two or three axes as the C ABI takes them, 0
    along an axis of one, whose stride says nothing."""
    n, s = t.shape, t.stride()
    if axes == 2:
        return _int64s(s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0)
    return _int64s(s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0)


def evenly(step):
    """The strides of rows `step` elements apart, in one group."""
    return _int64s(step, 0)


def none_if_empty(t):
    """Optional outputs travel through the ops as 0-element tensors."""
    return None if t is None or t.numel() == 0 else t


def new_like(t):
    """A contiguous tensor of t's shape and dtype (1.3 us of host time, against
    2.3 of torch.empty by shape)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def empty_like_dev(ref, *shape, dtype=None):
    return ref.new_empty(shape, dtype=ref.dtype if dtype is None else dtype)
