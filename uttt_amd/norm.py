"""Layer norm with weight and bias over the last axis, forward and backward
(the learned norm in front of a layer; the parameter-free norms of the
fast-weight inputs are uttt_amd.moe.rows_preprocess).  No CPU path."""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import _lib as L
from ._ops import first_order_only, new_like, none_if_empty, run_function, traced_op

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _code(t: Optional[Tensor]) -> int:
    return L.F32 if t is None else L.dtype_code(t.dtype)


def _launch_fwd(x, weight, bias, eps, y, stats):
    L.call_on(x, "uttt_layer_norm_fwd", L.ptr(x), L.dtype_code(x.dtype), x.stride(0), x.shape[0],
              x.shape[1], L.ptr(weight), _code(weight), L.ptr(bias), _code(bias), eps, L.ptr(y),
              L.ptr(stats), L.stream_of(x))


def _infer_fake(x, weight, bias, eps):
    return new_like(x)


@traced_op("layer_norm_infer", _infer_fake)
def _infer(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float) -> Tensor:
    """y of x [rows, N] with any row stride."""
    y = _infer_fake(x, weight, bias, eps)
    _launch_fwd(x, weight, bias, eps, y, None)
    return y


def _fwd_fake(x, weight, bias, eps):
    return _infer_fake(x, weight, bias, eps), x.new_empty((2, x.shape[0]), dtype=torch.float32)


@traced_op("layer_norm_fwd", _fwd_fake)
def _fwd(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor],
         eps: float) -> Tuple[Tensor, Tensor]:
    """y, and the fp32 mean and 1 / deviation of each row for the backward."""
    y, stats = _fwd_fake(x, weight, bias, eps)
    _launch_fwd(x, weight, bias, eps, y, stats)
    return y, stats


def _bwd_fake(x, dy, weight, bias, stats, want_dw, want_db):
    return [new_like(x), new_like(weight) if want_dw else x.new_empty((0,)),
            new_like(bias) if want_db else x.new_empty((0,))]


@traced_op("layer_norm_bwd", _bwd_fake)
def _bwd(x: Tensor, dy: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor,
         want_dw: bool, want_db: bool) -> List[Tensor]:
    rows, N = x.shape
    grads = _bwd_fake(x, dy, weight, bias, stats, want_dw, want_db)
    size = L.lib().uttt_layer_norm_bwd_workspace_bytes(rows, N) if want_dw or want_db else 0
    ws = torch.empty(size, dtype=torch.uint8, device=x.device)
    L.call_on(x, "uttt_layer_norm_bwd", L.ptr(x), L.dtype_code(x.dtype), x.stride(0), L.ptr(dy),
              dy.stride(0), rows, N, L.ptr(weight), _code(weight), L.ptr(stats), L.ptr(grads[0]),
              L.ptr(grads[1]) if want_dw else None, L.ptr(grads[2]) if want_db else None, _code(bias),
              L.ptr(ws), size, L.stream_of(x))
    return grads


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        if not keep:
            return _infer(x, weight, bias, eps)
        y, stats = _fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        _, want_dw, want_db = ctx.needs_input_grad[:3]
        dy = dy if dy.stride(-1) == 1 or dy.shape[-1] == 1 else dy.contiguous()
        grads = _bwd(x, dy, weight, bias, stats, want_dw, want_db)
        dx, dw, db = first_order_only("layer_norm", grads, x, weight, bias, dy)
        return dx, none_if_empty(dw), none_if_empty(db), None, None


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None,
               eps: float = 1e-5) -> Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis, of up to
    2^27 elements; mean, variance and the products in fp32, rounded once to x's dtype.

    x [..., N] in fp32, bf16 or fp16; weight and bias [N], each None or in any
    of the three (fp32 weights with bf16 activations included).  Gradients have
    their inputs' dtypes; those of weight and bias are summed over the rows in
    fp32, in an order that the shape and the 16-byte alignment of tensors and
    rows decide.  x may be a view whose rows are evenly spaced (a slice of the
    last axis); other views are copied.  Gradients of its gradients are refused."""
    L.require_device(x, weight, bias)
    assert x.dim() >= 1 and x.shape[-1] >= 1, "layer_norm: x must be [..., N] with N of 1 or more"
    assert x.dtype in _TYPES, f"layer_norm: dtype {x.dtype}"
    N = x.shape[-1]
    keep = x.requires_grad
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            assert t.shape == (N,), f"layer_norm: {name} must be [{N}], got {tuple(t.shape)}"
            assert t.dtype in _TYPES, f"layer_norm: {name} has dtype {t.dtype}"
            assert t.get_device() == x.get_device(), f"layer_norm: {name} is on {t.device}, x on {x.device}"
            keep = keep or t.requires_grad
    rows = x if x.dim() == 2 else x.reshape(-1, N)   # a view wherever the rows are evenly spaced
    if (rows.stride(1) != 1 and N > 1) or rows.stride(0) < 0:
        rows = rows.contiguous()
    keep = keep and torch.is_grad_enabled()
    y = run_function(_LayerNorm, rows, None if weight is None else weight.contiguous(),
                     None if bias is None else bias.contiguous(), float(eps), keep, graph=keep)
    return y if x.dim() == 2 else y.view(x.shape)
