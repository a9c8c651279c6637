"""Layer norm with weight and bias over the last axis, and the RMS norms before
and after a block with the residual sum, gate and scale that stand next to them,
forward and backward (the parameter-free norms of the fast-weight inputs are
uttt_amd.moe.rows_preprocess).  No CPU path."""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import _lib as L
from ._ops import evenly, first_order_only, new_like, none_if_empty, run_function, strides_of, traced_op

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


# ------------------------------------------------- the norms around a block --
MAX_BLOCK_ROW = 8192


def _grouped(t: Tensor):
    """t as [groups, rows of a group, N] with contiguous rows, a view wherever it can
    be: groups of the second to last axis."""
    N = t.shape[-1]
    if t.stride(-1) != 1 and N > 1:
        t = t.contiguous()
    return t.reshape(-1, t.shape[-2] if t.dim() > 2 else 1, N)


def _block_args(x: Tensor, *others: Optional[Tensor]):
    """([(tensor, its row strides), ...] of x and the others, rows, rows of a group)."""
    N, tensors = x.shape[-1], (x, *others)
    if x.numel() == 0 or all(t is None or t.is_contiguous() for t in tensors):
        return [(t, evenly(N)) for t in tensors], x.numel() // N, 1
    tensors = [None if t is None else _grouped(t) for t in tensors]
    return [(t, None if t is None else strides_of(t, 2)) for t in tensors], x.numel() // N, tensors[0].shape[1]


def _rstd(x):
    return x.new_empty((x.numel() // x.shape[-1],), dtype=torch.float32)


def _after_fake(x, weight, gate, residual, scale, alpha, eps, keep):
    return new_like(x if residual is None else residual), _rstd(x) if keep else x.new_empty((0,), dtype=torch.float32)


@traced_op("norm_after_fwd", _after_fake)
def _after_fwd(x: Tensor, weight: Optional[Tensor], gate: Optional[Tensor], residual: Optional[Tensor],
               scale: Optional[Tensor], alpha: float, eps: float, keep: bool) -> Tuple[Tensor, Tensor]:
    """(y, 1 / rms of each row for the backward, empty where nobody keeps it)."""
    y, rstd = _after_fake(x, weight, gate, residual, scale, alpha, eps, keep)
    ((x, xs), (gate, gs), (residual, rs)), rows, heads = _block_args(x, gate, residual)
    L.call_on(x, "uttt_norm_after_fwd", L.ptr(x), xs, _code(x), L.ptr(weight), _code(weight), L.ptr(gate),
              gs, L.ptr(residual), rs, _code(y), L.ptr(scale), _code(scale), alpha, rows,
              heads, x.shape[-1], eps, L.ptr(y), L.ptr(rstd) if keep else None, L.stream_of(x))
    return y, rstd


def _sums_like(x, weight, scale, want_dw, want_ds):
    return (new_like(weight) if want_dw else x.new_empty((0,)), new_like(scale) if want_ds else x.new_empty((0,)))


def _sums_workspace(x, rows, wanted):
    size = L.lib().uttt_norm_bwd_workspace_bytes(rows, x.shape[-1]) if wanted else 0
    return torch.empty(size, dtype=torch.uint8, device=x.device), size


def _after_bwd_fake(x, weight, gate, scale, alpha, rstd, dy, want_dw, want_ds):
    return [new_like(x), x.new_empty((0,)) if gate is None else new_like(gate),
            *_sums_like(x, weight, scale, want_dw, want_ds)]


@traced_op("norm_after_bwd", _after_bwd_fake)
def _after_bwd(x: Tensor, weight: Optional[Tensor], gate: Optional[Tensor], scale: Optional[Tensor], alpha: float,
               rstd: Tensor, dy: Tensor, want_dw: bool, want_ds: bool) -> List[Tensor]:
    grads = _after_bwd_fake(x, weight, gate, scale, alpha, rstd, dy, want_dw, want_ds)
    dx, dgate, dw, ds = grads
    ((x, xs), (gate, gs), (dy, ys)), rows, heads = _block_args(x, gate, dy)
    ws, size = _sums_workspace(x, rows, want_dw or want_ds)
    L.call_on(x, "uttt_norm_after_bwd", L.ptr(x), xs, _code(x), L.ptr(weight), _code(weight), L.ptr(gate),
              gs, L.ptr(scale), _code(scale), alpha, rows, heads, x.shape[-1], L.ptr(rstd), L.ptr(dy),
              ys, _code(dy), L.ptr(dx), None if gate is None else L.ptr(dgate), L.ptr(dw) if want_dw else None,
              L.ptr(ds) if want_ds else None, L.ptr(ws), size, L.stream_of(x))
    return grads


class _NormAfter(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, gate, residual, scale, alpha, eps, keep):
        y, rstd = _after_fwd(x, weight, gate, residual, scale, alpha, eps, keep)
        ctx.save_for_backward(x, weight, gate, scale, rstd)
        ctx.alpha, ctx.residual = alpha, residual is not None
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, gate, scale, rstd = ctx.saved_tensors
        _, want_dw, _, want_dr, want_ds = ctx.needs_input_grad[:5]
        grads = _after_bwd(x, weight, gate, scale, ctx.alpha, rstd, dy, want_dw, want_ds)
        dx, dgate, dw, ds = first_order_only("norm_after_block", grads, x, weight, gate, scale, dy)
        return (dx, dw if want_dw else None, None if gate is None else dgate, dy if want_dr else None,
                ds if want_ds else None, None, None, None)


def _before_fake(x, residual, weight, scale, alpha, eps, keep):
    return new_like(x), new_like(residual), _rstd(x) if keep else x.new_empty((0,), dtype=torch.float32)


@traced_op("norm_before_fwd", _before_fake)
def _before_fwd(x: Tensor, residual: Tensor, weight: Optional[Tensor], scale: Optional[Tensor], alpha: float,
                eps: float, keep: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """(y, the sum, 1 / rms of each row for the backward, empty where nobody keeps it)."""
    y, total, rstd = _before_fake(x, residual, weight, scale, alpha, eps, keep)
    ((x, xs), (residual, rs)), rows, heads = _block_args(x, residual)
    L.call_on(x, "uttt_norm_before_fwd", L.ptr(x), xs, _code(x), L.ptr(residual), rs,
              _code(residual), L.ptr(weight), _code(weight), L.ptr(scale), _code(scale), alpha, rows, heads,
              x.shape[-1], eps, L.ptr(y), L.ptr(total), L.ptr(rstd) if keep else None, L.stream_of(x))
    return y, total, rstd


def _before_bwd_fake(x, residual, weight, scale, alpha, rstd, dy, dtotal, want_dw, want_ds):
    return [new_like(x), new_like(residual), *_sums_like(x, weight, scale, want_dw, want_ds)]


@traced_op("norm_before_bwd", _before_bwd_fake)
def _before_bwd(x: Tensor, residual: Tensor, weight: Optional[Tensor], scale: Optional[Tensor], alpha: float,
                rstd: Tensor, dy: Optional[Tensor], dtotal: Optional[Tensor], want_dw: bool,
                want_ds: bool) -> List[Tensor]:
    grads = _before_bwd_fake(x, residual, weight, scale, alpha, rstd, dy, dtotal, want_dw, want_ds)
    dx, dr, dw, ds = grads
    ((x, xs), (residual, rs), (dy, ys), (dtotal, ts)), rows, heads = _block_args(x, residual, dy, dtotal)
    ws, size = _sums_workspace(x, rows, want_dw or want_ds)
    L.call_on(x, "uttt_norm_before_bwd", L.ptr(x), xs, _code(x), L.ptr(residual), rs,
              _code(residual), L.ptr(weight), _code(weight), L.ptr(scale), _code(scale), alpha, rows, heads,
              x.shape[-1], L.ptr(rstd), L.ptr(dy), ys, L.ptr(dtotal), ts, L.ptr(dx), L.ptr(dr),
              L.ptr(dw) if want_dw else None, L.ptr(ds) if want_ds else None, L.ptr(ws), size, L.stream_of(x))
    return grads


class _NormBefore(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, scale, alpha, eps, keep):
        y, total, rstd = _before_fwd(x, residual, weight, scale, alpha, eps, keep)
        if not keep:
            return y, total
        ctx.save_for_backward(x, residual, weight, scale, rstd)
        ctx.alpha = alpha
        ctx.set_materialize_grads(False)
        return y, total

    @staticmethod
    def backward(ctx, dy, dtotal):
        x, residual, weight, scale, rstd = ctx.saved_tensors
        _, _, want_dw, want_ds = ctx.needs_input_grad[:4]
        grads = _before_bwd(x, residual, weight, scale, ctx.alpha, rstd, dy, dtotal, want_dw, want_ds)
        dx, dr, dw, ds = first_order_only("norm_before_block", grads, x, residual, weight, scale, dy, dtotal)
        return dx, dr, dw if want_dw else None, ds if want_ds else None, None, None, None


def _check_block(what, x, weight, scale, same):
    """Checks of the norms around a block; (weight, scale tensor, alpha) as the kernels take them."""
    alpha = 1.0
    if scale is not None and not isinstance(scale, Tensor):
        scale, alpha = None, float(scale)
    L.require_device(x, weight, scale, *(t for _, t in same))
    assert x.dim() >= 1 and 1 <= x.shape[-1] <= MAX_BLOCK_ROW, (
        f"{what}: x must be [..., N] with N of 1 to {MAX_BLOCK_ROW}, got {tuple(x.shape)}")
    assert x.dtype in _TYPES, f"{what}: dtype {x.dtype}"
    N = x.shape[-1]
    for name, t in same:
        if t is not None:
            assert t.shape == x.shape, f"{what}: {name} must have x's shape {tuple(x.shape)}, got {tuple(t.shape)}"
            assert t.dtype in _TYPES, f"{what}: {name} has dtype {t.dtype}"
    for name, t in (("weight", weight), ("scale", scale)):
        if t is not None:
            assert t.shape == (N,), f"{what}: {name} must be [{N}], got {tuple(t.shape)}"
            assert t.dtype in _TYPES, f"{what}: {name} has dtype {t.dtype}"
    for name, t in (*same, ("weight", weight), ("scale", scale)):
        assert t is None or t.device == x.device, f"{what}: {name} is on {t.device}, x on {x.device}"
    return None if weight is None else weight.contiguous(), None if scale is None else scale.contiguous(), alpha


def norm_after_block(x: Tensor, weight: Tensor | None = None, *, gate: Tensor | None = None,
                     residual: Tensor | None = None, scale: Tensor | float | None = None,
                     eps: float = 1e-5) -> Tensor:
    """residual + scale * (x / rms(x) * weight * silu(gate)) over the last axis, with rms(x) =
    sqrt(mean(x^2) + eps) and without what is None; in the residual's dtype, in x's without one.

    x [..., N] in fp32, bf16 or fp16, N up to 8192 (a head's width for a norm by heads); gate of
    x's shape and dtype, residual of x's shape in any of the three; weight [N] and scale, [N] or
    a number, in any of the three.  Computed in fp32 and rounded once; the gradients of weight
    and scale are summed over the rows in an order that the sizes and the 16-byte alignment of
    tensors and rows decide.  Views are taken where rows are contiguous and evenly spaced up to
    the second to last axis (heads of a slice of a projection), others are copied.
    Differentiable once in all tensors."""
    what = "norm_after_block"
    weight, scale, alpha = _check_block(what, x, weight, scale, (("gate", gate), ("residual", residual)))
    assert gate is None or gate.dtype is x.dtype, f"{what}: gate must have x's dtype {x.dtype}, got {gate.dtype}"
    keep = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, weight, gate, residual, scale))
    return run_function(_NormAfter, x, weight, gate, residual, scale, alpha, float(eps), keep, graph=keep)


def norm_before_block(x: Tensor, residual: Tensor, weight: Tensor | None = None, *,
                      scale: Tensor | float | None = None, eps: float = 1e-5) -> Tuple[Tensor, Tensor]:
    """The last block's outputs x into the residual stream and the next block's norm: total =
    residual + scale * x, y = total / rms(total) * weight over the last axis.  Returns (y in x's
    dtype, total in the residual's); y is made of the sum before it is rounded.  Arguments as in
    norm_after_block.  Differentiable once in all tensors."""
    what = "norm_before_block"
    weight, scale, alpha = _check_block(what, x, weight, scale, (("residual", residual),))
    keep = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, scale))
    return run_function(_NormBefore, x, residual, weight, scale, alpha, float(eps), keep, graph=keep)
