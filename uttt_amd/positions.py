"""Rotary embedding over several position axes (view, row and column of image
tokens; time, row and column of video), forward and backward.  One scalar
position per token, from tables, is uttt_amd.moe.Rope.  No CPU path."""
from __future__ import annotations

import ctypes
import functools
from typing import List, Sequence

import torch
from torch import Tensor

from . import _lib as L
from ._ops import new_like, run_function, traced_op

MAX_AXES = 8


def axis_frequencies(sections: Sequence[int], base: float = 10000.0, *, per_axis: bool = False,
                     device=None) -> Tensor:
    """The fp32 frequencies of sum(sections) pairs: base^(-j / R), over all pairs
    in one falling row that the axes share out (R = sum(sections)), or with
    `per_axis` a whole row for each axis (R = its section)."""
    rows = [(j, m) for m in sections for j in range(m)] if per_axis else [
        (j, sum(sections)) for j in range(sum(sections))]
    return torch.tensor([float(base) ** (-j / m) for j, m in rows], dtype=torch.float32, device=device)


@functools.lru_cache(maxsize=256)
def _host(ctype, *values):
    """Host integers as the C ABI takes them (read during a call, never written)."""
    return (ctype * len(values))(*values)


def _turn_fake(x, positions, inv_freq, sections, interleaved, inverse):
    return new_like(x)


@traced_op("rotary_axes", _turn_fake)
def _turn(x: Tensor, positions: Tensor, inv_freq: Tensor, sections: List[int], interleaved: bool,
          inverse: bool) -> Tensor:
    B, Lx, H, D = x.shape
    if x.stride(3) != 1 and D > 1:
        x = x.contiguous()
    y = _turn_fake(x, positions, inv_freq, sections, interleaved, inverse)
    L.call_on(x, "uttt_rotary_axes", L.ptr(x), L.dtype_code(x.dtype),
              _host(ctypes.c_int64, *x.stride()[:3]), B, Lx, H, D, L.ptr(positions),
              int(positions.dtype == torch.int64), _host(ctypes.c_int64, *positions.stride()),
              L.ptr(inv_freq), _host(ctypes.c_int, *sections), len(sections),
              int(interleaved), int(inverse), L.ptr(y), L.stream_of(x))
    return y


class _RotaryAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, inv_freq, sections, interleaved, inverse):
        ctx.save_for_backward(positions, inv_freq)
        ctx.args = (sections, interleaved, inverse)
        return _turn(x, positions, inv_freq, sections, interleaved, inverse)

    @staticmethod
    def backward(ctx, dy):
        """The turn back, itself differentiable in dy."""
        positions, inv_freq = ctx.saved_tensors
        sections, interleaved, inverse = ctx.args
        turn = _RotaryAxes.apply if torch.is_grad_enabled() else _turn
        return turn(dy, positions, inv_freq, sections, interleaved, not inverse), None, None, None, None, None


def rotary_axes(x: Tensor, positions: Tensor, inv_freq: Tensor, sections: Sequence[int], *,
                interleaved: bool = False) -> Tensor:
    """x [B, L, H, D] turned by the positions of its tokens, in x's dtype (fp32,
    bf16 or fp16; rotated in fp32 and rounded once).

    positions   [B, L, A] or, the same for every batch row, [L, A] int32 or int64; any
                values, negative and far ones included (to the end of int64 angles keep fp32's precision).
    sections    the pairs of each of the A axes (up to 8), R = sum(sections) in all, 2R <= D:
                the first sections[0] pairs turn by the first axis' position, and so on.
    inv_freq    [R] fp32: pair j turns by position * inv_freq[j] (axis_frequencies); no gradient
                flows to it.
    interleaved pairs are features (2j, 2j + 1) instead of (j, j + R).

    Features from 2R on pass through.  Differentiable in x, any number of times.
    x may be a view with contiguous features (one of a fused projection's parts)."""
    what = "rotary_axes"
    L.require_device(x, positions, inv_freq)
    assert x.dim() == 4, f"{what}: x must be [B, L, H, D]"
    assert x.dtype in (torch.float32, torch.bfloat16, torch.float16), f"{what}: dtype {x.dtype}"
    B, Lx, H, D = x.shape
    sections = [int(s) for s in sections]
    A, R = len(sections), sum(sections)
    assert 1 <= A <= MAX_AXES and min(sections) >= 0, f"{what}: 1 to {MAX_AXES} sections of 0 or more pairs"
    assert 1 <= R and 2 * R <= D, f"{what}: {R} pairs do not fit {D} features"
    assert positions.dtype in (torch.int32, torch.int64), f"{what}: positions must be int32 or int64"
    assert positions.shape == (B, Lx, A) or positions.shape == (Lx, A), (
        f"{what}: positions must be [{B}, {Lx}, {A}] or [{Lx}, {A}], got {tuple(positions.shape)}")
    assert inv_freq.shape == (R,) and inv_freq.dtype == torch.float32, (
        f"{what}: inv_freq must be [{R}] fp32")
    assert not (inv_freq.requires_grad and torch.is_grad_enabled()), (
        f"{what}: no gradient flows to inv_freq; detach it")
    assert positions.get_device() == inv_freq.get_device() == x.get_device(), f"{what}: tensors on several devices"
    if positions.dim() == 2:
        positions = positions.expand(B, Lx, A)
    return run_function(_RotaryAxes, x, positions, inv_freq.contiguous(), sections, bool(interleaved),
                        False, graph=x.requires_grad)
