"""The state space memory layer: a short causal convolution per channel and the
selective scan, over whole sequences (training, prefill) and token by token
against states kept in place (generation).

The scan's memory is a state h [N] per channel, written by the token's B and read
by its C, with a step dt that the token chooses:

  h_t = e^{dt_t A} h_{t-1} + dt_t x_t B_t,   y_t = C_t . h_t + D x_t

The reference ships models of this layer beside uTTT
(uttt_llm/flame/custom_models/mamba2_swa/) on kernels that are not uTTT's own,
with decays shared by a head, which are an A with equal entries here, and more
states than the 64 that are taken here in their usual size; the convolution also
stands before its gated delta layers.

`causal_conv` and `selective_scan` are differentiable once in all their tensors
(gradients of their gradients are refused).  There is no CPU path.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import _lib as L
from ._ops import (first_order_only, new_like, no_gradient, none_if_empty, run_function, strides_of,
                   traced_op)

MAX_STATES = 64
MAX_CHANNELS = 1 << 24
MIN_WIDTH, MAX_WIDTH = 2, 8
TILE = 16   # tokens between the states that a backward keeps

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_ACTIVATIONS = {None: 0, "silu": 1}


def _inner(t: Optional[Tensor]) -> Optional[Tensor]:
    """t itself where its last axis is contiguous and its tokens are not too far
    apart (a tile's offsets are 32 bits), else a copy."""
    if t is None or ((t.stride(-1) == 1 or t.shape[-1] == 1) and (t.stride(1) < 1 << 24 or t.shape[1] == 1)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _on16(t: Optional[Tensor]) -> Optional[Tensor]:
    """A contiguous t that starts on 16 bytes, t itself where it does."""
    if t is None or (t.is_contiguous() and not t.data_ptr() % 16):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _seqs(x, cu_seqlens):
    return x.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1


def _is64(t: Optional[Tensor]) -> int:
    return int(t is not None and t.dtype == torch.int64)


def _check_sequences(what, x, cu_seqlens):
    assert x.shape[0] >= 1, f"{what}: an empty batch"
    assert x.shape[0] * x.shape[1] < 1 << 30, f"{what}: {x.shape[0] * x.shape[1]} tokens, fewer than 2^30 are taken"
    if cu_seqlens is None:
        return None
    assert x.shape[0] == 1, f"{what}: packed sequences have a batch of 1, got {x.shape[0]}"
    assert cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 2, f"{what}: cu_seqlens must be [N + 1]"
    assert cu_seqlens.dtype in (torch.int32, torch.int64), f"{what}: cu_seqlens must be int32 or int64"
    assert cu_seqlens.device == x.device, f"{what}: cu_seqlens is on {cu_seqlens.device}"
    return cu_seqlens.contiguous()


def _check_slots(what, B, state, shape, dtype, device, state_indices):
    """Checks of a step's states; the indices as the C ABI takes them."""
    assert state.dim() == 3 and state.shape[1:] == shape, (
        f"{what}: state must be [slots, {shape[0]}, {shape[1]}], got {tuple(state.shape)}")
    assert state.dtype == dtype and state.device == device, f"{what}: state must be {dtype} on {device}"
    size = shape[0] * shape[1]
    inner = [s for s, n in zip(state.stride()[1:], shape) if n > 1]
    assert size == 0 or (inner == [s for s, n in zip((shape[1], 1), shape) if n > 1]
                         and (state.shape[0] <= 1 or state.stride(0) >= size)), (
        f"{what}: each slot's state must be contiguous and apart from the others")
    if state_indices is None:
        assert B <= state.shape[0], f"{what}: {B} rows, {state.shape[0]} states"
        return None
    assert state_indices.shape == (B,), f"{what}: state_indices must be [{B}]"
    assert state_indices.dtype in (torch.int32, torch.int64), f"{what}: state_indices must be int32 or int64"
    assert state_indices.device == device, f"{what}: state_indices is on {state_indices.device}"
    return state_indices.contiguous()


def _apart(state):
    """Elements between slots; of one slot its stride says nothing."""
    return state.stride(0) if state.shape[0] > 1 else state.shape[1] * state.shape[2]


# ------------------------------------------------------------- convolution --
def _code(t: Optional[Tensor]) -> int:
    return L.F32 if t is None else L.dtype_code(t.dtype)


def _conv_state(x, weight, cu_seqlens, wanted):
    return x.new_empty((_seqs(x, cu_seqlens), weight.shape[1] - 1, x.shape[2]) if wanted else (0,))


def _conv_fwd_fake(x, weight, bias, silu, initial_state, cu_seqlens, want_state):
    return new_like(x), _conv_state(x, weight, cu_seqlens, want_state)


@traced_op("causal_conv_fwd", _conv_fwd_fake)
def _conv_fwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], silu: bool, initial_state: Optional[Tensor],
              cu_seqlens: Optional[Tensor], want_state: bool) -> Tuple[Tensor, Tensor]:
    """(y, the inputs that the next tokens need, empty where not wanted)."""
    y, state = _conv_fwd_fake(x, weight, bias, silu, initial_state, cu_seqlens, want_state)
    B, T, D = x.shape
    x, weight, bias = _inner(x), weight.contiguous(), None if bias is None else bias.contiguous()
    h0 = None if initial_state is None else initial_state.contiguous()
    L.call_on(x, "uttt_causal_conv_fwd", L.ptr(x), strides_of(x, 2), _code(x), L.ptr(weight), _code(weight),
              L.ptr(bias), _code(bias), int(silu), L.ptr(h0), L.ptr(cu_seqlens), _is64(cu_seqlens), B, T,
              _seqs(x, cu_seqlens), D, weight.shape[1], L.ptr(y), L.ptr(state) if want_state else None,
              L.stream_of(x))
    return y, state


def _conv_bwd_fake(x, weight, bias, silu, initial_state, cu_seqlens, dy, dstate, want_dw, want_db, want_dh0):
    none = x.new_empty((0,))
    return [new_like(x), torch.empty_like(weight, memory_format=torch.contiguous_format) if want_dw else none,
            new_like(bias) if want_db else x.new_empty((0,)),
            _conv_state(x, weight, cu_seqlens, want_dh0)]


@traced_op("causal_conv_bwd", _conv_bwd_fake)
def _conv_bwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], silu: bool, initial_state: Optional[Tensor],
              cu_seqlens: Optional[Tensor], dy: Tensor, dstate: Optional[Tensor], want_dw: bool, want_db: bool,
              want_dh0: bool) -> List[Tensor]:
    grads = _conv_bwd_fake(x, weight, bias, silu, initial_state, cu_seqlens, dy, dstate, want_dw, want_db, want_dh0)
    B, T, D = x.shape
    n, W = _seqs(x, cu_seqlens), weight.shape[1]
    x, dy = _inner(x), _inner(dy)
    weight, bias = weight.contiguous(), None if bias is None else bias.contiguous()
    h0 = None if initial_state is None else initial_state.contiguous()
    dstate = None if dstate is None else dstate.contiguous()
    size = (L.lib().uttt_causal_conv_bwd_workspace_bytes(B, T, n, int(cu_seqlens is not None), D, W)
            if want_dw or want_db else 0)
    ws = torch.empty(size, dtype=torch.uint8, device=x.device)
    dx, dw, db, dh0 = grads
    L.call_on(x, "uttt_causal_conv_bwd", L.ptr(x), strides_of(x, 2), _code(x), L.ptr(weight), _code(weight),
              L.ptr(bias), _code(bias), int(silu), L.ptr(h0), L.ptr(cu_seqlens), _is64(cu_seqlens), B, T, n, D, W,
              L.ptr(dy), strides_of(dy, 2), L.ptr(dstate), L.ptr(dx), L.ptr(dw) if want_dw else None,
              L.ptr(db) if want_db else None, L.ptr(dh0) if want_dh0 else None, L.ptr(ws), size, L.stream_of(x))
    return grads


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, silu, initial_state, cu_seqlens, want_state):
        ctx.save_for_backward(x, weight, bias, initial_state, cu_seqlens)
        ctx.silu = silu
        return _conv_fwd(x, weight, bias, silu, initial_state, cu_seqlens, want_state)

    @staticmethod
    def backward(ctx, dy, dstate):
        x, weight, bias, h0, cu = ctx.saved_tensors
        _, want_dw, want_db, _, want_dh0 = ctx.needs_input_grad[:5]
        dstate = none_if_empty(dstate)
        grads = _conv_bwd(x, weight, bias, ctx.silu, h0, cu, dy, dstate, want_dw, want_db, want_dh0)
        dx, dw, db, dh0 = first_order_only("causal_conv", grads, x, weight, bias, h0, dy, dstate)
        return dx, dw if want_dw else None, db if want_db else None, None, dh0 if want_dh0 else None, None, None


def _check_conv(what, x, weight, bias, activation):
    L.require_device(x, weight, bias)
    assert x.dim() == 3 and x.shape[2] >= 1, f"{what}: x must be [B, T, D]"
    assert x.dtype in _TYPES, f"{what}: dtype {x.dtype}"
    D = x.shape[2]
    assert weight.dim() == 2 and weight.shape[0] == D and MIN_WIDTH <= weight.shape[1] <= MAX_WIDTH, (
        f"{what}: weight must be [{D}, W] with W of {MIN_WIDTH} to {MAX_WIDTH}, got {tuple(weight.shape)}")
    assert bias is None or bias.shape == (D,), f"{what}: bias must be [{D}], got {tuple(bias.shape)}"
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            assert t.dtype in _TYPES, f"{what}: {name} has dtype {t.dtype}"
            assert t.device == x.device, f"{what}: {name} is on {t.device}, x on {x.device}"
    assert activation in _ACTIVATIONS, f"{what}: activation must be None or 'silu', got {activation!r}"
    return (weight.shape[1] - 1, D)


def causal_conv(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, activation: str | None = None,
                initial_state: Tensor | None = None, output_final_state: bool = False,
                cu_seqlens: Tensor | None = None):
    """A causal convolution of each channel with its own short kernel: y_t =
    act(bias + sum_k weight[:, k] x_{t-W+1+k}).  Returns (y [B, T, D] in x's dtype,
    the last W - 1 inputs of each sequence [N, W - 1, D] or None).

    x              [B, T, D] in fp32, bf16 or fp16; a view whose channels are contiguous will do,
                   others are copied.
    weight, bias   [D, W] with W of 2 to 8, the last column for the token itself, and [D] or
                   None, each in any of the three types.
    activation     None or "silu".
    initial_state  [N, W - 1, D] in x's dtype, the inputs before a sequence's first, the oldest
                   first; zeros if None.  N = B, or the packed sequences.
    cu_seqlens     [N + 1] int32 or int64 on the GPU: B is 1 and sequence n is the tokens
                   cu_seqlens[n] to cu_seqlens[n + 1], none at all allowed.  Offsets must
                   ascend; tokens of no sequence get zeros as outputs and gradients.

    Products and sums are fp32, each result rounded once to its type; gradients of weight and
    bias are summed in an order that the sizes and the 16-byte alignment of rows decide.
    Tokens of no sequence are cleared by few threads: a buffer that is mostly padding takes
    longer than a full one.
    Differentiable once in x, weight, bias and initial_state."""
    what = "causal_conv"
    shape = _check_conv(what, x, weight, bias, activation)
    cu_seqlens = _check_sequences(what, x, cu_seqlens)
    if initial_state is not None:
        shape = (_seqs(x, cu_seqlens), *shape)
        assert initial_state.shape == shape, f"{what}: initial_state must be {shape}"
        assert initial_state.dtype == x.dtype and initial_state.device == x.device, (
            f"{what}: initial_state must be {x.dtype} on {x.device}")
    graph = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, weight, bias, initial_state))
    y, state = run_function(_CausalConv, x, weight, bias, activation == "silu", initial_state, cu_seqlens,
                            bool(output_final_state), graph=graph)
    return y, state if output_final_state else None


def _conv_step_fake(x, weight, bias, silu, state, state_indices):
    return new_like(x)


@traced_op("causal_conv_step", _conv_step_fake, mutates_args=("state",))
def _conv_step(x: Tensor, weight: Tensor, bias: Optional[Tensor], silu: bool, state: Tensor,
               state_indices: Optional[Tensor]) -> Tensor:
    y = new_like(x)
    B, T, D = x.shape
    x, weight, bias = _inner(x), weight.contiguous(), None if bias is None else bias.contiguous()
    L.call_on(x, "uttt_causal_conv_step", L.ptr(x), strides_of(x, 2), _code(x), L.ptr(weight), _code(weight),
              L.ptr(bias), _code(bias), int(silu), B, T, D, weight.shape[1], L.ptr(state), _apart(state),
              state.shape[0], L.ptr(state_indices), _is64(state_indices), L.ptr(y), L.stream_of(x))
    return y


def causal_conv_step(x: Tensor, weight: Tensor, state: Tensor, bias: Tensor | None = None, *,
                     activation: str | None = None, state_indices: Tensor | None = None) -> Tensor:
    """A few tokens per sequence (generation): y [B, T, D], and `state` holds the last W - 1
    inputs afterwards.

    x, weight, bias, activation as in causal_conv; T is 1 for plain generation, the tokens of a
    row follow one another.
    state          [slots, W - 1, D] in x's dtype, its last two axes contiguous (a layer's slice
                   of a pool that holds all layers will do).
    state_indices  [B] int32 or int64, the slot of each row; row b's is b if None.  A row whose
                   index is no slot (-1: padding) leaves every state alone and gets zeros.  Rows
                   that name one slot follow one another in row order.

    No gradient flows through it, backward or forward: tensors that have one are refused."""
    what = "causal_conv_step"
    shape = _check_conv(what, x, weight, bias, activation)
    L.require_device(state)
    state_indices = _check_slots(what, x.shape[0], state, shape, x.dtype, x.device, state_indices)
    no_gradient(what, x, weight, bias, state)
    return _conv_step(x, weight, bias, activation == "silu", state, state_indices)


# -------------------------------------------------------------------- scan --
def _launch_scan(x, dt, A, B, C, D, gate, dt_bias, softplus, initial_state, cu_seqlens, y, state, tiles):
    n, T, Dm = x.shape
    seqs, N, G = _seqs(x, cu_seqlens), A.shape[1], B.shape[2]
    x, dt, B, C, gate = _inner(x), _inner(dt), _inner(B), _inner(C), _inner(gate)
    A, initial_state = _on16(A), _on16(initial_state)
    D, dt_bias = None if D is None else D.contiguous(), None if dt_bias is None else dt_bias.contiguous()
    size = L.lib().uttt_selective_scan_fwd_workspace_bytes(n, T, seqs, int(cu_seqlens is not None), Dm, N, G)
    ws = torch.empty(size, dtype=torch.uint8, device=x.device)
    L.call_on(x, "uttt_selective_scan_fwd", L.ptr(x), strides_of(x, 2), _code(x), L.ptr(dt), strides_of(dt, 2),
              _code(dt), L.ptr(A), L.ptr(B), strides_of(B, 3), L.ptr(C), strides_of(C, 3), L.ptr(D), L.ptr(gate),
              None if gate is None else strides_of(gate, 2), L.ptr(dt_bias), int(softplus), L.ptr(initial_state),
              L.ptr(cu_seqlens), _is64(cu_seqlens), n, T, seqs, Dm, N, G, L.ptr(y), L.ptr(state), L.ptr(tiles),
              L.ptr(ws), size, L.stream_of(x))


def _scan_state(x, A, cu_seqlens, wanted):
    return x.new_empty((_seqs(x, cu_seqlens), *A.shape) if wanted else (0,), dtype=torch.float32)


def _scan_infer_fake(x, dt, A, B, C, D, gate, dt_bias, softplus, initial_state, cu_seqlens, want_state):
    return new_like(x), _scan_state(x, A, cu_seqlens, want_state)


@traced_op("selective_scan_infer", _scan_infer_fake)
def _scan_infer(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], gate: Optional[Tensor],
                dt_bias: Optional[Tensor], softplus: bool, initial_state: Optional[Tensor],
                cu_seqlens: Optional[Tensor], want_state: bool) -> Tuple[Tensor, Tensor]:
    """(y, final states, empty where not wanted)."""
    y, state = _scan_infer_fake(x, dt, A, B, C, D, gate, dt_bias, softplus, initial_state, cu_seqlens, want_state)
    _launch_scan(x, dt, A, B, C, D, gate, dt_bias, softplus, initial_state, cu_seqlens, y,
                 state if want_state else None, None)
    return y, state


def _kept_states(N):
    """N up to the next power of two of 4 or more, as the kernels keep states."""
    return 4 if N <= 4 else 8 if N <= 8 else 16 if N <= 16 else 32 if N <= 32 else 64


def _scan_fwd_fake(x, dt, A, B, C, D, gate, dt_bias, softplus, initial_state, cu_seqlens, want_state):
    n, T = x.shape[:2]
    tiles = T // TILE + _seqs(x, cu_seqlens) if cu_seqlens is not None else n * max(1, (T + TILE - 1) // TILE)
    return (*_scan_infer_fake(x, dt, A, B, C, D, gate, dt_bias, softplus, initial_state, cu_seqlens, want_state),
            x.new_empty((tiles, _kept_states(A.shape[1]), A.shape[0]), dtype=torch.float32))


@traced_op("selective_scan_fwd", _scan_fwd_fake)
def _scan_fwd(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], gate: Optional[Tensor],
              dt_bias: Optional[Tensor], softplus: bool, initial_state: Optional[Tensor],
              cu_seqlens: Optional[Tensor], want_state: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """_scan_infer, and the states at every 16th token, which the backward starts from."""
    y, state, tiles = _scan_fwd_fake(x, dt, A, B, C, D, gate, dt_bias, softplus, initial_state, cu_seqlens, want_state)
    _launch_scan(x, dt, A, B, C, D, gate, dt_bias, softplus, initial_state, cu_seqlens, y,
                 state if want_state else None, tiles)
    return y, state, tiles


def _scan_bwd_fake(x, dt, A, B, C, D, gate, dt_bias, softplus, cu_seqlens, tiles, dy, dstate, want_dh0):
    def like(t):
        return x.new_empty((0,)) if t is None else new_like(t)

    return [new_like(x), new_like(dt), new_like(A), new_like(B), new_like(C), like(D), like(gate), like(dt_bias),
            _scan_state(x, A, cu_seqlens, want_dh0)]


@traced_op("selective_scan_bwd", _scan_bwd_fake)
def _scan_bwd(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], gate: Optional[Tensor],
              dt_bias: Optional[Tensor], softplus: bool, cu_seqlens: Optional[Tensor], tiles: Tensor, dy: Tensor,
              dstate: Optional[Tensor], want_dh0: bool) -> List[Tensor]:
    grads = _scan_bwd_fake(x, dt, A, B, C, D, gate, dt_bias, softplus, cu_seqlens, tiles, dy, dstate, want_dh0)
    n, T, Dm = x.shape
    seqs, N, G = _seqs(x, cu_seqlens), A.shape[1], B.shape[2]
    x, dt, B, C, gate, dy = _inner(x), _inner(dt), _inner(B), _inner(C), _inner(gate), _inner(dy)
    A, dstate = _on16(A), _on16(dstate)
    D, dt_bias = None if D is None else D.contiguous(), None if dt_bias is None else dt_bias.contiguous()
    dx, ddt, dA, dB, dC, dD, dgate, dbias, dh0 = grads
    size = L.lib().uttt_selective_scan_bwd_workspace_bytes(n, T, seqs, int(cu_seqlens is not None), Dm, N, G)
    ws = torch.empty(size, dtype=torch.uint8, device=x.device)
    L.call_on(x, "uttt_selective_scan_bwd", L.ptr(x), strides_of(x, 2), _code(x), L.ptr(dt), strides_of(dt, 2),
              _code(dt), L.ptr(A), L.ptr(B), strides_of(B, 3), L.ptr(C), strides_of(C, 3), L.ptr(D), L.ptr(gate),
              None if gate is None else strides_of(gate, 2), L.ptr(dt_bias), int(softplus), L.ptr(cu_seqlens),
              _is64(cu_seqlens), n, T, seqs, Dm, N, G, L.ptr(tiles), L.ptr(dy), strides_of(dy, 2), L.ptr(dstate),
              L.ptr(dx), L.ptr(ddt), L.ptr(dA), L.ptr(dB), L.ptr(dC), None if D is None else L.ptr(dD),
              None if gate is None else L.ptr(dgate), None if dt_bias is None else L.ptr(dbias),
              L.ptr(dh0) if want_dh0 else None, L.ptr(ws), size, L.stream_of(x))
    return grads


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, gate, dt_bias, softplus, initial_state, cu_seqlens, want_state, keep):
        args = (x, dt, A, B, C, D, gate, dt_bias, softplus, initial_state, cu_seqlens, want_state)
        if not keep:
            return _scan_infer(*args)
        y, state, tiles = _scan_fwd(*args)
        ctx.save_for_backward(x, dt, A, B, C, D, gate, dt_bias, cu_seqlens, tiles)
        ctx.softplus = softplus
        # its values are not needed again (no saved tensor, which must not change)
        ctx.h0 = initial_state if initial_state is not None and initial_state.requires_grad else None
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    def backward(ctx, dy, dstate):
        x, dt, A, B, C, D, gate, dt_bias, cu, tiles = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(x)
        dstate, want_dh0 = none_if_empty(dstate), ctx.h0 is not None
        grads = _scan_bwd(x, dt, A, B, C, D, gate, dt_bias, ctx.softplus, cu, tiles, dy, dstate, want_dh0)
        grads = list(first_order_only("selective_scan", grads, x, dt, A, B, C, D, gate, dt_bias, ctx.h0, dy, dstate))
        given = (x, dt, A, B, C, D, gate, dt_bias)
        grads[:8] = [None if t is None else g for t, g in zip(given, grads)]
        return (*grads[:8], None, grads[8] if want_dh0 else None, None, None, None)


def _check_scan(what, x, dt, A, B, C, D, gate, dt_bias):
    L.require_device(x, dt, A, B, C, D, gate, dt_bias)
    assert x.dim() == 3 and x.shape[2] >= 1, f"{what}: x must be [B, T, D]"
    assert x.dtype in _TYPES, f"{what}: dtype {x.dtype}"
    n, T, Dm = x.shape
    assert dt.shape == x.shape, f"{what}: dt {tuple(dt.shape)} must have x's shape {tuple(x.shape)}"
    assert dt.dtype in (torch.float32, x.dtype), f"{what}: dt must be fp32 or of x's dtype {x.dtype}, got {dt.dtype}"
    assert Dm <= MAX_CHANNELS, f"{what}: {Dm} channels, at most {MAX_CHANNELS} are taken"
    assert A.dim() == 2 and A.shape[0] == Dm and 1 <= A.shape[1] <= MAX_STATES, (
        f"{what}: A must be [{Dm}, N] with N of 1 to {MAX_STATES}, got {tuple(A.shape)}")
    assert B.dim() == 4 and B.shape[:2] == (n, T) and B.shape[3] == A.shape[1], (
        f"{what}: B must be [{n}, {T}, G, {A.shape[1]}], got {tuple(B.shape)}")
    assert C.shape == B.shape, f"{what}: C {tuple(C.shape)} must have B's shape {tuple(B.shape)}"
    assert B.shape[2] >= 1 and Dm % B.shape[2] == 0, f"{what}: {Dm} channels must be a multiple of {B.shape[2]} groups"
    assert gate is None or gate.shape == x.shape, f"{what}: gate must have x's shape {tuple(x.shape)}"
    dtype, dev = x.dtype, x.get_device()
    for name, t in (("B", B), ("C", C), ("gate", gate)):
        assert t is None or t.dtype is dtype, f"{what}: {name} must have x's dtype {dtype}, got {t.dtype}"
    for name, t in (("D", D), ("dt_bias", dt_bias)):
        assert t is None or t.shape == (Dm,), f"{what}: {name} must be [{Dm}], got {tuple(t.shape)}"
    for name, t in (("A", A), ("D", D), ("dt_bias", dt_bias)):
        assert t is None or t.dtype is torch.float32, f"{what}: {name} must be fp32, got {t.dtype}"
    for name, t in (("dt", dt), ("A", A), ("B", B), ("C", C), ("D", D), ("gate", gate), ("dt_bias", dt_bias)):
        assert t is None or t.get_device() == dev, f"{what}: {name} is on {t.device}, x on {x.device}"


def selective_scan(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, *, D: Tensor | None = None,
                   gate: Tensor | None = None, dt_bias: Tensor | None = None, dt_softplus: bool = False,
                   initial_state: Tensor | None = None, output_final_state: bool = False,
                   cu_seqlens: Tensor | None = None):
    """The selective scan over whole sequences.  Returns (y [B, T, D] in x's dtype,
    final states [N_seqs, D, N] fp32 or None).

    x              [B, T, D] in fp32, bf16 or fp16; fewer than 2^30 tokens in all.
    dt             [B, T, D] steps in fp32 or x's dtype, to which dt_bias [D] is added and, with
                   dt_softplus, ln(1 + e^x) applied.
    A              [D, N] fp32, N up to 64: the states' rates, below zero where they decay.
    B, C           [B, T, G, N] in x's dtype; channels D / G * g onwards read group g.
    D              [D] fp32 or None, what of x goes past the states.
    gate           [B, T, D] in x's dtype or None: outputs are multiplied by silu(gate).
    initial_state  [N_seqs, D, N] fp32, zeros if None; N_seqs = B, or the packed sequences.
    cu_seqlens     [N_seqs + 1] int32 or int64 on the GPU: B is 1 and sequence n is the tokens
                   cu_seqlens[n] to cu_seqlens[n + 1], none at all allowed.  Offsets must
                   ascend; tokens of no sequence get zeros as outputs and gradients.

    x, dt, B, C and gate may be views whose last axis is contiguous (slices of one projection);
    others are copied.  All of it is computed in fp32, each result rounded once to its type;
    every sum has an order that the sizes decide.  A value that is not finite reaches the
    results of its token and later ones of its sequence (of x, dt and gate: in its channel), as
    in the recurrence, and no others.  An A of -inf counts as fp32's lowest value.  States may
    grow (dt A above zero): what is in fp32's range at every token stays right and zeros stay
    zero, but e^{dt A} of a single token is infinite past e^88, as in fp32.
    Differentiable once in all tensors; the backward keeps the states at every 16th token: N up
    to the next power of two of 4 or more, by 4 bytes, for each channel and 16 tokens (at 16
    states 4 bytes an element of x), and of a packed sequence once more at most.  Tokens of no
    sequence are cleared by few threads: a buffer that is mostly padding takes longer than a
    full one."""
    what = "selective_scan"
    _check_scan(what, x, dt, A, B, C, D, gate, dt_bias)
    cu_seqlens = _check_sequences(what, x, cu_seqlens)
    if initial_state is not None:
        shape = (_seqs(x, cu_seqlens), *A.shape)
        assert initial_state.shape == shape, f"{what}: initial_state must be {shape}"
        assert initial_state.dtype == torch.float32 and initial_state.device == x.device, (
            f"{what}: initial_state must be fp32 on {x.device}")
    keep = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, dt, A, B, C, D, gate, dt_bias, initial_state))
    y, state = run_function(_SelectiveScan, x, dt, A, B, C, D, gate, dt_bias, bool(dt_softplus), initial_state,
                            cu_seqlens, bool(output_final_state), keep, graph=keep)
    return y, state if output_final_state else None


def _scan_step_fake(x, dt, A, B, C, D, gate, dt_bias, softplus, state, state_indices):
    return new_like(x)


@traced_op("selective_scan_step", _scan_step_fake, mutates_args=("state",))
def _scan_step(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], gate: Optional[Tensor],
               dt_bias: Optional[Tensor], softplus: bool, state: Tensor, state_indices: Optional[Tensor]) -> Tensor:
    y = new_like(x)
    n, T, Dm = x.shape
    x, dt, B, C, gate = _inner(x), _inner(dt), _inner(B), _inner(C), _inner(gate)
    A = _on16(A)
    D, dt_bias = None if D is None else D.contiguous(), None if dt_bias is None else dt_bias.contiguous()
    L.call_on(x, "uttt_selective_scan_step", L.ptr(x), strides_of(x, 2), _code(x), L.ptr(dt), strides_of(dt, 2),
              _code(dt), L.ptr(A), L.ptr(B), strides_of(B, 3), L.ptr(C), strides_of(C, 3), L.ptr(D), L.ptr(gate),
              None if gate is None else strides_of(gate, 2), L.ptr(dt_bias), int(softplus), n, T, Dm, A.shape[1],
              B.shape[2], L.ptr(state), _apart(state), state.shape[0], L.ptr(state_indices), _is64(state_indices),
              L.ptr(y), L.stream_of(x))
    return y


def selective_scan_step(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, *,
                        D: Tensor | None = None, gate: Tensor | None = None, dt_bias: Tensor | None = None,
                        dt_softplus: bool = False, state_indices: Tensor | None = None) -> Tensor:
    """A few tokens per sequence against states in place (generation): y [B, T, D] in x's
    dtype, and `state` is as after the last token.

    x to C, D, gate, dt_bias and dt_softplus as in selective_scan; T is 1 for plain generation,
    the tokens of a row follow one another.
    state          [slots, D, N] fp32, its last two axes contiguous (a layer's slice of a pool
                   that holds all layers will do); where N is a multiple of 4, slots on 16 bytes.
    state_indices  [B] int32 or int64, the slot of each row; row b's is b if None.  A row whose
                   index is no slot (-1: padding) leaves every state alone and gets zeros.  Rows
                   that name one slot follow one another in row order.

    No gradient flows through it, backward or forward: tensors that have one are refused."""
    what = "selective_scan_step"
    _check_scan(what, x, dt, A, B, C, D, gate, dt_bias)
    L.require_device(state)
    state_indices = _check_slots(what, x.shape[0], state, tuple(A.shape), torch.float32, x.device, state_indices)
    no_gradient(what, x, dt, A, B, C, D, gate, dt_bias, state)
    return _scan_step(x, dt, A, B, C, D, gate, dt_bias, bool(dt_softplus), state, state_indices)
