"""The gated delta rule: a linear fast-weight memory with forgetting, as a
chunked pass over whole sequences (training, prefill) and token by token
against states kept in place (generation).

Per value head, with a state S [Dk, Dv] that starts from `initial_state`:

  S_t = e^{g_t} S_{t-1} + k_t u_t^T
  u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t)
  o_t = scale S_t^T q_t

which is one step of gradient descent with rate beta_t on |S^T k_t - v_t|^2 / 2
after the old state has decayed by e^{g_t}.  The reference ships models of
this layer beside uTTT (uttt_llm/flame/custom_models/gated_deltanet_swa/,
uttt_nvs/models/gated_deltanet_block.py) and takes its kernels from a package
that is not part of it.

`gated_delta_rule` is differentiable once in q, k, v, g, beta and initial_state
(gradients of its gradients are refused).
There is no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
from typing import List, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib as L
from ._ops import first_order_only, new_like, run_function, traced_op

MAX_KEY_DIM = 256


@functools.lru_cache(maxsize=256)
def _int64s(*values):
    """Host integers as the C ABI takes them (read during a call, never written)."""
    return (ctypes.c_int64 * len(values))(*values)


def _steps(t: Tensor):
    """Element strides of [B, T, H, D]'s first three axes, 0 along an axis of one,
    whose stride says nothing."""
    (B, T, H, _), (sb, st, sh, _) = t.shape, t.stride()
    return sb if B > 1 else 0, st if T > 1 else 0, sh if H > 1 else 0


def _strides(t: Tensor):
    return _int64s(*_steps(t))


def _rows16(t: Tensor) -> Tensor:
    """t itself where its rows can be read 16 bytes at a time and a chunk's by
    31-bit offsets, else a copy (contiguous() gives back a t that is contiguous
    and starts at another address)."""
    sb, st, sh = _steps(t)
    if t.stride(3) == 1 and not (sb | st | sh) % 8 and st < 1 << 23 and not t.data_ptr() % 16:
        return t
    return t.clone(memory_format=torch.contiguous_format)


_GATE_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(q, k, v, g, beta, what):
    L.require_device(q, k, v, g, beta)
    assert q.get_device() == k.get_device() == v.get_device() == g.get_device() == beta.get_device(), (
        f"{what}: q, k, v, g and beta must be on one device")
    assert q.dim() == 4 and v.dim() == 4, (
        f"{what}: q and k must be [B, T, Hk, Dk], v [B, T, Hv, Dv]")
    B, T, Hk, Dk = shape = q.shape
    Bv, Tv, Hv, Dv = v.shape
    assert k.shape == shape, f"{what}: k {tuple(k.shape)} must have q's shape {tuple(q.shape)}"
    assert Bv == B and Tv == T, f"{what}: v {tuple(v.shape)} must have q's batch and tokens"
    assert Hk > 0 and Hv % Hk == 0, f"{what}: {Hv} value heads must be a multiple of {Hk} key heads"
    assert g.shape == (B, T, Hv) and beta.shape == (B, T, Hv), (
        f"{what}: g and beta must be [B, T, Hv] = {(B, T, Hv)}")
    assert k.dtype is q.dtype and v.dtype is q.dtype, f"{what}: q, k and v must have one dtype"
    assert g.dtype in _GATE_TYPES, f"{what}: g must be fp32, bf16 or fp16, got {g.dtype}"
    assert beta.dtype in _GATE_TYPES, f"{what}: beta must be fp32, bf16 or fp16, got {beta.dtype}"
    return B, T, Hk, Hv, Dk, Dv


def _seqs(q, cu_seqlens):
    return q.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1


def _launch_fwd(q, k, v, g, beta, initial_state, cu_seqlens, scale, o, state, u, s0):
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    n = _seqs(q, cu_seqlens)
    packed = cu_seqlens is not None
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    g, beta = g.contiguous(), beta.contiguous()
    size = L.lib().uttt_gated_delta_workspace_bytes(B, T, n, Hk, Hv, Dk, Dv, int(packed), 0)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device)
    L.call_on(q, "uttt_gated_delta_fwd", L.ptr(q), _strides(q), L.ptr(k), _strides(k), L.ptr(v),
              _strides(v), L.ptr(g), L.dtype_code(g.dtype), L.ptr(beta), L.dtype_code(beta.dtype),
              L.ptr(cu_seqlens), int(packed and cu_seqlens.dtype == torch.int64), B, T, n, Hk, Hv,
              Dk, Dv, scale, L.ptr(initial_state), L.ptr(o), L.ptr(state), L.ptr(u), L.ptr(s0),
              L.ptr(ws), size, L.stream_of(q))


def _state_like(v, q, cu_seqlens, wanted):
    shape = (_seqs(q, cu_seqlens), v.shape[2], q.shape[3], v.shape[3]) if wanted else (0,)
    return torch.empty(shape, dtype=torch.float32, device=v.device)


def _infer_fake(q, k, v, g, beta, initial_state, cu_seqlens, scale, want_state):
    return (new_like(v),
            _state_like(v, q, cu_seqlens, want_state))


@traced_op("gated_delta_infer", _infer_fake)
def _infer(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, initial_state: Optional[Tensor],
           cu_seqlens: Optional[Tensor], scale: float, want_state: bool) -> Tuple[Tensor, Tensor]:
    """(o, final states, empty where not wanted)."""
    o, state = _infer_fake(q, k, v, g, beta, initial_state, cu_seqlens, scale, want_state)
    _launch_fwd(q, k, v, g, beta, initial_state, cu_seqlens, scale, o, state if want_state else None,
                None, None)
    return o, state


def _fwd_fake(q, k, v, g, beta, initial_state, cu_seqlens, scale, want_state):
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    slots = T // 64 + _seqs(q, cu_seqlens) + 2 if cu_seqlens is not None else B * ((T + 63) // 64)
    return (*_infer_fake(q, k, v, g, beta, initial_state, cu_seqlens, scale, want_state),
            v.new_empty((B, T, Hv, Dv), dtype=torch.float32),
            v.new_empty((slots, Hv, Dk, Dv), dtype=torch.float32))


@traced_op("gated_delta_fwd", _fwd_fake)
def _fwd(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, initial_state: Optional[Tensor],
         cu_seqlens: Optional[Tensor], scale: float,
         want_state: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """_infer, and what the backward reads: U and the states at the chunks'
    starts."""
    o, state, u, s0 = _fwd_fake(q, k, v, g, beta, initial_state, cu_seqlens, scale, want_state)
    _launch_fwd(q, k, v, g, beta, initial_state, cu_seqlens, scale, o, state if want_state else None,
                u, s0)
    return o, state, u, s0


def _bwd_fake(q, k, v, g, beta, cu_seqlens, scale, u, s0, do, dstate, want_dh0):
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    dh0 = v.new_empty((_seqs(q, cu_seqlens), Hv, Dk, Dv) if want_dh0 else (0,), dtype=torch.float32)
    return [new_like(q), new_like(q), new_like(v), new_like(g), new_like(beta), dh0]


@traced_op("gated_delta_bwd", _bwd_fake)
def _bwd(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, cu_seqlens: Optional[Tensor],
         scale: float, u: Tensor, s0: Tensor, do: Tensor, dstate: Optional[Tensor],
         want_dh0: bool) -> List[Tensor]:
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    n = _seqs(q, cu_seqlens)
    packed = cu_seqlens is not None
    q, k, v, do = _rows16(q), _rows16(k), _rows16(v), _rows16(do)
    g, beta = g.contiguous(), beta.contiguous()
    grads = _bwd_fake(q, k, v, g, beta, cu_seqlens, scale, u, s0, do, dstate, want_dh0)
    dq, dk, dv, dg, dbeta, dh0 = grads
    size = L.lib().uttt_gated_delta_workspace_bytes(B, T, n, Hk, Hv, Dk, Dv, int(packed), 1)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device)
    L.call_on(q, "uttt_gated_delta_bwd", L.ptr(q), _strides(q), L.ptr(k), _strides(k), L.ptr(v),
              _strides(v), L.ptr(g), L.dtype_code(g.dtype), L.ptr(beta), L.dtype_code(beta.dtype),
              L.ptr(cu_seqlens), int(packed and cu_seqlens.dtype == torch.int64), B, T, n, Hk, Hv,
              Dk, Dv, scale, L.ptr(u), L.ptr(s0), L.ptr(do), _strides(do), L.ptr(dstate), L.ptr(dq),
              L.ptr(dk), L.ptr(dv), L.ptr(dg), L.ptr(dbeta), L.ptr(dh0) if want_dh0 else None,
              L.ptr(ws), size, L.stream_of(q))
    return grads


class _GatedDeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial_state, cu_seqlens, scale, want_state, keep):
        args = (q, k, v, g, beta, initial_state, cu_seqlens, scale, want_state)
        if not keep:
            return _infer(*args)
        o, state, u, s0 = _fwd(*args)
        ctx.save_for_backward(q, k, v, g, beta, cu_seqlens, u, s0)
        ctx.scale = scale
        # its values are not needed again (no saved tensor, which must not change)
        ctx.h0 = initial_state if initial_state is not None and initial_state.requires_grad else None
        ctx.set_materialize_grads(False)
        return o, state

    @staticmethod
    def backward(ctx, do, dstate):
        q, k, v, g, beta, cu, u, s0 = ctx.saved_tensors
        if do is None:
            do = torch.zeros_like(v)
        if dstate is not None:
            dstate = dstate.contiguous()
        want_dh0 = ctx.h0 is not None
        grads = _bwd(q, k, v, g, beta, cu, ctx.scale, u, s0, do, dstate, want_dh0)
        dq, dk, dv, dg, dbeta, dh0 = first_order_only("gated_delta_rule", grads, q, k, v, g, beta,
                                                      ctx.h0, do, dstate)
        return (dq, dk, dv, dg, dbeta, dh0 if want_dh0 else None, None, None, None, None)


def gated_delta_rule(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, *,
                     scale: float | None = None, initial_state: Tensor | None = None,
                     output_final_state: bool = False, cu_seqlens: Tensor | None = None):
    """The gated delta rule over whole sequences.  Returns (o [B, T, Hv, Dv]
    bf16, final states [N, Hv, Dk, Dv] fp32 or None).

    q, k           [B, T, Hk, Dk] bf16; Dk a multiple of 8 up to 256.  Used as given: a model
                   normalises them (uttt_amd.moe.rows_preprocess) before.
    v              [B, T, Hv, Dv] bf16; Dv a multiple of 8.  Value heads Hv / Hk * h onwards
                   share key head h.
    g, beta        [B, T, Hv] log decays (0 or less; -inf forgets everything) and write
                   strengths, in fp32, bf16 or fp16; their gradients have their types.
    scale          of the outputs, Dk ** -0.5 if None.
    initial_state  [N, Hv, Dk, Dv] fp32, zeros if None; N = B, or the packed sequences.
    cu_seqlens     [N + 1] int32 or int64 on the GPU: B is 1 and sequence n is the tokens
                   cu_seqlens[n] to cu_seqlens[n + 1] of the token axis, none of them at all
                   allowed.  Offsets must ascend; tokens of no sequence get zeros as outputs
                   and gradients.

    A value that is not finite reaches the results of its token and later ones of its sequence
    (of q: of its token alone; of v: in its column alone), as in the recurrence, and no others:
    what lies behind a padded sequence's tokens does not matter to their outputs.  Of v this
    holds for the gradients too, where those given for the later outputs are zeros.

    q, k and v may be views with any strides of their first three axes that are multiples of
    8 elements; others are copied.  States, their gradients and those of fp32 g and beta are
    exact to fp32's order, outputs and the other gradients are rounded to their types once.
    The backward keeps U and the state at every 64th token, 4 bytes an element."""
    what = "gated_delta_rule"
    B, T, Hk, Hv, Dk, Dv = _check(q, k, v, g, beta, what)
    assert q.dtype == torch.bfloat16, f"{what}: q, k and v must be bf16, got {q.dtype}"
    assert 8 <= Dk <= MAX_KEY_DIM and Dk % 8 == 0 and Dv >= 8 and Dv % 8 == 0, (
        f"{what}: Dk = {Dk} must be a multiple of 8 up to {MAX_KEY_DIM}, Dv = {Dv} a multiple of 8")
    assert B >= 1, f"{what}: an empty batch"
    if cu_seqlens is not None:
        assert B == 1, f"{what}: packed sequences have a batch of 1, got {B}"
        assert cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 2, f"{what}: cu_seqlens must be [N + 1]"
        assert cu_seqlens.dtype in (torch.int32, torch.int64), f"{what}: cu_seqlens must be int32 or int64"
        assert cu_seqlens.device == q.device, f"{what}: cu_seqlens is on {cu_seqlens.device}"
        cu_seqlens = cu_seqlens.contiguous()
    if initial_state is not None:
        shape = (_seqs(q, cu_seqlens), Hv, Dk, Dv)
        assert initial_state.shape == shape, f"{what}: initial_state must be {shape}"
        assert initial_state.dtype == torch.float32, f"{what}: states are fp32"
        assert initial_state.device == q.device, f"{what}: initial_state is on {initial_state.device}"
        initial_state = initial_state.contiguous()
    scale = Dk ** -0.5 if scale is None else float(scale)
    keep = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_state))
    o, state = run_function(_GatedDeltaRule, q, k, v, g, beta, initial_state, cu_seqlens, scale,
                            bool(output_final_state), keep, graph=keep)
    return o, state if output_final_state else None


def _step_fake(q, k, v, g, beta, state, scale, state_indices):
    return new_like(v)


@traced_op("gated_delta_step", _step_fake, mutates_args=("state",))
def _step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, state: Tensor, scale: float,
          state_indices: Optional[Tensor]) -> Tensor:
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    q, k, v = (t if t.stride(3) == 1 else t.contiguous() for t in (q, k, v))
    g, beta = g.contiguous(), beta.contiguous()
    o = _step_fake(q, k, v, g, beta, state, scale, state_indices)
    slots = state.shape[0]
    apart = state.stride(0) if slots > 1 else Hv * Dk * Dv   # of one slot it says nothing
    L.call_on(q, "uttt_gated_delta_step", L.ptr(q), _strides(q), L.ptr(k), _strides(k), L.ptr(v),
              _strides(v), L.dtype_code(q.dtype), L.ptr(g), L.dtype_code(g.dtype), L.ptr(beta),
              L.dtype_code(beta.dtype), B, T, Hk, Hv, Dk, Dv, scale, L.ptr(state), apart,
              slots, L.ptr(state_indices),
              int(state_indices is not None and state_indices.dtype == torch.int64), L.ptr(o),
              L.stream_of(q))
    return o


def gated_delta_step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, state: Tensor, *,
                     scale: float | None = None, state_indices: Tensor | None = None) -> Tensor:
    """A few tokens per sequence against states in place (generation): o
    [B, T, Hv, Dv] in q's dtype, and `state` is as after the last token.

    q, k           [B, T, Hk, Dk], v [B, T, Hv, Dv]: one dtype of bf16, fp16, fp32; Dk up to
                   256, Dv a multiple of 4; g, beta [B, T, Hv] as in gated_delta_rule.  T is 1
                   for plain generation; the tokens of a row follow one another.
    state          [slots, Hv, Dk, Dv] fp32, its last three axes contiguous (a layer's slice of
                   a pool that holds all layers will do).
    state_indices  [B] int32 or int64, the slot of each row; row b's is b if None.  A row whose
                   index is no slot (-1: padding) leaves every state alone and gets zeros.  Rows
                   that name one slot follow one another in row order.

    No gradient flows through it, backward or forward: tensors that have one are refused."""
    what = "gated_delta_step"
    B, T, Hk, Hv, Dk, Dv = _check(q, k, v, g, beta, what)
    assert q.dtype in (torch.float32, torch.bfloat16, torch.float16), f"{what}: dtype {q.dtype}"
    assert 1 <= Dk <= MAX_KEY_DIM and Dv >= 4 and Dv % 4 == 0, (
        f"{what}: Dk = {Dk} must be at most {MAX_KEY_DIM}, Dv = {Dv} a multiple of 4")
    assert state.dim() == 4 and state.shape[1:] == (Hv, Dk, Dv), (
        f"{what}: state must be [slots, {Hv}, {Dk}, {Dv}], got {tuple(state.shape)}")
    assert state.dtype == torch.float32 and state.device == q.device, f"{what}: state must be fp32 on {q.device}"
    ss, sh, sk, sd = state.stride()
    assert state.is_contiguous() or (sd == 1 and sk == Dv and sh == Dk * Dv and ss % 4 == 0
                                     and (ss >= Hv * Dk * Dv or state.shape[0] <= 1)), (
        f"{what}: each slot's state must be contiguous and apart from the others")
    if state_indices is not None:
        assert state_indices.shape == (B,), f"{what}: state_indices must be [{B}]"
        assert state_indices.dtype in (torch.int32, torch.int64), f"{what}: state_indices must be int32 or int64"
        assert state_indices.device == q.device, f"{what}: state_indices is on {state_indices.device}"
        state_indices = state_indices.contiguous()
    else:
        assert B <= state.shape[0], f"{what}: {B} rows, {state.shape[0]} states"
    tensors = (q, k, v, g, beta, state)
    assert not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)) and not (
        forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)), (
        f"{what}: no gradient flows through a state that is updated in place")
    return _step(q, k, v, g, beta, state, Dk ** -0.5 if scale is None else float(scale), state_indices)
