"""The gated delta rule token by token in 64 bits (CPU): the definition that
the chunked and the single-token kernels are checked against.  Gradients come
from torch's autograd through the recurrence."""
from __future__ import annotations

import torch


def recurrence(q, k, v, g, beta, state, scale):
    """One sequence: q, k [T, Hk, Dk], v [T, Hv, Dv], g, beta [T, Hv], state
    [Hv, Dk, Dv]; returns (o [T, Hv, Dv], the state after the last token)."""
    group = torch.arange(v.shape[1]) // (v.shape[1] // q.shape[1])
    out = []
    for t in range(q.shape[0]):
        kt, qt = k[t, group], q[t, group]
        # e^-inf is a state forgotten altogether, and takes no gradient
        state = state * torch.exp(g[t])[:, None, None]
        u = beta[t][:, None] * (v[t] - (kt[:, :, None] * state).sum(1))
        state = state + kt[:, :, None] * u[:, None, :]
        out.append(scale * (qt[:, :, None] * state).sum(1))
    o = torch.stack(out) if out else v.new_zeros(v.shape)
    return o, state


def gated_delta_rule(q, k, v, g, beta, scale, initial_state=None, cu_seqlens=None):
    """Batched [B, T, ...] or packed [1, T, ...] inputs in 64 bits; tokens of no
    sequence get zeros."""
    B, T = q.shape[:2]
    spans = [(b, 0, T) for b in range(B)] if cu_seqlens is None else [
        (0, s, e) for s, e in zip(cu_seqlens[:-1], cu_seqlens[1:])]
    o = [torch.zeros_like(v[b]) for b in range(B)]
    states = []
    for n, (b, s, e) in enumerate(spans):
        S = torch.zeros(v.shape[2], q.shape[3], v.shape[3], dtype=v.dtype) if (
            initial_state is None) else initial_state[n]
        y, S = recurrence(q[b, s:e], k[b, s:e], v[b, s:e], g[b, s:e], beta[b, s:e], S, scale)
        o[b] = torch.cat([o[b][:s], y, o[b][e:]])
        states.append(S)
    return torch.stack(o), torch.stack(states)
