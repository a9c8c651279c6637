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


def gradients(q, k, v, g, beta, state, do, dstate, scale):
    """The recurrence's gradients token by token, without autograd, for rows of
    equal length: q, k [N, T, H, Dk] (a key head per value head), v, do
    [N, T, H, Dv], g, beta [N, T, H], state, dstate [N, H, Dk, Dv].

    Returns a dict of dq, dk (per value head), dv, dg, dbeta, dh0; `u`, `du` and
    the states `S` [N, T + 1, H, Dk, Dv] before each token with their gradients
    `dS`; and `size_g`, `size_beta` [N, T, H]: the 2-norms whose product the sums
    for dg and dbeta are made of, those of <S, dS> and of du.(v - S^T k)."""
    T, Dk = q.shape[1], q.shape[3]
    norm = lambda x, d: x.square().sum(d).sqrt()  # noqa: E731
    S, P, u, err = [state], [], [], []
    for t in range(T):
        P.append(S[-1] * torch.exp(g[:, t])[..., None, None])
        err.append(v[:, t] - (k[:, t, ..., None] * P[-1]).sum(-2))
        u.append(beta[:, t, :, None] * err[-1])
        S.append(P[-1] + k[:, t, ..., None] * u[-1][..., None, :])
    D, out, dS = dstate, [], [dstate]
    for t in reversed(range(T)):
        kt, dot = k[:, t, ..., None], do[:, t, :, None, :]
        dq = scale * (S[t + 1] * dot).sum(-1)
        D = D + scale * q[:, t, ..., None] * dot
        du = (kt * D).sum(-2)
        db = (du * err[t]).sum(-1)
        dv = beta[:, t, :, None] * du
        dP = D - kt * dv[..., None, :]
        dk = (D * u[t][..., None, :]).sum(-1) - (P[t] * dv[..., None, :]).sum(-1)
        whole = norm(P[t], (-2, -1)) * norm(kt, (-2, -1)) / Dk ** 0.5   # the order of S^T k
        size_b = norm(D, (-2, -1)) * norm(kt, (-2, -1)) / Dk ** 0.5 * norm(err[t], -1) + norm(du, -1) * whole
        out.append((dq, dk, dv, (P[t] * dP).sum((-2, -1)), db, du,
                    norm(P[t], (-2, -1)) * norm(dP, (-2, -1)), size_b))
        D = torch.exp(g[:, t])[..., None, None] * dP
        dS.append(D)
    names = ("dq", "dk", "dv", "dg", "dbeta", "du", "size_g", "size_beta")
    got = {n: torch.stack([x[i] for x in reversed(out)], 1) for i, n in enumerate(names)}
    return dict(got, dh0=D, u=torch.stack(u, 1), S=torch.stack(S, 1), dS=torch.stack(dS[::-1], 1))
