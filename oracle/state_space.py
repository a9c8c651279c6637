"""The state space layer's operators in 64 bits (CPU): the short causal
convolution, the selective scan token by token and the norms around a block, the
definitions that the kernels are checked against.  Gradients of the convolution
and the norms come from torch's autograd; the scan's are formulas, token by
token, next to bounds of what fp32 arithmetic leaves of them."""
from __future__ import annotations

import torch

U = 2.0 ** -24   # half an ulp of fp32


def spans(B, T, cu_seqlens=None):
    """(row, first token, end) of each sequence."""
    if cu_seqlens is None:
        return [(b, 0, T) for b in range(B)]
    return [(0, s, e) for s, e in zip(cu_seqlens[:-1], cu_seqlens[1:])]


def causal_conv(x, weight, bias=None, silu=False, initial_state=None, cu_seqlens=None):
    """x [B, T, D], weight [D, W]: (y, the last W - 1 inputs of each sequence).
    Tokens of no sequence get zeros."""
    B, T, D = x.shape
    W = weight.shape[1]
    y, states = [torch.zeros_like(x[b]) for b in range(B)], []
    for n, (b, s, e) in enumerate(spans(B, T, cu_seqlens)):
        before = x.new_zeros(W - 1, D) if initial_state is None else initial_state[n]
        full = torch.cat([before, x[b, s:e]])
        p = sum(weight[:, k] * full[k:k + e - s] for k in range(W))
        p = p if bias is None else p + bias
        p = p * torch.sigmoid(p) if silu else p
        y[b] = torch.cat([y[b][:s], p, y[b][e:]])
        states.append(full[e - s:])
    return torch.stack(y), torch.stack(states)


def _by_group(t, G):
    """[D, N] summed over the channels of each group: [G, N]."""
    return t.reshape(G, -1, t.shape[-1]).sum(1)


def scan_sequence(x, dt, A, B, C, D=None, z=None, bias=None, softplus=False, h0=None, dy=None, dhT=None):
    """One sequence: x, dt, z, dy [T, D]; A, h0, dhT [D, N]; B, C [T, G, N]; D, bias
    [D].  Returns ({name: value}, {name: bound}) of y and state, and with dy or
    dhT of the gradients d_x, d_dt, d_A, d_B, d_C, d_D, d_z, d_bias and d_h0.

    A bound is of the error of fp32 arithmetic to the first order, without the
    last rounding to a result's type: each operation adds U of its operands'
    magnitudes (sums of absolute values run beside the sums), softplus and
    sigmoid are off by 8 U of themselves, a decay by what its step is off by
    times |A|, by 4 U of its exponent, by T U of it where steps were summed over a
    run, and by 4 U; sums over n values by (n + 16) U."""
    T, Dm = x.shape
    N, G = A.shape[1], B.shape[1]
    r = Dm // G
    zero = x.new_zeros(Dm)
    raw = dt if bias is None else dt + bias
    if softplus:
        step, slope = torch.logaddexp(raw, torch.zeros_like(raw)), torch.sigmoid(raw)
        e_step = 8 * U * step + 2 * U * raw.abs() * slope
    else:
        step, slope = raw, torch.ones_like(raw)
        e_step = U * raw.abs() if bias is not None else torch.zeros_like(raw)
    u = step * x
    e_u = e_step * x.abs() + U * u.abs()
    Bx, Cx = B.repeat_interleave(r, 1), C.repeat_interleave(r, 1)   # [T, D, N]
    h = x.new_zeros(Dm, N) if h0 is None else h0
    M, E = h.abs(), torch.zeros_like(h)
    hs, Ms, Es, decay, e_decay, y, e_y, core, e_core, M_core = [h], [M], [E], [], [], [], [], [], [], []
    for t in range(T):
        a = torch.exp(step[t][:, None] * A)
        da = A.abs() * e_step[t][:, None] + (step[t][:, None] * A).abs() * (4 + T) * U + 4 * U
        ub = u[t][:, None] * Bx[t]
        E = a * E + a * M * da + e_u[t][:, None] * Bx[t].abs() + 3 * U * (a * M + ub.abs())
        M = a * M + ub.abs()
        h = a * h + ub
        dx = zero if D is None else D * x[t]
        v, Mv = (Cx[t] * h).sum(-1) + dx, (Cx[t].abs() * M).sum(-1) + dx.abs()
        ev = (Cx[t].abs() * E).sum(-1) + (N + 16) * U * Mv
        hs.append(h), Ms.append(M), Es.append(E), decay.append(a), e_decay.append(da)
        core.append(v), e_core.append(ev), M_core.append(Mv)
        if z is None:
            y.append(v), e_y.append(ev)
        else:
            s = z[t] * torch.sigmoid(z[t])
            y.append(v * s), e_y.append(ev * s.abs() + (16 + z[t].abs()) * U * Mv * s.abs())
    stack = lambda t: torch.stack(t) if t else x.new_zeros(0, Dm)  # noqa: E731
    val, err = dict(y=stack(y), state=h), dict(y=stack(e_y), state=E)
    if dy is None and dhT is None:
        return val, err
    dy = torch.zeros_like(x) if dy is None else dy
    q = torch.zeros_like(h) if dhT is None else dhT      # the adjoint as it enters a token from behind
    Q, Eq = q.abs(), torch.zeros_like(q)
    g = {n: torch.zeros_like(t) for n, t in dict(x=x, dt=x, A=A, B=B, C=C, D=zero, z=x, bias=zero).items()}
    b = {n: torch.zeros_like(t) for n, t in g.items()}
    MA, MD, Mb = torch.zeros_like(A), zero.clone(), zero.clone()
    for t in reversed(range(T)):
        s = torch.ones_like(zero) if z is None else z[t] * torch.sigmoid(z[t])
        gt = dy[t] * s
        e_g = (0 if z is None else 8 * U) * gt.abs()
        col = lambda v: v[:, None]  # noqa: E731
        q = col(gt) * Cx[t] + q
        Eq = col(e_g) * Cx[t].abs() + Eq
        Q = (col(gt) * Cx[t]).abs() + Q
        Eq = Eq + 2 * U * Q
        g["C"][t] = _by_group(col(gt) * hs[t + 1], G)
        mC = _by_group(col(gt.abs()) * Ms[t + 1], G)
        b["C"][t] = _by_group(col(e_g) * Ms[t + 1] + col(gt.abs()) * Es[t + 1], G) + (r + 16) * U * mC
        g["B"][t] = _by_group(col(u[t]) * q, G)
        b["B"][t] = _by_group(col(u[t].abs()) * Eq + col(e_u[t]) * Q, G) + (r + 16) * U * _by_group(col(u[t].abs()) * Q, G)
        du, Mu = (q * Bx[t]).sum(-1), (Q * Bx[t].abs()).sum(-1)
        e_du = (Eq * Bx[t].abs()).sum(-1) + (N + 16) * U * Mu
        a, da = decay[t], e_decay[t]
        Eq = a * Eq + a * Q * da + U * a * Q
        q, Q = a * q, a * Q
        w, Mw = q * hs[t], Q * Ms[t]
        e_w = Eq * Ms[t] + Q * Es[t] + 2 * U * Mw
        skip = zero if D is None else D
        g["x"][t] = du * step[t] + skip * gt
        b["x"][t] = (e_du * step[t].abs() + Mu * e_step[t] + skip.abs() * e_g
                     + 3 * U * (Mu * step[t].abs() + (skip * gt).abs()))
        pre = (A * w).sum(-1) + du * x[t]
        Mp = (A.abs() * Mw).sum(-1) + Mu * x[t].abs()
        e_pre = (A.abs() * e_w).sum(-1) + e_du * x[t].abs() + (N + 16) * U * Mp
        g["dt"][t] = pre * slope[t]
        # the slope is off by 8 U of itself and by its input's rounding
        e_dt = e_pre * slope[t] + Mp * slope[t] * (10 + raw[t].abs()) * U
        b["dt"][t] = e_dt
        if z is not None:
            sig = torch.sigmoid(z[t])
            ds = sig * (1 + z[t] * (1 - sig))
            g["z"][t] = dy[t] * core[t] * ds
            b["z"][t] = dy[t].abs() * (ds.abs() * e_core[t] + M_core[t] * sig * (1 + z[t].abs()) * 24 * U)
        g["A"] += col(step[t]) * w
        b["A"] += col(step[t].abs()) * e_w + col(e_step[t]) * Mw
        MA += col(step[t].abs()) * Mw
        g["D"] += gt * x[t]
        b["D"] += e_g * x[t].abs()
        MD += (gt * x[t]).abs()
        g["bias"] += g["dt"][t]
        b["bias"] += e_dt
        Mb += Mp * slope[t]
    for n, m in (("A", MA), ("D", MD), ("bias", Mb)):
        b[n] += (T + 16) * U * m
    val.update({"d_" + n: t for n, t in g.items()}, d_h0=q)
    err.update({"d_" + n: t for n, t in b.items()}, d_h0=Eq)
    return val, err


def selective_scan(x, dt, A, B, C, D=None, z=None, bias=None, softplus=False, h0=None, dy=None, dhT=None,
                   cu_seqlens=None):
    """Batched or packed inputs; values and bounds as scan_sequence's, zeros for the
    tokens of no sequence."""
    rows, T, _ = x.shape
    at = lambda t, b, s, e: None if t is None else t[b, s:e]  # noqa: E731
    total = [{}, {}]
    for n, (b, s, e) in enumerate(spans(rows, T, cu_seqlens)):
        outs = scan_sequence(x[b, s:e], dt[b, s:e], A, B[b, s:e], C[b, s:e], D, at(z, b, s, e), bias, softplus,
                             None if h0 is None else h0[n], at(dy, b, s, e), None if dhT is None else dhT[n])
        for all_, one in zip(total, outs):
            for name, v in one.items():
                if name in ("state", "d_h0"):
                    all_.setdefault(name, []).append(v)
                elif name in ("d_A", "d_D", "d_bias"):
                    all_[name] = all_.get(name, 0) + v
                else:
                    if name not in all_:
                        all_[name] = x.new_zeros(rows, T, *v.shape[1:])
                    all_[name][b, s:e] = v
    for all_ in total:
        for name in ("state", "d_h0"):
            if name in all_:
                all_[name] = torch.stack(all_[name])
    return total


def rms(v, eps):
    return (v.square().mean(-1, keepdim=True) + eps).sqrt()


def norm_after_block(x, weight=None, gate=None, residual=None, scale=None, eps=1e-5):
    y = x / rms(x, eps)
    y = y if weight is None else y * weight
    y = y if gate is None else y * gate * torch.sigmoid(gate)
    y = y if scale is None else y * scale
    return y if residual is None else y + residual


def norm_before_block(x, residual, weight=None, scale=None, eps=1e-5):
    total = residual + (x if scale is None else x * scale)
    y = total / rms(total, eps)
    return (y if weight is None else y * weight), total
