"""The sequence operators from their definitions, step by step, in fp64 on the CPU; differentiable by torch.autograd."""
import math

import torch


def act(x, name):
    if name in (None, "none"):
        return x
    if name == "tanh":
        return torch.tanh(x)
    if name == "gelu":
        return x * 0.5 * torch.erfc(-x / math.sqrt(2.0))
    p = 1 / (1 + torch.exp(-x))
    return p if name == "sigmoid" else x * p


def _ends(lengths, nb, steps):
    return [steps] * nb if lengths is None else [min(max(int(n), 0), steps) for n in lengths]


def causal_conv(u, w, bias=None, name=None, start=None, lengths=None):
    """-> y [nb, L, D], window [nb, W-1, D]"""
    nb, steps, d = u.shape
    taps = w.shape[1]
    ys, windows = [], []
    for b, n in enumerate(_ends(lengths, nb, steps)):
        head = torch.zeros(taps - 1, d, dtype=u.dtype) if start is None else start[b]
        line = torch.cat([head, u[b, :n]], 0)
        rows = [sum((w[:, j] * line[t + j] for j in range(taps)), 0 * line[t] if bias is None else bias) for t in range(n)]
        rows = [act(r, name) for r in rows] + [torch.zeros(d, dtype=u.dtype)] * (steps - n)
        ys.append(torch.stack(rows) if rows else torch.zeros(0, d, dtype=u.dtype))
        windows.append(line[n:])
    return torch.stack(ys), torch.stack(windows)


def softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x)))


def lpv_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, use_softplus=True, start=None, lengths=None):
    """x_t = exp(delta_t A) x_{t-1} + delta_t B_t u_t,  y_t = (C_t . x_t + D u_t) silu(z_t) -> y [nb, L, D], x_L [nb, D, N]"""
    nb, steps, d = u.shape
    groups, n = B.shape[2:]
    ys, states = [], []
    for b, end in enumerate(_ends(lengths, nb, steps)):
        x = torch.zeros(d, n, dtype=u.dtype) if start is None else start[b]
        rows = []
        for t in range(end):
            raw = dt[b, t] if dt_bias is None else dt[b, t] + dt_bias
            delta = softplus(raw) if use_softplus else raw
            Bt, Ct = (v[b, t].repeat_interleave(d // groups, 0) for v in (B, C))
            x = torch.exp(delta[:, None] * A) * x + (delta * u[b, t])[:, None] * Bt
            y = (x * Ct).sum(1)
            if D is not None:
                y = y + D * u[b, t]
            rows.append(y if z is None else y * act(z[b, t], "silu"))
        rows += [torch.zeros(d, dtype=u.dtype)] * (steps - end)
        ys.append(torch.stack(rows) if rows else torch.zeros(0, d, dtype=u.dtype))
        states.append(x)
    return torch.stack(ys), torch.stack(states)


def gated_ffn(x, w_gate, w_up, name="silu"):
    return act(x @ w_gate.T, name) * (x @ w_up.T)
