"""The operators of moc/blocks.py in 64 bits on the CPU, one token after the other, from
their definitions; used only by tests.

Each gradient is written out by hand (tests/test_blocks_cpu.py holds them to autograd and
to differences), so that the same recurrences on absolute values give what a sum's
rounding errors are relative to."""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def spans(n_tokens: int, seq_len: int | None, cu: list[int] | None) -> list[tuple[int, int]]:
    """The sequences of a flat token axis: seq_len tokens each, or the packed axis cut at
    0, every cu entry and its end."""
    if cu is None:
        return [(a, a + seq_len) for a in range(0, n_tokens, seq_len)]
    edges = [0, *cu, n_tokens]
    return [(a, b) for a, b in zip(edges[:-1], edges[1:]) if b > a]


def norm(x, w, b, eps, dy=None):
    """y, or (y, dx, dw, db); w, b may be None (1 and 0)."""
    x = x.to(F64)
    D = x.shape[-1]
    w = torch.ones(D, dtype=F64) if w is None else w.to(F64)
    b = torch.zeros(D, dtype=F64) if b is None else b.to(F64)
    d = x - x.sum(-1, keepdim=True) / D
    rstd = 1.0 / torch.sqrt((d * d).sum(-1, keepdim=True) / D + eps)
    xh = d * rstd
    y = xh * w + b
    if dy is None:
        return y
    dy = dy.to(F64)
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    lead = tuple(range(x.ndim - 1))
    return y, dx, (dy * xh).sum(lead), dy.sum(lead)


def conv(x, w, b, act, seqs, dy=None, history=None):
    """x [N, D] flat, w [S, D], b [D] or None; history [len(seqs), S, D]: the inputs before
    each sequence (slot S - 1 the newest).  y, or (y, dx, dw, db)."""
    x, w = x.to(F64), w.to(F64)
    S, D = w.shape
    b = torch.zeros(D, dtype=F64) if b is None else b.to(F64)
    y, dx, dw, db = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros(D, dtype=F64)
    for q, (lo, hi) in enumerate(seqs):
        old = torch.zeros(S, D, dtype=F64) if history is None else history[q].to(F64)
        xs = torch.cat((old, x[lo:hi]), 0)  # row S + t is token t
        T = hi - lo
        p = b.repeat(T, 1)
        for s in range(S):
            p = p + w[s] * xs[s + 1:s + 1 + T]
        sg = 1 / (1 + torch.exp(-p))
        y[lo:hi] = p * sg if act else p
        if dy is None:
            continue
        g = dy[lo:hi].to(F64)
        if act:
            g = g * sg * (1 + p * (1 - sg))
        full = torch.zeros_like(xs)
        for s in range(S):
            full[s + 1:s + 1 + T] += w[s] * g
            dw[s] += (g * xs[s + 1:s + 1 + T]).sum(0)
        db += g.sum(0)
        dx[lo:hi] = full[S:]
    return y if dy is None else (y, dx, dw, db)


def step_lengths(dt, bias, softplus):
    v = dt.to(F64) + (0 if bias is None else bias.to(F64))
    return torch.log1p(torch.exp(-v.abs())) + v.clamp(min=0) if softplus else v


def scan(x, u, A, B, C, D, seqs, init=None, dy=None, dfin=None):
    """x [n, H, P], u [n, H] (step_lengths), A [H], B, C [n, G, N], D [H] or None, init
    [len(seqs), H, P, N] or None.  (y, final states), or with dy also the gradients
    (dx, du, dA, dB, dC, dD, dinit, da), du that of u, da that of the exponents u A."""
    x, u, A, B, C = (t.to(F64) for t in (x, u, A, B, C))
    n, H, P = x.shape
    G, N = B.shape[1:]
    Dv = torch.zeros(H, dtype=F64) if D is None else D.to(F64)
    a = torch.exp(u * A)
    Bh, Ch = (t.repeat_interleave(H // G, 1) for t in (B, C))
    y = Dv[:, None] * x
    states = torch.zeros(n, H, P, N, dtype=F64)  # behind each token
    starts = torch.zeros(len(seqs), H, P, N, dtype=F64) if init is None else init.to(F64)
    fin = torch.zeros_like(starts)
    for q, (lo, hi) in enumerate(seqs):
        h = starts[q]
        for t in range(lo, hi):
            h = a[t, :, None, None] * h + (u[t, :, None] * x[t])[:, :, None] * Bh[t][:, None]
            states[t] = h
        fin[q] = h
    y = y + (states * Ch[:, :, None]).sum(-1)
    if dy is None:
        return y, fin
    dy = dy.to(F64)
    dx, du, da = Dv[:, None] * dy, torch.zeros_like(u), torch.zeros_like(u)
    dBh, dCh, dinit = torch.zeros_like(Bh), torch.zeros_like(Ch), torch.zeros_like(starts)
    for q, (lo, hi) in enumerate(seqs):
        dh = torch.zeros(H, P, N, dtype=F64) if dfin is None else dfin[q].to(F64)
        for t in range(hi - 1, lo - 1, -1):
            dh = dh + dy[t][:, :, None] * Ch[t][:, None]
            dCh[t] = (dy[t][:, :, None] * states[t]).sum(1)
            dBh[t] = (u[t, :, None, None] * x[t][:, :, None] * dh).sum(1)
            hb = (dh * Bh[t][:, None]).sum(-1)
            dx[t] += u[t, :, None] * hb
            du[t] = (x[t] * hb).sum(-1)
            dh = dh * a[t, :, None, None]
            da[t] = (dh * (states[t - 1] if t > lo else starts[q])).sum((-1, -2))
        dinit[q] = dh
    to_groups = [t.unflatten(1, (G, H // G)).sum(2) for t in (dBh, dCh)]
    return (y, fin), (dx, du + A * da, (u * da).sum(0), *to_groups, (dy * x).sum((0, 2)), dinit, da)


def sigmoid_of(u, softplus):
    """d softplus(v) / dv from u = softplus(v)."""
    return -torch.expm1(-u) if softplus else torch.ones_like(u)


def half_step(dtype: torch.dtype) -> float:
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


F32_HALF = math.ldexp(1.0, -24)
