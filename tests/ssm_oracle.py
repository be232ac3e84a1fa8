"""The state space layer's operators in 64 bits on the CPU, from their
definitions, with bounds on what fewer bits may cost (test infrastructure).

Everywhere: a rounding to 32 bits is off by 2^-24 of the value, half a step of
an output's type by HALF; matrix instructions may cut a sum's terms instead of
rounding them (2^-23 each). The hardware's exponential and reciprocal are a few
steps of 2^-24 off: 2^-22 each below, beside what the argument's own rounding
does (|v| 2^-23, v log2 e)."""
from __future__ import annotations

import torch
from cache_oracle import HALF, TINY, assert_within  # noqa: F401


def _silu(v, e):
    """silu of v off by e: its slope is at most 1.1, and the factor sigmoid is
    off by (1 - sigmoid) times its exponent's error."""
    s = v * torch.sigmoid(v)
    return s, 1.1 * e + s.abs() * (v.abs() * 2.0 ** -22 + 2.0 ** -21)


def _rounded(y, e, dtype):
    return e + (y.abs() + e) * HALF[dtype] + TINY[dtype]


def _slot(slots, n_slots, b):
    s = b if slots is None else int(slots[b])
    return s if 0 <= s < n_slots else -1


def conv(x, w, bias, silu=True, state=None, n_slots=0, lengths=None, slots=None, rounded=True):
    """(y, bound, state_out [n_slots, taps - 1, C] or None): rows behind a
    sequence's length 0. taps products and as many sums in 32 bits."""
    B, L, C = x.shape
    taps = w.shape[1]
    dt = x.dtype
    x, w = x.double().cpu(), w.double().cpu()
    bias = torch.zeros(C, dtype=torch.float64) if bias is None else bias.double().cpu()
    y, e = torch.zeros(B, L, C, dtype=torch.float64), torch.zeros(B, L, C, dtype=torch.float64)
    after = torch.zeros(n_slots, taps - 1, C, dtype=torch.float64) if n_slots else None
    if state is not None:
        state = state.double().cpu()
        after = state.clone()
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        s = _slot(slots, n_slots, b)
        before = state[s] if state is not None and s >= 0 else torch.zeros(taps - 1, C, dtype=torch.float64)
        rows = torch.cat([before, x[b, :n]])
        for t in range(n):
            p = rows[t:t + taps].T * w
            v = p.sum(1) + bias
            d = (taps + 1) * 2.0 ** -24 * (p.abs().sum(1) + bias.abs())
            y[b, t], e[b, t] = _silu(v, d) if silu else (v, d)
        if after is not None and s >= 0:
            after[s] = rows[n:]
    return y, _rounded(y, e, dt) * (e != 0) if rounded else e, after


def time_step(raw, bias, softplus, lo, hi):
    """(dt, its relative error's bound): a sum, an exponential and a logarithm
    in 32 bits; where v cancels, the sum's rounding counts against it."""
    r = raw.double().cpu()
    b = torch.zeros(raw.shape[-1], dtype=torch.float64) if bias is None else bias.double().cpu()
    v, dv = r + b, (r.abs() + b.abs()) * 2.0 ** -24
    if softplus:
        y = torch.logaddexp(v, torch.zeros_like(v))
        e = dv * torch.sigmoid(v) + y * 2.0 ** -21
    else:
        y, e = v, dv
    y = y.clamp(lo, hi)
    return y, e / y.abs().clamp_min(1e-300)


def scan(x, dt, dt_rel, a, b, c, d=None, state=None, n_slots=0, lengths=None, slots=None, x_err=None, b_err=None,
         c_err=None, rounded=None):
    """(y, bound, state_out, its bound). x [B, L, nh, hd], dt [B, L, nh] the
    time steps themselves (relative error dt_rel), b and c [B, L, g, N].

    Sa is the scan of magnitudes. A state's error E: each token, the decay is
    off by |dt a| (dt_rel + 2^-22) + 2^-21 of itself, what comes in by dt_rel +
    2^-21, and a sum's roundings by 2^-22 of Sa; where 64 tokens are summed by
    matrix instructions, three products each (the incoming rows in three parts
    of 8 bits, 24 in all), 3 * 64 * 2^-23 of Sa once more. An output: sums of N
    terms (2^-23 each), and 2^-16 of the magnitudes, which is more than the
    state and the weights of a chunk's tokens need, whose bits are held by
    numbers that cancel in tests of their own."""
    B, L, nh, hd = x.shape
    N = b.shape[3]
    rep = nh // b.shape[2]
    xd, bd, cd = x.double().cpu(), b.double().cpu(), c.double().cpu()
    zero = torch.zeros(1, dtype=torch.float64)
    xe, be, ce = (zero.expand_as(t) if err is None else err for t, err in ((xd, x_err), (bd, b_err), (cd, c_err)))
    a = a.double().cpu()
    dd = torch.zeros(nh, dtype=torch.float64) if d is None else d.double().cpu()
    y, yb = torch.zeros(B, L, nh, hd, dtype=torch.float64), torch.zeros(B, L, nh, hd, dtype=torch.float64)
    after = None
    if state is not None:
        state = state.double().cpu()
        after, after_b = state.clone(), torch.zeros_like(state)
    elif n_slots:
        after = torch.zeros(n_slots, nh, hd, N, dtype=torch.float64)
        after_b = torch.zeros_like(after)
    for q in range(B):
        n = L if lengths is None else min(max(int(lengths[q]), 0), L)
        s = _slot(slots, n_slots, q)
        S = state[s].clone() if state is not None and s >= 0 else torch.zeros(nh, hd, N, dtype=torch.float64)
        Sa, E = S.abs(), torch.zeros_like(S)
        for t in range(n):
            bt, ct, bet, cet = (v[q, t].repeat_interleave(rep, 0) for v in (bd, cd, be, ce))
            h = dt[q, t]
            f = torch.exp(h * a)[:, None, None]
            fe = ((h * a).abs() * (dt_rel[q, t] + 2.0 ** -22) + 2.0 ** -21)[:, None, None]
            u = h[:, None, None] * xd[q, t][:, :, None] * bt[:, None]
            ue = (u.abs() * (dt_rel[q, t][:, None, None] + 2.0 ** -21)
                  + h[:, None, None] * (xe[q, t][:, :, None] * (bt.abs() + bet)[:, None]
                                        + xd[q, t].abs()[:, :, None] * bet[:, None]))
            E = f * (E + fe * Sa) + ue
            S, Sa = f * S + u, f * Sa + u.abs()
            E = E + 2.0 ** -22 * Sa
            full = E + 3 * min(n, 64) * 2.0 ** -23 * Sa
            skip = dd[:, None] * xd[q, t]
            y[q, t] = (S * ct[:, None]).sum(-1) + skip
            yb[q, t] = (((full + (2.0 ** -16 + N * 2.0 ** -23) * Sa) * ct.abs()[:, None] + (Sa + full) * cet[:, None]).sum(-1)
                        + skip.abs() * 2.0 ** -22 + dd.abs()[:, None] * xe[q, t] + y[q, t].abs() * 2.0 ** -22)
        if after is not None and s >= 0:
            after[s], after_b[s] = S, E + 3 * min(n, 64) * 2.0 ** -23 * Sa + TINY[torch.float32]
    if rounded is not None:
        live = torch.zeros(B, L, 1, 1, dtype=torch.bool)
        for q in range(B):
            live[q, :L if lengths is None else min(max(int(lengths[q]), 0), L)] = True
        yb = torch.where(live, _rounded(y, yb, rounded), yb)
    return (y, yb, after, after_b) if after is not None else (y, yb, None, None)


def gated_norm(x, w, z, eps, groups, gate_first, dtype, x_err=None):
    """(y, bound). The group's products are off by e each; its RMS by their
    norm over the group's, by size 2^-24 for the sum and 2^-21 for root and
    quotient; two more products."""
    x = x.double().cpu()
    C = x.shape[-1]
    w = torch.ones(C, dtype=torch.float64) if w is None else w.double().cpu()
    e = torch.zeros_like(x) if x_err is None else x_err
    u, ue = x, e
    if z is not None:
        z = z.double().cpu()
        g, ge = _silu(z, torch.zeros_like(z))
        if gate_first:
            u, ue = x * g, e * (g.abs() + ge) + x.abs() * ge + (x * g).abs() * 2.0 ** -24
    ug, ueg = u.unflatten(-1, (groups, -1)), ue.unflatten(-1, (groups, -1))
    size = C // groups
    rms = torch.sqrt(ug.square().mean(-1, keepdim=True) + eps)
    rel = torch.sqrt(ueg.square().mean(-1, keepdim=True)) / rms + size * 2.0 ** -24 + 2.0 ** -21
    y = (ug / rms).flatten(-2) * w
    yb = (ueg / rms).flatten(-2) * w.abs() + y.abs() * (rel.expand_as(ug).flatten(-2) + 2.0 ** -22)
    if z is not None and not gate_first:
        y, yb = y * g, yb * (g.abs() + ge) + y.abs() * ge + (y * g).abs() * 2.0 ** -24
    return y, _rounded(y, yb, dtype)
