"""The cache's long-context operators in 64 bits on the CPU, from their
definitions, with bounds on what fewer bits may cost (test infrastructure)."""
from __future__ import annotations

import math

import torch

# half a step of rounding, relative to the value
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


def rotate(x, positions, freqs, factor, dims, interleaved, inverse=False):
    """(y, bound): x [B, L, nh, hd] turned to positions [B, L], 64 bits. The
    bound: an angle exact to 2^-51 of itself (a product of three roundings in
    64 bits) and 2^-21 (its turn rounded to 32 bits, pi 2^-24, cosine and sine
    a few steps of 2^-24), two products and a sum in 32 bits, one rounding."""
    y = x.double().cpu().clone()
    ang = positions.double().cpu()[..., None] * torch.as_tensor(freqs, dtype=torch.float64)
    if inverse:
        ang = -ang
    c, s = (ang.cos() * factor)[:, :, None], (ang.sin() * factor)[:, :, None]
    n = dims // 2
    ia = torch.arange(n) * 2 if interleaved else torch.arange(n)
    ib = ia + 1 if interleaved else ia + n
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    err = torch.zeros_like(y)
    e = (a.abs() + b.abs()) * abs(factor) * (ang.abs()[:, :, None] * 2.0 ** -51 + 2.0 ** -20)
    err[..., ia], err[..., ib] = e, e
    turned = torch.zeros(y.shape[-1], dtype=torch.bool)
    turned[:dims] = True
    bound = torch.where(turned, err + y.abs() * HALF[x.dtype] + TINY[x.dtype], torch.zeros_like(y))
    return y, bound


def attention(q, kc, vc, offsets, scale, slots=None, kp=None, vp=None):
    """dict of out, lse, weights ([slots, nkv, S], this call's alone) and
    their bounds. q [B, L, nh, hd], caches [slots, nkv, S, hd], prefix
    [nkv, P, hd].

    Bounds. A score is a sum of hd exact products in 32 bits: off by at most
    hd 2^-23 of the sum of their magnitudes (any order, truncation included),
    and 2^-22 of itself by its scaling; two such errors (its own and the
    maximum's or the sum's) and 2^-20 for the exponentials are d, the relative
    error of a probability before rounding. The probabilities are rounded to
    the inputs' type for their product with the values, half a step h; sums
    over n keys in 32 bits n 2^-24 at most, of magnitudes: out is off by
    (d + 2 h + n 2^-24) sum p |v| and its own rounding."""
    B, L, nh, hd = q.shape
    nkv, S = kc.shape[1], kc.shape[2]
    rep = nh // nkv
    P = kp.shape[1] if kp is not None else 0
    h = HALF[q.dtype]
    q, kc, vc = q.double().cpu(), kc.double().cpu(), vc.double().cpu()
    offs = offsets.tolist()
    out = torch.zeros(B, L, nh, hd, dtype=torch.float64)
    out_b = torch.zeros_like(out)
    lse = torch.full((B, L, nh), -math.inf, dtype=torch.float64)
    lse_b = torch.zeros_like(lse)
    w = torch.zeros(kc.shape[:3], dtype=torch.float64)
    w_b = torch.zeros_like(w)
    for b in range(B):
        slot = b if slots is None else int(slots[b])
        live = 0 <= slot < kc.shape[0]
        for l in range(L):
            n = min(max(offs[b] + l + 1, 0), S) if live else 0
            if P + n == 0:
                continue
            for g in range(nkv):
                k, v = kc[slot, g, :n] if live else kc[0, g, :0], vc[slot, g, :n] if live else vc[0, g, :0]
                if P:
                    k, v = torch.cat([kp[g].double().cpu(), k]), torch.cat([vp[g].double().cpu(), v])
                qg = q[b, l, g * rep:(g + 1) * rep]
                s = (qg @ k.T) * scale
                mag = (qg.abs() @ k.abs().T) * scale
                d = 2 * (hd * 2.0 ** -23 * mag.amax(-1) + 2.0 ** -22 * s.abs().amax(-1)) + 2.0 ** -20  # [rep]
                z = torch.logsumexp(s, -1)
                p = torch.exp(s - z[:, None])
                hs = slice(g * rep, (g + 1) * rep)
                out[b, l, hs] = p @ v
                out_b[b, l, hs] = ((d + 2 * h + (P + n) * 2.0 ** -24)[:, None] * (p @ v.abs())
                                   + h * out[b, l, hs].abs() + TINY_OUT)
                lse[b, l, hs] = z
                lse_b[b, l, hs] = d + (P + n) * 2.0 ** -24 + 2.0 ** -22 * z.abs()
                if not live:
                    continue
                w[slot, g, :n] += p[:, P:].sum(0)
                w_b[slot, g, :n] += (p[:, P:] * (d + (P + n + L * rep) * 2.0 ** -24)[:, None]).sum(0)
    return dict(out=out, out_b=out_b, lse=lse, lse_b=lse_b, w=w, w_b=w_b + w * 2.0 ** -23 + 1e-37)


# a value's own rounding below the smallest normal number of float16
TINY_OUT = 2.0 ** -24


def kept_positions(w, n, budget, sinks, recent):
    """The positions kept of one row's n, in order."""
    if n <= budget:
        return list(range(n))
    sure = set(range(sinks)) | set(range(n - recent, n))

    def rank(j):
        v = float(w[j])
        return (0 if math.isnan(v) else 1, 0.0 if math.isnan(v) else -v, j)

    rest = sorted((j for j in range(n) if j not in sure), key=rank)
    return sorted(sure | set(rest[:budget - sinks - recent]))


def assert_within(got, want, bound, what):
    got = got.double().cpu()
    assert torch.isfinite(got[torch.isfinite(want)]).all(), f"{what}: not finite"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities"
    err = (got - want).abs()[~inf]
    over = err > bound[~inf]
    assert not over.any(), (f"{what}: {int(over.sum())} of {over.numel()} outside the bound, worst "
                            f"{float((err / bound[~inf].clamp_min(1e-300)).max()):.3g} of it")
