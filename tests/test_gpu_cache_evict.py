"""Eviction by accumulated weight (fmx_cache_evict) against its definition:
out of place and in place, ragged lengths, ties, zeros of both signs, NaN and
infinities, budgets of one, protected ends alone, odd rows; the rest of the
arrays left as they were. And the operators' run together: decode steps with
append, scored attention and periodic eviction."""
from __future__ import annotations

import math

import pytest
import torch

import cache_oracle as R

pytestmark = pytest.mark.gpu


def _randn(shape, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)


def _check(k, v, w, lens, budget, sinks, recent, slots, got_k, got_v, got_w, before, lengths, kept):
    """got_*: the arrays written (before: what they held)."""
    n_slots, nkv, S, hd = k.shape
    S_out = got_k.shape[2]
    seen = set()
    gk, gv, gw = got_k.cpu(), got_v.cpu(), got_w.cpu()
    k, v, w = k.cpu(), v.cpu(), w.cpu()
    bk, bv, bw = (t.cpu() for t in before)
    kept = kept.cpu()
    for b, n in enumerate(lens):
        s = b if slots is None else slots[b]
        if not 0 <= s < n_slots:
            assert int(lengths[b]) == 0 and bool((kept[b] == -1).all())
            continue
        seen.add(s)
        n = min(max(n, 0), S)
        c = min(n, budget)
        assert int(lengths[b]) == c
        for g in range(nkv):
            idx = R.kept_positions(w[s, g], n, budget, sinks, recent)
            assert kept[b, g].tolist() == idx + [-1] * (budget - c), (b, g)
            assert torch.equal(gk[s, g, :c], k[s, g, idx]) and torch.equal(gv[s, g, :c], v[s, g, idx]), (b, g)
            assert torch.equal(torch.nan_to_num(gw[s, g, :c], nan=-7.0), torch.nan_to_num(w[s, g, idx], nan=-7.0))
            assert bool((gw[s, g, c:] == 0).all())
            assert torch.equal(gk[s, g, c:S_out], bk[s, g, c:S_out]) and torch.equal(gv[s, g, c:], bv[s, g, c:])
    for s in set(range(n_slots)) - seen:
        assert torch.equal(gk[s], bk[s]) and torch.equal(gv[s], bv[s]) and torch.equal(gw[s], bw[s])


def _both_ways(fmx, k, v, w, lens, budget, sinks, recent, slots=None, S_out=None):
    n_slots, nkv, S, hd = k.shape
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    sl = None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda")
    S_out = S_out or min(budget, S)
    out = (_randn((n_slots, nkv, S_out, hd), k.dtype, 90), _randn((n_slots, nkv, S_out, hd), k.dtype, 91),
           _randn((n_slots, nkv, S_out), torch.float32, 92))
    before, src = [t.clone() for t in out], [t.clone() for t in (k, v, w)]
    got, kept = fmx.cache_evict(k, v, w, lengths, budget, sinks=sinks, recent=recent, slots=sl, out=out)
    for t, s in zip((k, v, w), src):
        assert torch.equal(t.nan_to_num(), s.nan_to_num())  # the source is left alone
    _check(k, v, w, lens, budget, sinks, recent, slots, *out, before, got, kept)
    ki, vi, wi = (t.clone() for t in src)
    got2, kept2 = fmx.cache_evict(ki, vi, wi, lengths, budget, sinks=sinks, recent=recent, slots=sl,
                                  lengths_out=lengths)
    assert got2 is lengths and torch.equal(kept, kept2)
    _check(*src, lens, budget, sinks, recent, slots, ki, vi, wi, src, lengths, kept2)


@pytest.mark.parametrize("B,nkv,S,hd,budget,sinks,recent", [
    (1, 1, 1, 8, 1, 0, 0), (3, 2, 70, 64, 1, 0, 0), (3, 2, 70, 64, 1, 1, 0), (3, 2, 70, 64, 1, 0, 1),
    (2, 4, 1030, 128, 500, 4, 100), (2, 1, 5000, 128, 4000, 0, 1), (4, 3, 200, 80, 64, 64, 0),
    (4, 3, 200, 80, 64, 30, 34), (2, 2, 300, 33, 100, 3, 7), (2, 2, 64, 256, 200, 4, 4), (1, 2, 20000, 16, 9000, 1, 9),
    (2, 1, 3000, 1024, 1500, 0, 0)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_evict(gpu, fmx, dt, B, nkv, S, hd, budget, sinks, recent):
    k, v = _randn((B, nkv, S, hd), dt, 1), _randn((B, nkv, S, hd), dt, 2)
    w = torch.exp(2 * _randn((B, nkv, S), torch.float32, 3))
    lens = [[S, S - 1, budget, budget + 1][b % 4] for b in range(B)]
    _both_ways(fmx, k, v, w, lens, budget, sinks, recent, S_out=min(budget, S) + 3)


@pytest.mark.parametrize("hd", [511, 513, 769, 1023])
def test_evict_odd_wide_heads(gpu, fmx, hd):
    """Rows of an odd number of elements, longer than a workgroup."""
    B, nkv, S, budget = 2, 2, 90, 50
    k, v = _randn((B, nkv, S, hd), torch.bfloat16, 1), _randn((B, nkv, S, hd), torch.bfloat16, 2)
    _both_ways(fmx, k, v, _randn((B, nkv, S), torch.float32, 3), [S, 60], budget, 2, 8)


@pytest.mark.parametrize("kind", ["equal", "zeros", "few", "special", "negative", "close"])
def test_evict_ties_and_special_weights(gpu, fmx, kind):
    B, nkv, S, hd, budget = 2, 2, 2100, 16, 700
    k, v = _randn((B, nkv, S, hd), torch.bfloat16, 1), _randn((B, nkv, S, hd), torch.bfloat16, 2)
    w = _randn((B, nkv, S), torch.float32, 3)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "zeros":
        w = torch.where(w > 0, 0.0, -0.0)
    elif kind == "few":
        w = torch.round(w * 2)
    elif kind == "special":
        w[:, :, ::7], w[:, :, 3::50], w[:, :, 5::11] = math.nan, math.inf, -math.inf
        w[:, 0, 100:110] = -math.nan
    elif kind == "negative":
        w = -w.abs() - 1
    else:  # neighbouring floats
        w = (torch.full_like(w, 1.0).view(torch.int32) + (w * 3).to(torch.int32)).view(torch.float32)
    _both_ways(fmx, k, v, w, [S, S - 5], budget, 4, 100)


def test_evict_slots(gpu, fmx):
    n, nkv, S, hd = 6, 2, 90, 64
    k, v, w = _randn((n, nkv, S, hd), torch.float16, 1), _randn((n, nkv, S, hd), torch.float16, 2), _randn((n, nkv, S), torch.float32, 3)
    _both_ways(fmx, k, v, w, [90, 50, -3, 200, 40, 0], 41, 2, 8, slots=[4, 0, 2, 1, -1, 5], S_out=50)
    _both_ways(fmx, k, v, w, [90, 90], 41, 2, 8, slots=[6, 3])


def test_evict_strided(gpu, fmx):
    """Positions before heads, rows at odd elements, the caches of one layer
    of a [layers, 2, slots, ...] array."""
    n, nkv, S, hd = 2, 3, 60, 20
    big = _randn((2, 2, n, S, nkv, hd + 1), torch.bfloat16, 1)
    ref = big.clone()
    k, v = big[1, 0, ..., 1:].transpose(1, 2), big[1, 1, ..., 1:].transpose(1, 2)
    w = _randn((n, nkv, S), torch.float32, 2)
    w0, k0, v0 = w.clone(), k.clone(), v.clone()
    lens = torch.tensor([60, 44], dtype=torch.int32, device="cuda")
    got, kept = fmx.cache_evict(k, v, w, lens, 20, sinks=1, recent=3)
    _check(k0, v0, w0, [60, 44], 20, 1, 3, None, k, v, w, (k0, v0, w0), got, kept)
    assert torch.equal(big[0], ref[0]) and torch.equal(big[..., 0], ref[..., 0])


@pytest.mark.parametrize("nh,nkv,interleaved", [(8, 2, False), (4, 4, True)])
def test_decode_with_eviction(gpu, fmx, nh, nkv, interleaved):
    """A run of all the operators: a prompt's attention sets the weights, then
    decode steps append at the caches' own offsets (positions run on), attend,
    add weights and cut the cache back to the budget every few steps; against
    a 64-bit run of the same steps with the kernel's choice of positions, and
    in one captured step against the eager one."""
    B, L, hd, budget, sinks, recent, room = 3, 50, 64, 40, 2, 8, 6
    S = L + room
    dt, scale = torch.float16, 0.125
    rope = fmx.Rope(fmx.RopeConfig(dims=hd, interleaved=interleaved, scaling="yarn", factor=4.0))
    kc, vc = (torch.zeros(B, nkv, S, hd, dtype=dt, device="cuda") for _ in range(2))
    w = torch.zeros(B, nkv, S, dtype=torch.float32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    step = [0]

    def qkv(n):
        step[0] += 1
        return (_randn((B, n, nh, hd), dt, 1000 + step[0]), _randn((B, n, nkv, hd), dt, 2000 + step[0]),
                _randn((B, n, nkv, hd), dt, 3000 + step[0]))

    def forward(q, k, v, pos):
        qr = rope.append(q, k, v, pos, lens, kc, vc)
        return qr, fmx.attention_scored(qr, kc, vc, lens, scale, weights=w, weights_out=w)[0]

    def check(qr, got, w_before):
        r = R.attention(qr, kc, vc, lens, scale)
        R.assert_within(got, r["out"], r["out_b"], "out")
        R.assert_within(w, r["w"] + w_before.double().cpu(), r["w_b"] + w_before.abs().cpu() * 2.0 ** -23, "weights")

    pos = torch.arange(L, dtype=torch.int32, device="cuda").expand(B, L).contiguous()
    w0 = w.clone()
    check(*forward(*qkv(L), pos), w0)
    lens += L
    pos = torch.full((B, 1), L, dtype=torch.int32, device="cuda")
    for i in range(12):
        if int(lens.max()) + 1 > S or i == 0:
            k0, v0, wb, l0 = kc.clone(), vc.clone(), w.clone(), lens.tolist()
            _, kept = fmx.cache_evict(kc, vc, w, lens, budget, sinks=sinks, recent=recent, lengths_out=lens)
            _check(k0, v0, wb, l0, budget, sinks, recent, None, kc, vc, w, (k0, v0, wb), lens, kept)
        args, w0 = qkv(1), w.clone()
        check(*forward(*args, pos), w0)
        lens += 1
        pos += 1
    # one captured step, cut included, replayed against eager copies
    args = qkv(1)
    state = [t.clone() for t in (kc, vc, w, lens)]

    def whole():
        fmx.cache_evict(kc, vc, w, lens, budget, sinks=sinks, recent=recent, lengths_out=lens)
        return forward(*args, pos)[1]

    whole()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out_g = whole()
    for _ in range(3):
        results = []
        for run in (lambda: (g.replay(), out_g)[1], whole):
            for t, s in zip((kc, vc, w, lens), state):
                t.copy_(s)
            o = run()
            torch.cuda.synchronize()
            results.append([o.clone()] + [t.clone() for t in (kc, vc, w, lens)])
        assert all(torch.equal(a, b) for a, b in zip(*results))
