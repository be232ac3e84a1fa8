"""The cache's long-context operators at the edges of their range: empty
batches, loads past the caches, eviction without the kept positions."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

import cache_oracle as R

pytestmark = pytest.mark.gpu


def _randn(shape, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)


@pytest.mark.parametrize("B,L", [(0, 1), (0, 40), (3, 0), (0, 0)])
@pytest.mark.parametrize("P,S", [(0, 9), (20, 9), (20, 0)])
def test_empty_batches(gpu, fmx, B, L, P, S):
    """No sequences, or no new tokens: empty results, caches and weights as they were."""
    nh, nkv, hd, n, dt = 8, 2, 64, 3, torch.bfloat16
    q, k = _randn((B, L, nh, hd), dt, 1), _randn((B, L, nkv, hd), dt, 2)
    kc, vc = _randn((n, nkv, S, hd), dt, 3), _randn((n, nkv, S, hd), dt, 4)
    kp = vp = _randn((nkv, P, hd), dt, 5) if P else None
    offs = torch.zeros(B, dtype=torch.int32, device="cuda")
    pos = torch.zeros((B, L), dtype=torch.int32, device="cuda")
    out, lse = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 0.1)
    assert out.shape == q.shape and lse.shape == (B, L, nh)
    rope = fmx.Rope(fmx.RopeConfig(dims=hd))
    assert rope(q, pos).shape == q.shape
    if S:
        before = kc.clone(), vc.clone()
        assert rope.append(q, k, k, pos, offs, kc, vc).shape == q.shape
        w = _randn((n, nkv, S), torch.float32, 6)
        out, w_out = fmx.attention_scored(q, kc, vc, offs, 0.1, weights=w)
        assert out.shape == q.shape and torch.equal(w_out, w)
        assert bool((fmx.attention_scored(q, kc, vc, offs, 0.1)[1] == 0).all())
        if B == 0:
            lengths, kept = fmx.cache_evict(kc, vc, w, offs, 4)
            assert lengths.shape == (0,) and kept.shape == (0, nkv, 4)
        assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


@pytest.mark.parametrize("S", [1, 300])
@pytest.mark.parametrize("given", [False, True])
def test_no_queries_keep_the_weights(gpu, fmx, given, S):
    """seq_len 0 adds an empty sum: a weights array of its own gets what was
    there (or 0) in the sequences' slots, and only there."""
    n, nkv, hd, dt = 4, 2, 64, torch.bfloat16
    q = torch.empty((3, 0, 8, hd), dtype=dt, device="cuda")
    kc, vc = _randn((n, nkv, S, hd), dt, 1), _randn((n, nkv, S, hd), dt, 2)
    w, w_out = _randn((n, nkv, S), torch.float32, 3), _randn((n, nkv, S), torch.float32, 4)
    slots = torch.tensor([2, -1, 0], dtype=torch.int32, device="cuda")
    offs = torch.full((3,), 5, dtype=torch.int32, device="cuda")
    want = w_out.clone()
    want[[2, 0]] = w[[2, 0]] if given else 0.0
    _, got = fmx.attention_scored(q, kc, vc, offs, 0.1, weights=w if given else None, weights_out=w_out, slots=slots)
    assert got is w_out and torch.equal(w_out, want)
    fmx.attention_scored(q, kc, vc, offs, 0.1, weights=w_out, weights_out=w_out, slots=slots)
    assert torch.equal(w_out, want)


def test_rope_of_the_most_rows(gpu, fmx):
    """2^24 rows of a workgroup each are more threads than one launch takes."""
    B, L, hd = 1 << 12, 1 << 12, 514  # (an odd number of 16-byte vectors: one pair per thread)
    x = _randn((1, 1, 1, hd), torch.bfloat16, 1)
    pos = torch.arange(B * L, dtype=torch.int32, device="cuda").view(B, L)
    rope = fmx.Rope(fmx.RopeConfig(dims=hd))
    out = rope(x.expand(B, L, 1, hd), pos)
    for b, l in ((0, 0), (B // 2, 7), (B - 1, L - 2), (B - 1, L - 1)):
        assert torch.equal(out[b, l], rope(x, pos[b:b + 1, l:l + 1].contiguous())[0, 0]), (b, l)
    # (every row but position 0's turns some element)
    assert int((out[:, :, 0, 0] == 0).sum()) == int((x[..., 0] == 0).sum()) * B * L
    del out
    torch.cuda.empty_cache()


def _long_cache(B, L, nh, nkv, hd, P, S, seen, dt, seed):
    """Caches of S positions of which sequences use up to `seen`; the rest are
    NaN keys and infinite values."""
    q = _randn((B, L, nh, hd), dt, seed)
    kc = torch.full((B, nkv, S, hd), math.nan, dtype=dt, device="cuda")
    vc = torch.full((B, nkv, S, hd), math.inf, dtype=dt, device="cuda")
    marks = [seen, 0, 1, seen - 1, seen // 2, 17, 130, 33]
    lens = [min(marks[b % len(marks)], seen) for b in range(B)]
    for b, n in enumerate(lens):
        kc[b, :, :n], vc[b, :, :n] = _randn((nkv, n, hd), dt, seed + 10 + b), _randn((nkv, n, hd), dt, seed + 500 + b)
    offs = torch.tensor([n - L for n in lens], dtype=torch.int32, device="cuda")
    kp, vp = (_randn((nkv, P, hd), dt, seed + 1), _randn((nkv, P, hd), dt, seed + 2)) if P else (None, None)
    small = [torch.nan_to_num(t[:, :, :seen], nan=0.0, posinf=0.0) for t in (kc, vc)]
    return q, kp, vp, kc, vc, small, offs


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("B,L,nh,nkv,hd,P,S,seen", [
    # narrow tiles alone: one row set, one query (heads of a template and others) and several
    (3, 1, 16, 4, 128, 0, 50000, 700), (4, 1, 4, 4, 64, 70, 70000, 500), (2, 1, 8, 2, 256, 33, 70000, 400),
    (2, 1, 8, 2, 80, 0, 220000, 300), (2, 3, 8, 2, 64, 40, 270000, 333), (2, 2, 6, 3, 96, 515, 120000, 290),
    (2, 2, 8, 2, 256, 20, 70000, 260),
    # two row sets
    (2, 5, 8, 2, 128, 0, 140000, 700), (2, 5, 8, 2, 72, 0, 240000, 300), (3, 1, 24, 1, 64, 0, 360000, 400),
    # beside a prefix in wide tiles
    (40, 1, 8, 2, 128, 300, 7000, 600), (36, 1, 4, 4, 64, 200, 8000, 260), (40, 2, 8, 4, 80, 150, 6000, 200),
    (10, 5, 8, 2, 64, 400, 60000, 300), (10, 5, 8, 2, 128, 150, 30000, 280), (36, 1, 2, 2, 256, 100, 4000, 150)])
def test_caches_beyond_256_mb(gpu, fmx, dt, B, L, nh, nkv, hd, P, S, seen):
    """From 256 MB of prefix and caches on, narrow tiles load past the caches."""
    assert (P + B * S) * nkv * hd * 4 > 256 << 20
    q, kp, vp, kc, vc, small, offs = _long_cache(B, L, nh, nkv, hd, P, S, seen, dt, hd + B)
    scale = hd ** -0.5
    out, lse = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, scale)
    r = R.attention(q, *small, offs, scale, kp=kp, vp=vp)
    R.assert_within(out, r["out"], r["out_b"], "out")
    R.assert_within(lse, r["lse"], r["lse_b"], "lse")
    if P:
        r = R.attention(q, *small, offs, scale)
    out, w = fmx.attention_scored(q, kc, vc, offs, scale)
    R.assert_within(out, r["out"], r["out_b"], "out of the scored call")
    R.assert_within(w[:, :, :seen], r["w"], r["w_b"], "weights")
    assert bool((w[:, :, seen:] == 0).all())


@pytest.mark.parametrize("own_workspace", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_without_kept_positions(gpu, fmx, in_place, own_workspace):
    """kept NULL: the positions stay in the workspace, the caller's or the call's own."""
    from flashmlx_amd import _lib
    from flashmlx_amd._lib import FmxHeads
    lib = _lib.load()
    B, nkv, S, hd, budget = 3, 2, 700, 64, 300
    k, v = _randn((B, nkv, S, hd), torch.bfloat16, 1), _randn((B, nkv, S, hd), torch.bfloat16, 2)
    w = _randn((B, nkv, S), torch.float32, 3)
    lens = torch.tensor([700, 250, 301], dtype=torch.int32, device="cuda")

    def outputs():
        if in_place:
            return k.clone(), v.clone(), w.clone()
        return tuple(torch.zeros((B, nkv, budget) + t, dtype=d, device="cuda")
                     for t, d in (((hd,), k.dtype), ((hd,), k.dtype), ((), w.dtype)))

    want = outputs()
    src = want if in_place else (k, v, w)
    lens_want, _ = fmx.cache_evict(*src, lens, budget, sinks=4, recent=20, out=None if in_place else want)
    got = outputs()
    src = got if in_place else (k, v, w)

    def heads(t):
        return C.byref(FmxHeads(t.data_ptr(), t.stride(0), t.stride(2), t.stride(1)))

    need = lib.fmx_cache_evict_workspace_size(B, nkv, budget)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    lens_got = torch.empty_like(lens)
    to = (None, None, None, 0) if in_place else (heads(got[0]), heads(got[1]), got[2].data_ptr(), budget)
    _lib.check(lib.fmx_cache_evict(
        _lib.FMX_BF16, B, nkv, hd, heads(src[0]), heads(src[1]), src[2].data_ptr(), B, S, lens.data_ptr(), None, budget, 4,
        20, *to, lens_got.data_ptr(), None, ws.data_ptr() if own_workspace else None, need if own_workspace else 0,
        torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(lens_got, lens_want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("budget", [0, -1, (1 << 24) + 1, 1 << 40])
def test_evict_refuses_a_budget_before_memory_is_taken(gpu, fmx, budget):
    kc = torch.zeros((2, 2, 9, 8), dtype=torch.bfloat16, device="cuda")
    w, lens = torch.zeros((2, 2, 9), device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    with pytest.raises(ValueError, match="budget"):
        fmx.cache_evict(kc, kc.clone(), w, lens, budget)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
