"""The cache's long-context operators at the edges of their range: empty
batches, loads past the caches, eviction without the kept positions."""
from __future__ import annotations

import pytest
import torch

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
