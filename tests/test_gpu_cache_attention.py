"""Attention over a shared prefix and over own caches with the keys' weights
(fmx_attention_shared_prefix, fmx_attention_scored) against 64 bits: head
layouts, sizes on both sides of the tiles', one to many queries per sequence,
ragged lengths, rows that see nothing, strides, slots, NaN and infinities
where no query may look; captured calls; more than 2^32 bytes of cache."""
from __future__ import annotations

import math

import pytest
import torch

import cache_oracle as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _randn(shape, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)


def _lengths(B, S, L):
    """Own positions per sequence, from none to all of the cache."""
    marks = [S, 0, 1, S - 1, S // 2, 17, 64, 3, 33, 16, 32, 15, 63, 65]
    return [min(max(marks[b % len(marks)], 0), S) for b in range(B)]


def _inputs(dt, B, L, nh, nkv, hd, P, S, seed=0):
    q = _randn((B, L, nh, hd), dt, seed + 1)
    kc, vc = _randn((B, nkv, S, hd), dt, seed + 2), _randn((B, nkv, S, hd), dt, seed + 3)
    kp, vp = (_randn((nkv, P, hd), dt, seed + 4), _randn((nkv, P, hd), dt, seed + 5)) if P else (None, None)
    offs = torch.tensor([n - L for n in _lengths(B, S, L)], dtype=torch.int32, device="cuda")
    return q, kp, vp, kc, vc, offs


def _blank(kc, vc, offs, L):
    """Cache positions that no query sees: NaN keys and infinite values."""
    for b, off in enumerate(offs.tolist()):
        n = max(off + L, 0)
        kc[b, :, n:] = math.nan
        vc[b, :, n:] = math.inf


def _finite(t):
    return torch.nan_to_num(t, nan=0.0, posinf=0.0, neginf=0.0)


SHAPES = [
    # B, L, nh, nkv, hd
    (1, 1, 1, 1, 64), (3, 1, 16, 16, 128), (6, 1, 32, 4, 128), (14, 1, 8, 1, 64), (2, 1, 14, 2, 256),
    (3, 1, 20, 1, 80), (2, 1, 4, 4, 8), (4, 5, 8, 2, 64), (3, 2, 40, 2, 96), (2, 3, 6, 3, 128),
]


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("P,S", [(0, 70), (1, 1), (17, 33), (200, 0), (515, 130)])
def test_shared_prefix(gpu, fmx, dt, shape, P, S):
    B, L, nh, nkv, hd = shape
    q, kp, vp, kc, vc, offs = _inputs(DT[dt], B, L, nh, nkv, hd, P, S)
    _blank(kc, vc, offs, L)
    scale = 1 / math.sqrt(hd)
    out, lse = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, scale)
    r = R.attention(q, _finite(kc), _finite(vc), offs, scale, kp=kp, vp=vp)
    R.assert_within(out, r["out"], r["out_b"], "out")
    R.assert_within(lse, r["lse"], r["lse_b"], "lse")


@pytest.mark.parametrize("B,L,nh,nkv,hd,P,S", [
    (40, 1, 32, 4, 128, 300, 40),     # many rows over the prefix
    (9, 16, 8, 4, 64, 129, 70),
    (1, 150, 4, 2, 128, 0, 150),      # a prompt
    (2, 77, 7, 1, 64, 40, 200),       # chunks behind a prefix and a context
    (1, 65, 2, 2, 256, 33, 65),
    (1, 40, 3, 3, 72, 5, 64),
    (2, 1, 4, 4, 128, 4111, 5000),    # long, few rows
])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_shared_prefix_many_rows(gpu, fmx, dt, B, L, nh, nkv, hd, P, S):
    q, kp, vp, kc, vc, _ = _inputs(DT[dt], B, L, nh, nkv, hd, P, S, seed=50)
    offs = torch.tensor([(S - L) * (b + 1) // B for b in range(B)], dtype=torch.int32, device="cuda")
    _blank(kc, vc, offs, L)
    scale = 1 / math.sqrt(hd)
    out, lse = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, scale)
    r = R.attention(q, _finite(kc), _finite(vc), offs, scale, kp=kp, vp=vp)
    R.assert_within(out, r["out"], r["out_b"], "out")
    R.assert_within(lse, r["lse"], r["lse_b"], "lse")


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("S", [1, 70, 515])
def test_scored(gpu, fmx, dt, shape, S):
    B, L, nh, nkv, hd = shape
    q, _, _, kc, vc, offs = _inputs(DT[dt], B, L, nh, nkv, hd, 0, S, seed=9)
    _blank(kc, vc, offs, L)
    w = _randn((B, nkv, S), torch.float32, 77)
    scale = 1 / math.sqrt(hd)
    r = R.attention(q, _finite(kc), _finite(vc), offs, scale)
    out, w_out = fmx.attention_scored(q, kc, vc, offs, scale, weights=w)
    R.assert_within(out, r["out"], r["out_b"], "out")
    R.assert_within(w_out, r["w"] + w.double().cpu(), r["w_b"] + w.abs().cpu() * 2.0 ** -23, "weights")
    out2, w_new = fmx.attention_scored(q, kc, vc, offs, scale)
    R.assert_within(w_new, r["w"], r["w_b"], "weights from nothing")
    w2 = w.clone()
    out3, w3 = fmx.attention_scored(q, kc, vc, offs, scale, weights=w2, weights_out=w2)
    assert w3 is w2 and torch.equal(w2, w_out)  # in place, equal bits
    assert torch.equal(out, out2) and torch.equal(out, out3)


@pytest.mark.parametrize("B,L,nh,nkv,hd,S", [(1, 150, 4, 2, 128, 150), (2, 77, 7, 1, 64, 200), (1, 65, 2, 2, 256, 65),
                                             (3, 33, 8, 2, 80, 100), (1, 300, 16, 1, 128, 310)])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_scored_prompt(gpu, fmx, dt, B, L, nh, nkv, hd, S):
    q, _, _, kc, vc, _ = _inputs(DT[dt], B, L, nh, nkv, hd, 0, S, seed=21)
    offs = torch.tensor([(S - L) * (b + 1) // B for b in range(B)], dtype=torch.int32, device="cuda")
    _blank(kc, vc, offs, L)
    scale = 1 / math.sqrt(hd)
    r = R.attention(q, _finite(kc), _finite(vc), offs, scale)
    out, w = fmx.attention_scored(q, kc, vc, offs, scale)
    R.assert_within(out, r["out"], r["out_b"], "out")
    R.assert_within(w, r["w"], r["w_b"], "weights")


@pytest.mark.parametrize("L,rep", [(3, 2), (40, 4)])
def test_later_keys_do_not_reach_earlier_queries(gpu, fmx, L, rep):
    """The newest token's key and value are NaN and infinite: every query but
    the newest is as without them, to the bit of a call that has zeros there."""
    hd, S = 64, 48
    q, _, _, kc, vc, _ = _inputs(torch.bfloat16, 1, L, 2 * rep, 2, hd, 0, S, seed=31)
    offs = torch.tensor([S - L], dtype=torch.int32, device="cuda")
    kz, vz = kc.clone(), vc.clone()
    kz[:, :, S - 1], vz[:, :, S - 1] = 0, 0
    for bad_k, bad_v in ((math.nan, math.nan), (math.inf, math.inf), (0.0, -math.inf)):
        kc[:, :, S - 1], vc[:, :, S - 1] = bad_k, bad_v
        out, lse = fmx.attention_shared_prefix(q, None, None, kc, vc, offs, 0.125)
        want, lse_z = fmx.attention_shared_prefix(q, None, None, kz, vz, offs, 0.125)
        assert torch.equal(out[:, :L - 1], want[:, :L - 1]) and torch.equal(lse[:, :L - 1], lse_z[:, :L - 1])
        if bad_k == 0.0:
            assert bool((out[:, L - 1] == -math.inf).all())
        else:
            assert not bool(torch.isfinite(out[:, L - 1]).any())


@pytest.mark.parametrize("B,L,nh,nkv,hd,P,S", [
    (300, 1, 4, 1, 64, 40, 20),       # more sequences than threads in a workgroup
    (300, 1, 32, 4, 64, 200, 12),     # more rows than the join has waves
    (1, 1, 2, 1, 64, 20000, 300),     # more pieces than lanes
    (2, 1, 2, 1, 128, 0, 30000),
    (1, 40, 4, 1, 64, 50, 2100),      # own keys of wide tiles in several pieces
    (2, 9, 8, 2, 256, 700, 1100),
    (36, 1, 2, 2, 256, 600, 40),      # wide prefix, narrow own keys, wide heads
    (20, 3, 16, 2, 80, 500, 70),
])
def test_shared_prefix_plans(gpu, fmx, B, L, nh, nkv, hd, P, S):
    """Both sides of every choice of tiles, pieces and joins."""
    q, kp, vp, kc, vc, offs = _inputs(torch.float16, B, L, nh, nkv, hd, P, S, seed=80)
    _blank(kc, vc, offs, L)
    scale = 1 / math.sqrt(hd)
    out, lse = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, scale)
    r = R.attention(q, _finite(kc), _finite(vc), offs, scale, kp=kp, vp=vp)
    R.assert_within(out, r["out"], r["out_b"], "out")
    R.assert_within(lse, r["lse"], r["lse_b"], "lse")


@pytest.mark.parametrize("B,L,nh,nkv,hd,S", [
    (300, 1, 4, 1, 64, 20), (300, 1, 32, 4, 64, 12), (2, 1, 2, 1, 128, 30000), (1, 40, 4, 1, 64, 2100),
    (2, 9, 8, 2, 256, 1100), (2, 600, 4, 1, 64, 900)])
def test_scored_plans(gpu, fmx, B, L, nh, nkv, hd, S):
    q, _, _, kc, vc, offs = _inputs(torch.bfloat16, B, L, nh, nkv, hd, 0, S, seed=81)
    _blank(kc, vc, offs, L)
    scale = 1 / math.sqrt(hd)
    r = R.attention(q, _finite(kc), _finite(vc), offs, scale)
    out, w = fmx.attention_scored(q, kc, vc, offs, scale)
    R.assert_within(out, r["out"], r["out_b"], "out")
    R.assert_within(w, r["w"], r["w_b"], "weights")


def test_slots_and_unused_sequences(gpu, fmx):
    B, nh, nkv, hd, S, n = 5, 8, 2, 64, 50, 7
    q = _randn((B, 1, nh, hd), torch.bfloat16, 1)
    kc, vc = _randn((n, nkv, S, hd), torch.bfloat16, 2), _randn((n, nkv, S, hd), torch.bfloat16, 3)
    kp, vp = _randn((nkv, 20, hd), torch.bfloat16, 4), _randn((nkv, 20, hd), torch.bfloat16, 5)
    slots = torch.tensor([6, -1, 2, n, 0], dtype=torch.int32, device="cuda")
    offs = torch.tensor([49, 3, -7, 2, 60], dtype=torch.int32, device="cuda")  # 60: ends at the cache's end
    r = R.attention(q, kc, vc, offs, 0.2, slots=slots, kp=kp, vp=vp)
    out, lse = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 0.2, slots=slots)
    R.assert_within(out, r["out"], r["out_b"], "out")
    R.assert_within(lse, r["lse"], r["lse_b"], "lse")
    r = R.attention(q, kc, vc, offs, 0.2, slots=slots)
    w = _randn((n, nkv, S), torch.float32, 6)
    out, w_out = fmx.attention_scored(q, kc, vc, offs, 0.2, weights=w, slots=slots)
    R.assert_within(out, r["out"], r["out_b"], "out")
    assert bool((out[1] == 0).all()) and bool((out[2] == 0).all()) and bool((out[3] == 0).all())
    R.assert_within(w_out, r["w"] + w.double().cpu(), r["w_b"] + w.abs().cpu() * 2.0 ** -23, "weights")
    for s in (1, 2, 3, 4, 5):
        assert torch.equal(w_out[s], w[s])
    # the same cache read by two sequences
    both = torch.tensor([3, 3, 3, 4, 4], dtype=torch.int32, device="cuda")
    r = R.attention(q, kc, vc, offs, 0.2, slots=both, kp=kp, vp=vp)
    out, _ = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 0.2, slots=both)
    R.assert_within(out, r["out"], r["out_b"], "out")


def test_strided_arrays(gpu, fmx):
    """q inside a fused row, caches with positions before heads, a prefix that
    is a slot of a larger cache, out heads before tokens; what lies between
    the rows is left alone."""
    B, L, nh, nkv, hd, S, P = 3, 2, 8, 4, 128, 40, 50
    fused = _randn((B, L, (nh + 2) * hd), torch.float16, 1)
    q = fused[:, :, hd:-hd].unflatten(2, (nh, hd))
    kc, vc = (_randn((B, S, nkv, hd), torch.float16, i).transpose(1, 2) for i in (2, 3))
    pool = _randn((2, 2, nkv, P + 9, hd), torch.float16, 4)
    kp, vp = pool[0, 1, :, 4:P + 4], pool[1, 0, :, :P]
    offs = torch.tensor([S - L, 5, -1], dtype=torch.int32, device="cuda")
    buf = torch.full((B, nh + 1, L + 1, hd), 3.0, dtype=torch.float16, device="cuda")
    out = buf[:, 1:, 1:].transpose(1, 2)
    fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 0.1, out=out)
    r = R.attention(q, kc, vc, offs, 0.1, kp=kp, vp=vp)
    R.assert_within(out, r["out"], r["out_b"], "out")
    want, _ = fmx.attention_shared_prefix(q.contiguous(), kp.contiguous(), vp.contiguous(), kc.contiguous(),
                                          vc.contiguous(), offs, 0.1)
    assert torch.equal(out, want)
    out.fill_(3.0)
    assert bool((buf == 3.0).all())


@pytest.mark.parametrize("L", [1, 40])
def test_large_scores(gpu, fmx, L):
    """Scores in the hundreds, one key far above the rest, equal keys."""
    hd, S = 128, 300
    q, _, _, kc, vc, _ = _inputs(torch.bfloat16, 2, L, 4, 2, hd, 0, S, seed=3)
    offs = torch.tensor([S - L, S - L - 60], dtype=torch.int32, device="cuda")
    q, kc = q * 8, kc * 4
    kc[1] = kc[1, :, :1]
    r = R.attention(q, kc, vc, offs, 0.5)
    out, w = fmx.attention_scored(q, kc, vc, offs, 0.5)
    R.assert_within(out, r["out"], r["out_b"], "out")
    R.assert_within(w, r["w"], r["w_b"], "weights")


@pytest.mark.parametrize("L,own", [(1, 700), (4, 90), (70, 500)])
def test_captured_calls_follow_device_lengths(gpu, fmx, L, own):
    """Both calls in one graph with workspaces shared between two graphs;
    every replay, with the lengths advanced in between, equals an eager call."""
    B, nh, nkv, hd, S, P = 3, 8, 2, 64, own + 20, 100
    q, kp, vp, kc, vc, _ = _inputs(torch.bfloat16, B, L, nh, nkv, hd, P, S, seed=60)
    offs = torch.tensor([own - L, 5, -1], dtype=torch.int32, device="cuda")
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    out, out2 = torch.empty_like(q), torch.empty_like(q)
    w = torch.zeros((B, nkv, S), dtype=torch.float32, device="cuda")
    w_out = torch.empty_like(w)

    def calls():
        lse = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 0.125, out=out, workspace=ws)[1]
        fmx.attention_scored(q, kc, vc, offs, 0.125, weights=w, weights_out=w_out, out=out2, workspace=ws)
        return lse

    calls()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            lse = calls()
        graphs.append((g, lse))
    for i in range(4):
        g, lse = graphs[i % 2]
        for t in (out, out2, w_out):
            t.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        e1, elin = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 0.125)
        e2, ew = fmx.attention_scored(q, kc, vc, offs, 0.125, weights=w)
        assert torch.equal(out, e1) and torch.equal(lse, elin) and torch.equal(out2, e2) and torch.equal(w_out, ew)
        offs += 3


def test_other_stream(gpu, fmx):
    q, kp, vp, kc, vc, offs = _inputs(torch.bfloat16, 4, 1, 8, 2, 64, 300, 70)
    want = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 0.125)[0]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 0.125)[0]
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("B,L,P,S", [(4, 1, 300, 700), (40, 1, 700, 300), (2, 150, 60, 300)])
def test_two_streams_at_once(gpu, fmx, B, L, P, S):
    """Both attentions in flight on two streams over the same inputs."""
    q, kp, vp, kc, vc, offs = _inputs(torch.bfloat16, B, L, 8, 2, 64, P, S, seed=70)
    want = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 0.125)
    want_s = fmx.attention_scored(q, kc, vc, offs, 0.125)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append((fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 0.125),
                        fmx.attention_scored(q, kc, vc, offs, 0.125)))
    torch.cuda.synchronize()
    for shared, scored in got:
        assert all(torch.equal(x, y) for x, y in zip(shared + scored, want + want_s))


@pytest.mark.parametrize("L", [1, 70])
def test_offsets_beyond_32_bits(gpu, fmx, L):
    """Slots and positions more than 2^32 elements apart: two heads of one
    sequence 2^32 + 8 elements apart in one allocation (zero but for them)."""
    hd, S = 64, 96
    far = 2 ** 32 + 64
    base = torch.zeros(far + 2 * S * hd, dtype=torch.bfloat16, device="cuda")
    kc = torch.as_strided(base, (1, 2, S, hd), (0, far, hd, 1), 0)
    vc = torch.as_strided(base, (1, 2, S, hd), (0, far, hd, 1), S * hd)
    small_k, small_v = _randn((1, 2, S, hd), torch.bfloat16, 1), _randn((1, 2, S, hd), torch.bfloat16, 2)
    kc.copy_(small_k)
    vc.copy_(small_v)
    q = _randn((1, L, 4, hd), torch.bfloat16, 3)
    offs = torch.tensor([S - L], dtype=torch.int32, device="cuda")
    a = fmx.attention_scored(q, kc, vc, offs, 0.125)
    b = fmx.attention_scored(q, small_k, small_v, offs, 0.125)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    del base, kc, vc
    torch.cuda.empty_cache()
