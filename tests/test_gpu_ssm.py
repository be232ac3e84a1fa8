"""The state space layer's operators on the GPU against their definitions in
64 bits: every type, odd sizes, ragged batches, slots, strides, and a layer's
prompts and steps run together."""
from __future__ import annotations

import math

import pytest
import torch

import ssm_oracle as O

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
LIMITS = (0.001, 0.5)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype)


def _cut(t, pad, dtype):
    """t as a slice of wider rows filled with NaN."""
    wide = torch.full((*t.shape[:-1], t.shape[-1] + 2 * pad), math.nan, dtype=dtype)
    wide[..., pad:pad + t.shape[-1]] = t
    return wide.cuda()[..., pad:pad + t.shape[-1]]


def _lens(lengths):
    return None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")


def _untouched(out, lengths):
    for b, n in enumerate(lengths or []):
        assert (out[b, max(n, 0):] == 7.0).all(), "rows behind a sequence"


# ------------------------------------------------------------------ convolution

@pytest.mark.parametrize("dtype,B,L,C,taps,silu,lengths,slots,pad", [
    (BF16, 1, 1, 64, 4, True, None, None, 0), (BF16, 3, 29, 96, 4, True, [29, 1, 0], [2, 0, 1], 8),
    (F16, 2, 17, 40, 3, True, [2, 16], [4, -1], 8), (F32, 2, 9, 12, 2, False, [1, 9], None, 4),
    (BF16, 2, 13, 37, 4, True, [13, 2], None, 3), (F16, 1, 8, 8, 1, True, None, None, 0),
    (F32, 2, 21, 20, 8, True, [3, 21], [1, 0], 1), (BF16, 2, 1, 264, 8, True, None, [0, 9], 0),
    (F16, 4, 5, 7, 5, False, [0, 1, 4, 5], [3, 2, 1, 0], 2), (BF16, 2, 19, 96, 4, True, [19, 6], None, 2),
    (F16, 2, 10, 8, 7, True, None, None, 6)])
@pytest.mark.parametrize("begun,keep", [(False, "out"), (True, "in place"), (True, "no")])
def test_conv(gpu, fmx, dtype, B, L, C, taps, silu, lengths, slots, pad, begun, keep):
    g = _gen(L * C + taps)
    x = _cut(_randn(g, B, L, C, dtype=dtype), pad, dtype)
    w, bias = _randn(g, C, taps, dtype=dtype).cuda(), _randn(g, C, dtype=dtype).cuda()
    state = _randn(g, 5, taps - 1, C, dtype=dtype).cuda()
    first = state if begun else None
    sl = None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda")
    want, bound, after = O.conv(x, w, bias, silu, first, 5, lengths, slots)
    out = torch.full((B, L, C), 7.0, dtype=dtype, device="cuda")
    for b, n in enumerate(lengths or []):
        x[b, n:] = math.nan
    s_out = {"out": torch.full_like(state, 3.0), "in place": state, "no": None}[keep]
    print("conv", dtype, B, L, C, taps, flush=True)
    fmx.causal_conv(x, w, bias, first, s_out, _lens(lengths), sl, "silu" if silu else None, out)
    torch.cuda.synchronize()
    _untouched(out, lengths)
    for b in range(B):
        n = L if lengths is None else lengths[b]
        O.assert_within(out[b, :n], want[b, :n], bound[b, :n], f"row {b}")
    if keep == "no" or taps == 1:
        return
    used = [O._slot(slots, 5, b) for b in range(B)]
    for s in range(5):
        if s in used:
            assert torch.equal(s_out[s].double().cpu(), after[s]), f"state {s}"
        elif keep == "out":
            assert (s_out[s] == 3.0).all()


def test_conv_in_chunks_is_the_whole(gpu, fmx):
    """Any cut into chunks gives the bits of one call."""
    g = _gen(5)
    x, w = _randn(g, 2, 41, 72, dtype=BF16).cuda(), _randn(g, 72, 4, dtype=BF16).cuda()
    whole = fmx.causal_conv(x, w)
    state = torch.zeros(2, 3, 72, dtype=BF16, device="cuda")
    parts, t = [], 0
    for n in (1, 2, 1, 8, 9, 20):
        parts.append(fmx.causal_conv(x[:, t:t + n], w, state=state, state_out=state))
        t += n
    assert t == 41 and torch.equal(torch.cat(parts, 1), whole)
    assert torch.equal(state, x[:, -3:])


@pytest.mark.parametrize("dtype,B,L,C,taps", [
    (BF16, 20, 65, 8192, 4), (F16, 1, 1301, 1023, 3), (F32, 20, 61, 4096, 2), (BF16, 16, 70, 8192, 8)])
def test_conv_of_many(gpu, fmx, dtype, B, L, C, taps):
    """Enough work for runs of 8 tokens, vectors and single elements."""
    g = _gen(C)
    x = _randn(g, B, L, C, dtype=dtype).cuda()
    w, bias = _randn(g, C, taps, dtype=dtype).cuda(), _randn(g, C, dtype=dtype).cuda()
    lengths = [L - 3 * (b % 3) for b in range(B)]
    want, bound, after = O.conv(x, w, bias, True, None, B, lengths)
    state = torch.full((B, taps - 1, C), 3.0, dtype=dtype, device="cuda")
    print("conv", dtype, B, L, C, taps, flush=True)
    out = fmx.causal_conv(x, w, bias, None, state, _lens(lengths))
    for b, n in enumerate(lengths):
        O.assert_within(out[b, :n], want[b, :n], bound[b, :n], f"row {b}")
    assert torch.equal(state.double().cpu(), after)


# ------------------------------------------------------------------ scan

def _scan_inputs(seed, dtype, B, L, nh, hd, groups, N, slots=6):
    g = _gen(seed)
    inner, n = nh * hd, groups * N
    v = torch.nn.functional.silu(_randn(g, B, L, inner + 2 * n)).to(dtype).cuda()
    dt = _cut(_randn(g, B, L, nh, dtype=dtype), 3, dtype)
    step = torch.exp(torch.empty(nh).uniform_(math.log(0.001), math.log(0.1), generator=g))
    bias = (step + torch.log(-torch.expm1(-step))).cuda()
    a = -torch.empty(nh).uniform_(1, 16, generator=g).cuda()
    return dict(x=v[..., :inner].view(B, L, nh, hd), b=v[..., inner:inner + n].view(B, L, groups, N),
                c=v[..., inner + n:].view(B, L, groups, N), dt=dt, dt_bias=bias, a=a, d=_randn(g, nh).cuda(),
                state=(0.5 * _randn(g, slots, nh, hd, N)).cuda())


def _check_scan(fmx, p, lengths=None, slots=None, begun=True, keep="out", limits=LIMITS, softplus=True, **kw):
    B, L, nh, hd = p["x"].shape
    steps, rel = O.time_step(p["dt"], p["dt_bias"], softplus, *limits)
    first = p["state"] if begun else None
    n_slots = p["state"].shape[0]
    want, bound, after, after_b = O.scan(p["x"], steps, rel, p["a"], p["b"], p["c"], p["d"], first, n_slots, lengths,
                                         slots, rounded=p["x"].dtype)
    out = torch.full_like(p["x"], 7.0, memory_format=torch.contiguous_format)
    sl = None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lengths or []):
        for k in ("x", "b", "c", "dt"):
            p[k][b, n:] = math.nan
    s_out = {"out": torch.full_like(p["state"], 3.0), "in place": p["state"], "no": None}[keep]
    print("scan", p["x"].dtype, tuple(p["x"].shape), tuple(p["b"].shape), lengths, flush=True)
    fmx.ssm_scan(p["x"], p["dt"], p["a"], p["b"], p["c"], p["d"], p["dt_bias"], first, s_out, _lens(lengths), sl,
                 softplus, limits, out, **kw)
    torch.cuda.synchronize()
    _untouched(out, lengths)
    for b in range(B):
        n = L if lengths is None else lengths[b]
        O.assert_within(out[b, :n], want[b, :n], bound[b, :n], f"sequence {b}")
    if s_out is not None:
        used = [O._slot(slots, n_slots, b) for b in range(B)]
        for s in range(n_slots):
            if s in used:
                O.assert_within(s_out[s], after[s], after_b[s], f"state {s}")
            elif keep == "out":
                assert (s_out[s] == 3.0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L", [1, 2, 7, 8, 17, 63, 64, 65, 129, 200])
def test_scan_lengths(gpu, fmx, dtype, L):
    _check_scan(fmx, _scan_inputs(L, dtype, 2, L, 4, 64, 2, 128))


@pytest.mark.parametrize("dtype,nh,hd,groups,N", [
    (BF16, 1, 8, 1, 8), (F16, 3, 24, 1, 16), (BF16, 4, 80, 2, 48), (BF16, 2, 128, 1, 64), (F16, 2, 256, 2, 32),
    (BF16, 2, 64, 2, 256), (BF16, 6, 40, 3, 200), (F16, 2, 32, 1, 104), (F16, 1, 200, 1, 256)])
@pytest.mark.parametrize("L", [1, 6, 70])
def test_scan_shapes(gpu, fmx, dtype, nh, hd, groups, N, L):
    _check_scan(fmx, _scan_inputs(hd + N, dtype, 2, L, nh, hd, groups, N), keep="in place")


@pytest.mark.parametrize("lengths,slots,begun,keep", [
    ([100, 0, 1, 65], [3, 0, 5, 1], True, "out"), ([64, 99, 100, 3], [0, -1, 6, 2], True, "in place"),
    ([5, 2, 0, 9], None, False, "out"), ([100, 37, 64, 1], None, True, "no"), ([0, 0, 0, 0], [1, 2, 3, 4], False, "out")])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scan_ragged(gpu, fmx, lengths, slots, begun, keep, dtype):
    _check_scan(fmx, _scan_inputs(11, dtype, 4, 100, 4, 64, 2, 128), lengths, slots, begun, keep)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L", [3, 150])
def test_scan_options(gpu, fmx, dtype, L):
    p = _scan_inputs(2, dtype, 1, L, 4, 64, 1, 64)
    p["d"], p["dt_bias"] = None, None
    _check_scan(fmx, p, begun=False)
    p = _scan_inputs(3, dtype, 1, L, 4, 64, 1, 64)
    p["dt"] = p["dt"].abs()
    _check_scan(fmx, p, softplus=False, limits=(0.0, math.inf), begun=False)
    # steps that forget everything at once, and ones that forget nothing
    p = _scan_inputs(4, dtype, 1, L, 4, 64, 1, 64)
    p["a"] = torch.tensor([-1e4, 0.0, -1e-6, -300.0], device="cuda")
    _check_scan(fmx, p)


@pytest.mark.parametrize("dtype,nh,hd,groups,N", [
    (BF16, 4, 64, 2, 128), (F16, 4, 64, 2, 128), (F16, 2, 64, 2, 64), (BF16, 3, 64, 1, 32), (F16, 2, 128, 1, 256),
    (BF16, 1, 40, 1, 120), (BF16, 2, 32, 2, 256)])
@pytest.mark.parametrize("lengths,slots,keep", [
    (None, None, "out"), ([700, 385], [4, 2], "in place"), ([0, 513], None, "in place"), ([640, 64], [-1, 5], "out")])
def test_scan_segments(gpu, fmx, dtype, nh, hd, groups, N, lengths, slots, keep):
    """Long sequences of few heads: cut, with a state to start from."""
    _check_scan(fmx, _scan_inputs(N + nh, dtype, 2, 700, nh, hd, groups, N), lengths, slots, True, keep)


@pytest.mark.parametrize("dtype,nh,hd,groups,N,L,lengths,keep", [
    (BF16, 258, 8, 2, 128, 100, None, "out"), (F16, 258, 8, 2, 64, 130, None, "in place"), (BF16, 300, 16, 3, 256, 70, None, "no"),
    (F16, 260, 64, 4, 16, 65, [33], "out"), (F16, 128, 64, 1, 32, 660, [651], "in place"),
    (BF16, 127, 8, 1, 128, 700, None, "in place"), (F16, 126, 8, 2, 256, 660, [640], "out"), (BF16, 66, 72, 2, 64, 645, None, "out")])
def test_scan_of_many_heads(gpu, fmx, dtype, nh, hd, groups, N, L, lengths, keep):
    """Enough items for two to a workgroup, an odd one alone in its group among them."""
    _check_scan(fmx, _scan_inputs(nh + N, dtype, 1, L, nh, hd, groups, N, slots=2), lengths, [1], True, keep)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L", [9, 300])
def test_scan_rows_of_all_sizes(gpu, fmx, dtype, L):
    """A head's rows from 2^-12 to 2^8: each keeps its own bits."""
    p = _scan_inputs(6, dtype, 1, L, 2, 64, 1, 128)
    by = 2.0 ** (torch.randperm(128, generator=_gen(1)) % 21 - 12).float().cuda().view(2, 64)
    p["x"] = (p["x"].float() * by).to(dtype)
    p["state"] *= by[..., None]
    _check_scan(fmx, p)


@pytest.mark.parametrize("L", [40, 100])
def test_scan_f16_tokens_of_all_sizes(gpu, fmx, L):
    """A token 2^24 times the others, alone in its column of the state. What
    tokens bring is scaled to its largest and taken as two numbers of float16,
    2^13 .. 2^14 at most and cut at 2^-24: off by 2^-37 of the largest, as the
    state is where it goes into outputs."""
    p = _scan_inputs(13, F16, 1, L, 1, 64, 1, 32, slots=1)
    p["x"][:, 1:] *= 2.0 ** -13
    p["x"][:, 0] *= 2.0 ** 11
    p["b"][:, 0, :, 1:] = 0
    p["b"][:, 1:, :, 0] = 0
    steps, rel = O.time_step(p["dt"], p["dt_bias"], True, *LIMITS)
    want, bound, after, after_b = O.scan(p["x"], steps, rel, p["a"], p["b"], p["c"], p["d"], None, 1, rounded=F16)
    most = (steps[0, :, :, None] * p["x"][0].double().cpu().abs()).sum(0)[..., None]  # [1, 64, 1], of what tokens bring
    b, c = p["b"][0, :, 0].double().cpu().abs(), p["c"][0, :, 0].double().cpu().abs()
    lost = 2.0 ** -37 * most * b.sum(0)
    s_out = torch.empty(1, 1, 64, 32, device="cuda")
    y = fmx.ssm_scan(p["x"], p["dt"], p["a"], p["b"], p["c"], p["d"], p["dt_bias"], None, s_out, dt_limits=LIMITS)
    O.assert_within(s_out[0], after[0], after_b[0] + lost, "state")
    more = (lost[None] * c[:, None, None]).sum(-1) + 2.0 ** -37 * (most * b.max())[None, ..., 0] * c.sum(-1)[:, None, None]
    O.assert_within(y[0], want[0], bound[0] + more, "out")
    assert (lost[0, :, 1:] < 2.0 ** -9 * after[0, 0, :, 1:].abs().max()).all()  # (far from what a missing second number would lose)


@pytest.mark.parametrize("L", [5, 130])
def test_scan_views(gpu, fmx, L):
    """b shared by the groups, c by the sequences, tokens in another order than
    memory's, a token's dt 17 elements apart."""
    p = _scan_inputs(7, BF16, 2, L, 4, 64, 2, 64)
    p["b"] = p["b"][:, :, :1].expand(2, L, 2, 64)
    p["c"] = p["c"][:1].expand(2, L, 2, 64)
    p["x"] = p["x"].permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)
    p["dt"] = torch.randn(2, 4, L, 17, generator=_gen(2)).to(BF16).cuda()[..., 5].permute(0, 2, 1)
    _check_scan(fmx, p)


@pytest.mark.parametrize("L", [12, 20])
def test_scan_of_far_tokens(gpu, fmx, L):
    """Tokens 2^24 elements apart, more than the chunks' lanes address."""
    p = _scan_inputs(8, BF16, 1, L, 2, 16, 1, 16)
    x = torch.empty(L * 2 ** 24, dtype=BF16, device="cuda").as_strided((1, L, 2, 16), (8, 2 ** 24, 16, 1))
    x.copy_(p["x"])
    p["x"] = x
    _check_scan(fmx, p, begun=False)


def test_scan_slots_beyond_32_bits(gpu, fmx):
    p = _scan_inputs(10, F16, 2, 70, 64, 64, 1, 128, slots=2)
    slots = [8200, 3]
    pool = torch.empty(8201, 64, 64, 128, device="cuda")  # 2^32 elements before the last slot
    assert slots[0] * pool.stride(0) > 2 ** 32
    pool[8200], pool[3] = p["state"][0], p["state"][1]
    sl = torch.tensor(slots, dtype=torch.int32, device="cuda")
    for L in (70, 4):
        q = {k: v[:, :L] if k in "xbc" or k == "dt" else v for k, v in p.items()}
        want_state = p["state"].clone()
        args = (q["x"], q["dt"], q["a"], q["b"], q["c"], q["d"], q["dt_bias"])
        want = fmx.ssm_scan(*args, want_state, want_state, dt_limits=LIMITS)
        got = fmx.ssm_scan(*args, pool, pool, slots=sl, dt_limits=LIMITS)
        assert torch.equal(got, want) and torch.equal(pool[8200], want_state[0]) and torch.equal(pool[3], want_state[1])
        p["state"] = want_state


def test_rows_beyond_32_bits(gpu, fmx):
    """The second sequence's rows 2^32 elements behind the first one's."""
    g, C, L = _gen(15), 64, 21
    far = [torch.empty(2 ** 32 + 2 * L * C, dtype=BF16, device="cuda").as_strided((2, L, C), (2 ** 32 + C, C, 1))
           for _ in range(2)]
    x, w = _randn(g, 2, L, C, dtype=BF16).cuda(), _randn(g, C, 4, dtype=BF16).cuda()
    far[0].copy_(x)
    assert torch.equal(fmx.causal_conv(far[0], w, out=far[1]), fmx.causal_conv(x, w))
    assert torch.equal(fmx.gated_norm(far[0], None, far[0], groups=4, out=far[1]), fmx.gated_norm(x, None, x, groups=4))
    p = _scan_inputs(16, BF16, 2, L, 1, 64, 1, 8)
    far[0].copy_(p["x"].flatten(2))
    args = (p["dt"], p["a"], p["b"], p["c"], p["d"], p["dt_bias"])
    for n in (L, 3):
        cut = tuple(t[:, :n] if t.dim() > 1 else t for t in args)
        got = fmx.ssm_scan(far[0].unflatten(2, (1, 64))[:, :n], *cut, out=far[1].unflatten(2, (1, 64))[:, :n])
        assert torch.equal(got, fmx.ssm_scan(p["x"][:, :n], *cut))


def test_nothing_to_do(gpu, fmx):
    """No sequences, no tokens: outputs of that shape; without tokens states are carried over."""
    p = _scan_inputs(17, BF16, 2, 3, 2, 16, 1, 16, slots=2)
    for B, L in ((0, 3), (2, 0)):
        q = {k: v[:B, :L] if k in "xbc" or k == "dt" else v for k, v in p.items()}
        s_out = torch.full_like(p["state"], 3.0)
        y = fmx.ssm_scan(q["x"], q["dt"], q["a"], q["b"], q["c"], q["d"], q["dt_bias"], p["state"], s_out)
        assert y.shape == (B, L, 2, 16)
        assert torch.equal(s_out, p["state"] if B else torch.full_like(s_out, 3.0))
        x, w = torch.randn(B, L, 16, device="cuda"), torch.randn(16, 4, device="cuda")
        c_in, c_out = torch.randn(2, 3, 16, device="cuda"), torch.full((2, 3, 16), 3.0, device="cuda")
        assert fmx.causal_conv(x, w, None, c_in, c_out).shape == x.shape
        assert torch.equal(c_out, c_in if B else torch.full_like(c_out, 3.0))
        assert fmx.gated_norm(x).shape == x.shape
    none = torch.empty(0, 2, 16, 16, device="cuda")  # a pool of no slots: from 0, nothing kept
    args = (p["x"], p["dt"], p["a"], p["b"], p["c"])
    assert torch.equal(fmx.ssm_scan(*args, state=none, state_out=none), fmx.ssm_scan(*args))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L", [4, 100])
def test_scan_from_a_state_with_infinities(gpu, fmx, dtype, L):
    """They stay in their rows."""
    p = _scan_inputs(18, dtype, 1, L, 2, 64, 1, 128, slots=1)
    args = (p["x"], p["dt"], p["a"], p["b"], p["c"], p["d"], p["dt_bias"])
    after, after_bad = torch.empty_like(p["state"]), torch.empty_like(p["state"])
    clean = fmx.ssm_scan(*args, p["state"], after, dt_limits=LIMITS)
    bad = p["state"].clone()
    bad[0, 1, 5, 7], bad[0, 0, 63, 0] = math.inf, math.nan
    y = fmx.ssm_scan(*args, bad, after_bad, dt_limits=LIMITS)
    for h, r in ((1, 5), (0, 63)):
        assert not torch.isfinite(y[0, :, h, r]).any() and not torch.isfinite(after_bad[0, h, r]).all()
        y[0, :, h, r], after_bad[0, h, r] = clean[0, :, h, r], after[0, h, r]
    assert torch.equal(y, clean) and torch.equal(after_bad, after)


def test_scan_graphs_share_a_workspace(gpu, fmx):
    """Two captured scans of several segments with one workspace, replayed in
    turn on one stream, with eager ones between."""
    ps = [_scan_inputs(19 + i, BF16, 1, 700 - 60 * i, 2, 64, 1, 128, slots=1) for i in range(2)]
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    run = [lambda p=p, out=torch.zeros_like(p["x"], memory_format=torch.contiguous_format): fmx.ssm_scan(
        p["x"], p["dt"], p["a"], p["b"], p["c"], p["d"], p["dt_bias"], p["state"], p["state"], dt_limits=LIMITS, out=out,
        workspace=ws) for p in ps]
    first = [p["state"].clone() for p in ps]
    want = []
    for i in range(2):
        want.append([(run[i]().clone(), ps[i]["state"].clone()) for _ in range(3)])
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = run[i]()
        graphs.append((g, y))
        ps[i]["state"].copy_(first[i])
    for k in range(3):
        for i in range(2):
            graphs[i][0].replay()
            fmx.ssm_scan(ps[i]["x"], ps[i]["dt"], ps[i]["a"], ps[i]["b"], ps[i]["c"], workspace=ws)
            torch.cuda.synchronize()
            assert torch.equal(graphs[i][1], want[i][k][0]) and torch.equal(ps[i]["state"], want[i][k][1])


def test_scan_infinities_come_late(gpu, fmx):
    """What is not finite in a token reaches it and later tokens, none before."""
    for at in (0, 5, 66, 127):
        for what in ("x", "b", "c", "dt"):
            p = _scan_inputs(9, BF16, 1, 128, 2, 64, 1, 128)
            clean = fmx.ssm_scan(p["x"], p["dt"], p["a"], p["b"], p["c"], p["d"], p["dt_bias"], dt_limits=LIMITS)
            for v in (math.inf, math.nan):
                p[what][:, at] = v
                y = fmx.ssm_scan(p["x"], p["dt"], p["a"], p["b"], p["c"], p["d"], p["dt_bias"], dt_limits=LIMITS)
                early, late = y[:, :at].float(), y[:, at + 1:].float()
                ref = clean[:, :at].float()
                # the same values in another order of sums at most: two roundings of the type
                assert ((early - ref).abs() <= 2.0 ** -7 * ref.abs() + 2.0 ** -10).all(), (at, what, v)
                if what == "c":  # a token's own
                    refl = clean[:, at + 1:].float()
                    assert ((late - refl).abs() <= 2.0 ** -7 * refl.abs() + 2.0 ** -10).all(), (at, what, v)
                elif what != "dt" or math.isnan(v):
                    assert not torch.isfinite(late).any(), (at, what, v)


# ------------------------------------------------------------------ norm

@pytest.mark.parametrize("dtype,B,L,C,groups,lengths,pad", [
    (BF16, 1, 1, 4096, 8, None, 8), (F16, 2, 5, 960, 3, [5, 0], 8), (F32, 2, 3, 512, 1, [1, 3], 4),
    (BF16, 1, 4, 4096, 1, None, 0), (F16, 1, 2, 37, 1, None, 3), (F32, 3, 2, 66, 2, None, 1), (BF16, 2, 3, 24, 3, None, 8),
    (BF16, 1, 2, 20000, 1, None, 0), (F32, 1, 2, 9000, 1, None, 0), (BF16, 1, 3, 128, 8, None, 16),
    (F16, 1, 3, 1536, 1, None, 0), (F32, 1, 1, 1, 1, None, 0), (BF16, 2, 5, 768, 4, [4, 5], 2), (F16, 1, 7, 768, 2, None, 6),
    (BF16, 2, 3, 320, 5, [3, 1], 2), (F32, 1, 9, 320, 10, None, 1), (F16, 3, 11, 640, 8, None, 2), (BF16, 1, 5, 4104, 1, None, 2)])
@pytest.mark.parametrize("gate", ["first", "last", "none"])
def test_gated_norm(gpu, fmx, dtype, B, L, C, groups, lengths, pad, gate):
    g = _gen(C + L)
    x, z = (_cut(_randn(g, B, L, C, dtype=dtype), pad, dtype) for _ in range(2))
    w = None if gate == "none" else (1 + 0.1 * _randn(g, C)).to(dtype).cuda()
    want, bound = O.gated_norm(x, w, None if gate == "none" else z, 1e-5, groups, gate == "first", dtype)
    print("norm", dtype, B, L, C, groups, gate, flush=True)
    out = torch.full((B, L, C), 7.0, dtype=dtype, device="cuda")
    kw = dict(z=None if gate == "none" else z, groups=groups, gate_first=gate == "first", lengths=_lens(lengths))
    fmx.gated_norm(x, w, out=out, **kw)
    torch.cuda.synchronize()
    _untouched(out, lengths)
    live = [L if lengths is None else lengths[b] for b in range(B)]
    for b in range(B):
        O.assert_within(out[b, :live[b]], want[b, :live[b]], bound[b, :live[b]], f"row {b}")
    fmx.gated_norm(x, w, out=x, **kw)  # in place: the same bits
    for b in range(B):
        assert torch.equal(x[b, :live[b]], out[b, :live[b]])


@pytest.mark.parametrize("dtype,B,L,C,groups", [
    (BF16, 1, 262145, 32, 1), (F16, 3, 2731, 1024, 8), (BF16, 2, 1025, 4096, 8), (F16, 1, 2051, 8192, 8),
    (F32, 3, 5462, 64, 4), (BF16, 1, 16400, 36, 1)])
@pytest.mark.parametrize("gate_first", [True, False])
def test_gated_norm_of_many(gpu, fmx, dtype, B, L, C, groups, gate_first):
    """Enough groups for two at a time, and the last ones left over."""
    g = _gen(C)
    x, z = _randn(g, B, L, C, dtype=dtype).cuda(), _randn(g, B, L, C, dtype=dtype).cuda()
    w = (1 + 0.1 * _randn(g, C)).to(dtype).cuda()
    want, bound = O.gated_norm(x, w, z, 1e-5, groups, gate_first, dtype)
    lengths = [L - 5 * b for b in range(B)]
    out = torch.full((B, L, C), 7.0, dtype=dtype, device="cuda")
    print("norm", dtype, B, L, C, groups, flush=True)
    fmx.gated_norm(x, w, z, groups=groups, gate_first=gate_first, lengths=_lens(lengths), out=out)
    _untouched(out, lengths)
    for b, n in enumerate(lengths):
        O.assert_within(out[b, :n], want[b, :n], bound[b, :n], f"row {b}")
    fmx.gated_norm(x, w, z, groups=groups, gate_first=gate_first, out=z)  # in place of the gate: the same bits
    for b, n in enumerate(lengths):
        assert torch.equal(z[b, :n], out[b, :n])


def test_gated_norm_of_zeros(gpu, fmx):
    x = torch.zeros(1, 2, 64, dtype=BF16, device="cuda")
    assert (fmx.gated_norm(x, None, eps=1e-6) == 0).all()


# ------------------------------------------------------------------ a layer

def _layer(fmx, seed, dtype, nh, hd, groups, N, taps, **kw):
    g = _gen(seed)
    C = nh * hd + 2 * groups * N
    p = _scan_inputs(seed, dtype, 1, 1, nh, hd, groups, N)
    w = dict(conv_weight=(_randn(g, C, taps) / math.sqrt(taps)).to(dtype).cuda(),
             conv_bias=(0.1 * _randn(g, C)).to(dtype).cuda(), a=p["a"], d=p["d"], dt_bias=p["dt_bias"],
             norm_weight=(1 + 0.1 * _randn(g, nh * hd)).to(dtype).cuda())
    return fmx.SsmLayer(head_dim=hd, groups=groups, state_dim=N, dt_limits=LIMITS, **w, **kw)


def _project(seed, dtype, shape, layer):
    """Slices of a projection's rows: z, xbc, dt."""
    row = _randn(_gen(seed), *shape, 2 * layer.inner + 2 * layer.groups * layer.state_dim + layer.heads,
                 dtype=dtype).cuda()
    C = layer.channels
    return row[..., layer.inner:layer.inner + C], row[..., layer.inner + C:], row[..., :layer.inner]


@pytest.mark.parametrize("dtype,B,nh,hd,groups,N,taps,kw", [
    (BF16, 1, 4, 64, 2, 128, 4, {}), (F16, 5, 3, 80, 1, 48, 3, dict(norm_groups=1)),
    (BF16, 3, 2, 128, 1, 64, 2, dict(gate_first=False)), (F16, 2, 6, 24, 3, 256, 8, dict(activation=None, eps=1e-3)),
    (BF16, 2, 1, 8, 1, 8, 4, dict(softplus=True)), (BF16, 2, 64, 64, 8, 16, 4, dict(norm_groups=1)),
    (F16, 2, 160, 64, 1, 8, 4, {}), (BF16, 1, 4, 200, 4, 32, 5, dict(norm_groups=2))])
@pytest.mark.parametrize("pad", [0, 3, 2])
def test_step(gpu, fmx, dtype, B, nh, hd, groups, N, taps, kw, pad):
    layer = _layer(fmx, 3, dtype, nh, hd, groups, N, taps, **kw)
    xbc, dt, z = _project(4, dtype, (B,), layer)
    if pad:  # rows on no word, or on words only
        xbc, z = _cut(xbc.cpu(), pad, dtype), _cut(z.cpu(), pad + 2, dtype)
    conv_state, state = (torch.randn(*t.shape, generator=_gen(5)).to(t.dtype).cuda() for t in layer.new_states(7))
    slots = [6, 0, 9, 3, -1][:B]
    n = groups * N
    v, ve, conv_after = O.conv(xbc[:, None], layer.conv_weight, layer.conv_bias, layer.activation == "silu", conv_state,
                               7, None, slots, rounded=False)
    steps, rel = O.time_step(dt[:, None], layer.dt_bias, True, *LIMITS)
    cut = (lambda t: (t[..., :layer.inner].reshape(B, 1, nh, hd), t[..., layer.inner:layer.inner + n].reshape(B, 1, groups, N),
                      t[..., layer.inner + n:].reshape(B, 1, groups, N)))
    (x, b, c), (xe, be, ce) = cut(v), cut(ve)
    y, yb, after, after_b = O.scan(x, steps, rel, layer.a, b, c, layer.d, state, 7, None, slots, xe, be, ce)
    want, bound = O.gated_norm(y.reshape(B, -1), layer.norm_weight, z, layer.eps, layer.norm_groups, layer.gate_first,
                               dtype, yb.reshape(B, -1))
    print("step", dtype, B, nh, hd, groups, N, flush=True)
    conv_got, got = conv_state.clone(), state.clone()
    out = layer.step(xbc, dt, z, conv_got, got, torch.tensor(slots, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    O.assert_within(out, want, bound, "out")
    O.assert_within(got, after, after_b, "state")
    assert torch.equal(conv_got.double().cpu(), conv_after)


def test_prompt_then_steps_is_the_prompt(gpu, fmx):
    """A ragged batch's prompts, then tokens one by one, against one long
    prompt. The steps keep what the prompt's operators round in between (the
    convolution's rows and the scan's: 2^-9 each of bf16 beside the last
    rounding), so outputs agree to a few such steps of their row's scale."""
    layer = _layer(fmx, 8, BF16, 8, 64, 2, 128, 4)
    B, L, more = 3, 90, 6
    xbc, dt, z = _project(9, BF16, (B, L + more), layer)
    lengths = [90, 17, 64]
    slots = torch.tensor([2, 0, 4], dtype=torch.int32, device="cuda")
    conv_state, state = layer.new_states(5)
    out = layer.prompt(xbc[:, :L], dt[:, :L], z[:, :L], conv_state, state, _lens(lengths), slots)
    rows = [[out[b, :n]] for b, n in enumerate(lengths)]
    for i in range(more):
        at = [n + i for n in lengths]
        take = lambda t: torch.stack([t[b, m] for b, m in enumerate(at)])  # noqa: E731
        y = layer.step(take(xbc), take(dt), take(z), conv_state, state, slots)
        for b in range(B):
            rows[b].append(y[b:b + 1])
    cs, ss = layer.new_states(B)
    n = [m + more for m in lengths]
    whole = layer.prompt(xbc, dt, z, cs, ss, _lens(n))
    for b in range(B):
        got, ref = torch.cat(rows[b]).float(), whole[b, :n[b]].float()
        assert torch.equal(conv_state[slots[b]], cs[b])
        assert (got - ref).norm() <= 4 * 2.0 ** -8 * ref.norm()
        assert (state[slots[b]] - ss[b]).norm() <= 4 * 2.0 ** -8 * ss[b].norm()


def test_step_captured(gpu, fmx):
    """A captured step follows its inputs, slots and states; replayed with
    eager work of the same layer between."""
    layer = _layer(fmx, 12, BF16, 8, 64, 2, 128, 4)
    B = 3
    xbc, dt, z = (t.clone() for t in _project(13, BF16, (B,), layer))
    slots = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    conv_state, state = layer.new_states(4)
    out = torch.empty(B, layer.inner, dtype=BF16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layer.step(xbc, dt, z, conv_state, state, slots, out)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(xbc, dt, z, conv_state, state, slots, out)
    for t in (conv_state, state):
        t.zero_()
    ref_conv, ref_state = layer.new_states(4)
    for i in range(4):
        nx, nd, nz = _project(20 + i, BF16, (B,), layer)
        xbc.copy_(nx), dt.copy_(nd), z.copy_(nz)
        slots.copy_(torch.tensor([[0, 1, 2], [3, -1, 0], [2, 3, 1], [1, 0, 7]][i], dtype=torch.int32))
        graph.replay()
        want = layer.step(xbc, dt, z, ref_conv, ref_state, slots)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, ref_state) and torch.equal(conv_state, ref_conv), i


def test_prompt_captured_and_on_two_streams(gpu, fmx):
    layer = _layer(fmx, 14, F16, 8, 64, 1, 128, 4)
    ins = [tuple(t.clone() for t in _project(30 + i, F16, (2, 300), layer)) for i in range(2)]
    lens = _lens([300, 131])
    want = [layer.prompt(*p, *layer.new_states(2), lens) for p in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = []
    for s, p in zip(streams, ins):
        states = layer.new_states(2)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append((layer.prompt(*p, *states, lens), states))
    torch.cuda.synchronize()
    for (y, _), w in zip(got, want):
        for b, n in enumerate((300, 131)):
            assert torch.equal(y[b, :n], w[b, :n])
    buf, states = tuple(t.clone() for t in ins[0]), layer.new_states(2)
    out = torch.zeros(2, 300, layer.inner, dtype=F16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.prompt(*buf, *states, lens, out=out)
    for i in (0, 1, 0):
        for t, n in zip(buf, ins[i]):
            t.copy_(n)
        for t in states:
            t.zero_()
        graph.replay()
        layer.prompt(*ins[1 - i], *layer.new_states(2), lens)
        torch.cuda.synchronize()
        for b, n in enumerate((300, 131)):
            assert torch.equal(out[b, :n], want[i][b, :n])


def test_step_slots_beyond_32_bits(gpu, fmx):
    layer = _layer(fmx, 21, BF16, 64, 64, 1, 128, 4)
    xbc, dt, z = _project(22, BF16, (2,), layer)
    conv_small, small = (torch.randn(*t.shape, generator=_gen(5)).to(t.dtype).cuda() for t in layer.new_states(2))
    pool, slots = torch.empty(8201, 64, 64, 128, device="cuda"), [8200, 3]
    conv_pool = torch.empty(8201, 3, layer.channels, dtype=BF16, device="cuda")
    for i, s in enumerate(slots):
        pool[s], conv_pool[s] = small[i], conv_small[i]
    sl = torch.tensor(slots, dtype=torch.int32, device="cuda")
    got = layer.step(xbc, dt, z, conv_pool, pool, sl)
    want = layer.step(xbc, dt, z, conv_small, small)
    assert torch.equal(got, want)
    for i, s in enumerate(slots):
        assert torch.equal(pool[s], small[i]) and torch.equal(conv_pool[s], conv_small[i])


def test_step_graphs_share_a_workspace(gpu, fmx):
    """Two layers' steps captured with one workspace, replayed in turn."""
    layers = [_layer(fmx, 23 + i, BF16, 4, 64, 2, 64, 4) for i in range(2)]
    ins = [_project(25 + i, BF16, (5,), m) for i, m in enumerate(layers)]
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    states, refs = [m.new_states(5) for m in layers], [m.new_states(5) for m in layers]
    graphs = []
    for m, p, st in zip(layers, ins, states):
        m.step(*p, *st, workspace=ws)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = m.step(*p, *st, workspace=ws)
        graphs.append((g, y))
        for t in st:
            t.zero_()
    for _ in range(4):
        for m, p, st, ref, (g, y) in zip(layers, ins, states, refs, graphs):
            g.replay()
            want = m.step(*p, *ref)
            torch.cuda.synchronize()
            assert torch.equal(y, want) and all(torch.equal(s, r) for s, r in zip(st, ref))


def test_a_nan_stays_in_its_sequence(gpu, fmx):
    """A padded batch with one bad sequence: the others' bits are the same."""
    layer = _layer(fmx, 27, BF16, 4, 64, 2, 128, 4)
    xbc, dt, z = (t.clone() for t in _project(28, BF16, (3, 150), layer))
    lens = _lens([150, 90, 20])
    for t in (xbc, dt, z):
        t[2, 20:] = math.nan
    states, bad_states = layer.new_states(3), layer.new_states(3)
    clean = layer.prompt(xbc, dt, z, *states, lens)
    xbc[1, 30:40] = math.inf
    bad = layer.prompt(xbc, dt, z, *bad_states, lens)
    for b, n in ((0, 150), (2, 20)):
        assert torch.equal(bad[b, :n], clean[b, :n])
        assert all(torch.equal(s[b], t[b]) for s, t in zip(states, bad_states))
    # the tokens before it sum the same numbers in an order that depends on none of their values
    assert torch.equal(bad[1, :30], clean[1, :30]) and not torch.isfinite(bad[1, 34:90]).any()
