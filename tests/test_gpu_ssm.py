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
    (F16, 4, 5, 7, 5, False, [0, 1, 4, 5], [3, 2, 1, 0], 2)])
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
    (F16, 1, 3, 1536, 1, None, 0), (F32, 1, 1, 1, 1, None, 0)])
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
    (BF16, 2, 1, 8, 1, 8, 4, dict(softplus=True))])
def test_step(gpu, fmx, dtype, B, nh, hd, groups, N, taps, kw):
    layer = _layer(fmx, 3, dtype, nh, hd, groups, N, taps, **kw)
    xbc, dt, z = _project(4, dtype, (B,), layer)
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
