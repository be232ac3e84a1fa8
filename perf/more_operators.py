"""The operators of a selective state space layer, as a serving program calls them:

  conv  the short causal convolution of a prompt's rows, with its state (causal_conv)
  scan  the selective scan of a prompt or of a few tokens (ssm_scan)
  step  one decoded token through convolution, scan and gated norm, states in
        place in a pool of slots (SsmLayer.step)
  norm  the RMS norm of groups with its gate (gated_norm)

`own` false: the plain forms, elementary torch operations in 32 bits (the
scan's decays, sums over many tokens, in 64), rounded once at the end. `own`
true: the framework's operators.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases

def listed():
    wide = dict(heads=64, head_dim=64, groups=8, state=128)
    narrow = dict(heads=24, head_dim=64, groups=1, state=128)
    return [
        # an ordinary prompt, the first one of its slot
        dict(name="conv_prompt_2048", kind="conv", dtype="bf16", batch=1, seq_len=2048, lo=2048, taps=4, begun=False,
             **wide),
        # a ragged batch that goes on from earlier chunks
        dict(name="conv_ragged_7_f16", kind="conv", dtype="f16", batch=7, seq_len=777, lo=1, taps=4, begun=True,
             **narrow),
        # a long document's chunk in 32 bits, three taps
        dict(name="conv_long_f32", kind="conv", dtype="f32", batch=1, seq_len=8191, lo=8191, taps=3, begun=True,
             **wide),
        # a chat message: few tokens, latency
        dict(name="scan_chat_200", kind="scan", dtype="bf16", batch=1, seq_len=200, lo=200, begun=False, **wide),
        # a long prompt, alone
        dict(name="scan_prompt_8192", kind="scan", dtype="bf16", batch=1, seq_len=8192, lo=8192, begun=False, **wide),
        # a ragged batch of chunks that go on from their slots' states, one shared B and C
        dict(name="scan_ragged_16_f16", kind="scan", dtype="f16", batch=16, seq_len=1531, lo=3, begun=True, **narrow),
        # five drafted tokens per sequence to be checked
        dict(name="scan_drafts_32", kind="scan", dtype="bf16", batch=32, seq_len=5, lo=5, begun=True, heads=32,
             head_dim=128, groups=4, state=64),
        # one sequence's decode step: latency
        dict(name="step_1", kind="step", dtype="bf16", batch=1, slots=4, taps=4, **wide),
        # an ordinary server batch
        dict(name="step_32_f16", kind="step", dtype="f16", batch=32, slots=40, taps=4, heads=80, head_dim=64, groups=1,
             state=128),
        # the largest: a full server
        dict(name="step_256", kind="step", dtype="bf16", batch=256, slots=256, taps=4, **wide),
        # a decode batch's norm: the smallest call
        dict(name="norm_decode_8", kind="norm", dtype="bf16", batch=8, seq_len=1, lo=1, gate_first=True, norm_groups=8,
             **wide),
        # a long prompt's norm, the gate a part of the projection's row
        dict(name="norm_prompt_8192", kind="norm", dtype="bf16", batch=1, seq_len=8192, lo=8192, gate_first=True,
             norm_groups=8, **wide),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 5e14


def draw(rng):
    # no more than the largest listed case of its kind costs
    limits = {}
    for c in listed():
        limits[c["kind"]] = max(limits.get(c["kind"], 0.0), _cost(c))
    while True:
        case = _draw(rng)
        if _cost(case) <= limits[case["kind"]]:
            return case


def _draw(rng):
    kind = rng.choice(["conv", "scan", "scan", "step", "step", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    heads, head_dim, groups, state = rng.choice([
        (64, 64, 8, 128), (64, 64, 8, 128), (24, 64, 1, 128), (80, 64, 1, 128), (32, 128, 4, 64), (16, 32, 2, 16),
        (12, 80, 3, 48), (40, 64, 5, 256)])
    layer = dict(heads=heads, head_dim=head_dim, groups=groups, state=state)
    if kind == "step":
        B = _log_int(rng, 1, 256)
        return dict(kind="step", dtype=dtype, batch=B, slots=B + rng.choice([0, 1, 8]), taps=rng.choice([4, 4, 3, 2]),
                    **layer)
    if kind == "norm":
        B = rng.choice([1, 1, 2, 9])
        L = _log_int(rng, 1, 8192)
        return dict(kind="norm", dtype=rng.choice(["bf16", "f16", "f32"]), batch=B, seq_len=L, lo=rng.choice([1, L]),
                    gate_first=rng.random() < 0.7, norm_groups=rng.choice([1, groups]), **layer)
    B = _log_int(rng, 1, 32)
    if kind == "conv":
        L = _log_int(rng, 1, 8192)
        return dict(kind="conv", dtype=rng.choice(["bf16", "f16", "f32"]), batch=B, seq_len=L, lo=rng.choice([1, L]),
                    taps=rng.choice([4, 4, 3, 2]), begun=rng.random() < 0.5, **layer)
    L = rng.choice([1, 2, 5]) if rng.random() < 0.2 else _log_int(rng, 8, 8192)
    while B * L * heads > 8192 * 80:  # the plain form's decay matrices fit
        B = max(1, B // 2)
    return dict(kind="scan", dtype=dtype, batch=B, seq_len=L, lo=rng.choice([1, L]), begun=rng.random() < 0.5, **layer)


def _lengths(lo, hi, n):
    """n lengths from lo to hi, evenly spread (the seed puts them in an order)."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _sizes(case):
    """Elements of a row of x, of B or C, of what the convolution takes, of the projection."""
    d, n = case["heads"] * case["head_dim"], case["groups"] * case["state"]
    return d, n, d + 2 * n, 2 * d + 2 * n + case["heads"]


def work(case):
    kind, es, B = case["kind"], 4 if case["dtype"] == "f32" else 2, case["batch"]
    d, n, C, _ = _sizes(case)
    nh, hd, N = case["heads"], case["head_dim"], case["state"]
    state = 4 * nh * hd * N
    # of one token: its decay, update and output of every state element, its skip
    token = 5 * d * N + 2 * d
    if kind == "step":
        taps = case["taps"]
        conv = (2 * (taps - 1) + 1) * C * es
        return {"bytes": B * (2 * state + conv + (2 * d + nh) * es + 4) + C * (taps + 1) * es + d * es + 12 * nh,
                "flops": B * (token + 2 * taps * C + 10 * d)}
    T = sum(_lengths(case["lo"], case["seq_len"], B))
    if kind == "conv":
        taps = case["taps"]
        states = (2 if case["begun"] else 1) * B * (taps - 1) * C * es
        return {"bytes": 2 * T * C * es + states + C * (taps + 1) * es + 4 * B, "flops": T * C * (2 * taps + 4)}
    if kind == "scan":
        return {"bytes": T * (2 * d + 2 * n + nh) * es + (2 if case["begun"] else 1) * B * state + 12 * nh + 4 * B,
                "flops": T * token}
    return {"bytes": 3 * T * d * es + d * es + 4 * B, "flops": 10 * T * d}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(6151 * (seed + 1))


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _rand(g, shape, lo, hi):
    return lo + (hi - lo) * torch.rand(shape, generator=g, device="cuda", dtype=torch.float32)


_DT_LIMITS = (0.001, 0.5)
_EPS = 1e-5


def _inputs(case, seed):
    g, dt, kind, B = _gen(seed), _DT[case["dtype"]], case["kind"], case["batch"]
    d, n, C, row = _sizes(case)
    nh, hd, N = case["heads"], case["head_dim"], case["state"]
    L = case.get("seq_len", 1)
    # the projection's rows: the gate, what the convolution takes, the time steps
    proj = _randn(g, (B, L, row), dt)
    a = dict(z=proj[..., :d], xbc=proj[..., d:d + C], dt=proj[..., d + C:])
    if kind != "step":
        lens = torch.tensor(_lengths(case["lo"], L, B), dtype=torch.int32, device="cuda")
        a["lengths"] = lens[torch.randperm(B, generator=g, device="cuda")]
    if kind in ("conv", "step"):
        taps = case["taps"]
        a["conv_w"], a["conv_b"] = _randn(g, (C, taps), dt) / math.sqrt(taps), 0.1 * _randn(g, (C,), dt)
        slots = case["slots"] if kind == "step" else B
        a["conv_state"] = _randn(g, (slots, taps - 1, C), dt)
    if kind in ("scan", "step"):
        # time steps around 0.001 to 0.1 before their input moves them, decays of 1 to 16
        step = torch.exp(_rand(g, (nh,), math.log(0.001), math.log(0.1)))
        a["dt_bias"] = step + torch.log(-torch.expm1(-step))
        a["a"], a["d"] = -_rand(g, (nh,), 1.0, 16.0), _randn(g, (nh,))
        slots = case["slots"] if kind == "step" else B
        a["state"] = 0.5 * _randn(g, (slots, nh, hd, N))
    if kind == "scan":
        # what the convolution leaves
        v = _randn(g, (B, L, C))
        v = (v * torch.sigmoid(v)).to(dt)
        a["x"] = v[..., :d].view(B, L, nh, hd)
        a["b"] = v[..., d:d + n].view(B, L, case["groups"], N)
        a["c"] = v[..., d + n:].view(B, L, case["groups"], N)
    if kind == "step":
        a["slots"] = torch.randperm(case["slots"], generator=g, device="cuda")[:B].to(torch.int32)
        a["z"], a["xbc"], a["dt"] = (a[k][:, 0] for k in ("z", "xbc", "dt"))
    if kind in ("norm", "step"):
        a["norm_w"] = 1 + 0.1 * _randn(g, (d,), dt)
    if kind == "norm":
        a["y"] = _randn(g, (B, L, d), dt)
    return a


def prepare(case, seed):
    st = dict(case=case, **_inputs(case, seed))
    if case["kind"] == "conv":
        st["out"] = torch.zeros(st["xbc"].shape, dtype=st["xbc"].dtype, device="cuda")
        st["conv_state_out"] = torch.zeros_like(st["conv_state"])
    if case["kind"] == "scan":
        st["out"] = torch.zeros(st["x"].shape, dtype=st["x"].dtype, device="cuda")
        st["state_out"] = torch.zeros_like(st["state"])
    if case["kind"] == "norm":
        st["out"] = torch.zeros_like(st["y"])
    if case["kind"] == "step" and own:
        import flashmlx_amd as F
        st["layer"] = F.SsmLayer(conv_weight=st["conv_w"], conv_bias=st["conv_b"], a=st["a"], d=st["d"],
                                 dt_bias=st["dt_bias"], norm_weight=st["norm_w"], head_dim=case["head_dim"],
                                 groups=case["groups"], state_dim=case["state"], norm_groups=case["groups"], eps=_EPS,
                                 dt_limits=_DT_LIMITS)
    return st


# ------------------------------------------------------------------ the framework's calls

def _run_own(st):
    import flashmlx_amd as F
    case = st["case"]
    kind = case["kind"]
    if kind == "conv":
        F.causal_conv(st["xbc"], st["conv_w"], st["conv_b"], state=st["conv_state"] if case["begun"] else None,
                      state_out=st["conv_state_out"], lengths=st["lengths"], out=st["out"])
        return [st["out"], st["conv_state_out"]]
    if kind == "scan":
        F.ssm_scan(st["x"], st["dt"], st["a"], st["b"], st["c"], d=st["d"], dt_bias=st["dt_bias"],
                   dt_limits=_DT_LIMITS, state=st["state"] if case["begun"] else None, state_out=st["state_out"],
                   lengths=st["lengths"], out=st["out"])
        return [st["out"], st["state_out"]]
    if kind == "step":
        out = st["layer"].step(st["xbc"], st["dt"], st["z"], st["conv_state"], st["state"], slots=st["slots"])
        return [out, st["conv_state"], st["state"]]
    return F.gated_norm(st["y"], st["norm_w"], z=st["z"], eps=_EPS, groups=case["norm_groups"],
                        gate_first=case["gate_first"], lengths=st["lengths"], out=st["out"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ plain forms

def _silu(v):
    return v / (1 + torch.exp(-v))


def _step_sizes(raw, bias):
    v = raw.float() + bias
    return (v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))).clamp(*_DT_LIMITS)


def _live(st):
    L = st["case"]["seq_len"]
    return torch.arange(L, device="cuda") < st["lengths"].long()[:, None]


def _run_plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "conv":
        return _conv_plain(st, case)
    if kind == "scan":
        return _scan_plain(st, case)
    if kind == "step":
        return _step_plain(st, case)
    y = _norm_plain(st["y"].float(), st["z"], st["norm_w"], case["norm_groups"], case["gate_first"])
    return torch.where(_live(st)[..., None], y.to(st["y"].dtype), st["out"])


def _norm_plain(y, z, w, groups, gate_first):
    gate = _silu(z.float())
    v = y * gate if gate_first else y
    v = v.unflatten(-1, (groups, -1))
    v = (v / torch.sqrt(v.square().mean(-1, keepdim=True) + _EPS)).flatten(-2) * w.float()
    return v if gate_first else v * gate


def _conv_plain(st, case):
    taps, L = case["taps"], case["seq_len"]
    before = st["conv_state"] if case["begun"] else torch.zeros_like(st["conv_state"])
    rows = torch.cat([before, st["xbc"]], dim=1)
    y = _silu((rows.float().unfold(1, taps, 1) * st["conv_w"].float()).sum(-1) + st["conv_b"].float())
    last = st["lengths"].long()[:, None] + torch.arange(taps - 1, device="cuda")
    after = rows.gather(1, last[..., None].expand(-1, -1, rows.shape[-1]))
    return [torch.where(_live(st)[..., None], y.to(rows.dtype), st["out"]), after]


_CHUNK = 64


def _scan_plain(st, case):
    """The scan in chunks of 64 tokens: products within a chunk, and between
    chunks one product with the decays from each to each later one."""
    B, L, nh, hd = st["x"].shape
    g, N, Q = case["groups"], case["state"], _CHUNK
    nc, rep = -(-L // Q), nh // g
    pad = nc * Q - L
    live = _live(st)[..., None]
    dt = torch.where(live, _step_sizes(st["dt"], st["dt_bias"]), 0.0)

    def chunks(t, heads):  # [B, heads, nc, Q, ..]
        t = torch.nn.functional.pad(t, (0, 0) * (t.dim() - 2) + (0, pad))
        return t.view(B, nc, Q, heads, -1).permute(0, 3, 1, 2, 4)

    x = chunks(torch.where(live[..., None], st["x"].float(), 0.0), nh)
    b = chunks(torch.where(live[..., None], st["b"].float(), 0.0), g)
    c = chunks(torch.where(live[..., None], st["c"].float(), 0.0), g)
    dt = chunks(dt, nh)[..., 0]  # [B, nh, nc, Q]
    cum = (dt.double() * st["a"].double()[:, None, None]).cumsum(-1)
    total = cum[..., -1].cumsum(-1)  # [B, nh, nc]
    # within a chunk
    lower = torch.ones(Q, Q, dtype=torch.bool, device="cuda").tril()
    m = torch.exp((cum[..., :, None] - cum[..., None, :]).masked_fill(~lower, -math.inf)).float() * dt[..., None, :]
    cb = c.contiguous() @ b.transpose(-1, -2).contiguous()  # [B, g, nc, Q, Q]
    m = (m.unflatten(1, (g, rep)) * cb[:, :, None]).flatten(1, 2)
    y = m @ x.contiguous()
    # each chunk's own state, and the state before each chunk
    w = torch.exp(cum[..., -1:] - cum).float() * dt
    own_state = (x * w[..., None]).transpose(-1, -2).contiguous().unflatten(1, (g, rep)) @ b.contiguous()[:, :, None]
    first = st["state"] if case["begun"] else torch.zeros_like(st["state"])
    states = torch.cat([first[:, :, None], own_state.flatten(1, 2)], dim=2).flatten(3)  # [B, nh, 1 + nc, hd N]
    at = torch.nn.functional.pad(total, (1, 0))
    upto = torch.ones(1 + nc, 1 + nc, dtype=torch.bool, device="cuda").tril()
    carry = torch.exp((at[..., :, None] - at[..., None, :]).masked_fill(~upto, -math.inf)).float()
    states = (carry @ states).unflatten(-1, (hd, N))
    enter = states[:, :, :-1].transpose(-1, -2).contiguous().unflatten(1, (g, rep))
    y = y + (c.contiguous()[:, :, None] @ enter).flatten(1, 2) * torch.exp(cum).float()[..., None]
    y = y + x * st["d"][:, None, None, None]
    y = y.permute(0, 2, 3, 1, 4).reshape(B, nc * Q, nh, hd)[:, :L]
    return [torch.where(live[..., None], y.to(st["x"].dtype), st["out"]), states[:, :, -1].contiguous()]


def _step_plain(st, case):
    B, nh, hd, g, N = case["batch"], case["heads"], case["head_dim"], case["groups"], case["state"]
    d, n, C, _ = _sizes(case)
    slots = st["slots"].long()
    rows = torch.cat([st["conv_state"][slots], st["xbc"][:, None]], dim=1)
    v = _silu((rows.float().transpose(1, 2) * st["conv_w"].float()).sum(-1) + st["conv_b"].float())
    st["conv_state"][slots] = rows[:, 1:]
    x = v[:, :d].view(B, g, nh // g, hd, 1)
    b, c = (t.reshape(B, g, 1, 1, N) for t in (v[:, d:d + n], v[:, d + n:]))
    dt = _step_sizes(st["dt"], st["dt_bias"]).view(B, g, nh // g, 1, 1)
    s = st["state"][slots].view(B, g, nh // g, hd, N)
    s = s * torch.exp(dt * st["a"].view(g, nh // g, 1, 1)) + dt * x * b
    st["state"][slots] = s.view(B, nh, hd, N)
    y = (s * c).sum(-1) + x[..., 0] * st["d"].view(g, nh // g, 1)
    y = _norm_plain(y.reshape(B, d), st["z"], st["norm_w"], g, True)
    return [y.to(st["z"].dtype), st["conv_state"], st["state"]]


# ------------------------------------------------------------------ 64 bits

def _exact_norm(y, z, w, groups, gate_first):
    z = z.double()
    gate = z * torch.special.expit(z)
    out = torch.empty_like(y)
    size = y.shape[-1] // groups
    for k in range(groups):
        at = slice(k * size, (k + 1) * size)
        v = y[..., at] * gate[..., at] if gate_first else y[..., at]
        v = v * torch.rsqrt((v * v).sum(-1, keepdim=True) / size + _EPS) * w[at].double()
        out[..., at] = v if gate_first else v * gate[..., at]
    return out


def _exact_dt(raw, bias):
    v = raw.double() + bias.double()
    return torch.logaddexp(v, torch.zeros_like(v)).clamp(*_DT_LIMITS)


def _exact_conv(rows, w, b, L):
    """rows [B, taps - 1 + L, C]: the sums of the rows under each tap."""
    y = b.double().expand(rows.shape[0], L, -1).clone()
    for k in range(w.shape[1]):
        y += rows[:, k:k + L].double() * w[:, k].double()
    return y * torch.special.expit(y)


def _exact_scan(x, dt, a, b, c, d, state, live):
    """Token by token. x [B, L, nh, hd], dt [B, L, nh], b and c [B, L, g, N], live [B, L]."""
    rep = x.shape[2] // b.shape[2]
    y = torch.zeros_like(x, dtype=torch.float64)
    s = state.double().clone()
    decay = torch.where(live[..., None], torch.exp(dt * a.double()), 1.0)
    for t in range(x.shape[1]):
        bt = b[:, t].double().repeat_interleave(rep, dim=1)
        ct = c[:, t].double().repeat_interleave(rep, dim=1)
        u = torch.where(live[:, t, None, None], x[:, t].double() * dt[:, t, :, None], 0.0)
        s.mul_(decay[:, t, :, None, None]).add_(u[..., None] * bt[:, :, None])
        y[:, t] = torch.matmul(s, ct[..., None])[..., 0] + x[:, t].double() * d.double()[:, None]
    return y * live[..., None, None], s


def exact(case, seed):
    a, kind, B = _inputs(case, seed), case["kind"], case["batch"]
    d, n, C, _ = _sizes(case)
    if kind == "step":
        slots = a["slots"].long()
        rows = torch.cat([a["conv_state"][slots], a["xbc"][:, None]], dim=1)
        v = _exact_conv(rows, a["conv_w"], a["conv_b"], 1)
        b, c = (t.reshape(B, 1, case["groups"], case["state"]) for t in (v[..., d:d + n], v[..., d + n:]))
        dt = _exact_dt(a["dt"], a["dt_bias"])[:, None]
        y, s = _exact_scan(v[..., :d].reshape(B, 1, case["heads"], case["head_dim"]), dt, a["a"], b, c, a["d"],
                           a["state"][slots], torch.ones(B, 1, dtype=torch.bool, device="cuda"))
        state, conv_state = a["state"].double(), a["conv_state"].double()
        state[slots], conv_state[slots] = s, rows[:, 1:].double()
        return [_exact_norm(y.reshape(B, d), a["z"], a["norm_w"], case["groups"], True), conv_state, state]
    L, lens = case["seq_len"], a["lengths"].tolist()
    live = torch.zeros(B, L, dtype=torch.bool, device="cuda")
    for i, m in enumerate(lens):
        live[i, :m] = True
    if kind == "norm":
        y = _exact_norm(a["y"].double(), a["z"], a["norm_w"], case["norm_groups"], case["gate_first"])
        return y * live[..., None]
    if kind == "conv":
        before = a["conv_state"] if case["begun"] else torch.zeros_like(a["conv_state"])
        rows = torch.cat([before, a["xbc"]], dim=1)
        after = torch.stack([rows[i, m:m + case["taps"] - 1] for i, m in enumerate(lens)]).double()
        return [_exact_conv(rows, a["conv_w"], a["conv_b"], L) * live[..., None], after]
    first = a["state"] if case["begun"] else torch.zeros_like(a["state"])
    y, s = _exact_scan(a["x"], _exact_dt(a["dt"], a["dt_bias"]), a["a"], a["b"], a["c"], a["d"], first, live)
    return [y, s]
