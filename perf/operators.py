"""The long-context operators of the KV cache, as a serving program calls them:

  rope    rotary positions of a prompt's rows (Rope.__call__), forward or inverse
  append  one decode step's q, k and v rows: q and k rotated, k and v put into
          the caches (Rope.append)
  shared  attention of a batch behind one shared prefix (attention_shared_prefix)
  scored  attention that adds up what weight each cached key got (attention_scored)
  evict   the cache cut to a budget by those weights (cache_evict)

`own` false: the plain forms, elementary torch operations in 32 bits (angles
in 64), rounded once at the end. `own` true: the framework's operators.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # a decode step of eight sequences: the smallest call, latency
        dict(name="append_decode_8", kind="append", dtype="bf16", batch=8, q_len=1, heads=16, kv_heads=16,
             head_dim=128, dims=128, interleaved=False, scaling="none", factor=1.0, far=4096, max_seq=4096),
        # a long prompt far behind the trained length: part of the head, interleaved pairs
        dict(name="rope_prompt_4099_f16", kind="rope", dtype="f16", batch=1, q_len=4099, heads=32, head_dim=128,
             dims=64, interleaved=True, scaling="parts", factor=8.0, far=1 << 20, inverse=False),
        # the way back (the gradient of a prompt batch's queries), 32-bit rows
        dict(name="rope_back_2x777_f32", kind="rope", dtype="f32", batch=2, q_len=777, heads=16, head_dim=128,
             dims=128, interleaved=False, scaling="yarn", factor=4.0, far=1 << 17, inverse=True),
        # a few chats behind a short system prompt, one token each: latency
        dict(name="shared_decode_4", kind="shared", dtype="bf16", batch=4, q_len=1, heads=16, kv_heads=16,
             head_dim=128, prefix=512, own_lo=1, own_hi=64, max_seq=256),
        # an ordinary server batch behind a prompt of odd length
        dict(name="shared_decode_32_f16", kind="shared", dtype="f16", batch=32, q_len=1, heads=32, kv_heads=4,
             head_dim=128, prefix=4001, own_lo=1, own_hi=1000, max_seq=1024),
        # five drafted tokens per sequence to be checked, small heads
        dict(name="shared_drafts_16", kind="shared", dtype="bf16", batch=16, q_len=5, heads=20, kv_heads=5,
             head_dim=64, prefix=1537, own_lo=5, own_hi=513, max_seq=640),
        # the largest: a full server behind a document
        dict(name="shared_decode_128", kind="shared", dtype="bf16", batch=128, q_len=1, heads=32, kv_heads=4,
             head_dim=128, prefix=32768, own_lo=64, own_hi=2048, max_seq=2048),
        # one sequence at the end of the decoder stack's cache
        dict(name="scored_decode_1", kind="scored", dtype="bf16", batch=1, q_len=1, heads=16, kv_heads=16,
             head_dim=128, own_lo=4000, own_hi=4000, max_seq=4096),
        # a ragged batch of long contexts
        dict(name="scored_decode_16_f16", kind="scored", dtype="f16", batch=16, q_len=1, heads=32, kv_heads=4,
             head_dim=128, own_lo=37, own_hi=16001, max_seq=16384),
        # a prompt whose weights pick what is kept of it
        dict(name="scored_prompt_2000", kind="scored", dtype="bf16", batch=1, q_len=2000, heads=32, kv_heads=4,
             head_dim=128, own_lo=2000, own_hi=2000, max_seq=2048),
        # a periodic cut of four decoding sequences, some still below the budget
        dict(name="evict_decode_4", kind="evict", dtype="bf16", batch=4, kv_heads=16, head_dim=128, len_lo=900,
             len_hi=1152, max_seq=1152, out_seq=1152, budget=1024, sinks=4, recent=256),
        # long prompts cut down into a small cache
        dict(name="evict_prompt_16_f16", kind="evict", dtype="f16", batch=16, kv_heads=4, head_dim=128,
             len_lo=2000, len_hi=16384, max_seq=16384, out_seq=4096, budget=4000, sinks=4, recent=512),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    return rng.choice([(16, 16), (32, 4), (32, 8), (20, 5), (14, 2), (8, 1), (24, 8)])


def _angles(rng, hd):
    return dict(dims=rng.choice([hd, hd, hd // 2]), interleaved=rng.random() < 0.5,
                scaling=rng.choice(["none", "linear", "ntk", "parts", "yarn"]), factor=rng.choice([2.0, 4.0, 8.0]),
                far=_log_int(rng, 64, 1 << 20))


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 5e14


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= limit:
            return case


def _draw(rng):
    kind = rng.choice(["rope", "append", "shared", "shared", "scored", "scored", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    hd = rng.choice([64, 80, 128, 128, 128, 256])
    nh, nkv = _heads(rng)
    if kind == "rope":
        B = rng.choice([1, 1, 2, 5])
        return dict(kind="rope", dtype=rng.choice(["bf16", "f16", "f32"]), batch=B,
                    q_len=_log_int(rng, 1, 8192 // B), heads=nh, head_dim=hd, inverse=rng.random() < 0.3,
                    **_angles(rng, hd))
    if kind == "append":
        B, S = _log_int(rng, 1, 256), _log_int(rng, 64, 4096)
        while B * nkv * S * hd > 8 * 16 * 4096 * 128:  # no larger caches than the listed case has
            S //= 2
        return dict(kind="append", dtype=dtype, batch=B, q_len=rng.choice([1, 1, 1, 2, 5]), heads=nh, kv_heads=nkv,
                    head_dim=hd, max_seq=max(S, 8), **_angles(rng, hd))
    if kind == "shared":
        L, B = rng.choice([1, 1, 1, 1, 2, 5, 33]), _log_int(rng, 1, 128)
        hi = _log_int(rng, L, 2048)
        P, room = _log_int(rng, 1, 32768), rng.choice([0, 1, 100])
        while B * L * nh * P > 128 * 32 * 32768:  # no more scores than the largest listed case has
            P = max(1, P // 2)
        return dict(kind="shared", dtype=dtype, batch=B, q_len=L, heads=nh, kv_heads=nkv, head_dim=hd, prefix=P,
                    own_lo=rng.choice([L, hi]), own_hi=hi, max_seq=hi + room)
    if kind == "scored":
        if rng.random() < 0.7:
            L, B = rng.choice([1, 1, 1, 4]), _log_int(rng, 1, 64)
            hi = _log_int(rng, L, 16384)
            while B * hi > 16 * 16384:  # no more keys than the ragged listed batch holds
                hi = max(L, hi // 2)
        else:
            B = rng.choice([1, 1, 2])
            L = _log_int(rng, 16, 2000 // B)
            hi = L + rng.choice([0, 0, 200])
        return dict(kind="scored", dtype=dtype, batch=B, q_len=L, heads=nh, kv_heads=nkv, head_dim=hd,
                    own_lo=rng.choice([L, hi]), own_hi=hi, max_seq=hi + rng.choice([0, 1, 100]))
    B, hi = _log_int(rng, 1, 16), _log_int(rng, 16, 16384)
    budget = max(1, int(hi * rng.uniform(0.05, 1.0)))
    sinks, recent = min(rng.choice([0, 1, 4]), budget), rng.choice([0.0, 0.1, 0.5])
    return dict(kind="evict", dtype=dtype, batch=B, kv_heads=nkv, head_dim=hd, len_lo=rng.choice([1, hi]), len_hi=hi,
                max_seq=hi + rng.choice([0, 5]), out_seq=budget + rng.choice([0, 7]), budget=budget, sinks=sinks,
                recent=int((budget - sinks) * recent))


def _lengths(lo, hi, n):
    """n lengths from lo to hi, evenly spread (the seed puts them in an order)."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _own_lengths(case):
    return _lengths(case["own_lo"], case["own_hi"], case["batch"])


def work(case):
    kind, hd = case["kind"], case["head_dim"]
    es = 4 if case["dtype"] == "f32" else 2
    B = case["batch"]
    if kind == "rope":
        n = B * case["q_len"]
        pairs = n * case["heads"] * case["dims"] // 2
        return {"bytes": 2 * n * case["heads"] * hd * es + 4 * n, "flops": 6 * pairs + 4 * n * case["dims"] // 2}
    if kind == "append":
        n = B * case["q_len"]
        nq, nk = case["heads"], case["kv_heads"]
        return {"bytes": 2 * n * (nq + 2 * nk) * hd * es + 4 * n + 4 * B,
                "flops": 6 * n * (nq + nk) * case["dims"] // 2 + 4 * n * case["dims"] // 2}
    if kind == "evict":
        lens = _lengths(case["len_lo"], case["len_hi"], B)
        kept = sum(min(n, case["budget"]) for n in lens)
        nkv = case["kv_heads"]
        return {"bytes": nkv * (4 * sum(lens) + 4 * kept * hd * es + 4 * kept + 4 * B * case["budget"]) + 8 * B,
                "flops": nkv * sum(lens)}
    L, nq, nk = case["q_len"], case["heads"], case["kv_heads"]
    lens = _own_lengths(case)
    # keys seen by all the rows of a sequence: its newest L tokens see one more each
    seen = sum(sum(max(0, n - L + 1 + l) for l in range(L)) for n in lens)
    io = 2 * B * L * nq * hd * es + 4 * B
    own_keys = 2 * sum(lens) * nk * hd * es
    if kind == "shared":
        P = case["prefix"]
        return {"bytes": io + own_keys + 2 * P * nk * hd * es + 4 * B * L * nq,
                "flops": 4 * hd * nq * (B * L * P + seen)}
    return {"bytes": io + own_keys + 8 * B * nk * case["max_seq"], "flops": 4 * hd * nq * seen}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(7919 * (seed + 1))


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ordered(g, values):
    """The lengths in an order of the seed's, int32 on the device."""
    perm = torch.randperm(len(values), generator=g, device="cuda")
    return torch.tensor(values, dtype=torch.int32, device="cuda")[perm]


def _inputs(case, seed):
    g, dt, kind, B, hd = _gen(seed), _DT[case["dtype"]], case["kind"], case["batch"], case["head_dim"]
    if kind == "evict":
        nkv, S = case["kv_heads"], case["max_seq"]
        # weights that attention leaves: few keys with most of it, a long tail
        w = torch.exp(2.0 * torch.randn((B, nkv, S), generator=g, device="cuda", dtype=torch.float32) - 5.0)
        return dict(k=_randn(g, (B, nkv, S, hd), dt), v=_randn(g, (B, nkv, S, hd), dt), w=w,
                    lengths=_ordered(g, _lengths(case["len_lo"], case["len_hi"], B)))
    L = case["q_len"]
    a = dict(q=_randn(g, (B, L, case["heads"], hd), dt))
    if kind in ("rope", "append"):
        start = torch.randint(0, max(1, case["far"] - L), (B, 1), generator=g, device="cuda")
        a["positions"] = (start + torch.arange(L, device="cuda")).to(torch.int32)
    if kind == "rope":
        return a
    nkv, S = case["kv_heads"], case["max_seq"]
    if kind == "append":
        a["k"], a["v"] = _randn(g, (B, L, nkv, hd), dt), _randn(g, (B, L, nkv, hd), dt)
        a["offsets"] = torch.randint(0, S - L + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        a["kc"], a["vc"] = torch.zeros((B, nkv, S, hd), dtype=dt, device="cuda"), torch.zeros((B, nkv, S, hd), dtype=dt, device="cuda")
        return a
    # the cache holds the new tokens' keys already: sequence b's rows sit at offsets[b] .. offsets[b] + L - 1
    a["offsets"] = _ordered(g, _own_lengths(case)) - L
    a["kc"], a["vc"] = _randn(g, (B, nkv, S, hd), dt), _randn(g, (B, nkv, S, hd), dt)
    # the first key of a context draws much of the attention
    a["kc"][:, :, 0] *= 1.5
    if kind == "shared":
        a["kp"], a["vp"] = _randn(g, (nkv, case["prefix"], hd), dt), _randn(g, (nkv, case["prefix"], hd), dt)
        a["kp"][:, 0] *= 1.5
    else:
        a["w"] = torch.rand((B, nkv, S), generator=g, device="cuda", dtype=torch.float32)
    return a


_BASE, _TRAINED = 10000.0, 4096


def _rope_config(case):
    from flashmlx_amd import RopeConfig
    return RopeConfig(dims=case["dims"], base=_BASE, interleaved=case["interleaved"], scaling=case["scaling"],
                      factor=case["factor"], original_max=_TRAINED)


def _scale(case):
    return 1.0 / math.sqrt(case["head_dim"])


def prepare(case, seed):
    a = _inputs(case, seed)
    st = dict(case=case, **a)
    if case["kind"] == "evict":
        B, nkv, hd, S = case["batch"], case["kv_heads"], case["head_dim"], case["out_seq"]
        st["k_out"] = torch.zeros((B, nkv, S, hd), dtype=a["k"].dtype, device="cuda")
        st["v_out"] = torch.zeros_like(st["k_out"])
        st["w_out"] = torch.zeros((B, nkv, S), dtype=torch.float32, device="cuda")
    if case["kind"] in ("rope", "append"):
        if own:
            from flashmlx_amd import Rope
            st["rope"] = Rope(_rope_config(case))
        else:
            f, m = _frequencies(case)
            st["freqs"], st["m"] = f.to("cuda"), m
    return st


# ------------------------------------------------------------------ the framework's calls

def _run_own(st):
    import flashmlx_amd as F
    case = st["case"]
    kind = case["kind"]
    if kind == "rope":
        return st["rope"](st["q"], st["positions"], inverse=case["inverse"])
    if kind == "append":
        q = st["rope"].append(st["q"], st["k"], st["v"], st["positions"], st["offsets"], st["kc"], st["vc"])
        return [q, st["kc"], st["vc"]]
    if kind == "shared":
        return list(F.attention_shared_prefix(st["q"], st["kp"], st["vp"], st["kc"], st["vc"], st["offsets"],
                                              _scale(case)))
    if kind == "scored":
        return list(F.attention_scored(st["q"], st["kc"], st["vc"], st["offsets"], _scale(case), weights=st["w"]))
    lengths, kept = F.cache_evict(st["k"], st["v"], st["w"], st["lengths"], case["budget"], sinks=case["sinks"],
                                  recent=case["recent"], out=(st["k_out"], st["v_out"], st["w_out"]))
    return [lengths, kept, st["k_out"], st["v_out"], st["w_out"]]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ plain forms

def _frequencies(case):
    """Angle per position of each pair (64-bit) and the factor on the result."""
    n, s = case["dims"] // 2, case["factor"]
    i = torch.arange(n, dtype=torch.float64)
    f, m = _BASE ** (-i / n), 1.0
    if case["scaling"] == "linear":
        f = f / s
    elif case["scaling"] == "ntk":
        f = (_BASE * s ** (n / (n - 1))) ** (-i / n)
    elif case["scaling"] == "parts":
        # turns over the trained length: from 4 on unscaled, up to 1 scaled
        keep = ((_TRAINED * f / (2 * math.pi) - 1.0) / 3.0).clamp(0, 1)
        f = f * keep + f / s * (1 - keep)
    elif case["scaling"] == "yarn":
        # the pairs that turn 32 times and once, between them a ramp over the pairs
        lo = max(0, math.floor(n * math.log(_TRAINED / (32 * 2 * math.pi)) / math.log(_BASE)))
        hi = min(2 * n - 1, math.ceil(n * math.log(_TRAINED / (2 * math.pi)) / math.log(_BASE)))
        keep = 1 - ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f * keep + f / s * (1 - keep)
        m = 0.1 * math.log(s) + 1.0
    return f, m


def _rotate(x, positions, freqs, m, case, inverse):
    d = case["dims"]
    ang = positions.double()[..., None] * freqs
    cos, sin = (ang.cos() * m).float()[:, :, None], (ang.sin() * (-m if inverse else m)).float()[:, :, None]
    y = x.float().clone()
    a, b = (slice(0, d, 2), slice(1, d, 2)) if case["interleaved"] else (slice(0, d // 2), slice(d // 2, d))
    xa, xb = x[..., a].float(), x[..., b].float()
    y[..., a] = xa * cos - xb * sin
    y[..., b] = xa * sin + xb * cos
    return y.to(x.dtype)


def _rows(q, nkv):
    """[B, L, nh, hd] to [B, nkv, L * rep, hd] in 32 bits."""
    B, L, nh, hd = q.shape
    return q.float().view(B, L, nkv, nh // nkv, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, L * (nh // nkv), hd)


def _unrows(o, L, nh):
    """[B, nkv, L * rep, ..] back to [B, L, nh, ..]."""
    B, nkv = o.shape[:2]
    rest = o.shape[3:]
    o = o.reshape(B, nkv, L, nh // nkv, *rest)
    return o.transpose(1, 2).reshape(B, L, nh, *rest)


def _own_seen(st, L, rep, S):
    n = (st["offsets"].long()[:, None] + torch.arange(1, L + 1, device="cuda")).clamp(0, S)
    n = n[:, :, None].expand(-1, -1, rep).reshape(n.shape[0], 1, 1, L * rep)
    return torch.arange(S, device="cuda")[:, None] < n


def _run_plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "rope":
        return _rotate(st["q"], st["positions"], st["freqs"], st["m"], case, case["inverse"])
    if kind == "append":
        q = _rotate(st["q"], st["positions"], st["freqs"], st["m"], case, False)
        k = _rotate(st["k"], st["positions"], st["freqs"], st["m"], case, False)
        b = torch.arange(case["batch"], device="cuda")[:, None]
        row = st["offsets"].long()[:, None] + torch.arange(case["q_len"], device="cuda")
        st["kc"][b, :, row] = k
        st["vc"][b, :, row] = st["v"]
        return [q, st["kc"], st["vc"]]
    if kind == "evict":
        return _evict_plain(st, case)
    nkv, L, nh, S = case["kv_heads"], case["q_len"], case["heads"], case["max_seq"]
    q = _rows(st["q"], nkv) * _scale(case)
    R = q.shape[2]
    s = st["kc"].float() @ q.transpose(-1, -2).contiguous()
    s = s.masked_fill_(~_own_seen(st, L, nh // nkv, S), -math.inf)  # [B, nkv, S, R]
    m = s.amax(dim=2, keepdim=True)
    if kind == "shared":
        B, P = case["batch"], case["prefix"]
        qp = q.transpose(0, 1).reshape(nkv, B * R, -1)
        sp = st["kp"].float() @ qp.transpose(-1, -2).contiguous()  # [nkv, P, B R]
        mp = sp.amax(dim=1, keepdim=True).view(nkv, 1, B, R).permute(2, 0, 1, 3)
        m = torch.maximum(m, mp)
        e = torch.exp(s.sub_(m))
        ep = torch.exp(sp.sub_(m.permute(1, 2, 0, 3).reshape(nkv, 1, B * R)))
        z = e.sum(dim=2) + ep.sum(dim=1).view(nkv, B, R).transpose(0, 1)
        o = e.transpose(-1, -2).contiguous() @ st["vc"].float()
        op = ep.transpose(-1, -2).contiguous() @ st["vp"].float()
        o = (o + op.view(nkv, B, R, -1).transpose(0, 1)) / z[..., None]
        return [_unrows(o, L, nh).to(st["q"].dtype), _unrows(m[:, :, 0] + torch.log(z), L, nh)]
    e = torch.exp(s.sub_(m))
    p = e / e.sum(dim=2, keepdim=True)
    o = p.transpose(-1, -2).contiguous() @ st["vc"].float()
    return [_unrows(o, L, nh).to(st["q"].dtype), st["w"] + p.sum(dim=-1)]


def _evict_plain(st, case):
    S, budget = case["max_seq"], case["budget"]
    n = st["lengths"].long()[:, None, None]
    j = torch.arange(S, device="cuda")
    score = st["w"].masked_fill((j < case["sinks"]) | (j >= n - case["recent"]), math.inf).masked_fill(j >= n, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :budget]
    count = n.clamp(max=budget)
    live = torch.arange(order.shape[-1], device="cuda") < count
    kept = torch.where(live, order, S).sort(dim=-1).values
    pick = kept.clamp(max=S - 1)
    rows = live.expand_as(pick)
    C = pick.shape[-1]

    def move(src, dst):
        index = pick if src.dim() == 3 else pick[..., None].expand(-1, -1, -1, src.shape[-1])
        keep = rows if src.dim() == 3 else rows[..., None]
        dst[:, :, :C] = torch.where(keep, src.gather(2, index), dst[:, :, :C])

    move(st["k"], st["k_out"])
    move(st["v"], st["v_out"])
    move(st["w"], st["w_out"])
    kept = torch.where(live, kept, -1).to(torch.int32)
    if C < budget:
        kept = torch.nn.functional.pad(kept, (0, budget - C), value=-1)
    return [count.view(-1).to(torch.int32), kept, st["k_out"], st["v_out"], st["w_out"]]


# ------------------------------------------------------------------ 64 bits

def _exact_rotation(case, positions, x, inverse):
    """Each pair as a complex number times m e^(i p f)."""
    n, s, sc = case["dims"] // 2, case["factor"], case["scaling"]
    f, m = np.empty(n), 1.0
    for i in range(n):
        w = math.exp(-math.log(_BASE) * i / n)
        if sc == "linear":
            w /= s
        elif sc == "ntk":
            w = math.exp(-(math.log(_BASE) + math.log(s) * n / (n - 1)) * i / n)
        elif sc == "parts":
            turns = _TRAINED * w / (2 * math.pi)
            keep = 0.0 if turns < 1 else 1.0 if turns > 4 else (turns - 1) / 3
            w = keep * w + (1 - keep) * w / s
        elif sc == "yarn":
            def pair(turns):
                return n * math.log(_TRAINED / (turns * 2 * math.pi)) / math.log(_BASE)
            lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), 2 * n - 1)
            part = 0.0 if i <= lo else 1.0 if i >= hi else (i - lo) / (hi - lo)
            w = (1 - part) * w + part * w / s
            m = 0.1 * math.log(s) + 1
        f[i] = w
    ang = positions.double().unsqueeze(-1) * torch.from_numpy(f).to(positions.device)
    turn = torch.polar(torch.full_like(ang, m), -ang if inverse else ang).unsqueeze(2)
    y, d = x.double(), case["dims"]
    head = y[..., :d]
    if case["interleaved"]:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], n, 2).contiguous()) * turn
        head = torch.view_as_real(z).reshape(head.shape)
    else:
        z = torch.complex(head[..., :n].contiguous(), head[..., n:].contiguous()) * turn
        head = torch.cat([z.real, z.imag], dim=-1)
    return torch.cat([head, y[..., d:]], dim=-1)


def _exact_evict(case, a):
    B, nkv, budget = case["batch"], case["kv_heads"], case["budget"]
    kept = torch.full((B, nkv, budget), -1, dtype=torch.int32)
    w, lengths = a["w"].cpu().numpy(), a["lengths"].tolist()
    for b, n in enumerate(lengths):
        for h in range(nkv):
            if n <= budget:
                idx = np.arange(n)
            else:
                first, last = case["sinks"], max(case["sinks"], n - case["recent"])
                rest = np.arange(first, last)
                rest = rest[np.lexsort((rest, -w[b, h, first:last]))][:budget - first - (n - last)]
                idx = np.sort(np.concatenate([np.arange(first), rest, np.arange(last, n)]))
            kept[b, h, :len(idx)] = torch.from_numpy(idx.astype(np.int32))
    index, S = kept.cuda().long(), case["out_seq"]
    live = index >= 0

    def moved(t):
        d = torch.zeros((B, nkv, S, *t.shape[3:]), dtype=torch.float64, device="cuda")
        i = torch.nonzero(live, as_tuple=True)
        d[i[0], i[1], i[2]] = t[i[0], i[1], index[live]].double()
        return d

    lens = torch.tensor([min(n, budget) for n in lengths], dtype=torch.int32)
    return [lens, kept, moved(a["k"]), moved(a["v"]), moved(a["w"])]


def exact(case, seed):
    a, kind = _inputs(case, seed), case["kind"]
    if kind == "rope":
        return _exact_rotation(case, a["positions"], a["q"], case["inverse"])
    if kind == "append":
        q = _exact_rotation(case, a["positions"], a["q"], False)
        k = _exact_rotation(case, a["positions"], a["k"], False)
        kc, vc = a["kc"].double(), a["vc"].double()
        for b, row in enumerate(a["offsets"].tolist()):
            kc[b, :, row:row + case["q_len"]] = k[b].transpose(0, 1)
            vc[b, :, row:row + case["q_len"]] = a["v"][b].transpose(0, 1).double()
        return [q, kc, vc]
    if kind == "evict":
        return _exact_evict(case, a)
    B, L, nh, hd = a["q"].shape
    nkv, S = case["kv_heads"], case["max_seq"]
    rep = nh // nkv
    out = torch.zeros((B, L, nh, hd), dtype=torch.float64, device="cuda")
    lse = torch.zeros((B, L, nh), dtype=torch.float64, device="cuda")
    w = a["w"].double() if kind == "scored" else None
    for g in range(nkv):
        for b, off in enumerate(a["offsets"].tolist()):
            n = min(off + L, S)
            keys, vals = a["kc"][b, g, :n].double(), a["vc"][b, g, :n].double()
            if kind == "shared":
                keys, vals = torch.cat([a["kp"][g].double(), keys]), torch.cat([a["vp"][g].double(), vals])
            q = a["q"][b, :, g * rep:(g + 1) * rep].double()
            s = torch.matmul(q.reshape(L * rep, hd), keys.t().contiguous()).view(L, rep, -1) / math.sqrt(hd)
            # token l does not see the keys of the tokens after it
            j, first = torch.arange(keys.shape[0], device="cuda"), keys.shape[0] - n
            late = j > first + off + torch.arange(L, device="cuda")[:, None]
            s = s.masked_fill(late[:, None], -math.inf)
            lse[b, :, g * rep:(g + 1) * rep] = torch.logsumexp(s, dim=-1)
            p = torch.softmax(s, dim=-1)
            out[b, :, g * rep:(g + 1) * rep] = torch.matmul(p.view(L * rep, -1), vals).view(L, rep, hd)
            if w is not None:
                w[b, g, :n] += p.sum(dim=(0, 1))
    return [out, lse] if kind == "shared" else [out, w]
