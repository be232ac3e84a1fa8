"""Infinities and NaN in the selective scan's inputs: they reach their token,
their rows and what comes behind them, and change no bit of anything else; for
both types, by the walk (6 tokens), in chunks of one segment (128) and in
several segments (700), one head to a workgroup and two (many sequences)."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
HEADS, ROWS, GROUPS = 4, 64, 2


def _inputs(seed, dtype, B, L, N):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    p = dict(x=rand(B, L, HEADS, ROWS).to(dtype), dt=rand(B, L, HEADS).to(dtype), b=rand(B, L, GROUPS, N).to(dtype),
             c=rand(B, L, GROUPS, N).to(dtype), a=-rand(HEADS).abs(), d=rand(HEADS), dt_bias=rand(HEADS) - 3,
             state=rand(B, HEADS, ROWS, N))
    return {k: v.cuda() for k, v in p.items()}


def _run(fmx, p, limits):
    after = torch.empty_like(p["state"])
    y = fmx.ssm_scan(p["x"], p["dt"], p["a"], p["b"], p["c"], p["d"], p["dt_bias"], p["state"], after, dt_limits=limits)
    return y, after


SIZES = [(1, 6, 128, (0, 3, 5)), (1, 9, 64, (0, 8)), (2, 128, 128, (0, 15, 66, 127)), (1, 700, 128, (0, 70, 300, 699)),
         (1, 700, 64, (191, 192, 500)), (70, 130, 128, (1, 64, 129)), (70, 100, 32, (40,))]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,L,N,places", SIZES)
@pytest.mark.parametrize("v", [math.inf, -math.inf, math.nan])
def test_one_row_of_x(gpu, fmx, dtype, B, L, N, places, v):
    """One row of one head of one token: that row from that token on, and its
    state; every other row, of that head too, keeps its bits."""
    p = _inputs(L + N, dtype, B, L, N)
    clean, state = _run(fmx, p, (0.001, 0.5))
    assert torch.isfinite(clean).all() and torch.isfinite(state).all()
    for at in places:
        q, h, r = B - 1, 1 + at % 3, (17 * at + 5) % ROWS
        old = p["x"][q, at, h, r].clone()
        p["x"][q, at, h, r] = v
        print("scan", dtype, B, L, N, at, h, r, flush=True)
        y, after = _run(fmx, p, (0.001, 0.5))
        p["x"][q, at, h, r] = old
        assert not torch.isfinite(y[q, at:, h, r]).any() and not torch.isfinite(after[q, h, r]).any()
        y[q, at:, h, r], after[q, h, r] = clean[q, at:, h, r], state[q, h, r]
        assert torch.equal(y, clean) and torch.equal(after, state)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,L,N,places", SIZES)
@pytest.mark.parametrize("what", ["x", "b", "c", "dt"])
def test_a_token(gpu, fmx, dtype, B, L, N, places, what):
    """x of all rows of a head, b or c in one column of a group, a head's step
    without an upper limit."""
    p = _inputs(L + N + 1, dtype, B, L, N)
    limits = (0.001, math.inf)
    clean, state = _run(fmx, p, limits)
    for at in places:
        for v in (math.inf, math.nan):
            q, h = B - 1, 2 + at % 2
            heads = [2, 3] if what in "bc" else [h]  # (the second group's)
            part = p[what][q, at, 1, 3:4] if what in "bc" else p[what][q, at, h]
            old = part.clone()
            part.fill_(v)
            print("scan", dtype, B, L, N, what, at, v, flush=True)
            y, after = _run(fmx, p, limits)
            part.copy_(old)
            reached = slice(at, at + 1) if what == "c" else slice(at, L)
            assert not torch.isfinite(y[q, reached, heads]).any()
            y[q, reached, heads] = clean[q, reached, heads]
            assert torch.equal(y, clean)
            if what == "b":  # its column
                assert not torch.isfinite(after[q, heads, :, 3]).any()
                after[q, heads, :, 3] = state[q, heads, :, 3]
            elif what != "c":
                assert not torch.isfinite(after[q, heads]).any()
                after[q, heads] = state[q, heads]
            if what == "b" and dtype == F16 and L > 8:
                # (a row's power of two goes by its largest finite number, the lost column's no more among them: each of
                # the chunk's tokens, 64 at most, to 2^-37 of that, once either way)
                assert (after - state).abs().max() <= 2.0 ** -30 * state.abs().max()
            else:
                assert torch.equal(after, state)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L,at", [(6, 2), (100, 70), (200, 10), (700, 70), (700, 500)])
def test_what_a_token_brings_is_infinite(gpu, fmx, dtype, L, at):
    """A finite step of 3e38 and an x of 2: dt x is infinite in one row, and
    stays in it."""
    p = _inputs(5, dtype, 1, L, 64)
    p["x"].zero_(), p["dt"].zero_(), p["a"].zero_(), p["c"].zero_()
    p["dt_bias"].fill_(3e38)
    p["x"][:, at] = 0.25
    p["b"][:, at] = 2.0 ** -10
    p["d"] = None
    clean, state = _run(fmx, p, (0.0, math.inf))
    assert torch.isfinite(state).all() and (state.abs().amax(-1) > 1e33).all() and (clean == 0).all()
    p["x"][0, at, 1, 9] = 2.0
    print("scan", dtype, L, at, flush=True)
    y, after = _run(fmx, p, (0.0, math.inf))
    assert not torch.isfinite(after[0, 1, 9]).any()
    behind = at if L <= 8 else (at // 64 + 1) * 64  # (its own chunk's outputs take the token by (c . b) dt, which is 0, times x)
    assert not torch.isfinite(y[0, behind:, 1, 9]).any()
    y[0, at:, 1, 9], after[0, 1, 9] = clean[0, at:, 1, 9], state[0, 1, 9]
    assert torch.equal(y, clean) and torch.equal(after, state)
