"""The softmax weights of attention over many rows per kv head reach the value
product with more bits than the inputs' type has: where all keys have the same
value, the output is that value to the bit, whatever the weights are."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _setup(dt, B, L, nh, nkv, hd, P, S, late):
    """Key 0 scores 0 for every row, key `late`, in a later part of the same
    tile's keys, up to 6 log2 more (a raise of the maximum that a tile may put
    off), all others far less. Only element 0 of queries and keys is not 0, so
    a score is one exact product."""
    g = torch.Generator(device="cuda").manual_seed(hd + L)
    q = torch.zeros(B, L, nh, hd, dtype=dt, device="cuda")
    q[..., 0] = (0.5 + 3.6 * torch.rand(B, L, nh, generator=g, device="cuda")).to(dt)
    v = (1.0 + torch.rand(nkv, 1, hd, generator=g, device="cuda")).to(dt)

    def keys(*shape):
        k = torch.zeros(*shape, hd, dtype=dt, device="cuda")
        k[..., 0] = -8.0
        return k

    kp, kc = (keys(nkv, P) if P else None), keys(B, nkv, S)
    first = kp if P else kc
    first[..., 0, 0], first[..., late, 0] = 0.0, 1.0
    vp = v.expand(nkv, P, hd).contiguous() if P else None
    vc = v.expand(B, nkv, S, hd).contiguous()
    offs = torch.full((B,), S - L, dtype=torch.int32, device="cuda")
    want = v[:, 0].repeat_interleave(nh // nkv, dim=0).expand(B, L, nh, hd)
    return q, kp, vp, kc, vc, offs, want


SHAPES = [
    # B, L, nh, nkv, hd, P, S: many rows, own keys in one piece, in several
    (1, 40, 4, 1, 128, 0, 300), (2, 40, 4, 2, 64, 0, 300), (1, 40, 4, 1, 256, 0, 300), (1, 40, 4, 1, 72, 0, 300),
    (1, 40, 4, 1, 64, 0, 1030), (1, 1, 48, 1, 128, 0, 300),
    # few rows, which run in narrow tiles
    (1, 1, 4, 1, 128, 0, 300), (7, 1, 4, 1, 128, 200, 40), (8, 1, 4, 1, 64, 200, 40), (2, 5, 6, 2, 256, 200, 40),
    # a prefix with own keys in narrow tiles of one and two row sets, in wide ones, with none
    (40, 1, 4, 1, 128, 200, 40), (10, 5, 4, 1, 128, 200, 40), (3, 40, 4, 1, 64, 200, 60), (40, 1, 4, 1, 128, 200, 0),
    (40, 1, 4, 1, 256, 600, 40), (20, 2, 6, 3, 80, 300, 33),
]


@pytest.mark.parametrize("late", [17, 40, 63])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_equal_values_come_out_as_they_are(gpu, fmx, dt, shape, late):
    """sum w v / sum w with one v: a weight kept as two numbers of the type
    loses 2^-16 (2^-22) of it, sums of at most 1030 keys in 32 bits, with
    truncation, 3 n 2^-24 < 2^-12.3 on both sides together: less than the half
    step of 2^-9 (2^-12) of v at least that would show. One number's 2^-8
    (2^-11) does show."""
    q, kp, vp, kc, vc, offs, want = _setup(DT[dt], *shape, late)
    out, _ = fmx.attention_shared_prefix(q, kp, vp, kc, vc, offs, 1.0)
    assert torch.equal(out, want), f"{int((out != want).sum())} of {out.numel()} differ"
    if kp is None:
        out, _ = fmx.attention_scored(q, kc, vc, offs, 1.0)
        assert torch.equal(out, want)
