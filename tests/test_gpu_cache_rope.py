"""Rotary positions (fmx_rope, fmx_rope_append) against 64 bits: both
pairings, part of the head, every scaling, positions near, far and negative,
vector and single-element paths, strided rows; the gradient as the inverse
call and by differences; appends with slots, rows outside the cache."""
from __future__ import annotations

import pytest
import torch

import cache_oracle as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _randn(shape, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)


def _positions(B, L, far, seed):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    return torch.randint(-far, far, (B, L), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,L,nh,hd,dims", [
    (1, 1, 1, 2, 2), (3, 1, 16, 128, 128), (2, 37, 5, 64, 32), (1, 5, 3, 80, 80), (1, 9, 7, 96, 24),
    (2, 3, 2, 1024, 1024), (1, 4, 100, 256, 64), (1, 6, 3, 33, 18), (1, 700, 2, 16, 16)])
def test_rope(gpu, fmx, dt, interleaved, B, L, nh, hd, dims):
    x, pos = _randn((B, L, nh, hd), DT[dt], hd + L), _positions(B, L, 100000, L)
    rope = fmx.Rope(fmx.RopeConfig(dims=dims, interleaved=interleaved))
    freqs, m = rope.cfg.frequencies()
    for inverse in (False, True):
        y = rope(x, pos, inverse=inverse)
        R.assert_within(y, *R.rotate(x, pos, freqs, m, dims, interleaved, inverse), f"inverse {inverse}")
    z = x.clone()
    assert torch.equal(rope(z, pos, out=z), rope(x, pos))  # in place


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("parts", 8.0), ("yarn", 4.0)])
def test_rope_scaled_and_far(gpu, fmx, scaling, factor):
    x = _randn((2, 8, 3, 128), torch.float32, 3)
    pos = torch.tensor([[0, 1, -1, 4095, 4096, 131071, -131072, 2 ** 24],
                        [2 ** 31 - 1, -2 ** 31, 2 ** 20 + 1, 7, 8, 9, 10, 11]], dtype=torch.int32, device="cuda")
    rope = fmx.Rope(fmx.RopeConfig(dims=128, scaling=scaling, factor=factor))
    freqs, m = rope.cfg.frequencies()
    R.assert_within(rope(x, pos), *R.rotate(x, pos, freqs, m, 128, False), scaling)


def test_rope_strided_rows(gpu, fmx):
    """q and k as views of one fused row, heads before tokens, and rows that
    start at odd elements (the single-element path)."""
    qkv = _randn((2, 7, 12 * 64 + 1), torch.bfloat16, 5)
    pos = _positions(2, 7, 5000, 9)
    rope = fmx.Rope(fmx.RopeConfig(dims=64))
    freqs, m = rope.cfg.frequencies()
    for view in (qkv[:, :, :256].unflatten(2, (4, 64)), qkv[:, :, 257:].unflatten(2, (8, 64)),
                 qkv[:, :, :256].reshape(2, 7, 4, 64).transpose(1, 2).contiguous().transpose(1, 2),
                 qkv[:, :1, :64].unflatten(2, (1, 64)).expand(2, 7, 4, 64)):
        want = R.rotate(view, pos, freqs, m, 64, False)
        R.assert_within(rope(view, pos), *want, str(view.stride()))
        out = torch.full((2, 9, 10, 72), 7.0, dtype=torch.bfloat16, device="cuda")
        rope(view, pos, out=out[:, 1:8, 1:1 + view.shape[2], 8:])
        R.assert_within(out[:, 1:8, 1:1 + view.shape[2], 8:], *want, "into a view")
        out[:, 1:8, 1:1 + view.shape[2], 8:] = 7.0
        assert bool((out == 7.0).all())
    q = qkv[:, :, :256].unflatten(2, (4, 64))
    want = R.rotate(q, pos, freqs, m, 64, False)
    rest = qkv[:, :, 256:].clone()
    rope(q, pos, out=q)  # in place within the fused row
    R.assert_within(q, *want, "in place")
    assert torch.equal(qkv[:, :, 256:], rest)


def test_rope_gradient(gpu, fmx):
    """sum(c * rope(x)) has the gradient rope(c, inverse): the formula's (the
    transposed turn) and by differences, exact here up to rounding because the
    call is linear in x."""
    cfg = fmx.RopeConfig(dims=24, interleaved=True, scaling="yarn", factor=4.0)
    rope = fmx.Rope(cfg)
    freqs, m = cfg.frequencies()
    x, c = _randn((1, 3, 2, 40), torch.float32, 1), _randn((1, 3, 2, 40), torch.float32, 2)
    pos = _positions(1, 3, 9000, 4)
    grad = rope(c, pos, inverse=True)
    R.assert_within(grad, *R.rotate(c, pos, freqs, m, 24, True, inverse=True), "formula")
    for i in range(0, 40, 3):
        d = torch.zeros_like(x)
        d[..., i] = 0.5
        diff = ((rope(x + d, pos).double() - rope(x - d, pos).double()) * c.double()).sum(-1)
        # three roundings of 2^-24 in values of up to |x| + 1, times 1.2 |c| and 40 terms
        bound = 4 * 2.0 ** -22 * (x.abs().max() + 1) * c.abs().sum(-1).max()
        assert float((diff - grad[..., i].double()).abs().max()) <= float(bound)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,L,nh,nkv,hd,interleaved", [(3, 1, 4, 4, 128, False), (5, 3, 8, 2, 64, True),
                                                       (2, 2, 7, 1, 33, False), (1, 1, 32, 4, 256, True)])
def test_rope_append(gpu, fmx, dt, B, L, nh, nkv, hd, interleaved):
    S, slots_n, dt = 20, B + 2, DT[dt]
    q, k, v = _randn((B, L, nh, hd), dt, 1), _randn((B, L, nkv, hd), dt, 2), _randn((B, L, nkv, hd), dt, 3)
    kc, vc = _randn((slots_n, nkv, S, hd), dt, 4), _randn((slots_n, nkv, S, hd), dt, 5)
    pos = _positions(B, L, 50000, 6)
    dims = hd // 2 * 2
    rope = fmx.Rope(fmx.RopeConfig(dims=dims, interleaved=interleaved))
    freqs, m = rope.cfg.frequencies()
    offs = torch.tensor([S - 1, 0, 7, 3, -2][:B], dtype=torch.int32, device="cuda")
    slot = torch.tensor([2, 0, slots_n, 1, 3][:B], dtype=torch.int32, device="cuda")
    for slots in (None, slot):
        kr, vr = kc.clone(), vc.clone()
        y = rope.append(q, k, v, pos, offs, kr, vr, slots=slots)
        R.assert_within(y, *R.rotate(q, pos, freqs, m, dims, interleaved), "q")
        want, bound = R.rotate(k, pos, freqs, m, dims, interleaved)
        touched = torch.zeros(slots_n, S, dtype=torch.bool)
        for b in range(B):
            s = b if slots is None else int(slot[b])
            for l in range(L):
                j = int(offs[b]) + l
                if 0 <= s < slots_n and 0 <= j < S:
                    R.assert_within(kr[s, :, j], want[b, l], bound[b, l], "key")
                    assert torch.equal(vr[s, :, j], v[b, l])
                    touched[s, j] = True
        keep = ~touched.cuda()
        assert torch.equal(kr.transpose(1, 2)[keep], kc.transpose(1, 2)[keep])
        assert torch.equal(vr.transpose(1, 2)[keep], vc.transpose(1, 2)[keep])


def test_rope_append_from_fused_rows(gpu, fmx):
    """q, k and v as views of one qkv row, caches with positions before heads."""
    B, nh, nkv, hd, S = 4, 8, 2, 64, 6
    qkv = _randn((B, 1, (nh + 2 * nkv) * hd), torch.float16, 1)
    rows = qkv.unflatten(2, (nh + 2 * nkv, hd))
    q, k, v = rows.split([nh, nkv, nkv], dim=2)
    kc, vc = (torch.zeros(B, S, nkv, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    pos, offs = _positions(B, 1, 900, 2), torch.tensor([0, 5, 2, 1], dtype=torch.int32, device="cuda")
    rope = fmx.Rope(fmx.RopeConfig(dims=hd))
    y = rope.append(q, k, v, pos, offs, kc.transpose(1, 2), vc.transpose(1, 2))
    assert torch.equal(y, rope(q, pos))
    b = torch.arange(B, device="cuda")
    assert torch.equal(kc[b, offs.long()], rope(k, pos)[:, 0])
    assert torch.equal(vc[b, offs.long()], v[:, 0])
    assert int((kc != 0).any(-1).sum()) == B * nkv
