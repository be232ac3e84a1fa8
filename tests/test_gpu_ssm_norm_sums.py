"""Every element of a group counts in its norm: one at a time is 1 and all
others 0, so that a part left out of the sum of squares makes the output 1 /
sqrt(eps) in place of 1 / sqrt(1 / size + eps). By every number of lanes and
vectors that a group can be dealt to.

The bound: 1 / size and its sum with eps rounded (2^-24 each, half of that in
the root), the root and the quotient to 2^-23 each, a product with 1: 2^-21 of
the value together, and half a step of the output's type."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-9


def _places(size, most=600):
    """All elements of small groups; of large ones the first and last ones and some of every part between."""
    if size <= most:
        return torch.arange(size)
    some = torch.cat([torch.arange(64), torch.arange(size - 64, size), torch.arange(0, size, max(1, size // (most - 128)))])
    return some.unique()


def _check(got, places, size):
    want = torch.tensor(1.0 / size + EPS, dtype=torch.float64).rsqrt()
    rows = torch.arange(len(places))
    got = got.double().cpu()
    one = got[rows, places]
    off = want * (2.0 ** -21 + torch.finfo(F32).eps)
    return one, want, off, got


@pytest.mark.parametrize("dtype,size,groups,pad", [
    # vectors of 8: 1 to 12 by 4 lanes, to 48 by 16, to 128 by 64, then a workgroup, kept up to 1024 and read twice beyond
    *[(BF16, 8 * v, 3, 0) for v in (1, 3, 4, 5, 8, 9, 12, 13, 16, 17, 32, 33, 48, 49, 64, 65, 128, 129, 256, 257, 512, 513, 1024,
                                    1025, 2500)],
    # of 4
    *[(F32, 4 * v, 2, 0) for v in (1, 4, 12, 48, 100, 128, 130, 1000, 1030, 2250)],
    # single elements
    *[(F16, v, 3, 1) for v in (1, 3, 7, 11, 33, 47, 65, 127, 255, 511, 1023, 1025, 3001)]])
def test_every_element_counts(gpu, fmx, dtype, size, groups, pad):
    places = _places(size)
    x = torch.zeros(len(places), groups * size + pad, dtype=dtype)
    for g in range(groups):
        x[torch.arange(len(places)), g * size + places] = 1.0
    x = x.cuda()[:, :groups * size]
    print("norm", dtype, size, groups, flush=True)
    for many in (False, True):  # (two groups at a time)
        rows = x
        if many:
            times = -(-4096 * 64 // (len(places) * groups)) + 1
            if times * x.numel() > 1 << 28:
                continue
            rows = x.repeat(times, 1)
            if pad:
                rows = torch.nn.functional.pad(rows, (0, pad))[:, :-pad]
        out = fmx.gated_norm(rows[None], None, eps=EPS, groups=groups)[0].unflatten(1, (groups, size))
        if many:
            assert torch.equal(out, out[:len(places)].repeat(times, 1, 1))
        for g in range(groups):
            one, want, off, got = _check(out[:len(places), g], places, size)
            assert ((one - want).abs() <= off + want * torch.finfo(dtype).eps / 2).all()
            assert (got.sum(1) == one).all()


@pytest.mark.parametrize("dtype,nh,hd,norm_groups,pad", [
    (BF16, 4, 64, 1, 0), (F16, 4, 64, 2, 1), (BF16, 32, 64, 1, 0), (BF16, 48, 64, 1, 0), (F16, 33, 64, 3, 1), (BF16, 64, 128, 1, 0),
    (F16, 96, 96, 1, 0), (BF16, 64, 256, 1, 0), (F16, 5, 8, 5, 3), (BF16, 64, 256, 2, 1)])
def test_every_element_counts_in_a_step(gpu, fmx, dtype, nh, hd, norm_groups, pad):
    """The convolution hands x on, b and c are 0, the skip is 1: the norm's rows are x."""
    N, inner = 8, nh * hd
    C, size = inner + 2 * N, inner // norm_groups
    w = torch.zeros(C, 2, dtype=dtype)
    w[:, 1] = 1.0
    layer = fmx.SsmLayer(w.cuda(), -torch.ones(nh, device="cuda"), None, hd, 1, N, d=torch.ones(nh, device="cuda"),
                         norm_groups=norm_groups, eps=EPS, activation=None)
    places = _places(size)
    B = len(places)
    xbc = torch.zeros(B, C + pad, dtype=dtype)
    for g in range(norm_groups):
        xbc[torch.arange(B), g * size + places] = 1.0
    xbc = xbc.cuda()[:, :C]
    print("step", dtype, nh, hd, norm_groups, flush=True)
    out = layer.step(xbc, torch.zeros(B, nh, dtype=dtype, device="cuda"), None, *layer.new_states(B))
    for g in range(norm_groups):
        one, want, off, got = _check(out.unflatten(1, (norm_groups, size))[:, g], places, size)
        assert ((one - want).abs() <= off + want * torch.finfo(dtype).eps / 2).all()
        assert (got.sum(1) == one).all()
