"""Calls of the state space layer's operators near the limits that the header
gives, more than a count of rows, groups or elements as if each had a workgroup
or a thread of its own would let through. Inputs are one row or one sequence
many times over, so that every output is the same as of a small call."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def test_conv_of_2_34_elements(gpu, fmx):
    """4097 runs of 4 rows of 2^20 channels: more than 2^32 by single elements,
    2^28 threads of 8 rows and 8 channels."""
    C, L = 1 << 20, 4 * 4096 + 4
    row, w = _rand(1, 1, 1, C, dtype=BF16), _rand(2, C, 2, dtype=BF16)
    want = fmx.causal_conv(row.expand(1, 3, C), w)
    print("conv", L, C, flush=True)
    out = fmx.causal_conv(row.expand(1, L, C), w)
    assert torch.equal(out[:, 0], want[:, 0])
    for t in range(1, L, 512):
        assert (out[0, t:t + 512] == want[0, 1]).all(), t


@pytest.mark.parametrize("dtype,L,C,groups,pad", [
    (BF16, 1 << 21, 64, 8, 0), (BF16, (1 << 22) + 3, 40, 5, 8), (torch.float32, 1 << 20, 68, 17, 0), (BF16, 1 << 20, 51, 17, 1)])
def test_norm_of_2_24_groups(gpu, fmx, dtype, L, C, groups, pad):
    """As many groups as workgroups of a launch and more, 64 to a workgroup."""
    assert L * groups >= (1 << 24) - 1
    x, z = _rand(3, 1, 7, C + pad, dtype=dtype)[..., :C], _rand(4, 1, 7, C, dtype=dtype)
    n = L // 7 * 7
    many = x.expand(n // 7, 7, C)
    want = fmx.gated_norm(x, None, z, groups=groups)
    print("norm", dtype, L, C, groups, flush=True)
    out = fmx.gated_norm(many.expand(n // 7, 7, C), None, z.expand(n // 7, 7, C), groups=groups)
    assert (out == want).all()
    one = fmx.gated_norm(x[:, :1].expand(1, L, C), None, z[:, :1].expand(1, L, C), groups=groups)
    assert (one == want[:, :1]).all()


@pytest.mark.parametrize("B,L,nh,hd,N", [(40000, 9, 64, 64, 16), (70000, 3, 32, 128, 8)])
def test_scan_of_many_sequences(gpu, fmx, B, L, nh, hd, N):
    """More heads than workgroups of 4 rows each would allow: by chunks 64 rows
    of two heads to one, by the walk all rows of one."""
    assert B * nh * hd // 4 > 1 << 24
    x, dt = _rand(5, 1, L, nh, hd, dtype=BF16), _rand(6, 1, L, nh, dtype=BF16)
    b, c, a = _rand(7, 1, L, 1, N, dtype=BF16), _rand(8, 1, L, 1, N, dtype=BF16), -_rand(9, nh).abs()
    want = fmx.ssm_scan(x, dt, a, b, c)
    many = [t.expand(B, *t.shape[1:]) for t in (x, dt, b, c)]
    print("scan", B, L, nh, hd, N, flush=True)
    out = fmx.ssm_scan(many[0], many[1], a, many[2], many[3])
    for i in range(0, B, 4000):
        assert (out[i:i + 4000] == want).all(), i


def test_step_of_many_sequences(gpu, fmx):
    B, nh, hd, N = 17000, 64, 64, 8
    assert B * nh * hd // 4 > 1 << 24
    C = nh * hd + 2 * N
    layer = fmx.SsmLayer(_rand(1, C, 4, dtype=BF16), -_rand(2, nh).abs(), _rand(3, nh * hd, dtype=BF16), hd, 1, N, norm_groups=8)
    xbc, dt, z = _rand(4, 1, C, dtype=BF16), _rand(5, 1, nh, dtype=BF16), _rand(6, 1, nh * hd, dtype=BF16)
    small, states = layer.new_states(1), layer.new_states(B)
    print("step", B, flush=True)
    for _ in range(2):
        want = layer.step(xbc, dt, z, *small)
        out = layer.step(xbc.expand(B, C), dt.expand(B, nh), z.expand(B, nh * hd), *states)
        assert (out == want).all() and all((s == t).all() for s, t in zip(states, small))
