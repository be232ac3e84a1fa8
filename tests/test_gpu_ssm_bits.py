"""The bits of the selective scan's sums, states and outputs, where tolerances
that grow with the sums' lengths would hide a lost part.

The inputs make every product and every sum a multiple of 2^-23 below 2, so
that fp32 takes each of them exactly, in any order: decays of 1, one column of
the state at a time, x of 1 and -1. What is left after two numbers of 24 bits
cancel shows how many of their bits the kernels have kept. In bfloat16 that is
all of them. Float16 takes a state's numbers and what tokens bring, dt x times
a decay, as two numbers of its own, each rounded: the first leaves 12 bits and a
sign of 24, the second is off by half a step of 11 of those, 2^-23 of the power
of two below the value."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
STEP = 2.0 ** -23


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _inputs(dtype, L, nh, hd, groups, N):
    zeros = lambda *s: torch.zeros(*s, dtype=dtype)  # noqa: E731
    return dict(x=zeros(1, L, nh, hd), dt=zeros(1, L, nh), b=zeros(1, L, groups, N), c=zeros(1, L, groups, N),
                a=torch.zeros(nh))


def _scan(fmx, p, dt_bias=None, state=None):
    nh, hd, N = p["x"].shape[2], p["x"].shape[3], p["b"].shape[3]
    after = torch.empty(1, nh, hd, N, device="cuda")
    y = fmx.ssm_scan(*(p[k].cuda() for k in ("x", "dt", "a", "b", "c")), dt_bias=dt_bias, state=state, state_out=after,
                     softplus=False, dt_limits=(0.0, math.inf))
    return y.double().cpu()[0], after.double().cpu()[0]


def test_silu(gpu, fmx):
    """The documented bound, over the whole range: for negative v the rounded
    argument of e^-v counts |v| log2 e 2^-24 ln 2 and log2 e's own rounding half of
    that again, the exponential, the sum, the reciprocal and the product 3.5 2^-23."""
    v = torch.cat([torch.linspace(-87, 87, 65536), 2.0 ** torch.arange(-60.0, 7), -2.0 ** torch.arange(-60.0, 7)])
    y = fmx.causal_conv(v.cuda().view(1, -1, 1), torch.ones(1, 1, device="cuda")).double().cpu().flatten()
    v = v.double()
    want = v / (1 + torch.exp(-v))
    off = want.abs() * 2.0 ** -23 * (4 + (-v).clamp(min=0))
    live = v >= -87
    assert ((y - want).abs() <= off)[live].all()
    low = torch.tensor([-87.5, -88.0, -89.0, -100.0, -1e4, -3e38], device="cuda").view(1, -1, 1)
    assert (fmx.causal_conv(low, torch.ones(1, 1, device="cuda")).abs() < 1e-35).all()


SHAPES = [(6, 16, 2, 8), (6, 64, 2, 64), (4, 72, 1, 128), (2, 64, 1, 256)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L", [5, 9, 64, 100, 700])
@pytest.mark.parametrize("nh,hd,groups,N", SHAPES)
def test_a_state_keeps_its_bits_into_outputs(gpu, fmx, dtype, L, nh, hd, groups, N):
    """Two columns of numbers 1 + k 2^-23, one taken from the other: k - k'
    steps, at most 7 bits, which both types hold."""
    p = _inputs(dtype, L, nh, hd, groups, N)
    p["c"][..., 1], p["c"][..., N - 2] = 1.0, -1.0
    k = torch.randint(0, 2 ** 22, (1, nh, hd, N), generator=_gen(N + L), dtype=torch.float64)
    k[..., N - 2] = k[..., 1] + torch.randint(-100, 101, (1, nh, hd), generator=_gen(3), dtype=torch.float64)
    k = k.clamp(min=0)
    state = (1 + k * STEP).float().cuda()
    assert torch.equal(state.double().cpu(), 1 + k * STEP)
    want = ((k[..., 1] - k[..., N - 2]) * STEP)[0].expand(L, nh, hd)
    print("scan", dtype, L, nh, hd, groups, N, flush=True)
    y, after = _scan(fmx, p, state=state)
    assert torch.equal(after, state.double().cpu()[0])
    off = 2 * STEP if dtype == F16 and L > 8 else 0.0  # (two numbers from 1 to 2; multiples of 2^-24 are no rounding)
    assert ((y - want).abs() <= off).all(), (y - want).abs().max() / STEP


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L,first,second", [
    (8, 1, 3), (64, 0, 1), (64, 3, 9), (64, 3, 20), (64, 17, 60), (100, 5, 70), (200, 66, 100), (700, 3, 40), (700, 130, 500)])
@pytest.mark.parametrize("nh,hd,groups,N", SHAPES)
def test_tokens_keep_their_bits(gpu, fmx, dtype, L, first, second, nh, hd, groups, N):
    """Two tokens of opposite x whose steps 1 + j 2^-23 and 1 + j 2^-23 + i
    2^-20 differ by 7 bits: outputs between them are the first's step, those
    behind the second -i 2^-20, and the state at the end is that or, in a
    column that the second does not reach, the first's 24 bits."""
    p = _inputs(dtype, L, nh, hd, groups, N)
    # (below 2^21: the steps stay below 1.5, multiples of 2^-23)
    j = torch.randint(0, 2 ** 21, (nh,), generator=_gen(N + L + first)).double()
    i = torch.randint(1, 101, (nh,), generator=_gen(7)).double()
    bias = (1 + j * STEP).float()
    p["dt"][0, second] = (i * 2.0 ** -20).to(dtype)
    assert torch.equal(p["dt"][0, second].double(), i * 2.0 ** -20)
    p["x"][0, first], p["x"][0, second] = 1.0, -1.0
    col = 5
    p["b"][0, first, :, col], p["b"][0, second, :, col] = 1.0, 1.0
    p["b"][0, first, :, col + 1] = 1.0
    p["c"][..., col] = 1.0
    step = 1 + j * STEP
    want = torch.zeros(L, nh, hd, dtype=torch.float64)
    want[first:second] = step[:, None]
    want[second:] = (-i * 2.0 ** -20)[:, None]
    print("scan", dtype, L, first, second, nh, hd, groups, N, flush=True)
    y, after = _scan(fmx, p, dt_bias=bias.cuda())
    off = STEP if dtype == F16 and L > 8 else 0.0  # of a number from 1 to 2 each time that it is taken in two
    half = torch.finfo(dtype).eps / 2
    assert ((y[:second] - want[:second]).abs() <= 2 * off + (want[:second].abs() + 2 * off) * half).all()
    # (of the first into the state and from it, or of both into it)
    assert ((y[second:] - want[second:]).abs() <= 2 * off).all(), (y[second:] - want[second:]).abs().max() / STEP
    if dtype == F16 and L > 8:  # a chunk's own tokens go by weights, which keep all bits
        end = min(L, (first // 64 + 1) * 64)
        if second < end:
            assert torch.equal(y[second:end], want[second:end])
    assert ((after[..., col] + (i * 2.0 ** -20)[:, None]).abs() <= 2 * off).all()
    assert ((after[..., col + 1] - step[:, None]).abs() <= off).all()
    rest = [n for n in range(N) if n not in (col, col + 1)]
    assert (after[..., rest] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("first,second", [(3, 40), (70, 900), (300, 310), (511, 640)])
@pytest.mark.parametrize("nh,hd,groups,N", [(258, 8, 2, 64), (130, 16, 130, 128), (132, 24, 66, 256)])
def test_bits_over_many_chunks(gpu, fmx, dtype, first, second, nh, hd, groups, N):
    """16 chunks in a row, two heads to a workgroup and one."""
    test_tokens_keep_their_bits(gpu, fmx, dtype, 1000, first, second, nh, hd, groups, N)
    test_a_state_keeps_its_bits_into_outputs(gpu, fmx, dtype, 1000, nh, hd, groups, N)
