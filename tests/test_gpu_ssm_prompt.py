"""A layer's prompt moves both of its states or neither."""
from __future__ import annotations


import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rand(seed, *shape, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _layer(fmx, dtype, taps=4, **kw):
    """4 heads of 16 rows, 2 groups of 32 columns."""
    kw = {**dict(norm_groups=2, dt_limits=(0.001, 0.5)), **kw}
    return fmx.SsmLayer(_rand(1, 192, taps, dtype=dtype), -_rand(2, 4).abs(), _rand(3, 64, dtype=dtype), 16, 2, 32,
                        conv_bias=_rand(4, 192, dtype=dtype), d=_rand(5, 4), dt_bias=_rand(6, 4), **kw)


def _call(dtype, taps=4, L=21):
    return dict(xbc=_rand(7, 2, L, 192, dtype=dtype), dt=_rand(8, 2, L, 4, dtype=dtype), z=_rand(9, 2, L, 64, dtype=dtype),
                conv_state=_rand(10, 3, taps - 1, 192, dtype=dtype), state=_rand(11, 3, 4, 16, 32))


@pytest.mark.parametrize("what", ["dt", "dt type", "state", "state type", "state place", "z", "z type", "out", "out twice",
                                  "out over state", "eps", "limits", "norm groups", "float32"])
def test_a_refused_prompt_moves_nothing(gpu, fmx, what):
    dtype = F32 if what == "float32" else BF16
    layer = _layer(fmx, dtype, **{"eps": dict(eps=0.0), "limits": dict(dt_limits=(1.0, 0.5)),
                                  "norm groups": dict(norm_groups=3)}.get(what, {}))
    p = _call(dtype)
    if what == "state place":  # 4 bytes behind an aligned address
        p["state"] = torch.cat([p["state"].flatten()[:1], p["state"].flatten()])[1:].view(p["state"].shape)
    p.update({"dt": lambda: dict(dt=p["dt"][:, :20]), "dt type": lambda: dict(dt=p["dt"].float()),
              "state": lambda: dict(state=p["state"][..., :24].contiguous()), "state type": lambda: dict(state=p["state"].double()),
              "z": lambda: dict(z=p["z"][..., :32]), "z type": lambda: dict(z=p["z"].half()),
              "out": lambda: dict(out=torch.empty(2, 21, 32, dtype=BF16, device="cuda")),
              "out twice": lambda: dict(out=torch.empty(2, 1, 64, dtype=BF16, device="cuda").expand(2, 21, 64)),
              "out over state": lambda: dict(out=p["state"].view(BF16).flatten()[:2 * 21 * 64].view(2, 21, 64)),
              }.get(what, dict)())
    before = p["conv_state"].clone(), p["state"].clone()
    with pytest.raises((ValueError, TypeError, fmx.FmxError)):
        layer.prompt(**p)
    torch.cuda.synchronize()
    assert torch.equal(p["conv_state"], before[0]) and torch.equal(p["state"], before[1])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("taps,L,lengths,slots,gate", [
    (4, 21, [21, 3], [2, 0], True), (1, 5, None, None, True), (3, 200, [64, 199], None, False), (2, 1, None, [5, 1], True),
    (4, 0, None, None, True)])
def test_a_prompt_is_its_three_calls(gpu, fmx, dtype, taps, L, lengths, slots, gate):
    layer, p = _layer(fmx, dtype, taps, gate_first=False), _call(dtype, taps, L)
    at = [None if t is None else torch.tensor(t, dtype=torch.int32, device="cuda") for t in (lengths, slots)]
    z = p["z"] if gate else None
    conv_state, state = p["conv_state"].clone(), p["state"].clone()
    out = torch.full_like(p["z"], 7.0)
    print("prompt", dtype, taps, L, lengths, slots, flush=True)
    got = layer.prompt(p["xbc"], p["dt"], z, conv_state, state, *at, out=out)
    assert got is out
    v = fmx.causal_conv(p["xbc"], layer.conv_weight, layer.conv_bias, p["conv_state"], p["conv_state"], *at)
    y = fmx.ssm_scan(v[..., :64].view(2, L, 4, 16), p["dt"], layer.a, v[..., 64:128].view(2, L, 2, 32),
                     v[..., 128:].view(2, L, 2, 32), layer.d, layer.dt_bias, p["state"], p["state"], *at, dt_limits=(0.001, 0.5))
    want = fmx.gated_norm(y.flatten(2), layer.norm_weight, z, groups=2, gate_first=False, lengths=at[0],
                          out=torch.full_like(p["z"], 7.0))
    assert torch.equal(got, want) and torch.equal(conv_state, p["conv_state"]) and torch.equal(state, p["state"])
    if taps > 1 and L:  # pools of two sizes: the second sequence's slot is in one of them alone
        one, slot = torch.zeros_like(conv_state[:1]), torch.tensor([0, 2], dtype=torch.int32, device="cuda")
        layer.prompt(p["xbc"], p["dt"], z, one, state, at[0], slot, out=out)
        both = torch.zeros_like(conv_state), p["state"]
        assert torch.equal(layer.prompt(p["xbc"], p["dt"], z, *both, at[0], slot, out=want), out)
        assert torch.equal(one[0], both[0][0]) and torch.equal(state, both[1])
    if lengths is None:
        assert torch.equal(layer.prompt(p["xbc"], p["dt"], z, torch.zeros_like(conv_state), torch.zeros_like(state)),
                           layer.prompt(p["xbc"], p["dt"], z, None, None))
