"""Host side of the state space layer's operators (include/fmx_ssm.h), without
a GPU: what is refused, and with which status; empty calls; workspace sizes.
No call here launches a kernel."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

import flashmlx_amd as F
from flashmlx_amd import _lib

OK, ARG, SHAPE, DTYPE, UNSUP, WS = (_lib.FMX_OK, _lib.FMX_ERR_ARG, _lib.FMX_ERR_SHAPE, _lib.FMX_ERR_DTYPE,
                                    _lib.FMX_ERR_UNSUPPORTED, _lib.FMX_ERR_WORKSPACE)
BF16, F16, F32 = _lib.FMX_BF16, _lib.FMX_F16, _lib.FMX_F32


class Heads:
    """Distinct fake arrays: never read, the calls are refused first."""
    next = 1 << 40

    def __new__(cls, bs=1 << 16, ts=1 << 12, hs=1 << 8, data=None):
        if data is None:
            cls.next += 1 << 36
            data = cls.next
        return C.byref(_lib.FmxHeads(data, bs, ts, hs))


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


AT = 1 << 46


def _conv(lib, dtype=BF16, B=2, L=3, ch=64, taps=4, act=1, x=None, w=1 << 33, bias=1 << 34, s_in=1 << 35,
          s_out=1 << 36, n_slots=2, lens=None, slots=None, out=None):
    return lib.fmx_causal_conv(dtype, B, L, ch, taps, act, x or Heads(), w, bias, s_in, s_out, n_slots, lens, slots,
                               out or Heads(), None)


def test_conv_refusals(lib):
    assert _conv(lib, dtype=_lib.FMX_I32) == DTYPE
    for bad in (dict(B=-1), dict(L=1 << 25), dict(B=1 << 13, L=1 << 13), dict(ch=0), dict(ch=(1 << 20) + 1), dict(taps=0),
                dict(taps=9), dict(n_slots=-1), dict(x=Heads(ts=-1)), dict(out=Heads(bs=1 << 40))):
        assert _conv(lib, **bad) == SHAPE, bad
    for bad in (dict(act=2), dict(w=None), dict(x=Heads(data=0)), dict(x=Heads(data=AT + 1)), dict(bias=(1 << 34) + 1),
                dict(out=Heads(ts=0)), dict(out=Heads(bs=0)), dict(x=Heads(data=AT), out=Heads(data=AT)),
                dict(x=Heads(data=AT), out=Heads(data=AT + 64)), dict(s_out=(1 << 35) + 64), dict(x=Heads(data=1 << 36)),
                dict(lens=AT, out=Heads(data=AT)), dict(slots=1 << 36), dict(w=1 << 36), dict(bias=1 << 36)):
        assert _conv(lib, **bad) == ARG, bad
    # more threads than a launch takes
    assert _conv(lib, B=1 << 12, L=1 << 12, ch=1 << 20, x=Heads(1 << 32, 1 << 20, data=1 << 50),
                 out=Heads(1 << 32, 1 << 20, data=1 << 52)) == UNSUP
    # empty: nothing runs, no array needed
    assert _conv(lib, B=0, x=Heads(data=0), out=Heads(data=0), w=None) == OK
    assert _conv(lib, L=0, x=Heads(data=0), out=Heads(data=0), w=None, s_out=None) == OK
    assert _conv(lib, L=0, x=Heads(data=0), out=Heads(data=0), w=None, s_out=1 << 35) == OK


def test_conv_without_tokens_needs_its_weight(lib):
    """A call without tokens that carries states over runs the kernel, which
    reads the weights: none is refused, rather than read at address 0."""
    none = dict(L=0, x=Heads(data=0), out=Heads(data=0), w=None)
    assert _conv(lib, **none) == ARG  # state_out another array than state_in
    assert _conv(lib, s_in=None, **none) == ARG
    assert _conv(lib, s_in=None, s_out=None, **none) == OK  # (nothing runs)
    assert _conv(lib, taps=1, **none) == OK  # (one tap keeps no state)


def _shape(dtype=BF16, B=2, L=3, nh=4, hd=64, g=2, N=128, lo=0.0, hi=math.inf):
    return C.byref(_lib.FmxSsmShape(dtype, B, L, nh, hd, g, N, 1, lo, hi))


def _scan(lib, shape=None, x=None, dt=None, a=1 << 33, b=None, c=None, d=1 << 34, bias=1 << 35, s_in=1 << 36,
          s_out=1 << 37, n_slots=2, lens=None, slots=None, out=None, ws=None, ws_bytes=0):
    return lib.fmx_ssm_scan(shape or _shape(), x or Heads(), dt or Heads(hs=1), a, b or Heads(), c or Heads(), d, bias,
                            s_in, s_out, n_slots, lens, slots, out or Heads(), ws, ws_bytes, None)


def test_scan_refusals(lib):
    for bad in (_shape(dtype=F32), _shape(dtype=_lib.FMX_U32)):
        assert _scan(lib, bad) == DTYPE
    for bad in (_shape(B=-1), _shape(L=1 << 25), _shape(nh=0), _shape(nh=70000), _shape(g=0), _shape(g=3), _shape(hd=0),
                _shape(N=0)):
        assert _scan(lib, bad) == SHAPE
    for bad in (_shape(hd=12), _shape(hd=264), _shape(N=20), _shape(N=264)):
        assert _scan(lib, bad) == UNSUP
    for bad in (_shape(lo=math.nan), _shape(hi=math.nan), _shape(lo=1.0, hi=0.5), _shape(lo=-math.inf)):
        assert _scan(lib, bad) == ARG
    assert lib.fmx_ssm_scan(None, *[None] * 9, 0, *[None] * 4, 0, None) == ARG
    assert _scan(lib, n_slots=-1) == SHAPE
    for bad in (dict(x=Heads(ts=12)), dict(b=Heads(hs=4)), dict(c=Heads(bs=(1 << 16) + 1)), dict(out=Heads(ts=20))):
        assert _scan(lib, **bad) == UNSUP, bad
    assert _scan(lib, dt=Heads(ts=-1)) == SHAPE
    for bad in (dict(a=None), dict(x=Heads(data=AT + 2)), dict(dt=Heads(data=0)), dict(s_in=(1 << 36) + 4),
                dict(s_out=(1 << 37) + 8), dict(a=(1 << 33) + 2), dict(x=Heads(data=AT), out=Heads(data=AT)),
                dict(b=Heads(data=AT), out=Heads(data=AT + 128)), dict(s_out=(1 << 36) + 4096), dict(a=1 << 37),
                dict(c=Heads(data=1 << 37)), dict(out=Heads(data=1 << 36)), dict(out=Heads(hs=0)), dict(lens=1 << 37)):
        assert _scan(lib, **bad) == ARG, bad
    far = {k: Heads(1 << 17, data=1 << at) for k, at in (("x", 50), ("b", 51), ("c", 52), ("dt", 53), ("out", 54))}
    assert _scan(lib, _shape(B=1 << 24, L=1, nh=256, g=1), n_slots=0, s_in=None, s_out=None, **far) == UNSUP
    assert _scan(lib, _shape(B=0), a=None) == OK
    assert _scan(lib, _shape(L=0), a=None, s_out=None) == OK
    assert lib.fmx_ssm_scan_workspace_size(_shape(hd=12)) == 0
    assert lib.fmx_ssm_scan_workspace_size(_shape(B=0)) == 0


def _norm(lib, dtype=BF16, B=2, L=3, ch=64, groups=2, eps=1e-5, x=None, z=None, w=1 << 33, lens=None, out=None):
    return lib.fmx_gated_norm(dtype, B, L, ch, groups, eps, 1, x or Heads(), z, w, lens, out or Heads(), None)


def test_norm_refusals(lib):
    assert _norm(lib, dtype=_lib.FMX_U32) == DTYPE
    for bad in (dict(B=-1), dict(ch=0), dict(ch=1 << 21), dict(groups=0), dict(groups=3), dict(x=Heads(ts=-8))):
        assert _norm(lib, **bad) == SHAPE, bad
    for bad in (dict(eps=0.0), dict(eps=math.nan), dict(eps=math.inf), dict(x=Heads(data=0)), dict(w=(1 << 33) + 1),
                dict(x=Heads(data=AT), out=Heads(data=AT + 2)), dict(x=Heads(data=AT), out=Heads(data=AT, ts=1 << 11)),
                dict(z=Heads(data=AT), out=Heads(data=AT + 2)), dict(out=Heads(data=1 << 33)), dict(out=Heads(ts=0)),
                dict(lens=AT, out=Heads(data=AT))):
        assert _norm(lib, **bad) == ARG, bad
    assert _norm(lib, B=0, x=Heads(data=0)) == OK
    assert _norm(lib, L=0, x=Heads(data=0)) == OK


def _layer(dtype=BF16, nh=4, hd=64, g=2, N=128, taps=4, act=1, w=1 << 33, a=1 << 34, lo=0.0, hi=math.inf, ng=2, eps=1e-5):
    return C.byref(_lib.FmxSsmLayer(dtype, nh, hd, g, N, taps, act, w, None, a, None, None, 1, lo, hi, None, ng, eps, 1))


def _step(lib, layer=None, B=2, xbc=None, dt=None, z=None, cs=1 << 35, st=1 << 36, n_slots=4, slots=None, out=None,
          ws=None, ws_bytes=0):
    return lib.fmx_ssm_step(layer or _layer(), B, xbc or Heads(), dt or Heads(hs=1), z, cs, st, n_slots, slots,
                            out or Heads(), ws, ws_bytes, None)


def test_step_refusals(lib):
    assert _step(lib, _layer(dtype=F32)) == DTYPE
    for bad in (_layer(nh=0), _layer(g=3), _layer(taps=1), _layer(taps=9), _layer(ng=0), _layer(ng=3),
                _layer(nh=60000, g=1, hd=256)):
        assert _step(lib, bad) == SHAPE
    for bad in (_layer(hd=12), _layer(N=512)):
        assert _step(lib, bad) == UNSUP
    for bad in (_layer(act=5), _layer(eps=-1.0), _layer(w=None), _layer(a=None), _layer(lo=2.0, hi=1.0)):
        assert _step(lib, bad) == ARG
    assert lib.fmx_ssm_step(None, 1, *[None] * 5, 0, None, None, None, 0, None) == ARG
    assert _step(lib, B=-1) == SHAPE and _step(lib, n_slots=1 << 25) == SHAPE
    for bad in (dict(cs=None), dict(st=None), dict(cs=(1 << 35) + 2), dict(st=(1 << 36) + 4), dict(st=(1 << 35) + 16),
                dict(xbc=Heads(data=0)), dict(out=Heads(bs=0)), dict(out=Heads(data=1 << 35)), dict(z=Heads(data=1 << 36)),
                dict(z=Heads(data=AT), out=Heads(data=AT)), dict(slots=1 << 36), dict(ws=AT + 1, ws_bytes=1 << 20)):
        assert _step(lib, **bad) == ARG, bad
    assert _step(lib, ws=AT, ws_bytes=8) == WS
    assert _step(lib, B=0, xbc=Heads(data=0)) == OK
    assert lib.fmx_ssm_step_workspace_size(_layer(), 3) >= 3 * 4 * 64 * 4
    assert lib.fmx_ssm_step_workspace_size(_layer(), 0) == 0 and lib.fmx_ssm_step_workspace_size(_layer(hd=4), 1) == 0


def _prompt(lib, layer=None, B=2, L=3, xbc=None, dt=None, z=None, v=1 << 48, y=1 << 49, cs=1 << 35, st=1 << 36, n_slots=4,
            conv_slots=None, lens=None, slots=None, out=None):
    return lib.fmx_ssm_prompt_check(layer or _layer(), B, L, xbc or Heads(), dt or Heads(hs=1), z, v, y, cs,
                                    n_slots if conv_slots is None else conv_slots, st, n_slots, lens, slots, out or Heads())


def test_prompt_refusals(lib):
    """What any of a prompt's calls refuses, and outputs of one over another's
    arrays; nothing is launched either way."""
    assert _prompt(lib) == OK and _prompt(lib, z=Heads()) == OK and _prompt(lib, _layer(taps=1)) == OK
    assert _prompt(lib, cs=None, st=None, n_slots=0) == OK
    for empty in (dict(B=0), dict(L=0)):
        assert _prompt(lib, xbc=Heads(data=0), dt=Heads(data=0), v=None, y=None, out=Heads(data=0), **empty) == OK
    assert _prompt(lib, _layer(dtype=F32)) == DTYPE and _prompt(lib, _layer(dtype=_lib.FMX_U32)) == DTYPE
    for bad in (_layer(nh=0), _layer(g=3), _layer(taps=0), _layer(taps=9), _layer(ng=0), _layer(ng=3),
                _layer(nh=60000, g=1, hd=256)):
        assert _prompt(lib, bad) == SHAPE
    for bad in (_layer(hd=12), _layer(N=512)):
        assert _prompt(lib, bad) == UNSUP
    for bad in (_layer(act=5), _layer(eps=-1.0), _layer(w=None), _layer(a=None), _layer(lo=2.0, hi=1.0)):
        assert _prompt(lib, bad) == ARG
    assert lib.fmx_ssm_prompt_check(None, 1, 1, *[None] * 6, 0, None, 0, None, None, None) == ARG
    for bad in (dict(B=-1), dict(L=1 << 25), dict(n_slots=1 << 25), dict(conv_slots=-1), dict(dt=Heads(ts=-1)), dict(out=Heads(bs=-1))):
        assert _prompt(lib, **bad) == SHAPE, bad
    for bad in (dict(xbc=Heads(data=0)), dict(dt=Heads(data=0)), dict(z=Heads(data=0)), dict(out=Heads(data=0)), dict(v=None),
                dict(y=None), dict(v=(1 << 48) + 2), dict(y=(1 << 49) + 8), dict(st=(1 << 36) + 4), dict(cs=(1 << 35) + 1),
                dict(out=Heads(ts=0)), dict(z=Heads(data=AT), out=Heads(data=AT + 2)),
                # one call's outputs over another's arrays
                dict(cs=1 << 36), dict(st=(1 << 35) + 16), dict(z=Heads(data=1 << 35)), dict(z=Heads(data=1 << 36)),
                dict(dt=Heads(data=1 << 35)), dict(dt=Heads(data=1 << 36)), dict(out=Heads(data=1 << 35)),
                dict(out=Heads(data=1 << 36)), dict(cs=1 << 34), dict(st=1 << 33), dict(v=1 << 36), dict(y=1 << 35),
                dict(v=1 << 49), dict(out=Heads(data=1 << 33)), dict(out=Heads(data=1 << 34)), dict(lens=1 << 49)):
        assert _prompt(lib, **bad) == ARG, bad


class _Recorder:
    """The library's checks and sizes, and the names of what would be launched."""

    def __init__(self, lib):
        self.lib, self.launched = lib, []

    def __getattr__(self, name):
        if name not in ("fmx_causal_conv", "fmx_ssm_scan", "fmx_gated_norm", "fmx_ssm_step"):
            return getattr(self.lib, name)
        return lambda *args: self.launched.append(name) or OK


def test_a_refused_prompt_has_run_nothing(lib, monkeypatch):
    """On host arrays, with launches recorded instead of made: all three, or none."""
    import flashmlx_amd.ssm as S
    rec = _Recorder(lib)
    monkeypatch.setattr(_lib, "load", lambda: rec)
    monkeypatch.setattr(S, "_device", lambda t, *_: t.get_device())
    monkeypatch.setattr(S, "_stream", lambda dev: None)
    bf, f = torch.bfloat16, torch.float32
    make = lambda dtype=bf, **kw: S.SsmLayer(  # noqa: E731
        torch.zeros(48, 4, dtype=dtype), torch.zeros(2), None, **{**dict(head_dim=8, groups=1, state_dim=16), **kw})
    layer = make()
    good = dict(xbc=torch.zeros(2, 5, 48, dtype=bf), dt=torch.zeros(2, 5, 2, dtype=bf), z=torch.zeros(2, 5, 16, dtype=bf),
                conv_state=torch.zeros(3, 3, 48, dtype=bf), state=torch.zeros(3, 2, 8, 16))
    assert layer.prompt(**good).shape == (2, 5, 16)
    assert rec.launched == ["fmx_causal_conv", "fmx_ssm_scan", "fmx_gated_norm"]
    rec.launched.clear()
    wrong = [dict(dt=good["dt"][:, :4]), dict(dt=good["dt"].to(f)), dict(z=good["z"][..., :8]), dict(z=good["z"].half()),
             dict(conv_state=good["conv_state"][:, :2]), dict(conv_state=good["conv_state"][0]), dict(conv_state=good["conv_state"].half()),
             dict(state=good["state"][:, :1]), dict(state=good["state"].double()),
             dict(state=torch.zeros(3 * 256 + 1)[1:].view(3, 2, 8, 16)), dict(state=good["state"].transpose(2, 3)),
             dict(out=torch.zeros(2, 5, 8, dtype=bf)), dict(out=torch.zeros(2, 5, 16)),
             dict(out=torch.zeros(2, 1, 16, dtype=bf).expand(2, 5, 16)), dict(lengths=torch.zeros(2)),
             dict(slots=torch.zeros(3, dtype=torch.int32)), dict(dt=None), dict(z=3)]
    shared = torch.zeros(1 << 14, dtype=torch.uint8)  # (the state at its start and what else the call writes there)
    at = shared[-shared.data_ptr() % 256:]
    over = at[:good["state"].nbytes].view(f).view(3, 2, 8, 16)
    wrong += [dict(state=over, out=at[:320].view(bf).view(2, 5, 16)), dict(state=over, z=at[:320].view(bf).view(2, 5, 16)),
              dict(state=over, conv_state=at[:864].view(bf).view(3, 3, 48))]
    for bad in wrong:
        with pytest.raises((ValueError, TypeError, _lib.FmxError)):
            layer.prompt(**{**good, **bad})
        assert rec.launched == [], bad
    for other, kw in ((make(eps=0.0), {}), (make(norm_groups=3), {}), (make(dt_limits=(1.0, 0.5)), {}),
                      (make(f), {k: good[k].to(f) for k in ("xbc", "dt", "z", "conv_state")})):
        with pytest.raises(_lib.FmxError):
            other.prompt(**{**good, **kw})
        assert rec.launched == []


def test_python_refusals():
    x = torch.zeros(1, 2, 8)
    for call in (lambda: F.causal_conv(None, x), lambda: F.gated_norm(3), lambda: F.ssm_scan([], *[None] * 4),
                 lambda: F.SsmLayer(None, x, x, 8, 1, 8)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: F.causal_conv(x, x), lambda: F.causal_conv(x[0], x), lambda: F.gated_norm(x),
                 lambda: F.ssm_scan(x[None], x, x, x, x), lambda: F.causal_conv(x, x, activation="gelu")):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        F.gated_norm(x.int())


def test_scan_workspaces(lib):
    """Segments' states: none for few tokens or few chunks, a bounded number for
    long sequences; one too small, or on no 256 bytes, is refused."""
    size = lambda **kw: lib.fmx_ssm_scan_workspace_size(_shape(**kw))  # noqa: E731
    assert size(B=1, L=5) == 0 and size(B=1, L=64) == 0 and size(B=256, L=4096, nh=64, g=8) == 0
    need = size(B=1, L=8192, nh=64, g=8)
    assert 0 < need <= 33 * 64 * (64 * 128 + 1) * 4 and size(B=1, L=1 << 24, nh=64, g=8) <= 33 * 64 * (64 * 128 + 1) * 4
    long = dict(B=1, L=8192, nh=64, g=8)
    views = lambda: {k: Heads(1 << 34, 1 << 14, data=1 << at)  # noqa: E731
                     for k, at in (("x", 50), ("b", 51), ("c", 52), ("dt", 53), ("out", 54))}
    assert _scan(lib, _shape(**long), s_in=None, s_out=None, ws=AT, ws_bytes=need - 1, **views()) == WS
    assert _scan(lib, _shape(**long), s_in=None, s_out=None, ws=AT + 16, ws_bytes=need, **views()) == ARG


def test_header_is_c(tmp_path):
    import pathlib
    import subprocess
    include = pathlib.Path(__file__).parent.parent / "include"
    src = tmp_path / "h.c"
    src.write_text('#include "fmx_ssm.h"\nint main(void) { fmx_ssm_shape s = {FMX_BF16}; return s.dtype != FMX_BF16; }\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-fsyntax-only", f"-I{include}", str(src)], check=True)


def test_work_beyond_a_launch(lib):
    """Workgroups are counted as the kernels deal the work out: one more than a
    launch of fewer than 2^32 threads takes is refused."""
    far = {k: Heads(0, 1 << 12, data=1 << at) for k, at in (("x", 50), ("out", 58))}
    # groups of more than 128 vectors: a workgroup each; single elements: up to 192 of them in a wave's lanes, 4 a workgroup
    assert _norm(lib, B=1, L=1 << 24, ch=2048, groups=1, **far) == UNSUP
    assert _norm(lib, B=1, L=1 << 24, ch=600, groups=5, w=(1 << 33) + 2, **far) == UNSUP
    # the walk: 2^24 workgroups of one head each; chunks: 2^23 of 512 threads
    views = lambda: {k: Heads(1 << 17, 1 << 13, data=1 << at)  # noqa: E731
                     for k, at in (("x", 50), ("b", 51), ("c", 52), ("dt", 53), ("out", 54))}
    no = dict(s_in=None, s_out=None, n_slots=0)
    assert _scan(lib, _shape(B=1 << 18, L=1, nh=64, g=1), **no, **views()) == UNSUP
    assert _scan(lib, _shape(B=1 << 18, L=9, nh=64, g=1), **no, **views()) == UNSUP
