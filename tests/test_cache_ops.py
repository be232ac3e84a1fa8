"""Host side of the cache's long-context operators (include/fmx_cache.h),
without a GPU: what is refused, and with which status; empty calls; workspace
sizes; the rotary frequencies. No call here launches a kernel."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from flashmlx_amd import RopeConfig, _lib

OK, ARG, SHAPE, DTYPE, UNSUP, WS = (_lib.FMX_OK, _lib.FMX_ERR_ARG, _lib.FMX_ERR_SHAPE, _lib.FMX_ERR_DTYPE,
                                    _lib.FMX_ERR_UNSUPPORTED, _lib.FMX_ERR_WORKSPACE)
BF16, F16, F32 = _lib.FMX_BF16, _lib.FMX_F16, _lib.FMX_F32


class Heads:
    """Distinct fake arrays: never read, the calls are refused first."""
    next = 1 << 40

    def __new__(cls, bs=1 << 16, ts=1 << 10, hs=1 << 7, data=None):
        if data is None:
            cls.next += 1 << 36
            data = cls.next
        return C.byref(_lib.FmxHeads(data, bs, ts, hs))


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


# ------------------------------------------------------------------ frequencies

@pytest.mark.parametrize("dims,base", [(2, 10000.0), (64, 10000.0), (128, 1e6), (1024, 500.0)])
def test_plain_frequencies(lib, dims, base):
    f, m = RopeConfig(dims=dims, base=base).frequencies()
    np.testing.assert_allclose(f, base ** (-2.0 * np.arange(dims // 2) / dims), rtol=1e-15 * 8)
    assert m == 1.0


def test_scaled_frequencies(lib):
    dims, base, s, n0 = 128, 10000.0, 4.0, 4096
    i = np.arange(dims // 2)
    g = base ** (-2.0 * i / dims)
    kw = dict(dims=dims, base=base, factor=s, original_max=n0)
    f, m = RopeConfig(scaling="linear", **kw).frequencies()
    np.testing.assert_allclose(f, g / s, rtol=1e-14)
    f, m = RopeConfig(scaling="ntk", **kw).frequencies()
    # the fastest pair keeps its angle, the slowest turns s times slower
    assert f[0] == 1.0 and m == 1.0
    np.testing.assert_allclose(f[-1], g[-1] / s, rtol=1e-12)
    f, m = RopeConfig(scaling="parts", **kw).frequencies()
    turns = n0 * g / (2 * math.pi)
    # unscaled: two libraries' pow, each within a step of 2^-52
    np.testing.assert_allclose(f[turns > 4], g[turns > 4], rtol=1e-15)
    np.testing.assert_allclose(f[turns < 1], g[turns < 1] / s, rtol=1e-14)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and np.all(f[mid] < g[mid]) and np.all(f[mid] > g[mid] / s)
    f, m = RopeConfig(scaling="yarn", **kw).frequencies()
    np.testing.assert_allclose(m, 0.1 * math.log(s) + 1, rtol=1e-15)
    lo = math.floor(dims * math.log(n0 / (32 * 2 * math.pi)) / (2 * math.log(base)))
    hi = math.ceil(dims * math.log(n0 / (2 * math.pi)) / (2 * math.log(base)))
    np.testing.assert_allclose(f[:lo + 1], g[:lo + 1], rtol=1e-15)
    np.testing.assert_allclose(f[hi:], g[hi:] / s, rtol=1e-14)
    t = (i[lo:hi] - lo) / (hi - lo)
    np.testing.assert_allclose(f[lo:hi], (1 - t) * g[lo:hi] + t * g[lo:hi] / s, rtol=1e-13)
    assert RopeConfig(scaling="yarn", attention_factor=2.5, **kw).frequencies()[1] == 2.5
    # a trained length so short that no pair turns `high` times
    f, _ = RopeConfig(dims=16, scaling="yarn", factor=2.0, original_max=8).frequencies()
    assert np.all(np.isfinite(f)) and np.all(f > 0)


@pytest.mark.parametrize("status,kw", [
    (SHAPE, dict(dims=0)), (SHAPE, dict(dims=7)), (SHAPE, dict(dims=1026)), (ARG, dict(dims=8, base=1.0)),
    (ARG, dict(dims=8, base=math.nan)), (ARG, dict(dims=8, scaling="linear", factor=0.5)),
    (ARG, dict(dims=8, scaling="yarn", factor=math.inf)), (SHAPE, dict(dims=2, scaling="ntk", factor=2.0)),
    (ARG, dict(dims=8, scaling="parts", factor=2.0, original_max=0)),
    (ARG, dict(dims=8, scaling="parts", factor=2.0, low=4.0, high=4.0)),
    (ARG, dict(dims=8, scaling="yarn", factor=2.0, low=0.0)), (ARG, dict(dims=8, attention_factor=-1.0))])
def test_frequency_refusals(lib, status, kw):
    with pytest.raises(_lib.FmxError) as e:
        RopeConfig(**kw).frequencies()
    assert e.value.status == status
    with pytest.raises(ValueError):
        RopeConfig(dims=8, scaling="other").frequencies()


# ------------------------------------------------------------------ rope

def _angles(dims=64, freqs=1 << 33, factor=1.0):
    return C.byref(_lib.FmxRopeAngles(freqs, dims, factor, 0))


def _rope(lib, angles=None, dtype=BF16, B=2, L=3, nh=4, hd=128, x=None, pos=1 << 34, out=None):
    return lib.fmx_rope(angles or _angles(), dtype, B, L, nh, hd, x or Heads(), pos, 0, out or Heads(), None)


def test_rope_refusals(lib):
    assert _rope(lib, dtype=_lib.FMX_I32) == DTYPE
    for bad in (dict(B=-1), dict(L=1 << 25), dict(B=1 << 13, L=1 << 13), dict(nh=0), dict(hd=1), dict(hd=1025), dict(hd=32),
                dict(angles=_angles(dims=3)), dict(angles=_angles(dims=0))):
        assert _rope(lib, **bad) == SHAPE, bad
    for bad in (dict(angles=_angles(freqs=None)), dict(pos=None), dict(x=Heads(data=0)), dict(x=Heads(data=(1 << 41) + 1)),
                dict(angles=_angles(factor=math.inf)), dict(x=Heads(data=1 << 42), out=Heads(data=(1 << 42) + 64)),
                dict(x=Heads(data=1 << 42), out=Heads(data=1 << 42, ts=1 << 11))):
        assert _rope(lib, **bad) == ARG, bad
    assert _rope(lib, x=Heads(ts=-1)) == SHAPE
    assert _rope(lib, x=Heads(bs=1 << 40)) == SHAPE
    assert lib.fmx_rope(None, BF16, 1, 1, 1, 64, Heads(), 1, 0, Heads(), None) == ARG
    # empty: nothing runs, no array needed
    assert lib.fmx_rope(_angles(), BF16, 0, 5, 4, 64, None, None, 0, None, None) == OK
    assert lib.fmx_rope(_angles(), BF16, 5, 0, 4, 64, None, None, 0, None, None) == OK


def _append(lib, angles=None, dtype=BF16, B=2, L=1, nh=4, nkv=2, hd=128, q=None, k=None, v=None, pos=1 << 34,
            offs=1 << 35, slots=None, n_slots=2, S=8, q_out=None, kc=None, vc=None):
    return lib.fmx_rope_append(angles or _angles(), dtype, B, L, nh, nkv, hd, q or Heads(), k or Heads(), v or Heads(),
                               pos, offs, slots, n_slots, S, q_out or Heads(), kc or Heads(), vc or Heads(), None)


def test_rope_append_refusals(lib):
    assert _append(lib, dtype=_lib.FMX_U32) == DTYPE
    for bad in (dict(nkv=0), dict(n_slots=1), dict(n_slots=-1), dict(S=-1), dict(S=1 << 25), dict(hd=2048),
                dict(kc=Heads(hs=-8))):
        assert _append(lib, **bad) == SHAPE, bad
    at = 1 << 42
    for bad in (dict(offs=None), dict(pos=None), dict(k=Heads(data=0)), dict(vc=Heads(data=at + 1)),
                dict(k=Heads(data=at), kc=Heads(data=at)), dict(q_out=Heads(data=at), vc=Heads(data=at)),
                dict(q=Heads(data=at), q_out=Heads(data=at + 256)), dict(v=Heads(data=at), q_out=Heads(data=at))):
        assert _append(lib, **bad) == ARG, bad
    assert lib.fmx_rope_append(_angles(), F32, 0, 1, 4, 2, 64, None, None, None, None, None, None, 0, 0, None, None, None,
                               None) == OK


# ------------------------------------------------------------------ attention

def _shape(dtype=BF16, B=2, L=1, nh=8, nkv=2, hd=128, scale=0.1):
    return C.byref(_lib.FmxAttentionShape(dtype, B, L, nh, nkv, hd, scale))


BAD_SHAPES = [(DTYPE, dict(dtype=F32)), (DTYPE, dict(dtype=9)), (SHAPE, dict(B=-1)), (SHAPE, dict(L=-1)),
              (SHAPE, dict(B=1 << 20, L=1 << 20)), (SHAPE, dict(nh=7)), (SHAPE, dict(nkv=0)), (SHAPE, dict(hd=0)),
              (UNSUP, dict(hd=12)), (UNSUP, dict(hd=264)), (ARG, dict(scale=0.0)), (ARG, dict(scale=-1.0)),
              (ARG, dict(scale=math.nan)), (ARG, dict(scale=math.inf))]


def _shared(lib, shape=None, q=None, kp=None, vp=None, P=5, kc=None, vc=None, n_slots=2, S=8, offs=1 << 35, slots=None,
            out=None, ws=None, ws_bytes=0):
    return lib.fmx_attention_shared_prefix(shape or _shape(), q or Heads(), kp or Heads(), vp or Heads(), P, kc or Heads(),
                                           vc or Heads(), n_slots, S, offs, slots, out or Heads(), None, ws, ws_bytes,
                                           None)


def _scored(lib, shape=None, q=None, kc=None, vc=None, n_slots=2, S=8, offs=1 << 35, slots=None, w_in=None,
            w_out=1 << 36, out=None, ws=None, ws_bytes=0):
    return lib.fmx_attention_scored(shape or _shape(), q or Heads(), kc or Heads(), vc or Heads(), n_slots, S, offs, slots,
                                    w_in, w_out, out or Heads(), ws, ws_bytes, None)


@pytest.mark.parametrize("status,kw", BAD_SHAPES, ids=str)
def test_attention_shape_refusals(lib, status, kw):
    assert _shared(lib, _shape(**kw)) == status
    assert _scored(lib, _shape(**kw)) == status
    assert lib.fmx_attention_shared_prefix_workspace_size(_shape(**kw), 5, 8) == 0
    assert lib.fmx_attention_scored_workspace_size(_shape(**kw), 8) == 0


def test_attention_refusals(lib):
    assert lib.fmx_attention_scored(None, Heads(), Heads(), Heads(), 1, 1, 1, None, None, 1, Heads(), None, 0, None) == ARG
    odd = Heads(data=(1 << 42) + 8)
    for call in (_shared, _scored):
        for bad in (dict(n_slots=1), dict(n_slots=-2), dict(S=1 << 25), dict(q=Heads(ts=-8))):
            assert call(lib, **bad) == SHAPE, bad
        for bad in (dict(offs=None), dict(q=odd), dict(kc=odd), dict(vc=Heads(data=0)), dict(out=Heads(data=0))):
            assert call(lib, **bad) == ARG, bad
        for bad in (dict(q=Heads(hs=4)), dict(kc=Heads(ts=130)), dict(out=Heads(bs=12))):
            assert call(lib, **bad) == UNSUP, bad
    assert _shared(lib, P=-1) == SHAPE
    assert _shared(lib, P=(1 << 24) + 1) == SHAPE
    assert _shared(lib, kp=odd) == ARG
    assert _scored(lib, S=0) == SHAPE
    assert _scored(lib, w_out=None) == ARG
    assert _scored(lib, w_out=(1 << 36) + 2) == ARG
    assert _scored(lib, w_in=(1 << 36) + 4) == ARG  # overlaps weights_out in part
    # no sequences or no queries: nothing runs, no array needed
    none = [None] * 3
    for kw in (dict(B=0), dict(L=0)):
        n = 0 if kw.get("B") == 0 else 2
        assert lib.fmx_attention_shared_prefix(_shape(**kw), *none, 5, None, None, n, 8, *none, None, None, 0, None) == OK
        assert lib.fmx_attention_scored(_shape(**kw), *none, n, 8, None, None, None, None, None, None, 0, None) == OK


@pytest.mark.parametrize("kw", [dict(), dict(B=64, nh=32), dict(L=7), dict(L=500, B=1), dict(hd=256, nkv=8)], ids=str)
def test_attention_workspaces(lib, kw):
    """A call with a workspace short by one byte, or not aligned, is refused."""
    sh = _shape(**kw)
    B = kw.get("B", 2)
    for size, call, more in ((lib.fmx_attention_shared_prefix_workspace_size(sh, 20000, 9000), _shared, dict(P=20000)),
                             (lib.fmx_attention_scored_workspace_size(sh, 9000), _scored, {})):
        if size:
            more = dict(more, S=9000, n_slots=B)
            assert call(lib, sh, ws=1 << 20, ws_bytes=size - 1, **more) == WS
            assert call(lib, sh, ws=(1 << 20) + 16, ws_bytes=size, **more) == ARG


def test_attention_limits(lib):
    """Token strides that 64 rows' byte offsets do not hold, positions and
    query rows beyond what one call counts, outputs among the inputs."""
    far = Heads(ts=(1 << 24) + 8)
    for call in (_shared, _scored):
        assert call(lib, kc=far) == UNSUP
        assert call(lib, vc=far) == UNSUP
        assert call(lib, _shape(B=1 << 13), n_slots=1 << 13, S=(1 << 23) + 1) == UNSUP
        assert call(lib, _shape(B=1 << 14, L=1 << 10, nh=128), n_slots=1 << 14) == UNSUP
    assert _shared(lib, kp=far) == UNSUP
    assert _shared(lib, vp=far) == UNSUP
    at = 1 << 50
    for call, names in ((_shared, ("q", "kc", "vc", "kp", "vp")), (_scored, ("q", "kc", "vc"))):
        for name in names:
            assert call(lib, **{name: Heads(data=at), "out": Heads(data=at)}) == ARG, name
            assert call(lib, **{name: Heads(data=at), "out": Heads(data=at + 256)}) == ARG, name


# ------------------------------------------------------------------ eviction

def _evict(lib, dtype=BF16, B=2, nkv=2, hd=64, k=None, v=None, w=1 << 35, n_slots=2, S=100, lens=1 << 33, slots=None,
           budget=50, sinks=4, recent=10, ko=None, vo=None, wo=None, S_out=0, lens_out=1 << 34, kept=1 << 36, ws=None,
           ws_bytes=0):
    return lib.fmx_cache_evict(dtype, B, nkv, hd, k or Heads(), v or Heads(), w, n_slots, S, lens, slots, budget, sinks,
                               recent, ko, vo, wo, S_out, lens_out, kept, ws, ws_bytes, None)


def test_evict_refusals(lib):
    assert _evict(lib, dtype=F32) == DTYPE
    for bad in (dict(B=-1), dict(nkv=0), dict(n_slots=1), dict(S=0), dict(hd=0), dict(hd=1025), dict(budget=0),
                dict(sinks=-1), dict(recent=-1), dict(sinks=51, recent=0), dict(sinks=4, recent=47),
                dict(budget=1 << 25), dict(k=Heads(ts=-1)),
                dict(ko=Heads(), vo=Heads(), wo=1 << 50, S_out=49)):
        assert _evict(lib, **bad) == SHAPE, bad
    at = 1 << 42
    for bad in (dict(lens=None), dict(lens_out=None), dict(w=None), dict(w=(1 << 35) + 1), dict(k=Heads(data=0)),
                dict(v=Heads(data=at + 1)), dict(ko=Heads()), dict(ko=Heads(), vo=Heads()),
                dict(k=Heads(data=at), ko=Heads(data=at), vo=Heads(), wo=1 << 50, S_out=60),
                dict(ko=Heads(), vo=Heads(), wo=1 << 35, S_out=60)):
        assert _evict(lib, **bad) == ARG, bad
    need = lib.fmx_cache_evict_workspace_size(2, 2, 50)
    assert need >= 2 * 2 * 50 * 4
    assert _evict(lib, kept=None, ws=1 << 20, ws_bytes=need - 1) == WS
    assert lib.fmx_cache_evict_workspace_size(2, 2, 0) == 0
    assert lib.fmx_cache_evict(BF16, 0, 2, 64, None, None, None, 0, 100, None, None, 50, 0, 0, None, None, None, 0, None,
                               None, None, 0, None) == OK


# ------------------------------------------------------------------ the Python face

def test_python_refusals(fmx):
    """Arrays that are not what a call takes: an exception names the argument,
    nothing is passed on (CPU tensors throughout)."""
    import torch
    q = torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16)
    kc = torch.zeros(2, 2, 10, 64, dtype=torch.bfloat16)
    offs = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        fmx.attention_scored(q, kc, kc, offs, 0.1)
    with pytest.raises(ValueError, match="batch, seq_len"):
        fmx.attention_scored(q[0], kc, kc, offs, 0.1)
    with pytest.raises(TypeError):
        fmx.attention_scored(q.int(), kc, kc, offs, 0.1)
    with pytest.raises(ValueError, match="HIP device"):
        fmx.cache_evict(kc, kc, torch.zeros(2, 2, 10), offs, 5)
    from flashmlx_amd import cache as M
    bf, dev = torch.bfloat16, -1  # (CPU tensors)
    with pytest.raises(ValueError, match="k_cache: shape"):
        M._cache(kc, "k_cache", (2, 4, 10, 64), bf, dev)
    with pytest.raises(TypeError, match="k_cache"):
        M._cache(kc.half(), "k_cache", kc.shape, bf, dev)
    with pytest.raises(ValueError, match="k_cache is on cpu"):
        M._cache(kc, "k_cache", kc.shape, bf, 0)
    with pytest.raises(ValueError, match="contiguous"):
        M._cache(torch.zeros(2, 2, 10, 128, dtype=bf)[..., ::2], "k_cache", kc.shape, bf, dev)
    for bad in (offs[:1], torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="offsets"):
            M._flat(bad, "offsets", (2,), torch.int32, dev)
    with pytest.raises(TypeError, match="offsets"):
        M._flat(offs.long(), "offsets", (2,), torch.int32, dev)
    with pytest.raises(TypeError, match="weights"):
        M._flat(torch.zeros(2, 2, 10).half(), "weights", (2, 2, 10), torch.float32, dev)
