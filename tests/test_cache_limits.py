"""Host side of the cache's long-context operators at the edges of their range,
without a GPU (no call here launches a kernel): counts that pass 32 bits,
empty calls, launches beyond what the device takes, arrays that overlap."""
from __future__ import annotations

import ctypes as C
import pathlib
import subprocess

import pytest

from flashmlx_amd import _lib

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_pieces_cover_the_keys():
    """The pieces that own keys are dealt to, for batches up to the limit of
    2^36 own positions (tests/c_abi/piece_check.cpp, built by
    __graft_entry__.build())."""
    prog = ROOT / "tests" / "c_abi" / "_build" / "piece_check"
    assert prog.exists(), f"{prog} missing: run __graft_entry__.build()"
    p = subprocess.run([str(prog)], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stdout + p.stderr


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _shape(dtype=_lib.FMX_BF16, B=2, L=1, nh=8, nkv=2, hd=128, scale=0.1):
    return C.byref(_lib.FmxAttentionShape(dtype, B, L, nh, nkv, hd, scale))


@pytest.mark.parametrize("kw", [dict(B=0), dict(L=0), dict(B=0, L=0), dict(B=0, L=1 << 24, nh=65535, nkv=1),
                                dict(B=0, L=40), dict(L=0, B=1 << 24)], ids=str)
def test_empty_calls_need_no_workspace(lib, kw):
    """No sequences or no queries: 0 bytes (the process ended before)."""
    for P, S in ((0, 0), (5, 0), (0, 8), (5, 8), (20000, 9000)):
        if S:
            assert lib.fmx_attention_scored_workspace_size(_shape(**kw), S) == 0
        assert lib.fmx_attention_shared_prefix_workspace_size(_shape(**kw), P, S) == 0


class Heads:
    """Distinct fake arrays: never read, the calls are refused first."""
    next = 1 << 40

    def __new__(cls, bs=1 << 13, ts=1 << 10, hs=1 << 7, data=None):
        if data is None:
            cls.next += 1 << 39
            data = cls.next
        return C.byref(_lib.FmxHeads(data, bs, ts, hs))


def _shared(lib, shape, P=5, n_slots=2, S=8, slots=None, lse=None, **at):
    h = {n: at.get(n) or Heads() for n in ("q", "kp", "vp", "kc", "vc", "out")}
    return lib.fmx_attention_shared_prefix(shape, h["q"], h["kp"], h["vp"], P, h["kc"], h["vc"], n_slots, S, 1 << 35,
                                           slots, h["out"], lse, None, 0, None)


def _scored(lib, shape, n_slots=2, S=8, slots=None, w_in=None, w_out=1 << 36, **at):
    h = {n: at.get(n) or Heads() for n in ("q", "kc", "vc", "out")}
    return lib.fmx_attention_scored(shape, h["q"], h["kc"], h["vc"], n_slots, S, 1 << 35, slots, w_in, w_out, h["out"],
                                    None, 0, None)


def _evict(lib, B=2, nkv=2, hd=64, w=1 << 36, n_slots=2, S=100, lens=1 << 33, slots=None, budget=50, out=None,
           S_out=0, lens_out=1 << 34, kept=1 << 37, **at):
    h = {n: at.get(n) or Heads() for n in ("k", "v")}
    ko, vo, wo = out or (None, None, None)
    return lib.fmx_cache_evict(_lib.FMX_BF16, B, nkv, hd, h["k"], h["v"], w, n_slots, S, lens, slots, budget, 0, 0, ko,
                               vo, wo, S_out, lens_out, kept, None, 0, None)


def test_launches_beyond_the_device(lib):
    """HIP takes launches of fewer than 2^32 threads: work that needs more is
    refused before anything runs (an in-place eviction had moved the weights
    before its second launch failed)."""
    unsup, one = _lib.FMX_ERR_UNSUPPORTED, 1 << 30
    for kw in (dict(B=1 << 20, nh=16, nkv=16), dict(B=1 << 17, nh=128, nkv=128), dict(B=1 << 19, nh=128, nkv=8, hd=8)):
        assert _shared(lib, _shape(**kw), n_slots=1, slots=one) == unsup, kw
        assert _scored(lib, _shape(**kw), n_slots=1, slots=one) == unsup, kw
    assert _scored(lib, _shape(B=1 << 10, L=0, nh=16, nkv=16), n_slots=1, S=1 << 24, slots=one) == unsup
    # the weights of a prompt in a cache far longer than it
    assert _scored(lib, _shape(B=1 << 10, L=64, nh=16, nkv=16, hd=8), n_slots=1, S=1 << 24, slots=one) == unsup
    assert _evict(lib, B=1 << 22, nkv=1, n_slots=1, slots=one) == unsup
    assert _evict(lib, B=1 << 20, nkv=4, n_slots=1, slots=one, out=(Heads(), Heads(), 1 << 38), S_out=60) == unsup
    assert lib.fmx_cache_evict_workspace_size(1 << 21, 2, 50) == 0
    # rows of an odd number of elements in four slices; many chunks of rows
    assert _evict(lib, B=1 << 21, nkv=1, hd=1023, n_slots=1, slots=one) == unsup
    far = dict(S=1 << 23, budget=1 << 23, S_out=1 << 23, out=(Heads(ts=64), Heads(ts=64), 1 << 38))
    assert _evict(lib, B=1 << 12, nkv=1, n_slots=1, slots=one, k=Heads(ts=64), v=Heads(ts=64), **far) == unsup


def _rope(lib, x=None, out=None, B=2, L=3, nh=4, hd=128):
    angles = C.byref(_lib.FmxRopeAngles(1 << 33, 64, 1.0, 0))
    return lib.fmx_rope(angles, _lib.FMX_BF16, B, L, nh, hd, x or Heads(), 1 << 34, 0, out or Heads(), None)


def _append(lib, q_out=None, kc=None, vc=None):
    angles = C.byref(_lib.FmxRopeAngles(1 << 33, 64, 1.0, 0))
    return lib.fmx_rope_append(angles, _lib.FMX_BF16, 2, 3, 4, 4, 128, Heads(), Heads(), Heads(), 1 << 34, 1 << 35, None, 2,
                               8, q_out or Heads(), kc or Heads(), vc or Heads(), None)


def test_outputs_that_overlap(lib):
    """Arrays that are written may lie over no other array of the call."""
    arg, at = _lib.FMX_ERR_ARG, 1 << 52
    # rows that are one row (a broadcast axis)
    for flat in (dict(bs=0), dict(ts=0), dict(hs=0)):
        for data in (None, at):
            v = Heads(data=data, **flat)
            assert _rope(lib, x=v, out=v) == arg
            assert _append(lib, q_out=v) == arg
            assert _append(lib, kc=v) == arg
            assert _append(lib, vc=v) == arg
            assert _shared(lib, _shape(L=2), out=v) == arg
            assert _scored(lib, _shape(L=2), out=v) == arg
            assert _evict(lib, k=v) == arg
            assert _evict(lib, out=(v, Heads(), 1 << 50), S_out=60) == arg
            assert _evict(lib, out=(Heads(), v, 1 << 50), S_out=60) == arg
    # keys over values
    for d in (0, 64):
        assert _append(lib, kc=Heads(data=at), vc=Heads(data=at + d)) == arg
        assert _evict(lib, k=Heads(data=at), v=Heads(data=at + d)) == arg
        assert _evict(lib, out=(Heads(data=at), Heads(data=at + d), 1 << 50), S_out=60) == arg
    # lse and weights
    for name in ("q", "kp", "vp", "kc", "vc", "out"):
        assert _shared(lib, _shape(), lse=at + 256, **{name: Heads(data=at)}) == arg, name
    assert _shared(lib, _shape(), lse=2) == arg
    for name in ("q", "kc", "vc", "out"):
        assert _scored(lib, _shape(), w_out=at + 256, **{name: Heads(data=at)}) == arg, name
    assert _scored(lib, _shape(), w_in=at + 256, out=Heads(data=at)) == arg
    # eviction's weights, positions and lengths
    for kw in (dict(k=Heads(data=at)), dict(v=Heads(data=at)), dict(out=(Heads(data=at), Heads(), 1 << 50), S_out=60),
               dict(out=(Heads(), Heads(data=at), 1 << 50), S_out=60)):
        assert _evict(lib, kept=at + 256, **kw) == arg, kw
        assert _evict(lib, lens_out=at + 256, **kw) == arg, kw
    assert _evict(lib, k=Heads(data=at), w=at + 256) == arg
    assert _evict(lib, out=(Heads(data=at), Heads(), at + 256), S_out=60) == arg
    assert _evict(lib, kept=1 << 36) == arg            # over the weights
    assert _evict(lib, lens_out=(1 << 36) + 8) == arg
    assert _evict(lib, kept=1 << 33) == arg            # over the lengths
    assert _evict(lib, kept=1 << 34) == arg            # over lengths_out
    assert _evict(lib, lens_out=(1 << 33) + 4) == arg  # over the lengths in part
    assert _evict(lib, n_slots=2, slots=at, kept=at) == arg


@pytest.mark.parametrize("bad", [None, [1, 2], 3.0, "numpy"], ids=str)
def test_python_arguments_that_are_no_tensors(fmx, bad):
    """A TypeError that names the argument."""
    import numpy as np
    import torch
    from flashmlx_amd import cache as M
    if bad == "numpy":
        bad = np.zeros((2, 1, 8, 64), dtype=np.float32)
    q = torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16)
    for f in (M._heads, M._cache, M._prefix):
        with pytest.raises(TypeError, match="some_array: a tensor expected"):
            f(bad, "some_array", (2, 1, 8, 64), torch.bfloat16, -1)
    if bad is not None:
        with pytest.raises(TypeError, match="some_array: a tensor expected"):
            M._flat(bad, "some_array", (2,), torch.int32, -1)
        with pytest.raises(TypeError, match="workspace: a tensor expected"):
            M._workspace(bad, 5, q)
    for call, name in ((lambda: fmx.attention_scored(bad, q, q, q, 0.1), "q"),
                       (lambda: fmx.attention_shared_prefix(bad, None, None, q, q, q, 0.1), "q"),
                       (lambda: fmx.cache_evict(bad, q, q, q, 4), "k_cache"), (lambda: M._pool(bad, 64), "k_cache")):
        with pytest.raises(TypeError, match=f"^{name}: a tensor expected"):
            call()


def test_keys_among_queries_in_place(lib):
    """Queries turned in place, new keys or values among their heads: a
    workgroup could read a key that another has turned already. Beside them in
    a fused row they are taken (that call ends at a later check here)."""
    angles = C.byref(_lib.FmxRopeAngles(1 << 33, 64, 1.0, 0))
    arg, at, row = _lib.FMX_ERR_ARG, 1 << 52, dict(bs=3 * 12 * 128, ts=12 * 128, hs=128)

    def call(k, v, cache=None):
        q = Heads(data=at, **row)
        caches = Heads(), cache or Heads()
        return lib.fmx_rope_append(angles, _lib.FMX_BF16, 2, 3, 4, 4, 128, q, Heads(data=at + 2 * k, **row),
                                   Heads(data=at + 2 * v, **row), 1 << 34, 1 << 35, None, 2, 8, q, *caches, None)

    for h in (0, 64, 128, 3 * 128):
        assert call(h, 8 * 128) == arg and b"overlaps k" in lib.fmx_last_error(), h
        assert call(4 * 128, h) == arg and b"overlaps v" in lib.fmx_last_error(), h
    assert call(4 * 128, 8 * 128, Heads(data=at)) == arg and b"a cache overlaps" in lib.fmx_last_error()
