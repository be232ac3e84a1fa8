"""The KV cache's long-context operators on libfmx (include/fmx_cache.h):
rotary positions of any layout with the caches' append (`Rope`), attention of
a batch behind one shared prefix, attention that adds up the weight each
cached key gets, and the eviction of keys by those weights.

Arrays: queries and new keys [batch, seq_len, heads, head_dim], caches
[slots, kv_heads, max_seq, head_dim], a prefix [kv_heads, length, head_dim],
weights fp32 [slots, kv_heads, max_seq]. Any strides with the head's elements
contiguous will do (16-byte steps for attention); weights, positions, offsets,
lengths and slots are contiguous. torch tensors only carry device memory and
the current stream into the C-ABI: no call is recorded for autograd, and a
result never requires a gradient, whatever its inputs do.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._lib import FmxAttentionShape, FmxHeads, FmxRopeAngles, FmxRopeConfig

_DT = {torch.bfloat16: _lib.FMX_BF16, torch.float16: _lib.FMX_F16, torch.float32: _lib.FMX_F32}
_SCALING = {"none": 0, "linear": 1, "ntk": 2, "parts": 3, "yarn": 4}
# (low, high) turns over the trained length where the config gives none
_TURNS = {"parts": (1.0, 4.0), "yarn": (1.0, 32.0)}


_byref = C.byref


def _tensor(t, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor expected, got {type(t).__name__}")


def _refuse(t, name: str, shape: tuple, dtype, dev: int) -> None:
    """Says which of an argument's shape, dtype, device or layout is wrong."""
    _tensor(t, name)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: {t.dtype}, expected {dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")
    raise ValueError(f"{name}: strides {t.stride()}, expected contiguous " +
                     ("elements of a head" if t.is_floating_point() and t.dim() > 2 else "memory"))


def _heads(t: torch.Tensor, name: str, shape, dtype, dev: int):
    """The view of a [batch, token, head, element] tensor."""
    try:
        s = t.stride()
    except AttributeError:
        _tensor(t, name)
        raise
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev or s[3] != 1 and shape[3] != 1:
        _refuse(t, name, shape, dtype, dev)
    return _byref(FmxHeads(t.data_ptr(), s[0], s[1], s[2]))


def _cache(t: torch.Tensor, name: str, shape, dtype, dev: int):
    """The view of a [slot, head, position, element] tensor."""
    try:
        s = t.stride()
    except AttributeError:
        _tensor(t, name)
        raise
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev or s[3] != 1 and shape[3] != 1:
        _refuse(t, name, shape, dtype, dev)
    return _byref(FmxHeads(t.data_ptr(), s[0], s[2], s[1]))


def _prefix(t: torch.Tensor, name: str, shape, dtype, dev: int):
    """The view of a [head, position, element] tensor."""
    try:
        s = t.stride()
    except AttributeError:
        _tensor(t, name)
        raise
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev or s[2] != 1 and shape[2] != 1:
        _refuse(t, name, shape, dtype, dev)
    return _byref(FmxHeads(t.data_ptr(), 0, s[1], s[0]))


def _flat(t: Optional[torch.Tensor], name: str, shape, dtype, dev: int) -> Optional[int]:
    """The address of a contiguous array, or None."""
    if t is None:
        return None
    try:
        wrong = t.shape != shape or t.dtype != dtype or t.get_device() != dev or not t.is_contiguous()
    except AttributeError:
        wrong = True
    if wrong:
        _refuse(t, name, shape, dtype, dev)
    return t.data_ptr()


def _device(t: torch.Tensor, name: str, dims: str) -> int:
    """The index of the current device, on which t, of four axes, has to be."""
    try:
        dims_there = t.dim()
    except AttributeError:
        _tensor(t, name)
        raise
    if dims_there != 4:
        raise ValueError(f"{name}: [{dims}] expected, got {tuple(t.shape)}")
    if t.dtype not in _DT:
        raise TypeError(f"{name}: {t.dtype} (bfloat16, float16 or float32)")
    dev = t.get_device()
    if dev < 0 or dev != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, which is not the current HIP device")
    return dev


_ROWS, _SLOTS = "batch, seq_len, heads, head_dim", "slots, kv_heads, positions, head_dim"


def _pool(k: torch.Tensor, hd: int) -> tuple:
    """(slots, kv heads, positions) of the caches."""
    try:
        wrong = k.dim() != 4 or k.shape[3] != hd
    except AttributeError:
        _tensor(k, "k_cache")
        raise
    if wrong:
        raise ValueError(f"k_cache: shape {tuple(k.shape)}, expected [slots, kv_heads, positions, {hd}]")
    return k.shape[0], k.shape[1], k.shape[2]


def _stream(dev: int) -> int:
    # (without torch's Stream object, whose making takes 2.4 us of an append's 13)
    return torch._C._cuda_getCurrentRawStream(dev)


def _workspace(ws: Optional[torch.Tensor], need: int, like: torch.Tensor) -> torch.Tensor:
    if ws is None:
        return like.new_empty(max(need, 1), dtype=torch.uint8)
    _tensor(ws, "workspace")
    if ws.get_device() != like.get_device() or not ws.is_contiguous() or ws.dtype != torch.uint8:
        raise ValueError(f"workspace: a contiguous uint8 tensor on {like.device} expected")
    return ws


# --------------------------------------------------------------------- rope

@dataclass
class RopeConfig:
    """fmx_rope_config: which elements of a head turn and by what angle per
    position. scaling: "none", "linear", "ntk", "parts" or "yarn"; low and
    high (turns over original_max) default to 1 and 4 for "parts", 1 and 32
    for "yarn"; attention_factor None: the scaling's own."""
    dims: int
    base: float = 10000.0
    interleaved: bool = False
    scaling: str = "none"
    factor: float = 1.0
    original_max: int = 4096
    low: Optional[float] = None
    high: Optional[float] = None
    attention_factor: Optional[float] = None

    def frequencies(self) -> tuple:
        """(angles per position, numpy float64 [dims / 2]; the factor on the
        results): fmx_rope_frequencies, host only."""
        if self.scaling not in _SCALING:
            raise ValueError(f"scaling {self.scaling!r}: one of {sorted(_SCALING)}")
        low, high = _TURNS.get(self.scaling, (1.0, 2.0))
        c = FmxRopeConfig(self.dims, self.base, _SCALING[self.scaling], self.factor, self.original_max,
                          low if self.low is None else self.low, high if self.high is None else self.high,
                          self.attention_factor or 0.0)
        freqs = np.empty(max(self.dims // 2, 1), dtype=np.float64)
        m = C.c_double()
        _lib.check(_lib.load().fmx_rope_frequencies(C.byref(c), freqs.ctypes.data, C.byref(m)))
        return freqs, m.value


class Rope:
    """Rotary positions of one layout: mx::fast::rope (server/src/model.cpp:
    875-876) with both pairings, part of the head, scaled frequencies and a
    position per token. Holds the frequencies on the device."""

    def __init__(self, cfg: RopeConfig, device: Optional[torch.device] = None):
        self.lib = _lib.load()
        self.cfg = cfg
        freqs, self.factor = cfg.frequencies()
        dev = device or torch.device("cuda", torch.cuda.current_device())
        self.freqs = torch.from_numpy(freqs).to(dev)
        self._c = FmxRopeAngles(self.freqs.data_ptr(), cfg.dims, self.factor, int(cfg.interleaved))
        self._dev = self.freqs.get_device()

    def _check(self, dev: int) -> None:
        if dev != self._dev:
            raise ValueError(f"the frequencies are on cuda:{self._dev}, the rows on cuda:{dev}")

    def __call__(self, x: torch.Tensor, positions: torch.Tensor, out: Optional[torch.Tensor] = None,
                 inverse: bool = False) -> torch.Tensor:
        """x [batch, seq_len, heads, head_dim] turned to positions [batch,
        seq_len] (int32); inverse: back, which is the gradient of the forward
        call with respect to x. out may be x."""
        dev, shape, dt = _device(x, "x", _ROWS), x.shape, x.dtype
        self._check(dev)
        B, L, nh, hd = shape
        if out is None:
            out = x.new_empty(shape)
        _lib.check(self.lib.fmx_rope(
            _byref(self._c), _DT[dt], B, L, nh, hd, _heads(x, "x", shape, dt, dev),
            _flat(positions, "positions", (B, L), torch.int32, dev), int(inverse),
            _heads(out, "out", shape, dt, dev), _stream(dev)))
        return out

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
               offsets: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
               slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One step's new tokens: returns q rotated; k, rotated, and v go to
        cache positions offsets[b] + l of slot slots[b] (or b). Rows outside
        the cache are not written. out may be q."""
        dev, shape, dt, i32 = _device(q, "q", _ROWS), q.shape, q.dtype, torch.int32
        self._check(dev)
        B, L, nh, hd = shape
        n_slots, nkv, S = _pool(k_cache, hd)
        new, pool = (B, L, nkv, hd), k_cache.shape
        if out is None:
            out = q.new_empty(shape)
        _lib.check(self.lib.fmx_rope_append(
            _byref(self._c), _DT[dt], B, L, nh, nkv, hd, _heads(q, "q", shape, dt, dev), _heads(k, "k", new, dt, dev),
            _heads(v, "v", new, dt, dev), _flat(positions, "positions", (B, L), i32, dev),
            _flat(offsets, "offsets", (B,), i32, dev), _flat(slots, "slots", (B,), i32, dev), n_slots, S,
            _heads(out, "out", shape, dt, dev), _cache(k_cache, "k_cache", pool, dt, dev),
            _cache(v_cache, "v_cache", pool, dt, dev), _stream(dev)))
        return out


# --------------------------------------------------------------------- attention

def attention_shared_prefix(q: torch.Tensor, k_prefix: Optional[torch.Tensor], v_prefix: Optional[torch.Tensor],
                            k_cache: torch.Tensor, v_cache: torch.Tensor, offsets: torch.Tensor, scale: float,
                            slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                            workspace: Optional[torch.Tensor] = None) -> tuple:
    """fmx_attention_shared_prefix: (out, lse fp32 [batch, seq_len, heads]).
    Queries are the newest seq_len tokens of each sequence (their keys at
    cache positions offsets[b] .. offsets[b] + seq_len - 1 already); all of
    them see the whole prefix (None: no prefix), and of their own slot the
    positions up to their own. A query that sees no key gets 0 and -inf."""
    lib = _lib.load()
    dev, shape, dt, i32 = _device(q, "q", _ROWS), q.shape, q.dtype, torch.int32
    B, L, nh, hd = shape
    n_slots, nkv, S = _pool(k_cache, hd)
    pool = k_cache.shape
    P, kp, vp = 0, None, None
    if (k_prefix is None) != (v_prefix is None):
        raise ValueError("k_prefix and v_prefix: both or neither")
    if k_prefix is not None:
        _tensor(k_prefix, "k_prefix")
        P = k_prefix.shape[1] if k_prefix.dim() == 3 else -1
        kp = _prefix(k_prefix, "k_prefix", (nkv, P, hd), dt, dev)
        vp = _prefix(v_prefix, "v_prefix", (nkv, P, hd), dt, dev)
    if out is None:
        out = q.new_empty(shape)
    lse = q.new_empty((B, L, nh), dtype=torch.float32)
    c = _byref(FmxAttentionShape(_DT[dt], B, L, nh, nkv, hd, scale))
    ws = _workspace(workspace, lib.fmx_attention_shared_prefix_workspace_size(c, P, S), q)
    _lib.check(lib.fmx_attention_shared_prefix(
        c, _heads(q, "q", shape, dt, dev), kp, vp, P, _cache(k_cache, "k_cache", pool, dt, dev),
        _cache(v_cache, "v_cache", pool, dt, dev), n_slots, S, _flat(offsets, "offsets", (B,), i32, dev),
        _flat(slots, "slots", (B,), i32, dev), _heads(out, "out", shape, dt, dev), lse.data_ptr(), ws.data_ptr(),
        ws.numel(), _stream(dev)))
    return out, lse


def attention_scored(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, offsets: torch.Tensor,
                     scale: float, weights: Optional[torch.Tensor] = None,
                     weights_out: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> tuple:
    """fmx_attention_scored: (out, weights_out), where weights_out is
    `weights` (None: 0) plus what the queries' softmax gives every cached
    position, summed over a kv head's query heads. weights_out may be weights;
    a new one made here holds `weights` (or 0) in the slots of no sequence."""
    lib = _lib.load()
    dev, shape, dt, i32, f32 = _device(q, "q", _ROWS), q.shape, q.dtype, torch.int32, torch.float32
    B, L, nh, hd = shape
    n_slots, nkv, S = _pool(k_cache, hd)
    pool, wsh = k_cache.shape, (n_slots, nkv, S)
    w_in = _flat(weights, "weights", wsh, f32, dev)
    if weights_out is None:
        if slots is None and n_slots == B and L > 0:
            weights_out = q.new_empty(wsh, dtype=f32)
        elif weights is not None:
            weights_out = weights.clone()
        else:
            weights_out = q.new_zeros(wsh, dtype=f32)
    if out is None:
        out = q.new_empty(shape)
    c = _byref(FmxAttentionShape(_DT[dt], B, L, nh, nkv, hd, scale))
    ws = _workspace(workspace, lib.fmx_attention_scored_workspace_size(c, S), q)
    _lib.check(lib.fmx_attention_scored(
        c, _heads(q, "q", shape, dt, dev), _cache(k_cache, "k_cache", pool, dt, dev),
        _cache(v_cache, "v_cache", pool, dt, dev), n_slots, S, _flat(offsets, "offsets", (B,), i32, dev),
        _flat(slots, "slots", (B,), i32, dev), w_in, _flat(weights_out, "weights_out", wsh, f32, dev),
        _heads(out, "out", shape, dt, dev), ws.data_ptr(), ws.numel(), _stream(dev)))
    return out, weights_out


# --------------------------------------------------------------------- eviction

def cache_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, weights: torch.Tensor, lengths: torch.Tensor,
                budget: int, sinks: int = 0, recent: int = 0, slots: Optional[torch.Tensor] = None,
                out: Optional[tuple] = None, lengths_out: Optional[torch.Tensor] = None) -> tuple:
    """fmx_cache_evict: cuts sequences of more than `budget` cached positions
    down to it (per kv head: the first `sinks`, the last `recent`, of the rest
    the largest weights), in place or into out = (k, v, weights). Returns
    (lengths_out int32 [batch], kept int32 [batch, kv_heads, budget]: the kept
    positions, -1 behind the last). lengths_out may be lengths."""
    lib = _lib.load()
    dev, pool, dt = _device(k_cache, "k_cache", _SLOTS), k_cache.shape, k_cache.dtype
    i32, f32 = torch.int32, torch.float32
    n_slots, nkv, S, hd = pool
    _tensor(lengths, "lengths")
    if lengths.dim() != 1:
        raise ValueError(f"lengths: shape {tuple(lengths.shape)}, expected [batch]")
    if not 1 <= budget <= 1 << 24:  # (before `kept` of so many positions is made)
        raise ValueError(f"budget {budget} (1 .. 2^24)")
    B = lengths.shape[0]
    ko = vo = wo = None
    S_out = 0
    if out is not None:
        k_out, v_out, w_out = out
        _tensor(k_out, "out[0]")
        S_out = k_out.shape[2] if k_out.dim() == 4 else -1
        to = (n_slots, nkv, S_out, hd)
        ko, vo = _cache(k_out, "out[0]", to, dt, dev), _cache(v_out, "out[1]", to, dt, dev)
        wo = _flat(w_out, "out[2]", to[:3], f32, dev)
    if lengths_out is None:
        lengths_out = lengths.new_empty((B,))
    kept = lengths.new_empty((B, nkv, budget))
    _lib.check(lib.fmx_cache_evict(
        _DT[dt], B, nkv, hd, _cache(k_cache, "k_cache", pool, dt, dev), _cache(v_cache, "v_cache", pool, dt, dev),
        _flat(weights, "weights", (n_slots, nkv, S), f32, dev), n_slots, S, _flat(lengths, "lengths", (B,), i32, dev),
        _flat(slots, "slots", (B,), i32, dev), budget, sinks, recent, ko, vo, wo, S_out,
        _flat(lengths_out, "lengths_out", (B,), i32, dev), kept.data_ptr(), None, 0, _stream(dev)))
    return lengths_out, kept
