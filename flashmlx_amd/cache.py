"""The KV cache's long-context operators on libfmx (include/fmx_cache.h):
rotary positions of any layout with the caches' append (`Rope`), attention of
a batch behind one shared prefix, attention that adds up the weight each
cached key gets, and the eviction of keys by those weights.

Arrays: queries and new keys [batch, seq_len, heads, head_dim], caches
[slots, kv_heads, max_seq, head_dim], a prefix [kv_heads, length, head_dim],
weights fp32 [slots, kv_heads, max_seq]. Any strides with the head's elements
contiguous will do (16-byte steps for attention); weights, positions, offsets,
lengths and slots are contiguous. torch tensors only carry device memory and
the current stream into the C-ABI.
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


def _heads(t: torch.Tensor, name: str, like: torch.Tensor, shape: tuple, order=(0, 1, 2)) -> FmxHeads:
    """The view of a 4-d tensor whose batch, token and head axes are `order`."""
    if tuple(t.shape) != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {shape}")
    if t.dtype != like.dtype:
        raise TypeError(f"{name}: {t.dtype}, expected {like.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, not {like.device}")
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        raise ValueError(f"{name}: the head's elements must be contiguous")
    st = t.stride()
    # the stride of an axis of one entry is never used: 0, whatever torch says
    b, l, h = (st[i] if t.shape[i] > 1 else 0 for i in order)
    return FmxHeads(t.data_ptr(), b, l, h)


def _cache(t: torch.Tensor, name: str, like: torch.Tensor, nkv: int, hd: int) -> FmxHeads:
    if t.dim() != 4 or t.shape[1] != nkv or t.shape[3] != hd:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected [slots, {nkv}, positions, {hd}]")
    return _heads(t, name, like, tuple(t.shape), (0, 2, 1))


def _ints(t: Optional[torch.Tensor], name: str, like: torch.Tensor, shape: tuple) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != like.device:
        raise ValueError(f"{name}: a contiguous int32 tensor {shape} on {like.device} expected")
    return t.data_ptr()


def _floats(t: Optional[torch.Tensor], name: str, like: torch.Tensor, shape: tuple) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != like.device:
        raise ValueError(f"{name}: a contiguous float32 tensor {shape} on {like.device} expected")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str) -> tuple:
    """(batch, seq_len, heads, head_dim) of a query-like tensor on the current device."""
    if t.dim() != 4:
        raise ValueError(f"{name}: [batch, seq_len, heads, head_dim] expected, got {tuple(t.shape)}")
    if t.dtype not in _DT:
        raise TypeError(f"{name}: {t.dtype} (bfloat16, float16 or float32)")
    _on_device(t, name)
    return tuple(t.shape)


def _on_device(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda or t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, which is not the current HIP device")


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _workspace(ws: Optional[torch.Tensor], need: int, like: torch.Tensor) -> torch.Tensor:
    if ws is None:
        return torch.empty(max(need, 1), dtype=torch.uint8, device=like.device)
    if ws.device != like.device or not ws.is_contiguous() or ws.dtype != torch.uint8:
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

    def _check(self, t: torch.Tensor) -> None:
        if t.device != self.freqs.device:
            raise ValueError(f"the frequencies are on {self.freqs.device}, the rows on {t.device}")

    def __call__(self, x: torch.Tensor, positions: torch.Tensor, out: Optional[torch.Tensor] = None,
                 inverse: bool = False) -> torch.Tensor:
        """x [batch, seq_len, heads, head_dim] turned to positions [batch,
        seq_len] (int32); inverse: back, which is the gradient of the forward
        call with respect to x. out may be x."""
        B, L, nh, hd = shape = _rows(x, "x")
        self._check(x)
        if out is None:
            out = torch.empty(shape, dtype=x.dtype, device=x.device)
        _lib.check(self.lib.fmx_rope(
            C.byref(self._c), _DT[x.dtype], B, L, nh, hd, C.byref(_heads(x, "x", x, shape)),
            _ints(positions, "positions", x, (B, L)), int(inverse), C.byref(_heads(out, "out", x, shape)), _stream()))
        return out

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
               offsets: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
               slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One step's new tokens: returns q rotated; k, rotated, and v go to
        cache positions offsets[b] + l of slot slots[b] (or b). Rows outside
        the cache are not written. out may be q."""
        B, L, nh, hd = shape = _rows(q, "q")
        self._check(q)
        nkv = k.shape[2] if k.dim() == 4 else 0
        if out is None:
            out = torch.empty(shape, dtype=q.dtype, device=q.device)
        kc, vc = _cache(k_cache, "k_cache", q, nkv, hd), _cache(v_cache, "v_cache", q, nkv, hd)
        if v_cache.shape[:3] != k_cache.shape[:3]:
            raise ValueError("k_cache and v_cache differ in shape")
        _lib.check(self.lib.fmx_rope_append(
            C.byref(self._c), _DT[q.dtype], B, L, nh, nkv, hd, C.byref(_heads(q, "q", q, shape)),
            C.byref(_heads(k, "k", q, (B, L, nkv, hd))), C.byref(_heads(v, "v", q, (B, L, nkv, hd))),
            _ints(positions, "positions", q, (B, L)), _ints(offsets, "offsets", q, (B,)),
            _ints(slots, "slots", q, (B,)), k_cache.shape[0], k_cache.shape[2],
            C.byref(_heads(out, "out", q, shape)), C.byref(kc), C.byref(vc), _stream()))
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
    B, L, nh, hd = shape = _rows(q, "q")
    nkv = k_cache.shape[1] if k_cache.dim() == 4 else 0
    kc, vc = _cache(k_cache, "k_cache", q, nkv, hd), _cache(v_cache, "v_cache", q, nkv, hd)
    if v_cache.shape[:3] != k_cache.shape[:3]:
        raise ValueError("k_cache and v_cache differ in shape")
    P, kp, vp = 0, None, None
    if (k_prefix is None) != (v_prefix is None):
        raise ValueError("k_prefix and v_prefix: both or neither")
    if k_prefix is not None:
        P = k_prefix.shape[1] if k_prefix.dim() == 3 else -1
        kp = C.byref(_heads(k_prefix.unsqueeze(0), "k_prefix", q, (1, nkv, P, hd), (0, 2, 1)))
        vp = C.byref(_heads(v_prefix.unsqueeze(0), "v_prefix", q, (1, nkv, P, hd), (0, 2, 1)))
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((B, L, nh), dtype=torch.float32, device=q.device)
    c = FmxAttentionShape(_DT[q.dtype], B, L, nh, nkv, hd, scale)
    S = k_cache.shape[2]
    ws = _workspace(workspace, lib.fmx_attention_shared_prefix_workspace_size(C.byref(c), P, S), q)
    _lib.check(lib.fmx_attention_shared_prefix(
        C.byref(c), C.byref(_heads(q, "q", q, shape)), kp, vp, P, C.byref(kc), C.byref(vc), k_cache.shape[0], S,
        _ints(offsets, "offsets", q, (B,)), _ints(slots, "slots", q, (B,)), C.byref(_heads(out, "out", q, shape)),
        lse.data_ptr(), ws.data_ptr(), ws.numel(), _stream()))
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
    B, L, nh, hd = shape = _rows(q, "q")
    nkv = k_cache.shape[1] if k_cache.dim() == 4 else 0
    kc, vc = _cache(k_cache, "k_cache", q, nkv, hd), _cache(v_cache, "v_cache", q, nkv, hd)
    if v_cache.shape[:3] != k_cache.shape[:3]:
        raise ValueError("k_cache and v_cache differ in shape")
    n_slots, S = k_cache.shape[0], k_cache.shape[2]
    w_in = _floats(weights, "weights", q, (n_slots, nkv, S))
    if weights_out is None:
        if slots is None and n_slots == B and L > 0:
            weights_out = torch.empty((n_slots, nkv, S), dtype=torch.float32, device=q.device)
        elif weights is not None:
            weights_out = weights.clone()
        else:
            weights_out = torch.zeros((n_slots, nkv, S), dtype=torch.float32, device=q.device)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    c = FmxAttentionShape(_DT[q.dtype], B, L, nh, nkv, hd, scale)
    ws = _workspace(workspace, lib.fmx_attention_scored_workspace_size(C.byref(c), S), q)
    _lib.check(lib.fmx_attention_scored(
        C.byref(c), C.byref(_heads(q, "q", q, shape)), C.byref(kc), C.byref(vc), n_slots, S,
        _ints(offsets, "offsets", q, (B,)), _ints(slots, "slots", q, (B,)), w_in,
        _floats(weights_out, "weights_out", q, (n_slots, nkv, S)), C.byref(_heads(out, "out", q, shape)),
        ws.data_ptr(), ws.numel(), _stream()))
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
    if k_cache.dim() != 4:
        raise ValueError(f"k_cache: shape {tuple(k_cache.shape)}, expected [slots, kv_heads, positions, head_dim]")
    if k_cache.dtype not in _DT:
        raise TypeError(f"k_cache: {k_cache.dtype}")
    _on_device(k_cache, "k_cache")
    n_slots, nkv, S, hd = k_cache.shape
    B = lengths.shape[0] if lengths.dim() == 1 else -1
    kc, vc = _cache(k_cache, "k_cache", k_cache, nkv, hd), _cache(v_cache, "v_cache", k_cache, nkv, hd)
    if v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache differ in shape")
    w = _floats(weights, "weights", k_cache, (n_slots, nkv, S))
    ko = vo = wo = None
    S_out = 0
    if out is not None:
        k_out, v_out, w_out = out
        S_out = k_out.shape[2] if k_out.dim() == 4 else -1
        want = (n_slots, nkv, S_out, hd)
        ko = C.byref(_heads(k_out, "out[0]", k_cache, want, (0, 2, 1)))
        vo = C.byref(_heads(v_out, "out[1]", k_cache, want, (0, 2, 1)))
        wo = _floats(w_out, "out[2]", k_cache, want[:3])
    if budget < 1:
        raise ValueError(f"budget {budget}")
    if lengths_out is None:
        lengths_out = torch.empty((max(B, 0),), dtype=torch.int32, device=k_cache.device)
    kept = torch.empty((max(B, 0), nkv, budget), dtype=torch.int32, device=k_cache.device)
    _lib.check(lib.fmx_cache_evict(
        _DT[k_cache.dtype], B, nkv, hd, C.byref(kc), C.byref(vc), w, n_slots, S,
        _ints(lengths, "lengths", k_cache, (B,)), _ints(slots, "slots", k_cache, (B,)), budget, sinks, recent, ko, vo,
        wo, S_out, _ints(lengths_out, "lengths_out", k_cache, (B,)), kept.data_ptr(), None, 0, _stream()))
    return lengths_out, kept
