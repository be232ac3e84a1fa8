"""The selective state space layer's operators on libfmx (include/fmx_ssm.h):
the short causal convolution, the selective scan, the norm of groups with its
gate, and a layer's own weights with one decoded token through all three
(`SsmLayer`): what NemotronHModel's Mamba-2 mixer (server/src/nemotron_h.cpp)
computes between its projections.

Arrays: rows [batch, seq_len, channels], heads [batch, seq_len, heads,
head_dim], states in pools of slots: the convolution's [slots, taps - 1,
channels], the scan's fp32 [slots, heads, head_dim, state_dim]. Any strides
with a row's (a head's) elements contiguous will do (16-byte steps for the
scan), so the parts of a projection's rows need no copies; states, weights,
lengths and slots are contiguous. torch tensors only carry device memory and
the current stream into the C-ABI: no call is recorded for autograd.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib
from ._lib import FmxHeads, FmxSsmLayer, FmxSsmShape
from .cache import _DT, _flat, _heads, _refuse, _stream, _tensor, _workspace

_ACT = {None: 0, "none": 0, "silu": 1}
_byref = C.byref
_F32, _I32 = torch.float32, torch.int32


def _device(t: torch.Tensor, name: str, dims: str, n: int) -> int:
    """The index of the current device, on which t, of n axes, has to be."""
    try:
        there = t.dim()
    except AttributeError:
        _tensor(t, name)
        raise
    if there != n:
        raise ValueError(f"{name}: [{dims}] expected, got {tuple(t.shape)}")
    if t.dtype not in _DT:
        raise TypeError(f"{name}: {t.dtype} (bfloat16, float16 or float32)")
    dev = t.get_device()
    if dev < 0 or dev != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, which is not the current HIP device")
    return dev


def _rows(t: torch.Tensor, name: str, shape, dtype, dev: int):
    """The view of a [batch, token, element] tensor."""
    try:
        s = t.stride()
    except AttributeError:
        _tensor(t, name)
        raise
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev or s[2] != 1 and shape[2] != 1:
        _refuse(t, name, shape, dtype, dev)
    return _byref(FmxHeads(t.data_ptr(), s[0], s[1], 0))


def _row(t: torch.Tensor, name: str, shape, dtype, dev: int):
    """The view of a [batch, element] tensor."""
    try:
        s = t.stride()
    except AttributeError:
        _tensor(t, name)
        raise
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev or s[1] != 1 and shape[1] != 1:
        _refuse(t, name, shape, dtype, dev)
    return _byref(FmxHeads(t.data_ptr(), s[0], 0, 0))


def _steps(t: torch.Tensor, name: str, shape, dtype, dev: int):
    """The view of a [batch, token, head] (or [batch, head]) tensor, any strides."""
    _tensor(t, name)
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev:
        _refuse(t, name, shape, dtype, dev)
    s = t.stride()
    return _byref(FmxHeads(t.data_ptr(), s[0], s[1] if len(s) == 3 else 0, s[-1]))


def _activation(activation: Optional[str]) -> int:
    if activation not in _ACT:
        raise ValueError(f"activation {activation!r}: one of {sorted(str(k) for k in _ACT)}")
    return _ACT[activation]


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                state: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                activation: Optional[str] = "silu", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fmx_causal_conv: the causal convolution of x [batch, seq_len, channels]
    per channel with weight [channels, taps], from the rows that `state`
    [slots, taps - 1, channels] holds (None: zeros), and its activation ("silu"
    or None). state_out, which may be state, receives each sequence's last
    taps - 1 rows. Rows of out behind a sequence's length are left as they are
    (those of one made here are not set)."""
    lib = _lib.load()
    act = _activation(activation)
    dev, shape, dt = _device(x, "x", "batch, seq_len, channels", 3), x.shape, x.dtype
    B, L, ch = shape
    _tensor(weight, "weight")
    taps = weight.shape[1] if weight.dim() == 2 else -1
    some = state if state_out is None else state_out
    n_slots = 0
    if some is not None:
        _tensor(some, "state")
        n_slots = some.shape[0] if some.dim() == 3 else -1
    pool = (n_slots, taps - 1, ch)
    if out is None:
        out = x.new_empty(shape)
    _lib.check(lib.fmx_causal_conv(
        _DT[dt], B, L, ch, taps, act, _rows(x, "x", shape, dt, dev), _flat(weight, "weight", (ch, taps), dt, dev),
        _flat(bias, "bias", (ch,), dt, dev), _flat(state, "state", pool, dt, dev),
        _flat(state_out, "state_out", pool, dt, dev), n_slots, _flat(lengths, "lengths", (B,), _I32, dev),
        _flat(slots, "slots", (B,), _I32, dev), _rows(out, "out", shape, dt, dev), _stream(dev)))
    return out


def ssm_scan(x: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor,
             d: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
             state: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None,
             lengths: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None, softplus: bool = True,
             dt_limits: tuple = (0.0, math.inf), out: Optional[torch.Tensor] = None,
             workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fmx_ssm_scan: the selective scan of x [batch, seq_len, heads, head_dim]
    with time steps dt [batch, seq_len, heads] (before bias, softplus and
    limits), rates a [heads] (negative, fp32), b and c [batch, seq_len, groups,
    state_dim] and the skip d [heads] (fp32), from `state` fp32 [slots, heads,
    head_dim, state_dim] (None: zeros); state_out, which may be state, receives
    the state behind each sequence's last token. Rows of out behind a
    sequence's length are left as they are."""
    lib = _lib.load()
    dev, shape, ty = _device(x, "x", "batch, seq_len, heads, head_dim", 4), x.shape, x.dtype
    B, L, nh, hd = shape
    _tensor(b, "b")
    groups, N = (b.shape[2], b.shape[3]) if b.dim() == 4 else (-1, -1)
    some = state if state_out is None else state_out
    n_slots = 0
    if some is not None:
        _tensor(some, "state")
        n_slots = some.shape[0] if some.dim() == 4 else -1
    pool, inner = (n_slots, nh, hd, N), (B, L, groups, N)
    if out is None:
        out = x.new_empty(shape)
    s = _byref(FmxSsmShape(_DT[ty], B, L, nh, hd, groups, N, int(softplus), dt_limits[0], dt_limits[1]))
    ws = _workspace(workspace, lib.fmx_ssm_scan_workspace_size(s), x)
    _lib.check(lib.fmx_ssm_scan(
        s, _heads(x, "x", shape, ty, dev), _steps(dt, "dt", (B, L, nh), ty, dev), _flat(a, "a", (nh,), _F32, dev),
        _heads(b, "b", inner, ty, dev), _heads(c, "c", inner, ty, dev), _flat(d, "d", (nh,), _F32, dev),
        _flat(dt_bias, "dt_bias", (nh,), _F32, dev), _flat(state, "state", pool, _F32, dev),
        _flat(state_out, "state_out", pool, _F32, dev), n_slots, _flat(lengths, "lengths", (B,), _I32, dev),
        _flat(slots, "slots", (B,), _I32, dev), _heads(out, "out", shape, ty, dev), ws.data_ptr(), ws.numel(),
        _stream(dev)))
    return out


def gated_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
               eps: float = 1e-5, groups: int = 1, gate_first: bool = True, lengths: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fmx_gated_norm: x [batch, seq_len, channels], times silu(z) before the
    norm (gate_first) or behind it (z None: no gate), over the RMS of each of
    `groups` runs of channels, times weight [channels]. out may be x or z. Rows
    of out behind a sequence's length are left as they are."""
    lib = _lib.load()
    dev, shape, dt = _device(x, "x", "batch, seq_len, channels", 3), x.shape, x.dtype
    B, L, ch = shape
    if out is None:
        out = x.new_empty(shape)
    _lib.check(lib.fmx_gated_norm(
        _DT[dt], B, L, ch, groups, eps, int(gate_first), _rows(x, "x", shape, dt, dev),
        None if z is None else _rows(z, "z", shape, dt, dev), _flat(weight, "weight", (ch,), dt, dev),
        _flat(lengths, "lengths", (B,), _I32, dev), _rows(out, "out", shape, dt, dev), _stream(dev)))
    return out


class SsmLayer:
    """A layer between its projections: its weights, checked once. The
    convolution's channels are x (heads * head_dim), b, then c (groups *
    state_dim each); norm_groups None: one per group. Holds no state."""

    def __init__(self, conv_weight: torch.Tensor, a: torch.Tensor, norm_weight: Optional[torch.Tensor],
                 head_dim: int, groups: int, state_dim: int, conv_bias: Optional[torch.Tensor] = None,
                 d: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                 norm_groups: Optional[int] = None, eps: float = 1e-5, gate_first: bool = True, softplus: bool = True,
                 dt_limits: tuple = (0.0, math.inf), activation: Optional[str] = "silu"):
        self.lib = _lib.load()
        dev, dt = _device(conv_weight, "conv_weight", "channels, taps", 2), conv_weight.dtype
        _tensor(a, "a")
        heads = a.numel()
        ch, taps = conv_weight.shape
        inner = heads * head_dim
        if ch != inner + 2 * groups * state_dim:
            raise ValueError(f"conv_weight: {ch} channels, expected {inner} + 2 * {groups * state_dim}")
        self.heads, self.head_dim, self.groups, self.state_dim = heads, head_dim, groups, state_dim
        self.channels, self.taps, self.inner, self.dtype, self._dev = ch, taps, inner, dt, dev
        self.conv_weight, self.conv_bias, self.a, self.d, self.dt_bias = conv_weight, conv_bias, a, d, dt_bias
        self.norm_weight, self.norm_groups = norm_weight, groups if norm_groups is None else norm_groups
        self.eps, self.gate_first, self.softplus, self.dt_limits = eps, gate_first, softplus, dt_limits
        self.activation = activation
        self._c = FmxSsmLayer(
            _DT[dt], heads, head_dim, groups, state_dim, taps, _activation(activation),
            _flat(conv_weight, "conv_weight", (ch, taps), dt, dev), _flat(conv_bias, "conv_bias", (ch,), dt, dev),
            _flat(a, "a", (heads,), _F32, dev), _flat(d, "d", (heads,), _F32, dev),
            _flat(dt_bias, "dt_bias", (heads,), _F32, dev), int(softplus), dt_limits[0], dt_limits[1],
            _flat(norm_weight, "norm_weight", (inner,), dt, dev), self.norm_groups, eps, int(gate_first))
        self._ref, self._bytes = _byref(self._c), {}  # (of the struct; workspace bytes by batch)

    def new_states(self, slots: int) -> tuple:
        """(conv_state, state) of a pool of so many slots, zeros."""
        dev = self.conv_weight.device
        return (torch.zeros((slots, self.taps - 1, self.channels), dtype=self.dtype, device=dev),
                torch.zeros((slots, self.heads, self.head_dim, self.state_dim), dtype=_F32, device=dev))

    def _here(self, dev: int) -> None:
        if dev != self._dev:
            raise ValueError(f"the weights are on cuda:{self._dev}, the rows on cuda:{dev}")

    def prompt(self, xbc: torch.Tensor, dt: torch.Tensor, z: Optional[torch.Tensor], conv_state: torch.Tensor,
               state: torch.Tensor, lengths: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Rows xbc [batch, seq_len, channels], dt [batch, seq_len, heads] and
        z [batch, seq_len, heads * head_dim] through causal_conv, ssm_scan and
        gated_norm, from the slots' states and with them moved on. A call that
        is refused has moved neither."""
        lib, ty = self.lib, self.dtype
        dev = _device(xbc, "xbc", "batch, seq_len, channels", 3)
        self._here(dev)
        B, L, _ = xbc.shape
        nh, hd, ch, inner = self.heads, self.head_dim, self.channels, self.inner
        n = self.groups * self.state_dim
        xbc_v, dt_v = _rows(xbc, "xbc", (B, L, ch), ty, dev), _steps(dt, "dt", (B, L, nh), ty, dev)
        z_v = None if z is None else _rows(z, "z", (B, L, inner), ty, dev)
        pools = []
        for t, name, dims in ((conv_state, "conv_state", 3), (state, "state", 4)):
            if t is not None:
                _tensor(t, name)
            pools.append(0 if t is None else t.shape[0] if t.dim() == dims else -1)
        conv_slots, n_slots = pools
        cs = _flat(conv_state, "conv_state", (conv_slots, self.taps - 1, ch), ty, dev)
        st = _flat(state, "state", (n_slots, nh, hd, self.state_dim), _F32, dev)
        lens, at = _flat(lengths, "lengths", (B,), _I32, dev), _flat(slots, "slots", (B,), _I32, dev)
        if out is None:
            out = xbc.new_empty((B, L, inner))
        out_v = _rows(out, "out", (B, L, inner), ty, dev)
        # between the calls: the convolution's rows and the scan's
        v, y = xbc.new_empty((B, L, ch)), xbc.new_empty((B, L, inner))
        vp, yp = v.data_ptr(), y.data_ptr()
        _lib.check(lib.fmx_ssm_prompt_check(self._ref, B, L, xbc_v, dt_v, z_v, vp, yp, cs, conv_slots, st, n_slots, lens, at,
                                            out_v))
        c = self._c
        shape = _byref(FmxSsmShape(c.dtype, B, L, nh, hd, self.groups, self.state_dim, c.dt_softplus, c.dt_min, c.dt_max))
        ws = _workspace(None, lib.fmx_ssm_scan_workspace_size(shape), xbc)
        es, stream = xbc.element_size(), _stream(dev)
        _lib.check(lib.fmx_causal_conv(
            c.dtype, B, L, ch, self.taps, c.activation, xbc_v, c.conv_weight, c.conv_bias, cs, cs, conv_slots, lens, at,
            _byref(FmxHeads(vp, L * ch, ch, 0)), stream))
        part = lambda first, size: _byref(FmxHeads(vp and vp + first * es, L * ch, ch, size))  # noqa: E731
        _lib.check(lib.fmx_ssm_scan(
            shape, part(0, hd), dt_v, c.a, part(inner, self.state_dim), part(inner + n, self.state_dim), c.d, c.dt_bias, st,
            st, n_slots, lens, at, _byref(FmxHeads(yp, L * inner, inner, hd)), ws.data_ptr(), ws.numel(), stream))
        _lib.check(lib.fmx_gated_norm(
            c.dtype, B, L, inner, c.norm_groups, c.eps, c.gate_first, _byref(FmxHeads(yp, L * inner, inner, 0)), z_v,
            c.norm_weight, lens, out_v, stream))
        return out

    def step(self, xbc: torch.Tensor, dt: torch.Tensor, z: Optional[torch.Tensor], conv_state: torch.Tensor,
             state: torch.Tensor, slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
             workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """fmx_ssm_step: one token of each sequence, xbc [batch, channels], dt
        [batch, heads] and z [batch, heads * head_dim] (None: no gate), the
        slots' states moved on in place."""
        dev, ty = _device(xbc, "xbc", "batch, channels", 2), self.dtype
        self._here(dev)
        B = xbc.shape[0]
        inner = (B, self.inner)
        _tensor(state, "state")
        n_slots = state.shape[0] if state.dim() == 4 else -1
        if out is None:
            out = xbc.new_empty(inner)
        need, c = self._bytes.get(B), self._ref
        if need is None:
            need = self._bytes[B] = self.lib.fmx_ssm_step_workspace_size(c, B)
        ws = _workspace(workspace, need, xbc)
        _lib.check(self.lib.fmx_ssm_step(
            c, B, _row(xbc, "xbc", (B, self.channels), ty, dev), _steps(dt, "dt", (B, self.heads), ty, dev),
            None if z is None else _row(z, "z", inner, ty, dev),
            _flat(conv_state, "conv_state", (n_slots, self.taps - 1, self.channels), ty, dev),
            _flat(state, "state", (n_slots, self.heads, self.head_dim, self.state_dim), _F32, dev), n_slots,
            _flat(slots, "slots", (B,), _I32, dev), _row(out, "out", inner, ty, dev), ws.data_ptr(), ws.numel(),
            _stream(dev)))
        return out
