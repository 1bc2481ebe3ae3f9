"""Recurrent layers' state: the short convolution's window and the gated delta rule's state of each sequence.

`GatedDeltaCache` stands where the reference's hybrid models keep a `MambaCache` (KVCache.swift:1307-1726) beside the KV caches
of their attention layers: two dense arrays of fixed size, which `causal_convolution` and `gated_delta_update`
(`gatedDeltaUpdate`, GatedDelta.swift:112) read and write in place.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from .cache import _DT, _ptr, _stream


def _on_current_device(*arrays):
    for t in arrays:
        if t is not None and (not t.is_cuda or t.device.index != torch._C._cuda_getDevice()):
            raise ValueError(f"an array lies on {t.device}, not on the current device")


def _per_sequence(t, batch, name):
    if t is None:
        return None
    if tuple(t.shape) != (batch,):
        raise ValueError(f"{name} is one number to each of {batch} sequences, not {tuple(t.shape)}")
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} is int32 or int64, not {t.dtype}")
    return _int32(t).to("cuda").contiguous()


def _int32(t):
    """Whole numbers as int32, those beyond its ends as its ends."""
    return t if t.dtype == torch.int32 else t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)


def _order(order, rows):
    if order.dtype not in (torch.int32, torch.int64) or tuple(order.shape) != (rows,):
        raise ValueError(f"an order is one row number to each of {rows} sequences, not {order.dtype} {tuple(order.shape)}")
    _on_current_device(order)
    return _int32(order).contiguous()


def _dense_rows(t):
    """`t` [B, L, ...] with everything behind the tokens dense: itself, or a copy."""
    want = 1
    for size, stride in zip(reversed(t.shape[2:]), reversed(t.stride()[2:])):
        if size != 1 and stride != want:
            return t.contiguous()
        want *= size
    return t


class GatedDeltaCache:
    """What a gated delta layer remembers of its sequences: `window` [B, conv_width - 1, C], the last inputs of its short
    convolution, and `delta_state` [B, Hv, Dv, Dk] in float32.  Both are None until the first call, or assigned (copied).  Like
    the reference's `ArraysCache` it cannot be trimmed; `copy` before a draft and go back to the copy instead."""

    is_trimmable = False
    max_size = None

    def __init__(self, conv_width=4):
        if not 1 <= int(conv_width) <= 8:
            raise ValueError(f"a convolution of 1 to 8 taps, not {conv_width}")
        self.conv_width = int(conv_width)
        self.offset = 0
        self._window = self._state = None
        self._made_on = {}

    # ---- protocol surface -------------------------------------------------
    @property
    def rope_offset(self):
        return self.offset

    def is_trimmable_after(self, positions):
        return False

    def trim(self, n):
        return 0

    def prepare(self, lengths=None):
        """Nothing to prepare: ragged calls say so themselves (`left_pad`, `lengths`)."""

    def finalize(self):
        """Nothing transient to clear."""

    def eval(self):
        L.check(L.load().kvhip_sync(_stream()))

    def _adopt(self, name, t):
        self._made_on[name] = None if t is None else _stream()
        setattr(self, name, t)

    def _held(self, name):
        """An array of the cache for a call on the current stream."""
        t = getattr(self, name)
        if t is not None and self._made_on[name] != _stream() and not torch.cuda.is_current_stream_capturing():
            t.record_stream(torch.cuda.current_stream())  # (its memory outlives what this stream still does with it)
        return t

    @property
    def window(self):
        return self._window

    @window.setter
    def window(self, t):
        if t is not None:
            if t.dim() != 3 or t.shape[1] != self.conv_width - 1 or t.dtype not in _DT:
                raise ValueError(f"a window is [B, {self.conv_width - 1}, C], not {t.dtype} {tuple(t.shape)}")
            _on_current_device(t)
            t = t.clone(memory_format=torch.contiguous_format)
        self._adopt("_window", t)

    @property
    def delta_state(self):
        return self._state

    @delta_state.setter
    def delta_state(self, t):
        if t is not None:
            if t.dim() != 4 or t.dtype != torch.float32:
                raise ValueError(f"a state is float32 [B, Hv, Dv, Dk], not {t.dtype} {tuple(t.shape)}")
            _on_current_device(t)
            t = t.clone(memory_format=torch.contiguous_format)
        self._adopt("_state", t)

    @property
    def state(self):
        """[window, delta_state], of those that there are."""
        return [t for t in (self._window, self._state) if t is not None]

    @state.setter
    def state(self, arrays):
        by_rank = {t.dim(): t for t in arrays}
        if len(by_rank) != len(arrays) or not set(by_rank) <= {3, 4}:
            raise ValueError("a state is a window [B, W - 1, C] and a delta state [B, Hv, Dv, Dk], or one of them")
        self.window, self.delta_state = by_rank.get(3), by_rank.get(4)

    def inner_state(self):
        return self.state

    @property
    def meta_state(self):
        return [str(self.conv_width), str(self.offset)]

    @meta_state.setter
    def meta_state(self, values):
        width, offset = (int(v) for v in values)
        if width != self.conv_width or offset < 0:
            raise ValueError(f"a cache of {self.conv_width} taps cannot take the metadata {list(values)}")
        self.offset = offset

    def copy(self):
        new = GatedDeltaCache(self.conv_width)
        new.offset, new.window, new.delta_state = self.offset, self._held("_window"), self._held("_state")
        return new

    def reorder(self, order, shared=0):
        """Sequence b becomes what sequence order[b] was (`beam_select`'s rows); an entry outside the batch leaves its own.  (A state has
        no positions that sequences could share: whatever `shared` says, all of it moves.)"""
        arrays = [t for t in (self._held("_window"), self._held("_state")) if t is not None and t.numel()]
        if not arrays:
            return
        rows = arrays[0].shape[0]
        if any(t.shape[0] != rows for t in arrays):
            raise ValueError("window and state hold different numbers of sequences")
        order = _order(order, rows)
        _on_current_device(*arrays)
        n = len(arrays)
        at = (C.c_void_p * n)(*[_ptr(t) for t in arrays])
        sizes = (C.c_size_t * n)(*[t.numel() // rows * t.element_size() for t in arrays])
        L.init()
        L.check(L.load().kvhip_reorder_rows(n, at, sizes, rows, _ptr(order), _stream()))

    # ---- the operators ------------------------------------------------------
    def convolve(self, x, weight, bias=None, silu=True, left_pad=None, lengths=None):
        """The short convolution of x [B, L, C] with weight [C, W] behind this cache's window, which moves on: [B, L, C]."""
        window = self._held("_window")
        if window is not None and left_pad is None and lengths is None:
            native, entry = L.native("convolve", "kvhip_short_convolution")  # (a step of the ordinary form, as one native call)
            out = native(entry, x, weight, bias, window, silu) if native else None
            if type(out) is int:
                L.check(out)
            if out is not None:
                return out
        if x.dim() != 3 or x.dtype not in _DT:
            raise ValueError(f"x is [B, L, C] in float16, bfloat16 or float32, not {x.dtype} {tuple(x.shape)}")
        B, n, c = x.shape
        W = self.conv_width
        if tuple(weight.shape) != (c, W) or weight.dtype != x.dtype:
            raise ValueError(f"weight is {x.dtype} {(c, W)}, not {weight.dtype} {tuple(weight.shape)}")
        if bias is not None and (tuple(bias.shape) != (c,) or bias.dtype != x.dtype):
            raise ValueError(f"bias is {x.dtype} {(c,)}, not {bias.dtype} {tuple(bias.shape)}")
        if window is not None and (tuple(window.shape) != (B, W - 1, c) or window.dtype != x.dtype):
            raise ValueError(f"x {x.dtype} {tuple(x.shape)} does not go with the window {window.dtype} {tuple(window.shape)}")
        _on_current_device(x, weight, bias, window)
        pad, ends = _per_sequence(left_pad, B, "left_pad"), _per_sequence(lengths, B, "lengths")
        x, weight, bias = _dense_rows(x), weight.contiguous(), None if bias is None else bias.contiguous()
        L.init()
        out = torch.empty((B, n, c), dtype=x.dtype, device=x.device)
        new = torch.empty((B, W - 1, c), dtype=x.dtype, device=x.device) if window is None else window
        if out.numel():
            L.check(L.load().kvhip_short_convolution(
                _ptr(x), x.stride(0), x.stride(1), _ptr(weight), None if bias is None else _ptr(bias), B, n, c, W, _DT[x.dtype],
                int(bool(silu)), None if pad is None else _ptr(pad), None if ends is None else _ptr(ends),
                None if window is None else _ptr(window), _ptr(new), _ptr(out), _stream()))
        elif window is None:
            return out
        if window is None:
            self._adopt("_window", new)
        return out

    def update(self, q, k, v, a, b, a_log=None, dt_bias=None, scale=None, norm_eps=1e-6, left_pad=None, lengths=None):
        """The gated delta rule over q, k [B, L, Hk, Dk] and v [B, L, Hv, Dv] from this cache's state on, which moves on: [B, L, Hv, Dv].
        a, b [B, L, Hv]: with a_log [Hv] what the decays exp(-exp(a_log) softplus(a + dt_bias)) and the rates sigmoid(b) come from, without
        it the decays' logarithms and the rates themselves.  `scale` defaults to Dk^-0.5; norm_eps 0 leaves q and k as they are."""
        state = self._held("_state")
        if state is not None and left_pad is None and lengths is None and a_log is not None and dt_bias is not None:
            native, entry, workspace = L.native("delta", "kvhip_gated_delta")  # (a step of the ordinary form, as one native call)
            out = native(entry, workspace, q, k, v, a, b, a_log, dt_bias, state, scale, norm_eps) if native else None
            if type(out) is int:
                L.check(out)
            if out is not None:
                self.offset += out.shape[1]
                return out
        if any(t.dim() != 4 for t in (q, k, v)) or q.shape != k.shape or q.shape[:2] != v.shape[:2]:
            raise ValueError(f"queries {tuple(q.shape)}, keys {tuple(k.shape)} and values {tuple(v.shape)} do not go together")
        B, n, Hk, Dk = k.shape
        Hv, Dv = v.shape[2:]
        if q.dtype not in _DT or k.dtype != q.dtype or v.dtype != q.dtype:
            raise TypeError(f"queries are {q.dtype}, keys {k.dtype}, values {v.dtype}")
        if tuple(a.shape) != (B, n, Hv) or tuple(b.shape) != (B, n, Hv) or a.dtype != b.dtype or a.dtype not in _DT:
            raise ValueError(f"a and b are {(B, n, Hv)} of one type, not {a.dtype} {tuple(a.shape)} and {b.dtype} {tuple(b.shape)}")
        for name, t in (("a_log", a_log), ("dt_bias", dt_bias)):
            if t is not None and tuple(t.shape) != (Hv,):
                raise ValueError(f"{name} is one number to each of {Hv} heads, not {tuple(t.shape)}")
        if dt_bias is not None and a_log is None:
            raise ValueError("dt_bias goes with a_log")
        if state is not None and tuple(state.shape) != (B, Hv, Dv, Dk):
            raise ValueError(f"keys {tuple(k.shape)} and values {tuple(v.shape)} do not go with the state {tuple(state.shape)}")
        _on_current_device(q, k, v, a, b, a_log, dt_bias, state)
        pad, ends = _per_sequence(left_pad, B, "left_pad"), _per_sequence(lengths, B, "lengths")
        q, k, v, a, b = (_dense_rows(t) for t in (q, k, v, a, b))
        a_log, dt_bias = (None if t is None else t.to(torch.float32).contiguous() for t in (a_log, dt_bias))
        L.init()
        out = torch.empty((B, n, Hv, Dv), dtype=v.dtype, device=v.device)
        if not out.numel():
            return out
        new = torch.empty((B, Hv, Dv, Dk), dtype=torch.float32, device=v.device) if state is None else state
        x = L.GatedDelta(
            q=_ptr(q), k=_ptr(k), v=_ptr(v), a=_ptr(a), b=_ptr(b), q_stride_b=q.stride(0), q_stride_l=q.stride(1), k_stride_b=k.stride(0),
            k_stride_l=k.stride(1), v_stride_b=v.stride(0), v_stride_l=v.stride(1), a_stride_b=a.stride(0), a_stride_l=a.stride(1),
            b_stride_b=b.stride(0), b_stride_l=b.stride(1), a_log=None if a_log is None else _ptr(a_log),
            dt_bias=None if dt_bias is None else _ptr(dt_bias), left_pad=None if pad is None else _ptr(pad),
            lengths=None if ends is None else _ptr(ends), state_in=None if state is None else _ptr(state), state_out=_ptr(new), out=_ptr(out),
            B=B, L=n, Hk=Hk, Hv=Hv, Dk=Dk, Dv=Dv, dtype=_DT[q.dtype], gate_dtype=_DT[a.dtype],
            scale=float(Dk ** -0.5 if scale is None else scale), norm_eps=float(norm_eps))
        lib = L.load()
        need = lib.kvhip_gated_delta_workspace(C.byref(x))
        scratch = torch.empty(need, dtype=torch.uint8, device=v.device) if need else None
        L.check(lib.kvhip_gated_delta(C.byref(x), None if scratch is None else _ptr(scratch), need, _stream()))
        if state is None:
            self._adopt("_state", new)
        self.offset += n
        return out


def causal_convolution(x, weight, cache: GatedDeltaCache, bias=None, silu=True, left_pad=None, lengths=None):
    """`GatedDeltaCache.convolve`: a gated delta layer's short convolution, its window kept in `cache`."""
    return cache.convolve(x, weight, bias, silu, left_pad, lengths)


def gated_delta_update(q, k, v, a, b, a_log, dt_bias, cache: GatedDeltaCache, scale=None, norm_eps=1e-6, left_pad=None, lengths=None):
    """`gatedDeltaUpdate` (GatedDelta.swift:112) over `cache`: `GatedDeltaCache.update`."""
    return cache.update(q, k, v, a, b, a_log, dt_bias, scale, norm_eps, left_pad, lengths)
