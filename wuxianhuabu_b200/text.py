"""The text side over libwx: what the layers of a decoder-only text model need between their
linears to make the hidden states that ``H3TextRefiner`` and ``H3DiT.step`` take (the reference
runs its text encoder once per generation, model/minimax h3/H3TextEncoder.swift).

* ``RopeTable``        — rotary positions of a token stream (interleaved or half layout, part of
  the head, scaled for long contexts, one or several position axes), with norms of the q and k heads
* ``PagePool``         — the pages of a cache dealt out to sequences, and a step's positions, slots
  and lengths, made on the device
* ``PagedKVCache``     — a paged K/V cache, quantised as it is written, read back on demand
* ``prompt_attention`` — whole prompts: causal, grouped heads, packed sequences
* ``paged_attention``  — new tokens (one per sequence or a chunk) over the cache
* ``prefix_attention`` — the same where all sequences stand behind one cached prefix

Tensors are torch CUDA tensors used as device buffers; calls are ordered on torch's current
stream, do not synchronise, and may be captured in CUDA graphs (whose replays must not overlap
one another: they share the context's captured scratch). q, k and v are [tokens, heads, head_dim] bf16 with contiguous
heads; the stride between tokens is free, so slices of a packed q|k|v projection need no copy.
Errors raise ``WxError``; wrong values in device-side arguments (positions, slots, lengths,
block entries) are caught by the kernels and raise at the next ``Context.check_device``.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from ._lib import (KV_BF16, KV_E4M3, KV_INT8, ROPE_BY_PARTS, ROPE_LINEAR, ROPE_PLAIN, AttnDims, KvCache, Rope, RopeAxes,
                   WxError, check)
from .h3 import _need_bf16_cuda, _p, context

__all__ = ["RopeScaling", "RopeTable", "rope_axes", "PagePool", "StepPlan", "PagedKVCache", "prompt_attention",
           "paged_attention", "prefix_attention"]

_FORMATS = {"bf16": (KV_BF16, torch.bfloat16), "int8": (KV_INT8, torch.int8), "e4m3": (KV_E4M3, torch.float8_e4m3fn)}
_SCALINGS = {"none": ROPE_PLAIN, "linear": ROPE_LINEAR, "by_parts": ROPE_BY_PARTS}


def _invalid(msg: str) -> WxError:
    return WxError(_lib.WX_ERR_INVALID, msg)


def _need_ints(dtype: torch.dtype, n: Optional[int], what: str, t: torch.Tensor) -> int:
    """The device pointer of a contiguous integer tensor of n entries."""
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise _invalid(f"{what} must be a contiguous CUDA {dtype} tensor, got {t.dtype} on {t.device}")
    if n is not None and t.numel() != n:
        raise _invalid(f"{what} must have {n} entries, got {t.numel()}")
    return t.data_ptr()


def _rows(t: torch.Tensor, what: str) -> tuple[int, int, int, int]:
    """tokens, heads, head_dim and the token stride of a [tokens, heads, head_dim] tensor."""
    if t.dtype != torch.bfloat16 or not t.is_cuda:
        _need_bf16_cuda(t)
    if t.dim() != 3:
        raise _invalid(f"{what} must be [tokens, heads, head_dim]")
    n, h, d = t.shape
    s0, s1, s2 = t.stride()
    if n and (s2 != 1 or (h > 1 and s1 != d)):
        raise _invalid(f"{what} must have contiguous heads")
    return n, h, d, s0 if n > 1 else max(s0, h * d)


def _same_device(*ts: torch.Tensor) -> int:
    dev = ts[0].get_device()
    for t in ts:
        if t.get_device() != dev:
            raise _invalid(f"tensors on {ts[0].device} and {t.device}")
    return dev


def _out_rows(like: torch.Tensor, n: int, h: int, d: int, out: Optional[torch.Tensor], msg: str):
    """The output tensor (a new one without ``out``) and its token stride."""
    if out is None:
        return torch.empty_like(like), h * d  # (rows of contiguous heads: never anything but contiguous)
    if out.shape != like.shape:
        raise _invalid(msg)
    return out, _rows(out, "out")[3]


@dataclass
class RopeScaling:
    """How the frequencies of a longer context follow from the original ones: "none", "linear"
    (all divided by ``factor``) or "by_parts" (pairs that turn at most ``low`` times over
    ``original_positions`` are divided, those that turn at least ``high`` times are kept, linear
    in between). ``magnitude`` multiplies cos and sin."""
    kind: str = "none"
    factor: float = 1.0
    original_positions: float = 8192.0
    low: float = 1.0
    high: float = 4.0
    magnitude: float = 1.0


def rope_axes(shares: Sequence[int], dealt: bool = False) -> tuple[int, ...]:
    """The position axis of each pair, from the pairs that each axis has: in runs (axis 0's pairs first),
    or ``dealt`` out in turn while an axis has pairs left."""
    left = [int(n) for n in shares]
    if not 1 <= len(left) <= 4 or min(left) < 0:
        raise _invalid("shares must be the pairs of 1 to 4 axes")
    if not dealt:
        return tuple(a for a, n in enumerate(left) for _ in range(n))
    return tuple(a for turn in range(max(left)) for a, n in enumerate(left) if turn < n)


class _Described:
    """An object whose tensors the library is told of in a struct, ``_desc``. It is made at the first call
    that needs it, checked, and made again after an attribute was assigned; copies make their own."""

    def __getattr__(self, name: str):  # (only where there is no such attribute)
        if name != "_desc":
            raise AttributeError(name)
        self.__dict__["_desc"] = made = C.byref(self._describe())
        return made

    def __setattr__(self, name: str, value) -> None:
        self.__dict__.pop("_desc", None)
        object.__setattr__(self, name, value)

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k != "_desc"}


def _head_norm(w: Optional[torch.Tensor], d: int, what: str) -> Optional[int]:
    """The device pointer of a head norm's weight [head_dim]."""
    if w is None:
        return None
    _need_bf16_cuda(w)
    if w.numel() != d or not w.is_contiguous():
        raise _invalid(f"{what} must be a contiguous [head_dim] tensor")
    return w.data_ptr()


class RopeTable(_Described):
    """cos / sin of every position, fp32 [positions, rot / 2] (angles in 64 bits). With ``axes`` (one
    axis a pair, ``rope_axes``) a token has a position on each axis: positions are [axes, tokens]
    then, instead of [tokens]; text's, the same on every axis, may be an expanded row."""
    axes: Optional[tuple] = None

    def __init__(self, rot: int, positions: int, base: float = 10000.0, interleaved: bool = False,
                 scaling: Optional[RopeScaling] = None, device: Optional[int] = None,
                 axes: Optional[Sequence[int]] = None):
        s = scaling or RopeScaling()
        if s.kind not in _SCALINGS:
            raise _invalid(f"unknown rope scaling {s.kind!r}")
        if rot <= 0 or rot % 8 or rot > 128 or positions <= 0:
            raise _invalid("rot must be a multiple of 8 in 8..128 and positions positive")
        inv = np.zeros(rot // 2, dtype=np.float64)
        check(_lib.load().wx_rope_inv_freq(rot, float(base), _SCALINGS[s.kind], float(s.factor),
                                           float(s.original_positions), float(s.low), float(s.high), inv.ctypes.data))
        ctx = context(device)
        dev = torch.device("cuda", ctx.device)
        self.inv_freq = inv
        self.interleaved = interleaved
        self.axes = axes
        self.cos = torch.empty((positions, rot // 2), dtype=torch.float32, device=dev)
        self.sin = torch.empty_like(self.cos)
        self._desc  # (checked)
        ctx.call("wx_rope_table", inv.ctypes.data, rot // 2, positions, float(s.magnitude), _p(self.cos), _p(self.sin))

    @classmethod
    def from_tables(cls, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool = False,
                    axes: Optional[Sequence[int]] = None) -> "RopeTable":
        """Over tables that exist already (not copied)."""
        self = cls.__new__(cls)
        self.cos, self.sin, self.interleaved, self.inv_freq = cos, sin, interleaved, None
        self.axes = axes
        self._desc  # (checked)
        return self

    def _describe(self) -> Rope:
        cos, sin = self.cos, self.sin
        for t in (cos, sin):
            if not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous() or t.dim() != 2:
                raise _invalid("cos and sin must be contiguous CUDA fp32 [positions, rot / 2]")
        if cos.shape != sin.shape:
            raise _invalid("cos and sin must have one shape")
        _same_device(cos, sin)
        n, half = cos.shape
        if self.axes is not None and len(self.axes) != half:
            raise _invalid(f"axes must have an entry for each of the {half} pairs, got {len(self.axes)}")
        return Rope(_p(cos), _p(sin), n, 2 * half, int(self.interleaved))

    def __setattr__(self, name: str, value) -> None:
        if name == "axes" and value is not None:
            value = tuple(int(a) for a in value)
            if not value or len(value) > 64 or min(value) < 0 or max(value) > 3:
                raise _invalid("axes must name one of 4 axes for each pair")
            # (as the library takes it, but for the positions' stride, which is the call's)
            object.__setattr__(self, "_axes_as_bytes", bytes(RopeAxes(max(value) + 1, (C.c_uint8 * 64)(*value), 0)))
        super().__setattr__(name, value)

    def _at(self, positions: torch.Tensor, n: int):
        """The device pointer of positions, and the axes of this call (None: one position a token)."""
        if self.axes is None:
            return _need_ints(torch.int32, n, "positions", positions), None
        axes = RopeAxes.from_buffer_copy(self._axes_as_bytes)
        if not positions.is_cuda or positions.dtype != torch.int32 or positions.dim() != 2 or \
                positions.shape[0] < axes.n_axes or positions.shape[1] != n:
            raise _invalid(f"positions must be a CUDA int32 [axes, tokens] tensor of {axes.n_axes} axes and {n} tokens")
        axes.position_stride, inner = positions.stride()
        if n > 1 and inner != 1:
            raise _invalid("positions of an axis must be contiguous")
        return positions.data_ptr(), C.byref(axes)

    def apply_qk(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, q_norm: Optional[torch.Tensor] = None,
                 k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
        """q and k of the same tokens, each head normalised by its root mean square and q_norm / k_norm
        [head_dim] where given, and turned, in one launch; outputs may be the inputs."""
        n, hq, d, qs = _rows(q, "q")
        nk, hk, dk, ks = _rows(k, "k")
        if (nk, dk) != (n, d):
            raise _invalid("k must have q's tokens and head_dim")
        qw, kw = _head_norm(q_norm, d, "q_norm"), _head_norm(k_norm, d, "k_norm")
        at, axes = self._at(positions, n)
        qo, qos = _out_rows(q, n, hq, d, q_out, "q_out must have q's shape")
        ko, kos = _out_rows(k, n, hk, d, k_out, "k_out must have k's shape")
        dev = _same_device(q, k, positions, qo, ko, self.cos, *(w for w in (q_norm, k_norm) if w is not None))
        context(dev).call("wx_norm_rope_apply", self._desc, axes, at, q.data_ptr(), qs, hq, qw, k.data_ptr(), ks, hk, kw,
                          eps, n, d, qo.data_ptr(), qos, ko.data_ptr(), kos)
        return qo, ko

    def apply(self, x: torch.Tensor, positions: torch.Tensor, out: Optional[torch.Tensor] = None,
              norm: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
        """x [tokens, heads, head_dim] with token t turned by positions[t] (int32); ``out`` may be x. With
        ``norm`` [head_dim] each head is normalised first, as in ``apply_qk``."""
        n, h, d, stride = _rows(x, "x")
        if self.axes is not None or norm is not None:
            weight = _head_norm(norm, d, "norm")
            at, axes = self._at(positions, n)
            o, ostride = _out_rows(x, n, h, d, out, "out must have x's shape")
            context(_same_device(x, positions, o, self.cos, x if norm is None else norm)).call(
                "wx_norm_rope_apply", self._desc, axes, at, x.data_ptr(), stride, h, weight, None, 0, 0, None, eps, n, d,
                o.data_ptr(), ostride, None, 0)
            return o
        at = _need_ints(torch.int32, n, "positions", positions)
        o, ostride = _out_rows(x, n, h, d, out, "out must have x's shape")
        context(_same_device(x, positions, o, self.cos)).call(
            "wx_rope_apply", self._desc, at, x.data_ptr(), stride, n, h, d, o.data_ptr(), ostride)
        return o


@dataclass
class StepPlan:
    """A step's arrays on the device: positions [tokens] int32, slots [tokens] int64 (-1: no token),
    cu_seqlens [batch + 1], kv_lens [batch] and the free list's height [1] int32."""
    positions: torch.Tensor
    slots: torch.Tensor
    cu_seqlens: torch.Tensor
    kv_lens: torch.Tensor
    taken: torch.Tensor


class PagePool(_Described):
    """The pages of a cache (or of several of one geometry) dealt out to the sequences of a batch, on the
    device. ``free`` [pages] int32 is a stack that grows downwards: its entries from ``taken`` [1] on
    are free. Sequence b has ``lens``[b] tokens in the pages ``table``[b] ([batch, blocks], the
    ``block_table`` of ``paged_attention``)."""

    def __init__(self, pages: int, page_size: int, batch: int, blocks: int, device: Optional[int] = None):
        dev = torch.device("cuda", context(device).device)
        if min(pages, blocks) <= 0 or batch < 0:
            raise _invalid("pages and blocks must be positive, batch not negative")
        self.page_size = page_size
        self.free = torch.arange(pages, dtype=torch.int32, device=dev)
        self.taken = torch.zeros(1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.table = torch.full((batch, blocks), -1, dtype=torch.int32, device=dev)
        self._desc  # (checked)

    @classmethod
    def from_tensors(cls, page_size: int, free: torch.Tensor, taken: torch.Tensor, lens: torch.Tensor,
                     table: torch.Tensor) -> "PagePool":
        """Over arrays that exist already (not copied)."""
        self = cls.__new__(cls)
        self.page_size, self.free, self.taken, self.lens, self.table = page_size, free, taken, lens, table
        self._desc  # (checked)
        return self

    def _describe(self) -> _lib.PagePool:
        batch = self.lens.numel()
        free = _need_ints(torch.int32, None, "free", self.free)
        taken = _need_ints(torch.int32, 1, "taken", self.taken)
        lens = _need_ints(torch.int32, None, "lens", self.lens)
        table = _need_ints(torch.int32, None, "table", self.table)
        if self.table.dim() != 2 or self.table.shape[0] != batch:
            raise _invalid("table must be [batch, blocks]")
        _same_device(self.free, self.taken, self.lens, self.table)
        return _lib.PagePool(free, taken, lens, table, self.free.numel(), self.table.shape[1], batch, self.page_size)

    def plan(self, new: torch.Tensor, tokens: int, keep: Optional[torch.Tensor] = None, first_position: int = 0,
             commit: bool = True) -> StepPlan:
        """One step: sequence b keeps its first keep[b] tokens (all without ``keep``) and gets new[b] more
        (int32, on the device), pages being given back and taken as that needs: an ended sequence keeps 0,
        rejected drafts are not kept. ``tokens``: entries of positions and slots, as many as the new tokens
        or more. Positions count from ``first_position`` (tokens that stand before every sequence). With
        ``commit`` lens and taken are brought up to date, and are the plan's kv_lens and taken; without, the
        plan has its own and the step can be planned again. A step that does not fit raises at the next
        ``check_device`` and changes nothing (no slots, no new tokens)."""
        batch = self.lens.numel()
        add = _need_ints(torch.int32, batch, "new", new)
        kept = None if keep is None else _need_ints(torch.int32, batch, "keep", keep)
        if not 0 <= tokens < _INT32 or not 0 <= first_position < _INT32:
            raise _invalid("tokens and first_position must be in 0..2^31 - 1")
        dev = _same_device(self.lens, new, new if keep is None else keep)
        desc = self._desc
        slots = new.new_empty(tokens, dtype=torch.int64)
        # (one allocation, cut up: each is a microsecond and more)
        if commit:
            pos, cu = new.new_empty(tokens + batch + 1).split_with_sizes((tokens, batch + 1))
            lens, taken = self.lens, self.taken
        else:
            pos, cu, lens, taken = new.new_empty(tokens + 2 * batch + 2).split_with_sizes((tokens, batch + 1, batch, 1))
        context(dev).call("wx_page_plan", desc, kept, add, tokens, first_position, pos.data_ptr(), slots.data_ptr(),
                          cu.data_ptr(), lens.data_ptr(), taken.data_ptr())
        return StepPlan(pos, slots, cu, lens, taken)


class PagedKVCache(_Described):
    """Pages of ``page_size`` tokens, [pages, kv_heads, page_size, head_dim] each for k and v in
    ``fmt`` ("bf16", "int8", "e4m3"); the 8-bit formats hold one fp32 scale per (token, head)
    row in [pages, kv_heads, page_size]. A slot is page * page_size + offset (int64)."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, fmt: str = "bf16",
                 device: Optional[int] = None):
        if fmt not in _FORMATS:
            raise _invalid(f"unknown cache format {fmt!r}")
        dev = torch.device("cuda", context(device).device)
        shape = (pages, kv_heads, page_size, head_dim)
        kind = _FORMATS[fmt][1]
        self.k, self.v = (torch.zeros(shape, dtype=kind if fmt == "bf16" else torch.uint8, device=dev).view(kind)
                          for _ in range(2))
        self.k_scale, self.v_scale = (None, None) if fmt == "bf16" else \
            (torch.zeros(shape[:3], dtype=torch.float32, device=dev) for _ in range(2))
        self._desc  # (checked)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                     v_scale: Optional[torch.Tensor] = None) -> "PagedKVCache":
        """Over buffers that exist already (not copied)."""
        self = cls.__new__(cls)
        self.k, self.v = k, v
        self.k_scale, self.v_scale = (k_scale, v_scale) if k.dtype != torch.bfloat16 else (None, None)
        self._desc  # (checked)
        return self

    def __setattr__(self, name: str, value) -> None:
        if name == "k":  # format and geometry are those of k
            fmt = next((f for f, (_, d) in _FORMATS.items() if d == value.dtype), None)
            if fmt is None or value.dim() != 4:
                raise _invalid("k must be [pages, kv_heads, page_size, head_dim] of a cache format")
            self.fmt = fmt
            self.pages, self.kv_heads, self.page_size, self.head_dim = value.shape
        super().__setattr__(name, value)

    def _describe(self) -> KvCache:
        k, v, scales = self.k, self.v, (self.k_scale, self.v_scale)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise _invalid("k and v must be [pages, kv_heads, page_size, head_dim] of one cache format")
        if not (k.is_cuda and k.is_contiguous() and v.is_contiguous()):
            raise _invalid("k and v must be contiguous CUDA tensors")
        _same_device(k, v)
        if self.fmt == "bf16":
            scales = None, None
        else:
            for s in scales:
                if s is None or s.dtype != torch.float32 or s.shape != k.shape[:3] or not s.is_contiguous():
                    raise _invalid("an 8-bit cache needs contiguous fp32 scales [pages, kv_heads, page_size]")
            _same_device(k, *scales)
        return KvCache(_p(k), _p(v), _p(scales[0]), _p(scales[1]), self.pages, self.page_size, self.kv_heads,
                       self.head_dim, _FORMATS[self.fmt][0])

    def _kv(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor):
        n, h, d, ks = _rows(k, "k")
        nv, hv, dv, vs = _rows(v, "v")
        if (n, h, d) != (nv, hv, dv) or (h, d) != (self.kv_heads, self.head_dim):
            raise _invalid("k and v must be [tokens, kv_heads, head_dim] of the cache")
        return n, ks, vs, _need_ints(torch.int64, n, "slots", slots)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Write k and v of each token to its slot (< 0: skipped), quantised to the format."""
        n, ks, vs, at = self._kv(k, v, slots)
        context(_same_device(self.k, k, v, slots)).call("wx_kv_append", self._desc, k.data_ptr(), ks, v.data_ptr(), vs,
                                                        n, at)

    def append_roped(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, rope: RopeTable,
                     positions: torch.Tensor, q_out: Optional[torch.Tensor] = None,
                     q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                     eps: float = 1e-6) -> torch.Tensor:
        """``rope.apply`` of q (returned) and k, and ``append`` of k and v, in one launch; with ``q_norm`` /
        ``k_norm`` [head_dim] the heads are normalised first, as in ``rope.apply_qk``."""
        n, ks, vs, at = self._kv(k, v, slots)
        nq, hq, dq, qs = _rows(q, "q")
        if (nq, dq) != (n, self.head_dim):
            raise _invalid("q must be [tokens, q_heads, head_dim] of k's tokens")
        o, ostride = _out_rows(q, n, hq, dq, q_out, "q_out must have q's shape")
        if rope.axes is not None or q_norm is not None or k_norm is not None:
            qw, kw = _head_norm(q_norm, dq, "q_norm"), _head_norm(k_norm, dq, "k_norm")
            pos, axes = rope._at(positions, n)
            dev = _same_device(self.k, q, k, v, slots, positions, o, rope.cos,
                               *(w for w in (q_norm, k_norm) if w is not None))
            context(dev).call("wx_norm_rope_kv_append", rope._desc, axes, pos, q.data_ptr(), qs, hq, qw, kw, eps,
                              self._desc, k.data_ptr(), ks, v.data_ptr(), vs, n, at, o.data_ptr(), ostride)
            return o
        pos = _need_ints(torch.int32, n, "positions", positions)
        context(_same_device(self.k, q, k, v, slots, positions, o, rope.cos)).call(
            "wx_rope_kv_append", rope._desc, pos, q.data_ptr(), qs, hq, self._desc, k.data_ptr(), ks, v.data_ptr(), vs,
            n, at, o.data_ptr(), ostride)
        return o

    def read(self, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """k and v of the slots as bf16 [tokens, kv_heads, head_dim] (< 0: zeros)."""
        at = _need_ints(torch.int64, None, "slots", slots)
        n, h, d = slots.numel(), self.kv_heads, self.head_dim
        k = slots.new_empty((n, h, d), dtype=torch.bfloat16)
        v = torch.empty_like(k)
        context(_same_device(self.k, slots)).call("wx_kv_read", self._desc, at, n, k.data_ptr(), v.data_ptr(), h * d)
        return k, v


def _attn_out(q: torch.Tensor, out: Optional[torch.Tensor], return_lse: bool):
    n, h, d, stride = _rows(q, "q")
    o, ostride = _out_rows(q, n, h, d, out, "out must have q's shape")
    lse = q.new_empty((n, h), dtype=torch.float32) if return_lse else None
    return n, h, d, stride, o, ostride, lse


def _batch_of(cu_seqlens: torch.Tensor) -> int:
    batch = cu_seqlens.numel() - 1
    if batch < 0:
        raise _invalid("cu_seqlens needs at least one entry")
    return batch


_INT32 = 1 << 31


def _dims(n: int, batch: int, max_len: int, h: int, hk: int, d: int, causal: bool, window: int,
          scale: Optional[float]):
    if window >= _INT32 or window < 0 or max_len >= _INT32 or max_len < 0:
        # (beyond 32 bits, the nearest int32: a struct's field would keep the low bits)
        window, max_len = (max(-_INT32, min(x, _INT32 - 1)) for x in (window, max_len))
    return C.byref(AttnDims(n, batch, max_len, h, hk, d, causal, window, d ** -0.5 if scale is None else scale))


def _first_keys(sinks: int) -> int:
    if sinks < 0:
        raise _invalid("sinks must not be negative")
    return min(sinks, _INT32 - 1)  # (more than any sequence has)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_len: int,
                     scale: Optional[float] = None, causal: bool = True, window: int = 0,
                     cu_seqlens_k: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                     return_lse: bool = False, sinks: int = 0):
    """Packed prompts: sequence b is rows cu_seqlens[b]..cu_seqlens[b + 1] (int32, on the device)
    of q [total, q_heads, head_dim] and k, v [total, kv_heads, head_dim] (of cu_seqlens_k for k
    and v where they differ, the last query row standing at the last key). ``max_len``: the
    longest query length. A ``window`` leaves a row the last ``window`` keys up to its own, and with
    ``sinks`` the sequence's first ``sinks`` keys too. Returns out [total, q_heads, head_dim], with
    ``return_lse`` also the log-sum-exp [total, q_heads] fp32."""
    n, h, d, qs, o, os_, lse = _attn_out(q, out, return_lse)
    nk, hk, dk, ks = _rows(k, "k")
    nv, hv, dv, vs = _rows(v, "v")
    if (nk, hk, dk) != (nv, hv, dv) or dk != d:
        raise _invalid("k and v must be [tokens, kv_heads, head_dim] of q's head_dim")
    batch = _batch_of(cu_seqlens)
    cu = _need_ints(torch.int32, None, "cu_seqlens", cu_seqlens)
    cu_k = None if cu_seqlens_k is None else _need_ints(torch.int32, batch + 1, "cu_seqlens_k", cu_seqlens_k)
    dev = _same_device(q, k, v, cu_seqlens, o, cu_seqlens if cu_k is None else cu_seqlens_k)
    dims = _dims(n, batch, max_len, h, hk, d, causal, window, scale)
    args = q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, nk, cu, cu_k, o.data_ptr(), os_, _p(lse)
    if sinks:
        context(dev).call("wx_prompt_attention_sinks", dims, _first_keys(sinks), *args)
    else:
        context(dev).call("wx_prompt_attention", dims, *args)
    return (o, lse) if return_lse else o


def paged_attention(q: torch.Tensor, cache: PagedKVCache, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
                    block_table: torch.Tensor, max_len: int, scale: Optional[float] = None, causal: bool = True,
                    window: int = 0, out: Optional[torch.Tensor] = None, return_lse: bool = False, sinks: int = 0):
    """New tokens over the cache that already holds them: query rows cu_seqlens[b]..[b + 1] of q
    are the last of the kv_lens[b] tokens cached in pages block_table[b] (int32, [batch, blocks];
    entries beyond the length are not read). ``max_len``: the longest query length; ``window`` and
    ``sinks`` as in ``prompt_attention``."""
    n, h, d, qs, o, os_, lse = _attn_out(q, out, return_lse)
    batch = _batch_of(cu_seqlens)
    cu = _need_ints(torch.int32, None, "cu_seqlens", cu_seqlens)
    lens = _need_ints(torch.int32, batch, "kv_lens", kv_lens)
    table = _need_ints(torch.int32, None, "block_table", block_table)
    if block_table.dim() != 2 or block_table.shape[0] != batch:
        raise _invalid("block_table must be [batch, blocks]")
    if d != cache.head_dim:
        raise _invalid("q must have the cache's head_dim")
    dev = _same_device(q, cache.k, cu_seqlens, kv_lens, block_table, o)
    dims = _dims(n, batch, max_len, h, cache.kv_heads, d, causal, window, scale)
    args = q.data_ptr(), qs, cache._desc, cu, lens, table, block_table.shape[1], o.data_ptr(), os_, _p(lse)
    if sinks:
        context(dev).call("wx_paged_attention_sinks", dims, _first_keys(sinks), *args)
    else:
        context(dev).call("wx_paged_attention", dims, *args)
    return (o, lse) if return_lse else o


def prefix_attention(q: torch.Tensor, cache: PagedKVCache, prefix_blocks: torch.Tensor, prefix_len: int,
                     cu_seqlens: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, max_len: int,
                     scale: Optional[float] = None, causal: bool = True, out: Optional[torch.Tensor] = None,
                     return_lse: bool = False):
    """``paged_attention`` where every sequence stands behind the same ``prefix_len`` cached tokens, in pages
    prefix_blocks (int32): these are walked once for the whole batch and seen by every row. kv_lens and
    block_table are of each sequence's own tokens behind them; block_table (one column at least) may be columns
    of a larger table (``prefix_attention(q, cache, table[0, :n], n * page_size, cu, lens - n * page_size,
    table[:, n:], ...)``) or one row expanded to all sequences."""
    n, h, d, qs, o, os_, lse = _attn_out(q, out, return_lse)
    batch = _batch_of(cu_seqlens)
    cu = _need_ints(torch.int32, None, "cu_seqlens", cu_seqlens)
    lens = _need_ints(torch.int32, batch, "kv_lens", kv_lens)
    prefix = _need_ints(torch.int32, None, "prefix_blocks", prefix_blocks)
    if not 0 <= prefix_len <= prefix_blocks.numel() * cache.page_size:
        raise _invalid(f"prefix_len must be in 0..{prefix_blocks.numel() * cache.page_size} (prefix_blocks' tokens)")
    if block_table.dim() != 2 or block_table.shape[0] != batch or not block_table.is_cuda or \
            block_table.dtype != torch.int32:
        raise _invalid("block_table must be a CUDA int32 [batch, blocks] tensor")
    blocks = block_table.shape[1]
    stride, inner = block_table.stride()
    if (blocks > 1 and inner != 1) or (batch > 1 and 0 < stride < blocks):
        raise _invalid("block_table must have contiguous rows, apart or one for all sequences")
    stride = stride if batch > 1 else blocks
    if d != cache.head_dim:
        raise _invalid("q must have the cache's head_dim")
    dev = _same_device(q, cache.k, cu_seqlens, kv_lens, block_table, prefix_blocks, o)
    context(dev).call("wx_prefix_attention", _dims(n, batch, max_len, h, cache.kv_heads, d, causal, 0, scale),
                      q.data_ptr(), qs, cache._desc, prefix, prefix_len, cu, lens, block_table.data_ptr(), blocks,
                      stride, o.data_ptr(), os_, _p(lse))
    return (o, lse) if return_lse else o
