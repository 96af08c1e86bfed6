"""The text side over libwx: what the layers of a decoder-only text model need between their
linears to make the hidden states that ``H3TextRefiner`` and ``H3DiT.step`` take (the reference
runs its text encoder once per generation, model/minimax h3/H3TextEncoder.swift).

* ``RopeTable``        — rotary positions of a token stream (interleaved or half layout, part of
  the head, scaled for long contexts)
* ``PagedKVCache``     — a paged K/V cache, quantised as it is written, read back on demand
* ``prompt_attention`` — whole prompts: causal, grouped heads, packed sequences
* ``paged_attention``  — new tokens (one per sequence or a chunk) over the cache

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
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._lib import (KV_BF16, KV_E4M3, KV_INT8, ROPE_BY_PARTS, ROPE_LINEAR, ROPE_PLAIN, AttnDims, KvCache, Rope, WxError,
                   check)
from .h3 import _need_bf16_cuda, _p, context

__all__ = ["RopeScaling", "RopeTable", "PagedKVCache", "prompt_attention", "paged_attention"]

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


class RopeTable(_Described):
    """cos / sin of every position, fp32 [positions, rot / 2] (angles in 64 bits)."""

    def __init__(self, rot: int, positions: int, base: float = 10000.0, interleaved: bool = False,
                 scaling: Optional[RopeScaling] = None, device: Optional[int] = None):
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
        self.cos = torch.empty((positions, rot // 2), dtype=torch.float32, device=dev)
        self.sin = torch.empty_like(self.cos)
        ctx.call("wx_rope_table", inv.ctypes.data, rot // 2, positions, float(s.magnitude), _p(self.cos), _p(self.sin))

    @classmethod
    def from_tables(cls, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool = False) -> "RopeTable":
        """Over tables that exist already (not copied)."""
        self = cls.__new__(cls)
        self.cos, self.sin, self.interleaved, self.inv_freq = cos, sin, interleaved, None
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
        return Rope(_p(cos), _p(sin), n, 2 * half, int(self.interleaved))

    def apply(self, x: torch.Tensor, positions: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [tokens, heads, head_dim] with token t turned by positions[t] (int32); ``out`` may be x."""
        n, h, d, stride = _rows(x, "x")
        at = _need_ints(torch.int32, n, "positions", positions)
        o, ostride = _out_rows(x, n, h, d, out, "out must have x's shape")
        context(_same_device(x, positions, o, self.cos)).call(
            "wx_rope_apply", self._desc, at, x.data_ptr(), stride, n, h, d, o.data_ptr(), ostride)
        return o


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
                     positions: torch.Tensor, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``rope.apply`` of q (returned) and k, and ``append`` of k and v, in one launch."""
        n, ks, vs, at = self._kv(k, v, slots)
        nq, hq, dq, qs = _rows(q, "q")
        if (nq, dq) != (n, self.head_dim):
            raise _invalid("q must be [tokens, q_heads, head_dim] of k's tokens")
        pos = _need_ints(torch.int32, n, "positions", positions)
        o, ostride = _out_rows(q, n, hq, dq, q_out, "q_out must have q's shape")
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


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_len: int,
                     scale: Optional[float] = None, causal: bool = True, window: int = 0,
                     cu_seqlens_k: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                     return_lse: bool = False):
    """Packed prompts: sequence b is rows cu_seqlens[b]..cu_seqlens[b + 1] (int32, on the device)
    of q [total, q_heads, head_dim] and k, v [total, kv_heads, head_dim] (of cu_seqlens_k for k
    and v where they differ, the last query row standing at the last key). ``max_len``: the
    longest query length. Returns out [total, q_heads, head_dim], with ``return_lse`` also the
    log-sum-exp [total, q_heads] fp32."""
    n, h, d, qs, o, os_, lse = _attn_out(q, out, return_lse)
    nk, hk, dk, ks = _rows(k, "k")
    nv, hv, dv, vs = _rows(v, "v")
    if (nk, hk, dk) != (nv, hv, dv) or dk != d:
        raise _invalid("k and v must be [tokens, kv_heads, head_dim] of q's head_dim")
    batch = _batch_of(cu_seqlens)
    cu = _need_ints(torch.int32, None, "cu_seqlens", cu_seqlens)
    cu_k = None if cu_seqlens_k is None else _need_ints(torch.int32, batch + 1, "cu_seqlens_k", cu_seqlens_k)
    dev = _same_device(q, k, v, cu_seqlens, o, cu_seqlens if cu_k is None else cu_seqlens_k)
    context(dev).call("wx_prompt_attention", _dims(n, batch, max_len, h, hk, d, causal, window, scale), q.data_ptr(), qs,
                      k.data_ptr(), ks, v.data_ptr(), vs, nk, cu, cu_k, o.data_ptr(), os_, _p(lse))
    return (o, lse) if return_lse else o


def paged_attention(q: torch.Tensor, cache: PagedKVCache, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
                    block_table: torch.Tensor, max_len: int, scale: Optional[float] = None, causal: bool = True,
                    window: int = 0, out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """New tokens over the cache that already holds them: query rows cu_seqlens[b]..[b + 1] of q
    are the last of the kv_lens[b] tokens cached in pages block_table[b] (int32, [batch, blocks];
    entries beyond the length are not read). ``max_len``: the longest query length."""
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
    context(dev).call("wx_paged_attention", _dims(n, batch, max_len, h, cache.kv_heads, d, causal, window, scale),
                      q.data_ptr(), qs, cache._desc, cu, lens, table, block_table.shape[1], o.data_ptr(), os_, _p(lse))
    return (o, lse) if return_lse else o
