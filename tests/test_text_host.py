"""Host side of the text operators: rotary frequencies against their definition, and refusals that
need no GPU.

The frequencies are a power and, scaled, a few products in double precision: a relative error of a
few 2^-53, to which pow adds under 2^-51; 1e-13 is 900 times 2^-53."""
import math

import numpy as np
import pytest

from wuxianhuabu_b200 import _lib


def _inv_freq(rot, base, kind, factor=1.0, original=8192.0, low=1.0, high=4.0):
    out = np.full(max(rot // 2, 1), -1.0)
    st = _lib.load().wx_rope_inv_freq(rot, base, kind, factor, original, low, high, out.ctypes.data)
    return st, out


def _expected(rot, base, kind, factor, original, low, high):
    want = []
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if kind == _lib.ROPE_LINEAR:
            f /= factor
        elif kind == _lib.ROPE_BY_PARTS:
            turns = original * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            f = (1 - keep) * f / factor + keep * f
        want.append(f)
    return np.array(want)


@pytest.mark.parametrize("rot", [8, 64, 96, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("kind,factor", [(_lib.ROPE_PLAIN, 1.0), (_lib.ROPE_LINEAR, 4.0), (_lib.ROPE_BY_PARTS, 8.0)])
def test_rope_inv_freq(rot, base, kind, factor):
    st, got = _inv_freq(rot, base, kind, factor)
    assert st == _lib.WX_OK
    want = _expected(rot, base, kind, factor, 8192.0, 1.0, 4.0)
    assert np.all(np.abs(got - want) <= 1e-13 * want)


def test_by_parts_keeps_and_divides():
    _, plain = _inv_freq(128, 10000.0, _lib.ROPE_PLAIN)
    _, parts = _inv_freq(128, 10000.0, _lib.ROPE_BY_PARTS, 8.0)
    assert parts[0] == plain[0]
    assert abs(parts[-1] * 8.0 / plain[-1] - 1) < 1e-13
    assert np.all((parts <= plain * (1 + 1e-15)) & (parts >= plain / 8 * (1 - 1e-13)))


@pytest.mark.parametrize("args", [
    (0, 10000.0, _lib.ROPE_PLAIN), (7, 10000.0, _lib.ROPE_PLAIN), (64, 0.0, _lib.ROPE_PLAIN),
    (64, math.nan, _lib.ROPE_PLAIN), (64, 10000.0, 17), (64, 10000.0, _lib.ROPE_LINEAR, 0.0),
    (64, 10000.0, _lib.ROPE_BY_PARTS, 8.0, 0.0), (64, 10000.0, _lib.ROPE_BY_PARTS, 8.0, 8192.0, 4.0, 1.0),
])
def test_rope_inv_freq_refusals(args):
    st, _ = _inv_freq(*args)
    assert st == _lib.WX_ERR_INVALID
    assert _lib.load().wx_rope_inv_freq(64, 10000.0, _lib.ROPE_PLAIN, 1.0, 8192.0, 1.0, 4.0, None) == _lib.WX_ERR_INVALID


def test_calls_without_a_context_are_refused():
    lib = _lib.load()
    assert lib.wx_rope_table(None, None, 32, 16, 1.0, None, None) == _lib.WX_ERR_INVALID
    assert lib.wx_rope_apply(None, None, None, None, 0, 0, 0, 0, None, 0) == _lib.WX_ERR_INVALID
    assert lib.wx_kv_append(None, None, None, 0, None, 0, 0, None) == _lib.WX_ERR_INVALID
    assert lib.wx_rope_kv_append(None, None, None, None, 0, 0, None, None, 0, None, 0, 0, None, None, 0) \
        == _lib.WX_ERR_INVALID
    assert lib.wx_kv_read(None, None, None, 0, None, None, 0) == _lib.WX_ERR_INVALID
    assert lib.wx_prompt_attention(None, None, None, 0, None, 0, None, 0, 0, None, None, None, 0, None) \
        == _lib.WX_ERR_INVALID
    assert lib.wx_paged_attention(None, None, None, 0, None, None, None, None, 0, None, 0, None) \
        == _lib.WX_ERR_INVALID


@pytest.mark.parametrize("make", [
    lambda t: t.RopeTable(12, 16), lambda t: t.RopeTable(256, 16), lambda t: t.RopeTable(64, 0),
    lambda t: t.RopeTable(64, 16, scaling=t.RopeScaling("cubic")), lambda t: t.PagedKVCache(2, 16, 2, 128, "int4"),
])
def test_python_refusals(make):
    from wuxianhuabu_b200 import text
    with pytest.raises(_lib.WxError) as e:
        make(text)
    assert e.value.status == _lib.WX_ERR_INVALID
