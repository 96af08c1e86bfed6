"""Host side of the text operators that plan steps, normalise heads and attend beside windows and
prefixes: refusals that need no GPU, and the pairs' axes."""
import ctypes as C

import pytest

from wuxianhuabu_b200 import _lib


def test_calls_without_a_context_are_refused():
    lib = _lib.load()
    assert lib.wx_norm_rope_apply(None, None, None, None, None, 0, 0, None, None, 0, 0, None, 0.0, 0, 0, None, 0, None, 0) \
        == _lib.WX_ERR_INVALID
    assert lib.wx_norm_rope_kv_append(None, None, None, None, None, 0, 0, None, None, 0.0, None, None, 0, None, 0, 0, None,
                                      None, 0) == _lib.WX_ERR_INVALID
    assert lib.wx_prompt_attention_sinks(None, None, 0, None, 0, None, 0, None, 0, 0, None, None, None, 0, None) \
        == _lib.WX_ERR_INVALID
    assert lib.wx_paged_attention_sinks(None, None, 0, None, 0, None, None, None, None, 0, None, 0, None) \
        == _lib.WX_ERR_INVALID
    assert lib.wx_prefix_attention(None, None, None, 0, None, None, 0, None, None, None, 0, 0, None, 0, None) \
        == _lib.WX_ERR_INVALID
    assert lib.wx_page_plan(None, None, None, None, 0, 0, None, None, None, None, None) == _lib.WX_ERR_INVALID


def test_structs_have_the_library_s_layout():
    assert C.sizeof(_lib.RopeAxes) == 80 and _lib.RopeAxes.position_stride.offset == 72
    assert C.sizeof(_lib.PagePool) == 56


def test_axes_of_the_pairs():
    from wuxianhuabu_b200 import text
    assert text.rope_axes((3, 2, 1)) == (0, 0, 0, 1, 1, 2)
    assert text.rope_axes((3, 2, 1), dealt=True) == (0, 1, 2, 0, 1, 0)
    assert text.rope_axes((24, 20, 20), dealt=True)[:6] == (0, 1, 2, 0, 1, 2)
    assert text.rope_axes((24, 20, 20), dealt=True)[60:] == (0, 0, 0, 0)
    assert text.rope_axes((2, 0, 1), dealt=True) == (0, 2, 0)
    for wrong in ((), (1, 1, 1, 1, 1), (2, -1)):
        with pytest.raises(_lib.WxError):
            text.rope_axes(wrong)
