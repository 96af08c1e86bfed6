"""The text side stays inside its buffers.

* On the bounds-checked build (libwx_checked.so) rope, cache writes and reads and both attention kernels, whole
  and in pieces, packed and paged in every format, record no bounds error, and give the normal build's bits.
* Memory around outputs and beside written slots keeps its sentinel on the normal build."""
import os
import subprocess
import sys
import tempfile
from pathlib import Path

import numpy as np
import pytest
import torch

from tests.test_gpu_text import BF16, _check_device, _cu, _gen, _paged, _randn, _text

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

CHILD = r'''
import sys
import numpy as np
sys.path.insert(0, sys.argv[1])
import torch
from tests.test_gpu_text import PAGED, PROMPTS, _cu, _gen, _paged, _randn, _text
from wuxianhuabu_b200 import h3
text, outs = _text(), {}
def keep(name, *ts):
    for i, t in enumerate(ts):
        outs[f"{name}.{i}"] = t.contiguous().view(torch.uint8).cpu().numpy()
for i, (lens, hq, hkv, hd, causal, window) in enumerate(PROMPTS):
    g = _gen(i)
    qkv = _randn(g, sum(lens), hq + 2 * hkv, hd)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    keep(f"prompt{i}", *text.prompt_attention(q, k, v, _cu(lens), max(lens), causal=causal, window=window, return_lse=True))
extra = [([90], [4100], 8, 2, 128, 64, 0), ([70, 0, 200, 66], [2049, 300, 1025, 0], 4, 1, 64, 16, 0),
         ([130, 66], [6000, 2048], 4, 4, 128, 32, 2500)]
for fmt in ("bf16", "int8", "e4m3"):
    for i, (q_lens, kv_lens, hq, hkv, hd, page, window) in enumerate(PAGED + extra):
        g = _gen(50 + i)
        cache, table, q, _, _ = _paged(g, fmt, q_lens, kv_lens, hq, hkv, hd, page)
        lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
        keep(f"{fmt}{i}", *text.paged_attention(q, cache, _cu(q_lens), lens, table, max(q_lens), window=window,
                                                return_lse=True))
    for i, (tokens, kv_heads, hd, page) in enumerate([(1, 1, 128, 16), (333, 8, 64, 32), (1500, 2, 128, 256)]):
        g = _gen(80 + i)
        cache = text.PagedKVCache((tokens + page - 1) // page, page, kv_heads, hd, fmt)
        x = _randn(g, tokens, 5 * kv_heads, hd)
        slots = torch.arange(tokens, device="cuda")
        tab = text.RopeTable(hd // 2, tokens)
        pos = slots.to(torch.int32)
        keep(f"cache{fmt}{i}", cache.append_roped(x[:, :3 * kv_heads], x[:, 3 * kv_heads:4 * kv_heads],
                                                  x[:, 4 * kv_heads:], slots, tab, pos), *cache.read(slots),
             tab.apply(x, pos))
h3.context().check_device()  # raises on a recorded device error (bounds: code 8)
np.savez(sys.argv[2], **outs)
print("ok")
'''


def _run(variant, path):
    env = dict(os.environ)
    env.pop("WX_LIB_VARIANT", None)
    if variant:
        env["WX_LIB_VARIANT"] = variant
    r = subprocess.run([sys.executable, "-c", CHILD, str(ROOT), path], env=env, capture_output=True, text=True,
                       timeout=600, cwd=str(ROOT))
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout[-2000:] + r.stderr[-2000:]
    return np.load(path)


def test_checked_build_finds_nothing_and_gives_the_same_bits():
    if not (ROOT / "wuxianhuabu_b200" / "libwx_checked.so").exists():
        pytest.fail("libwx_checked.so is missing: __graft_entry__.build() builds it")
    with tempfile.TemporaryDirectory() as d:
        a, b = _run("checked", os.path.join(d, "checked.npz")), _run("", os.path.join(d, "normal.npz"))
        assert sorted(a.files) == sorted(b.files)
        for k in a.files:
            assert np.array_equal(a[k], b[k]), k


SENTINEL = 123.0


def _framed(n, h, d):
    """An output [n, h, d] with rows before and behind it and a gap after each row, all of one value."""
    whole = torch.full((n + 6, h + 2, d), SENTINEL, dtype=BF16, device="cuda")
    return whole, whole[3:3 + n, :h]


def _frame_kept(whole, n, h):
    inside = torch.zeros(whole.shape[:2], dtype=torch.bool, device="cuda")
    inside[3:3 + n, :h] = True
    return bool((whole[~inside] == SENTINEL).all()) and not bool((whole[inside] == SENTINEL).all(-1).any())


@pytest.mark.parametrize("lens,hq,hkv,hd", [([1], 4, 2, 128), ([5, 0, 3], 8, 2, 64), ([129, 1, 40], 6, 3, 128),
                                            ([700], 7, 1, 64), ([60], 4, 4, 128)])
def test_prompt_attention_writes_only_its_rows(lens, hq, hkv, hd):
    text = _text()
    g = _gen(sum(lens))
    n = sum(lens)
    q, k, v = _randn(g, n, hq, hd), _randn(g, n, hkv, hd), _randn(g, n, hkv, hd)
    whole, out = _framed(n, hq, hd)
    text.prompt_attention(q, k, v, _cu(lens), max(lens), out=out)
    _check_device()
    assert _frame_kept(whole, n, hq)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,hd", [([1], [5000], 8, 2, 128), ([2, 0, 1], [700, 9, 0], 4, 4, 64),
                                                      ([90], [4100], 8, 2, 128), ([200, 17], [300, 17], 7, 1, 64)])
def test_paged_attention_writes_only_its_rows(fmt, q_lens, kv_lens, hq, hkv, hd):
    """Rows behind the last sequence (padding of a batch) stay as they are, and the cache is not written."""
    text = _text()
    g = _gen(sum(q_lens) + hd)
    cache, table, q, _, _ = _paged(g, fmt, q_lens, kv_lens, hq, hkv, hd, 16)
    before = cache.k.clone(), cache.v.clone()
    n = sum(q_lens)
    whole, out = _framed(n + 5, hq, hd)
    padded = torch.cat([q, _randn(g, 5, hq, hd)])
    lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    text.paged_attention(padded, cache, _cu(q_lens), lens, table, max(q_lens), out=out)
    _check_device()
    assert _frame_kept(whole, n, hq)
    for x, y in zip((cache.k, cache.v), before):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 64)])
def test_cache_writes_touch_only_their_slots(fmt, hd, page):
    text = _text()
    g = _gen(hd)
    cache = text.PagedKVCache(7, page, 3, hd, fmt)
    junk = _randn(g, 7 * page, 3, hd)
    cache.append(junk, junk, torch.arange(7 * page, device="cuda"))
    held = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    slots = torch.tensor([page - 1, page, 3 * page + 5, 7 * page - 1, -1], device="cuda")
    x = _randn(g, 5, 13, hd)
    tab = text.RopeTable(hd, 8)
    whole, out = _framed(5, 7, hd)
    cache.append_roped(x[:, :7], x[:, 7:10], x[:, 10:], slots, tab, torch.arange(5, dtype=torch.int32, device="cuda"), q_out=out)
    _check_device()
    assert _frame_kept(whole, 5, 7)
    other = torch.ones(7 * page, dtype=torch.bool, device="cuda")
    other[slots[:4]] = False
    now = [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    for a, b in zip(now, held):
        a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b))
        a, b = (t.transpose(1, 2).reshape(7 * page, 3, -1) for t in (a, b))
        assert torch.equal(a[other], b[other]) and not torch.equal(a[~other], b[~other])
