"""The objects of the text side: tensors assigned after they were made, copies."""
import copy

import pytest
import torch

from tests.test_gpu_text import BF16, _check_device, _cu, _gen, _randn, _text

pytestmark = pytest.mark.gpu


def test_a_table_follows_its_tensors():
    text = _text()
    g = _gen(1)
    a, b = text.RopeTable(64, 32, base=10000.0), text.RopeTable(128, 48, base=500.0, interleaved=True)
    x, pos = _randn(g, 20, 3, 128), torch.arange(20, dtype=torch.int32, device="cuda") + 12
    a.apply(x, pos)
    keep = a.cos, a.sin
    a.cos, a.sin, a.interleaved = b.cos, b.sin, True
    pos40 = pos + 16  # beyond the first table
    assert torch.equal(a.apply(x, pos40), b.apply(x, pos40))
    _check_device()
    a.cos = b.cos[:8].contiguous()  # cos and sin differ now
    from wuxianhuabu_b200 import h3
    with pytest.raises(h3.WxError):
        a.apply(x, pos)
    del keep


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
def test_a_cache_follows_its_tensors(fmt):
    """A cache that is grown by assigning larger tensors: writes, reads and attention use the new ones."""
    text = _text()
    g = _gen(2)
    small, large = text.PagedKVCache(2, 16, 2, 64, fmt), text.PagedKVCache(6, 32, 2, 64, fmt)
    k, v = _randn(g, 20, 2, 64), _randn(g, 20, 2, 64)
    first = torch.arange(20, device="cuda")
    small.append(k, v, first)
    old = small.k.clone(), small.k, small.v, small.k_scale, small.v_scale
    small.k, small.v = large.k, large.v
    if fmt != "bf16":
        small.k_scale, small.v_scale = large.k_scale, large.v_scale
    assert (small.pages, small.page_size) == (6, 32)
    slots = first + 100
    small.append(k, v, slots)
    got = small.read(slots)
    want = large.read(slots)
    assert got[0].any() and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(old[1].view(torch.uint8), old[0].view(torch.uint8))
    q = _randn(g, 1, 2, 64)
    table = torch.tensor([[3]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([20], dtype=torch.int32, device="cuda")
    a = text.paged_attention(q, small, _cu([1]), lens, table, 1)
    b = text.paged_attention(q, large, _cu([1]), lens, table, 1)
    assert torch.equal(a, b)
    _check_device()
    from wuxianhuabu_b200 import h3
    small.v = large.v[:4]
    with pytest.raises(h3.WxError):
        small.read(slots)


def test_tables_and_caches_can_be_copied():
    text = _text()
    g = _gen(3)
    tab = text.RopeTable(64, 32)
    cache = text.PagedKVCache(2, 16, 1, 64, "int8")
    x, slots = _randn(g, 10, 1, 64), torch.arange(10, device="cuda")
    cache.append(x, x, slots)
    tab2, cache2 = copy.deepcopy(tab), copy.deepcopy(cache)
    assert tab2.cos.data_ptr() != tab.cos.data_ptr() and cache2.k.data_ptr() != cache.k.data_ptr()
    pos = torch.arange(10, dtype=torch.int32, device="cuda")
    assert torch.equal(tab2.apply(x, pos), tab.apply(x, pos))
    before = cache.read(slots)
    assert torch.equal(cache2.read(slots)[0], before[0])
    cache2.append(x * 2, x * 2, slots)
    assert torch.equal(cache.read(slots)[0], before[0]) and not torch.equal(cache2.read(slots)[0], before[0])
    shallow = copy.copy(cache)
    assert torch.equal(shallow.read(slots)[0], before[0])
    _check_device()
    assert before[0].dtype == BF16
