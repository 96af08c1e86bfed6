"""Arrays that are only read may be views in which rows share their memory: the results are those of the
same values laid out in full, bit for bit."""
import pytest
import torch

from tests.test_gpu_text import BF16, _check_device, _cu, _gen, _randn, _slots, _text
from tests.test_gpu_text_prefix import _behind, _i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 2, 50, 1900])  # (the last: persistent warps)
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_that_all_axes_share(tokens, interleaved):
    text = _text()
    g = _gen(tokens)
    rope = text.RopeTable(128, 4000, interleaved=interleaved, axes=text.rope_axes((24, 20, 20), dealt=True))
    q, k, v = _randn(g, tokens, 32, 128), _randn(g, tokens, 8, 128), _randn(g, tokens, 8, 128)
    w = (1.0 + 0.1 * _randn(g, 128).float()).to(BF16)
    row = torch.randperm(4000, generator=g, device="cuda")[:tokens].to(torch.int32)
    shared, full = row.expand(3, -1), row.expand(3, -1).contiguous()
    assert shared.stride(0) == 0
    for a, b in zip(rope.apply_qk(q, k, shared, q_norm=w, k_norm=w), rope.apply_qk(q, k, full, q_norm=w, k_norm=w)):
        assert torch.equal(a, b)
    assert torch.equal(rope.apply(q, shared, norm=w), rope.apply(q, full, norm=w))
    assert torch.equal(rope.apply(q, shared), rope.apply(q, full))
    pages = -(-tokens // 16) + 1
    slots = _slots(g, tokens, pages, 16)
    for fmt in ("bf16", "int8", "e4m3"):
        got = []
        for pos in (shared, full):
            cache = text.PagedKVCache(pages, 16, 8, 128, fmt)
            got.append((cache.append_roped(q, k, v, slots, rope, pos, q_norm=w, k_norm=w), *cache.read(slots)))
        assert all(torch.equal(a, b) for a, b in zip(*got)), fmt
    _check_device()


def test_a_plan_s_positions_serve_every_axis():
    """A step's one row of positions goes straight into a model of several axes."""
    text = _text()
    g = _gen(9)
    pool = text.PagePool(20, 16, 3, 8)
    plan = pool.plan(torch.tensor([20, 1, 7], dtype=torch.int32, device="cuda"), 28, first_position=100)
    rope = text.RopeTable(64, 200, axes=text.rope_axes((12, 10, 10)))
    q, k, v = _randn(g, 28, 4, 64), _randn(g, 28, 2, 64), _randn(g, 28, 2, 64)
    cache = text.PagedKVCache(20, 16, 2, 64, "bf16")
    turned = cache.append_roped(q, k, v, plan.slots, rope, plan.positions.expand(3, -1))
    assert torch.equal(turned, rope.apply(q, plan.positions.expand(3, -1).contiguous()))
    _check_device()


def test_overlapping_axes_are_refused():
    text = _text()
    from wuxianhuabu_b200 import h3
    rope = text.RopeTable(64, 30, axes=text.rope_axes((12, 10, 10)))
    q = _randn(_gen(1), 5, 3, 64)
    pos = torch.zeros(30, dtype=torch.int32, device="cuda")
    for stride in (1, 4):
        with pytest.raises(h3.WxError):
            rope.apply(q, pos.as_strided((3, 5), (stride, 1)))
    _check_device()


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("q_lens", [[1] * 3, [1] * 40, [60, 3], [1]])
def test_own_pages_that_all_sequences_share(q_lens, fmt):
    """Sequences over the same own pages, to lengths of their own: one row of the table for all of them."""
    text = _text()
    prefix, kv_lens = 300, [60 + 3 * i for i in range(len(q_lens))]
    cache, front, table, q, _, _ = _behind(_gen(len(q_lens)), fmt, prefix, q_lens, kv_lens, 8, 2, 128, 16)
    row = table[-1]
    shared, full = row.expand(len(q_lens), -1), row.expand(len(q_lens), -1).contiguous()
    got = [text.prefix_attention(q, cache, front, prefix, _cu(q_lens), _i32(kv_lens), t, max(q_lens), return_lse=True)
           for t in (shared, full)]
    _check_device()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_block_tables_whose_rows_overlap_are_refused():
    text = _text()
    from wuxianhuabu_b200 import h3
    cache, front, table, q, _, _ = _behind(_gen(2), "bf16", 100, [1, 1], [5, 40], 4, 2, 128, 16)
    for stride in (1, 2):
        with pytest.raises(h3.WxError):
            text.prefix_attention(q, cache, front, 100, _cu([1, 1]), _i32([5, 40]),
                                  table.as_strided((2, 3), (stride, 1)), 1)
    _check_device()
