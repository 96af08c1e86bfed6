"""New prompts behind a shared prefix, whose items may be cut into pieces along their keys: the room that the
pieces' partial sums take, and the rows. Tolerances as in test_gpu_text_prefix."""
import pytest
import torch

from tests.test_gpu_text import _check_device, _cu, _gen, _paged, _text, assert_attention
from tests.test_gpu_text_prefix import _behind, _check, _i32
from tests.test_gpu_text_sinks import ref_seen

pytestmark = pytest.mark.gpu


def _with_new_context(call):
    """What the call returns, and the bytes that a context made for it holds afterwards."""
    from wuxianhuabu_b200 import h3
    dev = torch.cuda.current_device()
    h3.context()
    usual = h3._contexts[dev]
    h3._contexts[dev] = ctx = h3.Context(dev)
    try:
        got = call()
        held = ctx.lib.wx_ctx_workspace_bytes(ctx.h)
        ctx.check_device()
        ctx.close()
    finally:
        h3._contexts[dev] = usual
    return got, held


def _some_rows(got, q, lens, ks, vs, rows):
    """The given (sequence, row) pairs against the definition."""
    for b, r in rows:
        k, v = torch.cat([ks[0], ks[1 + b]]), torch.cat([vs[0], vs[1 + b]])
        at = sum(lens[:b]) + r
        see = (torch.arange(k.shape[0], device="cuda") <= k.shape[0] - lens[b] + r)[None]
        ref, rl, mag = ref_seen(q[at:at + 1], k, v, q.shape[2] ** -0.5, see)
        assert_attention(got[0][at:at + 1], got[1][at:at + 1], ref, rl, mag, f"row {r} of sequence {b}")


@pytest.mark.parametrize("lens,prefix", [([1000] * 6, 8000), ([1200] * 10, 16000)])
def test_many_rows_take_little_room(lens, prefix):
    """192,000 and 384,000 rows, five and ten rounds over the SMs: in pieces their partial sums would be 286 and 381 MB."""
    text = _text()
    cache, table, q, ks, vs = _paged(_gen(4), "bf16", [0] + lens, [prefix] + lens, 32, 8, 128, 128)
    args = q, cache, table[0, :-(-prefix // 128)].clone(), prefix, _cu(lens), _i32(lens), table[1:].contiguous(), lens[0]
    got, held = _with_new_context(lambda: text.prefix_attention(*args, return_lse=True))
    assert held <= 64 << 20, held
    last = len(lens) - 1
    _some_rows(got, q, lens, ks, vs, [(0, 0), (0, lens[0] - 1), (4, 500), (last, 1), (last, lens[0] - 1)])


def test_few_items_over_many_own_keys_are_cut():
    """40 new tokens, 30,000 own keys, a short prefix: 8 items, whose keys the SMs share."""
    text = _text()
    cache, front, table, q, ks, vs = _behind(_gen(5), "bf16", 128, [40], [30000], 32, 8, 128, 64)
    run = lambda: text.prefix_attention(q, cache, front, 128, _cu([40]), _i32([30000]), table, 40,  # noqa: E731
                                        return_lse=True)
    got, held = _with_new_context(run)
    _, one = _with_new_context(lambda: text.prefix_attention(q, cache, front, 128, _cu([40]), _i32([40]),
                                                                 table[:, :1], 40))
    assert held - one >= 8 * 40 * 32 * 128 * 4, (held, one)  # eight pieces' sums at least
    _check_device()
    _check(*got, q, [40], ks, vs)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("wide", [0, 3000])
@pytest.mark.parametrize("prefix,q_lens,kv_lens,hq,hkv,hd,page", [
    (300, [40, 33, 70, 1], [9000, 40, 70, 2500], 8, 2, 128, 64),      # the longest first
    (300, [65, 3, 0, 40], [65, 3, 0, 20001], 28, 4, 128, 32),         # an empty sequence, the longest last
    (2500, [200, 64], [200, 12000], 16, 4, 64, 16),                   # whole rounds of one, pieces of the other
    (0, [90, 50], [7000, 50], 4, 1, 128, 128)])
def test_long_and_short_sequences_in_one_call(prefix, q_lens, kv_lens, hq, hkv, hd, page, wide, fmt):
    text = _text()
    cache, front, table, q, ks, vs = _behind(_gen(prefix), fmt, prefix, q_lens, kv_lens, hq, hkv, hd, page)
    if wide:
        far = torch.full((len(q_lens), wide), -1, dtype=torch.int32, device="cuda")
        far[:, :table.shape[1]] = table
        table = far
    out = torch.full_like(q, float("nan"))
    got = text.prefix_attention(q, cache, front, prefix, _cu(q_lens), _i32(kv_lens), table, max(q_lens), out=out,
                                return_lse=True)
    _check_device()
    _check(*got, q, q_lens, ks, vs)
