"""A shared prefix that the kernel for few rows walks in chunks: the layers that are joined are those that
were written, whatever earlier calls left in the workspace. Tolerances as in test_gpu_text_prefix."""
import pytest
import torch

from tests.test_gpu_text import _check_device, _cu, _gen, _text
from tests.test_gpu_text_prefix import _behind, _check, _i32

pytestmark = pytest.mark.gpu


def _leave_sums():
    """A larger call: 2,048 rows' sums over parts of 8,011 keys (tens in magnitude) fill the workspace's front."""
    text = _text()
    kv_lens = [1 + 13 * i for i in range(64)]
    cache, front, table, q, _, _ = _behind(_gen(1), "bf16", 8011, [1] * 64, kv_lens, 32, 8, 128, 64)
    text.prefix_attention(q, cache, front, 8011, _cu([1] * 64), _i32(kv_lens), table, 1)


# prefixes whose chunks, rounded up to whole steps of 16 keys, are fewer than the most that a length has
@pytest.mark.parametrize("prefix,batch,hq,hkv,hd,fmt", [
    (2100, 5, 32, 8, 128, "bf16"), (2048, 3, 16, 16, 64, "bf16"), (3100, 8, 16, 16, 128, "bf16"),
    (5231, 5, 16, 16, 128, "bf16"), (4200, 16, 16, 16, 64, "bf16"), (3200, 8, 32, 8, 128, "e4m3"),
    (4096, 8, 32, 8, 64, "e4m3"), (5646, 8, 32, 8, 128, "int8"), (5646, 12, 32, 8, 64, "int8")])
def test_the_workspace_s_past_does_not_reach_the_rows(prefix, batch, hq, hkv, hd, fmt):
    text = _text()
    q_lens, kv_lens = [1] * batch, [1 + 29 * i % 150 for i in range(batch)]
    cache, front, table, q, ks, vs = _behind(_gen(prefix), fmt, prefix, q_lens, kv_lens, hq, hkv, hd, 64)
    run = lambda: text.prefix_attention(q, cache, front, prefix, _cu(q_lens), _i32(kv_lens), table, 1,  # noqa: E731
                                        return_lse=True)
    before = run()
    _leave_sums()
    after = run()
    _check_device()
    _check(*after, q, q_lens, ks, vs)
    _check(*before, q, q_lens, ks, vs)
    assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1])
