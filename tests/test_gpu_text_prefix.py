"""Attention of a batch behind one cached prefix, against the masked softmax over prefix and own keys in 64
bits. Tolerances as in test_gpu_text: one rounding to bf16 of the weights, one of the output."""
import math

import pytest
import torch

from tests.test_gpu_text import (BF16, F64, _check_device, _cu, _gen, _paged, _randn, _text, assert_attention)
from tests.test_gpu_text_sinks import ref_seen

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _behind(g, fmt, prefix, q_lens, kv_lens, hq, hkv, hd, page):
    """A cache whose first sequence is the prefix: the prefix's pages, the others' table, q, and all keys."""
    cache, table, q, ks, vs = _paged(g, fmt, [0] + list(q_lens), [prefix] + list(kv_lens), hq, hkv, hd, page)
    return cache, table[0, :-(-prefix // page)].clone(), table[1:].contiguous(), q, ks, vs


def _check(out, lse, q, q_lens, ks, vs, causal=True):
    hd, a = q.shape[2], 0
    for n, k, v in zip(q_lens, ks[1:], vs[1:]):
        if not n:
            continue
        p, m = ks[0].shape[0], k.shape[0]
        see = torch.ones((n, p + m), dtype=torch.bool, device="cuda")
        if causal:
            see[:, p:] = torch.arange(m, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (m - n)
        ref, rl, mag = ref_seen(q[a:a + n], torch.cat([ks[0], k]), torch.cat([vs[0], v]), hd ** -0.5, see)
        assert_attention(out[a:a + n], None if lse is None else lse[a:a + n], ref, rl, mag, f"{n} over {p} + {m}")
        a += n


CASES = [  # prefix, q_lens, kv_lens, q heads, kv heads, head_dim, page
    (1, [1], [1], 2, 1, 128, 16),
    (16, [1, 1], [1, 30], 4, 2, 64, 16),
    (333, [1, 1, 1], [1, 40, 17], 16, 16, 64, 16),
    (500, [1] * 5, [3, 700, 64, 65, 1], 8, 2, 128, 64),
    (0, [1, 1, 2], [5, 300, 40], 8, 2, 128, 32),            # no prefix
    (129, [1, 1], [0, 5], 8, 2, 128, 32),                   # no own keys
    (0, [1], [0], 2, 2, 64, 16),                            # nothing at all
    (2000, [1] * 33, [1 + 37 * i % 300 for i in range(33)], 8, 2, 128, 64),
    (3001, [1] * 70, [1 + 91 * i % 500 for i in range(70)], 14, 2, 128, 16),
    (127, [1] * 40, [9] * 40, 6, 1, 64, 128),
    (4100, [1] * 150, [1 + i % 60 for i in range(150)], 4, 4, 64, 32),
    (700, [3, 1, 0, 5], [50, 400, 0, 5], 7, 1, 128, 16),    # drafted tokens, an empty sequence
    (640, [4] * 20, [4 + 13 * i for i in range(20)], 16, 2, 128, 256),
    (200, [9, 30], [12, 20], 4, 2, 128, 32),                # 30 queries, 20 own keys: rows that see the prefix alone
    (1000, [100, 37, 1], [100, 37, 1], 8, 2, 128, 64),      # prompts behind it
    (1500, [260, 33], [900, 33], 4, 1, 64, 16),
    (77, [513], [513], 28, 4, 128, 16),
    (9000, [70], [70], 4, 1, 128, 64),                      # few items: pieces
    (5000, [2] * 3, [1000, 2, 30], 40, 2, 64, 64),
    (300, [1] * 9, [20] * 9, 64, 1, 128, 32),
    (200, [1] * 5, [1, 90, 17, 0, 300], 128, 1, 64, 64),                # as many query heads to a K/V head as there may be
    (513, [1] * 70, [5000 if i == 33 else 3 for i in range(70)], 8, 4, 128, 64),  # one long among short: longer chunks
    (900, [1] * 300, [1 + 7 * i % 200 for i in range(300)], 4, 4, 64, 16),       # fewer, longer chunks
    (3000, [1, 1], [40, 3000], 4, 1, 128, 16),                          # few items, long: a piece per CTA
]


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("prefix,q_lens,kv_lens,hq,hkv,hd,page", CASES)
def test_against_the_definition(prefix, q_lens, kv_lens, hq, hkv, hd, page, fmt):
    text = _text()
    g = _gen(prefix + len(q_lens))
    cache, front, table, q, ks, vs = _behind(g, fmt, prefix, q_lens, kv_lens, hq, hkv, hd, page)
    out = torch.full_like(q, math.nan)
    out, lse = text.prefix_attention(q, cache, front, prefix, _cu(q_lens), _i32(kv_lens), table, max(q_lens), out=out,
                                     return_lse=True)
    _check_device()
    _check(out, lse, q, q_lens, ks, vs)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [40, 0, 7]), ([50, 20], [60, 5]), ([1] * 30, [3] * 30)])
def test_without_causal(q_lens, kv_lens):
    text = _text()
    cache, front, table, q, ks, vs = _behind(_gen(3), "bf16", 190, q_lens, kv_lens, 4, 2, 128, 16)
    out, lse = text.prefix_attention(q, cache, front, 190, _cu(q_lens), _i32(kv_lens), table, max(q_lens), causal=False,
                                     return_lse=True)
    _check_device()
    _check(out, lse, q, q_lens, ks, vs, causal=False)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("q_lens,kv_lens", [([1] * 24, [1 + 17 * i for i in range(24)]), ([1, 1], [9, 300]),
                                            ([90, 40], [90, 77])])
def test_columns_of_a_whole_table(q_lens, kv_lens, fmt):
    """Tables that begin with the prefix's pages, as paged_attention takes them: the same rows."""
    text = _text()
    page, prefix = 16, 32 * 16
    cache, front, table, q, ks, vs = _behind(_gen(5), fmt, prefix, q_lens, kv_lens, 8, 2, 128, page)
    n = prefix // page
    whole = torch.cat([front.expand(len(q_lens), -1), table], 1).contiguous()
    a = text.prefix_attention(q, cache, whole[0, :n], prefix, _cu(q_lens), _i32(kv_lens), whole[:, n:], max(q_lens),
                              return_lse=True)
    b = text.prefix_attention(q, cache, front, prefix, _cu(q_lens), _i32(kv_lens), table, max(q_lens), return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c = text.paged_attention(q, cache, _cu(q_lens), _i32(kv_lens) + prefix, whole, max(q_lens), return_lse=True)
    _check_device()
    # (each is within its own tolerance of the definition, in which the same sums stand)
    _check(*a, q, q_lens, ks, vs)
    _check(*c, q, q_lens, ks, vs)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("q_lens", [[1, 1], [1] * 40, [60, 3]])
def test_what_stands_behind_the_prefix_s_end_is_not_seen(q_lens, fmt):
    """NaN in the rest of the prefix's last page and behind the own keys, infinities in the prefix itself."""
    text = _text()
    kv_lens = [n + 5 for n in q_lens]
    prefix, page = 150, 64
    cache, front, table, q, ks, vs = _behind(_gen(len(q_lens)), fmt, prefix, q_lens, kv_lens, 4, 2, 64, page)

    def poison(pages, j, value):
        for store, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            if fmt == "bf16":
                store[int(pages[j // page]), :, j % page] = value
            else:
                scale[int(pages[j // page]), :, j % page] = value

    for j in range(prefix, 3 * page):
        poison(front, j, math.nan)
    poison(table[0], kv_lens[0], math.inf)
    run = lambda: text.prefix_attention(q, cache, front, prefix, _cu(q_lens), _i32(kv_lens), table,  # noqa: E731
                                        max(q_lens), return_lse=True)
    out, lse = run()
    _check_device()
    _check(out, lse, q, q_lens, ks, vs)
    for j, value in ((3, math.inf), (149, -math.inf)):  # (in V, seen by every row)
        if fmt == "bf16":
            cache.v[int(front[j // page]), 1, j % page, 7] = value
        else:
            cache.v_scale[int(front[j // page]), 1, j % page] = math.nan
    again, lse2 = run()
    _check_device()
    assert torch.equal(lse2, lse)
    hurt = torch.zeros(64, dtype=torch.bool, device="cuda")
    hurt[7] = True
    if fmt != "bf16":
        hurt[:] = True
    assert torch.isnan(again[:, 2:][..., hurt]).all() and torch.equal(again[:, :2], out[:, :2])
    again[:, 2:] = torch.where(hurt, out[:, 2:], again[:, 2:])  # (the other columns, summed another way, stand)
    _check(again, lse2, q, q_lens, ks, vs)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("q_lens,kv_lens", [([1] * 40, [1 + 9 * i for i in range(40)]), ([1, 2], [30, 5]),
                                            ([100, 7], [100, 90])])
def test_tables_far_wider_than_the_lengths(q_lens, kv_lens, fmt):
    text = _text()
    cache, front, table, q, ks, vs = _behind(_gen(77), fmt, 800, q_lens, kv_lens, 8, 2, 128, 16)
    wide = torch.full((len(q_lens), 9000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    out, lse = text.prefix_attention(q, cache, front, 800, _cu(q_lens), _i32(kv_lens), wide, max(q_lens), return_lse=True)
    _check_device()
    _check(out, lse, q, q_lens, ks, vs)


def test_rows_behind_the_last_sequence_are_left():
    text = _text()
    cache, front, table, q, ks, vs = _behind(_gen(8), "bf16", 300, [1, 2], [5, 9], 4, 2, 128, 16)
    for rows, lens in ((1, [1, 1]), (40, [1, 2])):
        q2 = torch.cat([q, _randn(_gen(9), rows, 4, 128)])
        out = torch.full_like(q2, 5.0)
        out, lse = text.prefix_attention(q2, cache, front, 300, _cu([1, 2]), _i32([5, 9]), table, 2, out=out,
                                         return_lse=True)
        _check_device()
        _check(out[:3], lse[:3], q, [1, 2], ks, vs)
        assert (out[3:] == 5.0).all()


def test_captured_and_direct_calls_and_streams():
    """Two captured calls of different sizes, replayed among direct calls and on another stream."""
    text = _text()
    sets = []
    for i, (prefix, n) in enumerate(((2000, 40), (500, 3))):
        q_lens, kv_lens = [1] * n, [1 + 11 * j % 90 for j in range(n)]
        cache, front, table, q, ks, vs = _behind(_gen(20 + i), "bf16", prefix, q_lens, kv_lens, 8, 2, 128, 16)
        args = q, cache, front, prefix, _cu(q_lens), _i32(kv_lens), table, 1
        sets.append((args, text.prefix_attention(*args)))
    torch.cuda.synchronize()
    graphs = []
    for args, want in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = text.prefix_attention(*args)
        graphs.append((graph, out))
    for _ in range(3):
        for (graph, out), (args, want) in zip(graphs, sets):
            out.fill_(0)
            graph.replay()
            direct = text.prefix_attention(*args)
            assert torch.equal(out, want) and torch.equal(direct, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = text.prefix_attention(*sets[0][0])
    mine = text.prefix_attention(*sets[1][0])
    torch.cuda.synchronize()
    assert torch.equal(other, sets[0][1]) and torch.equal(mine, sets[1][1])
    _check_device()


def test_wrong_pages_and_lengths_are_reported():
    text = _text()
    from wuxianhuabu_b200 import h3
    cache, front, table, q, ks, vs = _behind(_gen(30), "bf16", 100, [1, 1], [5, 9], 4, 2, 128, 16)
    bad = front.clone()
    bad[2] = cache.pages
    cases = [(bad, _i32([5, 9]), table), (front, _i32([5, -1]), table), (front, _i32([5, 9]), table * 0 - 3),
             (front, _i32([5, 10 ** 6]), table)]
    for f, lens, t in cases:
        for rows in (1, 30):  # both kernels
            q2 = q.repeat_interleave(rows, 0)
            text.prefix_attention(q2, cache, f, 100, _cu([rows, rows]), lens, t.contiguous(), rows)
            with pytest.raises(h3.WxError):
                _check_device()
    out = text.prefix_attention(q, cache, front, 100, _cu([1, 1]), _i32([5, 9]), table, 1)
    _check_device()
    _check(out, None, q, [1, 1], ks, vs)


def test_refusals():
    text = _text()
    from wuxianhuabu_b200 import h3
    cache, front, table, q, _, _ = _behind(_gen(31), "bf16", 100, [1, 1], [5, 9], 4, 2, 128, 16)
    cu, lens = _cu([1, 1]), _i32([5, 9])
    for call in (lambda: text.prefix_attention(q, cache, front, 113, cu, lens, table, 1),
                 lambda: text.prefix_attention(q, cache, front, -1, cu, lens, table, 1),
                 lambda: text.prefix_attention(q, cache, front.long(), 100, cu, lens, table, 1),
                 lambda: text.prefix_attention(q, cache, front.cpu(), 100, cu, lens, table, 1),
                 lambda: text.prefix_attention(q, cache, front, 100, cu, lens, table[:1], 1),
                 lambda: text.prefix_attention(q, cache, front, 100, cu, lens, table.t().contiguous().t(), 1)
                 if table.shape[1] > 1 else text.prefix_attention(q, cache, front, 113, cu, lens, table, 1),
                 lambda: text.prefix_attention(q, cache, front, 100, cu, lens, table[:, :0], 1),
                 lambda: text.prefix_attention(q, cache, front, 100, cu, lens, table, 1, scale=-1.0),
                 lambda: text.prefix_attention(q[..., :64], cache, front, 100, cu, lens, table, 1)):
        with pytest.raises(h3.WxError):
            call()
    empty = text.prefix_attention(q[:0], cache, front, 100, _cu([0, 0]), lens, table, 0)
    assert empty.shape == (0, 4, 128)
    _check_device()
