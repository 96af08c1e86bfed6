"""Attention with a window beside which the first keys of a sequence stay visible, against the masked
softmax in 64 bits. Tolerances as in test_gpu_text: one rounding to bf16 of the weights, one of the output."""
import math

import pytest
import torch

from tests.test_gpu_text import (BF16, F64, _check_device, _cu, _gen, _paged, _randn, _text, assert_attention)

pytestmark = pytest.mark.gpu
BIG = 2 ** 31 - 1


def ref_seen(q, k, v, scale, see):
    """One sequence, 64 bits, ``see`` [lq, lk]: out, lse and sum w |v|."""
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    grp = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(grp, 1), v.repeat_interleave(grp, 1)
    s = (torch.einsum("ihd,jhd->hij", q, k) * scale).masked_fill(~see, -math.inf)
    none = torch.full(s.shape[:2], -math.inf, dtype=F64, device=q.device)
    lse = torch.logsumexp(s, -1) if k.shape[0] else none
    zero = torch.zeros((), dtype=F64, device=q.device)
    w = torch.where(see, (s - torch.where(lse == -math.inf, zero, lse)[..., None]).exp(), zero)
    if torch.isfinite(v).all():
        return torch.einsum("hij,jhd->ihd", w, v), lse.T, torch.einsum("hij,jhd->ihd", w, v.abs())
    prod = torch.where(see[None, :, :, None], w[..., None] * v.permute(1, 0, 2)[:, None], zero)
    return prod.sum(2).permute(1, 0, 2), lse.T, prod.abs().sum(2).permute(1, 0, 2)


def seen(lq, lk, window, sinks):
    at = torch.arange(lq, device="cuda")[:, None] + (lk - lq)
    j = torch.arange(lk, device="cuda")[None]
    return (j <= at) & ((j > at - window) | (j < sinks)) if window else j <= at


PROMPTS = [  # lens, q heads, kv heads, head_dim, window, sinks
    ([1], 4, 2, 128, 1, 1),
    ([300, 77], 8, 2, 128, 40, 4),
    ([700, 1, 33], 4, 4, 64, 64, 1),
    ([900], 5, 1, 128, 100, 127),
    ([900], 5, 1, 64, 100, 128),
    ([640, 500], 2, 2, 128, 1, 129),
    ([1300], 28, 4, 128, 130, 300),
    ([1025, 260], 3, 3, 64, 256, 16),
    ([2300], 2, 1, 128, 600, 5),
    ([400, 222], 6, 2, 128, 3, BIG),       # first keys are all keys
    ([400, 222], 6, 2, 64, BIG, 7),        # the window is
    ([513], 4, 2, 128, 0, 9),              # no window: nothing changes
    ([5, 3], 2, 1, 128, 2, 1),
    ([16, 9], 1, 1, 64, 4, 3),
    ([4100], 1, 1, 128, 200, 70),
]


@pytest.mark.parametrize("lens,hq,hkv,hd,window,sinks", PROMPTS)
def test_prompts(lens, hq, hkv, hd, window, sinks):
    text = _text()
    g = _gen(sum(lens) + sinks % 1000)
    qkv = _randn(g, sum(lens), hq + 2 * hkv, hd)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    out = torch.full((q.shape[0], hq, hd), math.nan, dtype=BF16, device="cuda")
    out, lse = text.prompt_attention(q, k, v, _cu(lens), max(lens), window=window, sinks=sinks, out=out, return_lse=True)
    _check_device()
    a = 0
    for n in lens:
        ref, rl, mag = ref_seen(q[a:a + n], k[a:a + n], v[a:a + n], hd ** -0.5, seen(n, n, window, sinks))
        assert_attention(out[a:a + n], lse[a:a + n], ref, rl, mag, f"len {n}")
        a += n


@pytest.mark.parametrize("lens_q,lens_k,hq,hkv,hd,window,sinks", [
    ([5, 40, 9], [9, 7, 0], 4, 2, 128, 2, 3),            # more queries than keys: rows that see nothing
    ([130, 1, 300], [20, 300, 1500], 8, 1, 64, 33, 150),
    ([64, 200], [2500, 130], 6, 3, 128, 70, 20),
    ([1, 1, 3], [2000, 15, 4000], 4, 2, 128, 100, 30),
])
def test_prompts_with_other_key_lengths(lens_q, lens_k, hq, hkv, hd, window, sinks):
    text = _text()
    g = _gen(sum(lens_q) + sum(lens_k))
    q, k, v = _randn(g, sum(lens_q), hq, hd), _randn(g, sum(lens_k), hkv, hd), _randn(g, sum(lens_k), hkv, hd)
    out, lse = text.prompt_attention(q, k, v, _cu(lens_q), max(lens_q), window=window, sinks=sinks,
                                     cu_seqlens_k=_cu(lens_k), return_lse=True)
    _check_device()
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        ref, rl, mag = ref_seen(q[a:a + n], k[b:b + m], v[b:b + m], hd ** -0.5, seen(n, m, window, sinks))
        assert_attention(out[a:a + n], lse[a:a + n], ref, rl, mag, f"{n} over {m}")
        a, b = a + n, b + m


PAGED = [  # q_lens, kv_lens, q heads, kv heads, head_dim, page, window, sinks
    ([1], [1], 2, 1, 128, 16, 4, 4),
    ([1], [0], 2, 1, 64, 16, 4, 4),
    ([1, 1, 1], [17, 2000, 33], 4, 4, 64, 16, 10, 4),
    ([1, 1], [5000, 129], 8, 1, 128, 64, 300, 1),
    ([1] * 9, [5, 700, 64, 63, 65, 1, 2000, 128, 300], 14, 2, 128, 32, 50, 17),
    ([1, 1, 1], [3000, 100, 511], 6, 2, 64, 128, 100, 16),
    ([3, 1, 5], [500, 400, 5], 7, 1, 128, 16, 20, 33),
    ([4, 0, 8], [1500, 77, 140], 8, 2, 64, 64, 1, 200),
    ([2], [9000], 16, 2, 128, 64, 4000, 4),
    ([1, 2], [3000, 700], 4, 2, 128, 32, BIG, 4),
    ([1, 2], [3000, 700], 4, 2, 128, 32, 9, BIG),
    ([9, 30], [12, 20], 4, 2, 128, 32, 5, 2),          # 30 queries, 20 keys: rows that see nothing
    ([100, 37], [1400, 37], 8, 2, 128, 64, 64, 4),
    ([260], [3900], 4, 1, 64, 256, 300, 130),
    ([130, 20], [300, 6000], 28, 4, 128, 16, 90, 500),
    ([90], [6100], 8, 2, 128, 64, 2200, 40),
    ([70, 0, 200, 66], [2049, 300, 3025, 0], 4, 1, 64, 16, 1100, 8),
]


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,hd,page,window,sinks", PAGED)
def test_paged(q_lens, kv_lens, hq, hkv, hd, page, window, sinks, fmt):
    text = _text()
    g = _gen(sum(kv_lens) + hq)
    cache, table, q, ks, vs = _paged(g, fmt, q_lens, kv_lens, hq, hkv, hd, page)
    lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    out, lse = text.paged_attention(q, cache, _cu(q_lens), lens, table, max(q_lens), window=window, sinks=sinks,
                                    return_lse=True)
    _check_device()
    a = 0
    for n, k, v in zip(q_lens, ks, vs):
        ref, rl, mag = ref_seen(q[a:a + n], k, v, hd ** -0.5, seen(n, k.shape[0], window, sinks))
        assert_attention(out[a:a + n], lse[a:a + n], ref, rl, mag, f"{n} over {k.shape[0]}")
        a += n


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("rows", [1, 2, 40])
def test_keys_between_first_keys_and_window_are_not_read_into_a_row(fmt, rows):
    """NaN and infinities in keys that no row sees, and in first keys and window edges that only some see."""
    text = _text()
    g = _gen(rows)
    n, page, window, sinks = 700, 16, 60, 21
    cache, table, q, _, _ = _paged(g, fmt, [rows], [n], 4, 2, 128, page)
    pg = table[0].long()

    def poison(j, what, where):
        store, scale = (cache.k, cache.k_scale) if what == "k" else (cache.v, cache.v_scale)
        if fmt == "bf16":
            store[pg[j // page], :, j % page] = where
        else:
            scale[pg[j // page], :, j % page] = where

    hidden = [j for j in (sinks, sinks + 1, 100, 333, n - rows - window) if sinks <= j <= n - rows - window]
    for j in hidden:
        poison(j, "k", math.nan)
        poison(j, "v", math.inf if j % 2 else math.nan)
    some = [n - rows - window + 1] + ([n - 1] if rows > 1 else [])  # seen by the first row, or the last, alone
    if rows > 1:
        for j in some:
            poison(j, "v", math.inf)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    out, lse = text.paged_attention(q, cache, _cu([rows]), lens, table, rows, window=window, sinks=sinks,
                                    return_lse=True)
    _check_device()
    j = torch.arange(n, device="cuda")
    k, v = (c.view(torch.int8 if fmt != "bf16" else BF16)[pg[j // page], :, j % page].view(c.dtype).float().to(F64)
            for c in (cache.k, cache.v))
    if fmt != "bf16":
        k, v = (x * s[pg[j // page], :, j % page].to(F64)[..., None] for x, s in ((k, cache.k_scale), (v, cache.v_scale)))
    see = seen(rows, n, window, sinks)
    unseen = ~see.any(0)
    k[unseen] = 0
    ref, rl, mag = ref_seen(q, k, v, 128 ** -0.5, see)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(out), fin)
    tol = 2.0 ** -8 * (ref.abs() + mag) * (1 + 2.0 ** -7) + 2.0 ** -14 * mag
    assert ((out.to(F64) - ref).abs() <= tol)[fin].all()
    assert torch.isfinite(lse).all() and float((lse.to(F64) - rl).abs().max()) < 1e-4


def test_a_captured_call_and_another_stream():
    text = _text()
    g = _gen(11)
    cache, table, q, _, _ = _paged(g, "bf16", [1, 1], [900, 300], 8, 2, 128, 16)
    lens = torch.tensor([900, 300], dtype=torch.int32, device="cuda")
    how = dict(window=70, sinks=4)
    want = text.paged_attention(q, cache, _cu([1, 1]), lens, table, 1, **how)
    cu = _cu([1, 1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = text.paged_attention(q, cache, cu, lens, table, 1, **how)
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = text.paged_attention(q, cache, cu, lens, table, 1, **how)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(other, want)
    _check_device()


def test_refusals():
    text = _text()
    from wuxianhuabu_b200 import h3
    g = _gen(1)
    q, k, v = _randn(g, 9, 2, 64), _randn(g, 9, 1, 64), _randn(g, 9, 1, 64)
    for how in (dict(window=4, sinks=-1), dict(window=-4, sinks=1), dict(window=4, sinks=1, causal=False)):
        with pytest.raises(h3.WxError):
            text.prompt_attention(q, k, v, _cu([9]), 9, **how)
    a = text.prompt_attention(q, k, v, _cu([9]), 9, window=3, sinks=2 ** 40)
    b = text.prompt_attention(q, k, v, _cu([9]), 9)
    assert torch.equal(a, b)
    _check_device()
