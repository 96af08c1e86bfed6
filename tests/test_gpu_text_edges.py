"""The text-side operators where a mask, a value or a length is extreme: windows near the integer
limit, infinities and NaN in keys and values that some rows see, NaN codes in an e4m3 cache.

Attention is compared with its definition in 64 bits; the tolerance of finite outputs is that of the
weights' and the output's rounding to bf16 (2^-8 of the sum of |w v|, 2^-8 of the output) and 2^-14 of the
weights for scores and exponentials in fp32. NaN, +inf and -inf have to stand exactly where the
definition puts them.
"""
import math

import pytest
import torch

from tests.test_gpu_text import BF16, F64, _check_device, _cu, _gen, _paged, _randn, _text, ref_attention

pytestmark = pytest.mark.gpu
INT_MAX = 2 ** 31 - 1


def assert_same(out, lse, ref, rlse, mag, what=""):
    for name, is_it in (("NaN", torch.isnan), ("+inf", torch.isposinf), ("-inf", torch.isneginf)):
        assert torch.equal(is_it(out), is_it(ref)), f"{what}: {name} at other places"
        if lse is not None:
            assert torch.equal(is_it(lse), is_it(rlse)), f"{what}: {name} of lse at other places"
    ok = torch.isfinite(ref)
    tol = 2.0 ** -8 * (ref.abs() + mag) * (1 + 2.0 ** -7) + 2.0 ** -14 * mag
    over = ((out.to(F64) - ref).abs() > tol) & ok
    assert not over.any(), f"{what}: {int(over.sum())} outputs off"
    if lse is not None:
        fin = torch.isfinite(rlse)
        e = (lse.to(F64) - rlse)[fin].abs()
        assert e.numel() == 0 or float((e - 2.0 ** -20 * rlse[fin].abs()).max()) < 2e-5, f"{what}: lse"


# ---------------------------------------------------------------------------------- windows
@pytest.mark.parametrize("window", [INT_MAX, INT_MAX - 7, 2 ** 30, 2 ** 31, 2 ** 32 + 3])
@pytest.mark.parametrize("lens_q,lens_k,hq,hkv,hd", [
    ([5, 3], [3, 3], 4, 2, 128),            # few rows
    ([16, 7, 2], [2, 0, 40], 2, 2, 64),
    ([130, 300], [20, 290], 8, 2, 128),     # many rows
    ([400], [130], 4, 4, 64),
])
def test_a_window_that_holds_every_key_hides_none(lens_q, lens_k, hq, hkv, hd, window):
    """More query than key rows (some see nothing) under windows up to and beyond the 32-bit limit."""
    text = _text()
    g = _gen(sum(lens_q) + hd)
    q = _randn(g, sum(lens_q), hq, hd)
    k, v = _randn(g, sum(lens_k), hkv, hd), _randn(g, sum(lens_k), hkv, hd)
    out, lse = text.prompt_attention(q, k, v, _cu(lens_q), max(lens_q), window=window, cu_seqlens_k=_cu(lens_k),
                                     return_lse=True)
    _check_device()
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        ref, rl, mag = ref_attention(q[a:a + n], k[b:b + m], v[b:b + m], 1 / math.sqrt(hd), True, 0)
        assert_same(out[a:a + n], lse[a:a + n], ref, rl, mag, f"{n} over {m}")
        a, b = a + n, b + m


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("q_lens,kv_lens", [([9, 30], [4, 20]), ([3], [1]), ([200], [150])])
def test_a_window_that_holds_the_whole_cache_hides_nothing(fmt, q_lens, kv_lens):
    text = _text()
    g = _gen(sum(q_lens))
    cache, table, q, ks, vs = _paged(g, fmt, q_lens, kv_lens, 4, 2, 128, 16)
    lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    out, lse = text.paged_attention(q, cache, _cu(q_lens), lens, table, max(q_lens), window=INT_MAX, return_lse=True)
    _check_device()
    a = 0
    for n, k, v in zip(q_lens, ks, vs):
        ref, rl, mag = ref_attention(q[a:a + n], k, v, 1 / math.sqrt(128), True, 0)
        assert_same(out[a:a + n], lse[a:a + n], ref, rl, mag, f"{n} over {k.shape[0]}")
        a += n


def test_windows_below_zero_are_refused_whatever_their_low_bits():
    text = _text()
    from wuxianhuabu_b200 import _lib, h3
    g = _gen(1)
    q = _randn(g, 4, 2, 64)
    for window in (-1, -2 ** 32, -2 ** 32 + 5):
        with pytest.raises(h3.WxError) as e:
            text.prompt_attention(q, q, q, _cu([4]), 4, window=window)
        assert e.value.status == _lib.WX_ERR_INVALID


# ------------------------------------------------------------- infinities and NaN in values
def _spoil(v, first, last):
    """Infinities and NaN in values at keys of [first, last): of one sign, of both in a column, NaN beside
    infinity, in the first and the last columns."""
    at = torch.linspace(first, last - 1, 7, device=v.device).long().tolist()
    v[at[0], 0, 0], v[at[1], 0, -1] = math.inf, -math.inf
    v[at[2], -1, 3], v[at[4], -1, 3] = math.inf, -math.inf
    v[at[2], -1, 33], v[at[3], -1, 33] = math.inf, math.inf
    v[at[4], 0, 40], v[at[6], 0, 40] = -math.inf, math.nan
    v[at[5], -1, -2], v[at[6], 0, 17] = -math.inf, math.inf


@pytest.mark.parametrize("hd,hq,hkv", [(128, 8, 2), (64, 4, 2), (64, 3, 3)])
@pytest.mark.parametrize("lens,causal,window,first,last", [
    ([300], True, 0, 0, 300),        # tiles that every row sees, and tiles under the diagonal
    ([300], True, 0, 250, 300),
    ([220, 260], True, 90, 0, 480),  # and tiles that the window cuts
    ([200], False, 0, 30, 200),
])
def test_prompt_attention_keeps_infinities(hd, hq, hkv, lens, causal, window, first, last):
    text = _text()
    g = _gen(sum(lens) + hd)
    n = sum(lens)
    q, k, v = _randn(g, n, hq, hd), _randn(g, n, hkv, hd), _randn(g, n, hkv, hd)
    _spoil(v, first, last)
    out, lse = text.prompt_attention(q, k, v, _cu(lens), max(lens), causal=causal, window=window, return_lse=True)
    _check_device()
    a = 0
    for m in lens:
        s = slice(a, a + m)
        ref, rl, mag = ref_attention(q[s], k[s], v[s], 1 / math.sqrt(hd), causal, window)
        assert_same(out[s], lse[s], ref, rl, mag, f"len {m}")
        a += m


@pytest.mark.parametrize("hd,hq,hkv,page", [(128, 4, 2, 16), (64, 4, 2, 64), (128, 16, 8, 32)])
@pytest.mark.parametrize("nq,n,window", [(1, 200, 0), (3, 200, 0), (7, 150, 60), (5, 4, 0), (100, 260, 0), (90, 2300, 0)])
def test_paged_attention_keeps_infinities(hd, hq, hkv, page, nq, n, window):
    """Values of the last keys, which only some of the new tokens see, and of keys that all of them see."""
    text = _text()
    g = _gen(nq + n + hd)
    cache, table, q, ks, vs = _paged(g, "bf16", [nq], [n], hq, hkv, hd, page)
    first = max(0, n - 2 * nq)
    _spoil(vs[0], first, n)
    j = torch.arange(n, device="cuda")
    cache.append(ks[0], vs[0], table[0].long()[j // page] * page + j % page)
    out, lse = text.paged_attention(q, cache, _cu([nq]), torch.tensor([n], dtype=torch.int32, device="cuda"), table, nq,
                                    window=window, return_lse=True)
    _check_device()
    # (the definition's product takes lq * lk * hd numbers a head: the keys before `first` are finite)
    ref, rl, mag = ref_attention(q, ks[0], vs[0], 1 / math.sqrt(hd), True, window)
    assert_same(out, lse, ref, rl, mag)


# --------------------------------------------------------------- NaN codes of an e4m3 cache
def _with_nan_codes(cache, table, page, ks, vs, spots):
    """NaN codes at spots (kind, key, head, column) of sequence 0; the expected values with them."""
    for i, (kind, j, h, c) in enumerate(spots):
        at = int(table[0, j // page])
        buf, ref = (cache.k, ks[0]) if kind == "k" else (cache.v, vs[0])
        buf.view(torch.uint8)[at, h, j % page, c] = 0x7f if i % 2 else 0xff
        ref[j, h, c] = math.nan


@pytest.mark.parametrize("hd,hq,hkv,page", [(128, 8, 2, 64), (64, 4, 4, 16), (128, 16, 2, 128)])
@pytest.mark.parametrize("nq,n,window", [(1, 150, 0), (2, 700, 0), (6, 150, 0), (6, 400, 130), (90, 150, 0), (300, 333, 0),
                                         (64, 3000, 0)])
@pytest.mark.parametrize("kind", ["v", "k"])
def test_nan_codes_of_an_e4m3_cache_are_nan(hd, hq, hkv, page, nq, n, window, kind):
    """Written by somebody else (this package's writes saturate): NaN for the rows that see them, in all
    columns for a key, in its own column for a value, and to nobody else; kv_read says the same."""
    text = _text()
    g = _gen(nq + n + hd)
    cache, table, q, ks, vs = _paged(g, "e4m3", [nq], [n], hq, hkv, hd, page)
    if kind == "v":
        spots = [("v", 0, 0, 0), ("v", n // 2, hkv - 1, 37), ("v", n // 2, hkv - 1, hd - 1), ("v", n - 1, 0, 5),
                 ("v", n - 1, hkv - 1, 16), ("v", max(0, n - nq // 2 - 1), 0, 63), ("v", n - n // 3, 0, 5)]
    else:
        spots = [("k", n - 1, 0, 9), ("k", max(0, n - nq // 2 - 1), hkv - 1, hd - 1), ("k", n - 2, hkv - 1, 0)]
    _with_nan_codes(cache, table, page, ks, vs, spots)
    last = int(table[0, (n - 1) // page])
    if n % page:  # behind the last key: NaN codes and scales that nobody sees
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[last, :, n % page:] = 0x7f
        cache.k_scale[last, :, n % page:] = math.nan
        cache.v_scale[last, :, n % page:] = math.nan
    out, lse = text.paged_attention(q, cache, _cu([nq]), torch.tensor([n], dtype=torch.int32, device="cuda"), table, nq,
                                    window=window, return_lse=True)
    j = torch.arange(n, device="cuda")
    kr, vr = cache.read(table[0].long()[j // page] * page + j % page)
    _check_device()
    assert torch.equal(torch.isnan(kr), torch.isnan(ks[0])) and torch.equal(torch.isnan(vr), torch.isnan(vs[0]))
    scale = 1 / math.sqrt(hd)
    if kind == "v":
        # the definition with zeros in those places, and NaN for the rows and columns that see one
        ref, rl, mag = ref_attention(q, ks[0], torch.nan_to_num(vs[0], nan=0.0), scale, True, window)
        i = torch.arange(nq, device="cuda")[:, None] + (n - nq)
        sees = (j[None] <= i) & ((j[None] > i - window) if window else torch.ones_like(j[None] <= i))
        hit = torch.einsum("ij,jhd->ihd", sees.float(), torch.isnan(vs[0]).float()) > 0
        ref[hit.repeat_interleave(hq // hkv, 1)] = math.nan
    else:
        ref, rl, mag = ref_attention(q, ks[0], vs[0], scale, True, window)
    assert_same(out, lse, ref, rl, mag)


def test_every_e4m3_code_reads_as_itself():
    """All 256 codes, in a cache made elsewhere: read back, and as the value of the only key of a sequence."""
    text = _text()
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(2, 1, 1, 128).expand(2, 1, 16, 128).contiguous()
    v = codes.view(torch.float8_e4m3fn)
    ones = torch.ones((2, 1, 16), dtype=torch.float32, device="cuda")
    zeros = torch.zeros_like(codes).view(torch.float8_e4m3fn)
    cache = text.PagedKVCache.from_tensors(zeros, v, ones, ones.clone())
    want = v.float()[:, 0, 0]
    got = cache.read(torch.tensor([3, 20], device="cuda"))[1][:, 0].float()
    q = torch.ones((2, 1, 128), dtype=BF16, device="cuda")
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    few = text.paged_attention(q, cache, _cu([1, 1]), lens, table, 1)[:, 0].float()
    many = text.paged_attention(torch.ones((200, 1, 128), dtype=BF16, device="cuda"), cache, _cu([100, 100]), lens, table,
                                100)[[99, 199], 0].float()
    _check_device()
    for x in (got, few, many):
        assert torch.equal(torch.nan_to_num(x, nan=1e9), torch.nan_to_num(want, nan=1e9))


# ------------------------------------------------------------------------- lengths that mislead
@pytest.mark.parametrize("lens", [[100, 7, 300], [1000]])
def test_a_longest_length_that_is_too_small_changes_nothing(lens):
    """It chooses the kernel: the one for few rows takes any number of them."""
    text = _text()
    g = _gen(sum(lens))
    q, k, v = (_randn(g, sum(lens), h, 128) for h in (8, 2, 2))
    for max_len in (0, 1, 2, -(-max(lens) // 2)):
        out, lse = text.prompt_attention(q, k, v, _cu(lens), max_len, return_lse=True)
        _check_device()
        a = 0
        for n in lens:
            s = slice(a, a + n)
            ref, rl, mag = ref_attention(q[s], k[s], v[s], 1 / math.sqrt(128), True, 0)
            assert_same(out[s], lse[s], ref, rl, mag, f"len {n}, longest {max_len}")
            a += n


def test_more_work_than_the_kernel_for_few_rows_can_count_is_an_error():
    """262,400 tokens that are announced as one: 64 heads of 32,800 tiles of 8 rows over 2,050 units of keys are
    more than 2^32. Nothing is computed, and the error word says so."""
    text = _text()
    from wuxianhuabu_b200 import h3
    n = 262400
    assert 64 * (n // 8) * (n // 128) > 2 ** 32
    q = torch.zeros((n, 64, 64), dtype=BF16, device="cuda")
    text.prompt_attention(q, q, q, _cu([n]), 1)
    with pytest.raises(h3.WxError):
        _check_device()
    small = _randn(_gen(1), 3, 64, 64)
    out, lse = text.prompt_attention(small, small, small, _cu([3]), 3, return_lse=True)
    _check_device()
    ref, rl, mag = ref_attention(small, small, small, 1 / 8, True, 0)
    assert_same(out, lse, ref, rl, mag)


# -------------------------------------------------------------------------- alone and in a batch
@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [3, 2, 1, 4], [70, 5, 33, 1]])
def test_a_sequence_alone_and_in_a_batch(fmt, q_lens):
    """The batch deals the keys to other CTAs and joins other pieces: both are within the definition's
    tolerance, and a sequence does not reach its neighbours' rows."""
    text = _text()
    g = _gen(sum(q_lens))
    kv = [4000, 900, 2222, 17]
    cache, table, q, ks, vs = _paged(g, fmt, q_lens, kv, 8, 2, 128, 64)
    lens = torch.tensor(kv, dtype=torch.int32, device="cuda")
    out, lse = text.paged_attention(q, cache, _cu(q_lens), lens, table, max(q_lens), return_lse=True)
    a = 0
    for i, n in enumerate(q_lens):
        s = slice(a, a + n)
        alone, lse1 = text.paged_attention(q[s], cache, _cu([n]), lens[i:i + 1], table[i:i + 1], n, return_lse=True)
        _check_device()
        ref, rl, mag = ref_attention(q[s], ks[i], vs[i], 1 / math.sqrt(128), True, 0)
        assert_same(out[s], lse[s], ref, rl, mag, f"{i} in the batch")
        assert_same(alone, lse1, ref, rl, mag, f"{i} alone")
        a += n
