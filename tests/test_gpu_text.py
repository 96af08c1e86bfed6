"""The text-side operators against plain 64-bit restatements of their definitions: rotary
positions, the paged (quantised) K/V cache, attention over packed prompts and attention of new
tokens over the cache.

Tolerances, set from the arithmetic:
* rope: both products and the sum are fp32 over fp32 tables (relative error 2^-24 each, at most
  4 of them), then one rounding to bf16 (8 significant bits: 2^-8 of the value): 2^-8 |y| + 2^-21 (|x1| + |x2|);
* cache: the stored value is the nearest of its format to x * (max / amax) formed with two fp32
  roundings: half a step of the format, plus 2^-22 relative, plus the bf16 rounding of the read;
* attention: the weights are rounded to bf16 once (2^-8 of each weight, so 2^-8 sum w|v|), the
  output once (2^-8 |o|); scores, maxima, sums and the exponential are fp32 with a total relative
  error of a weight below 2^-14 for these score magnitudes.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64
BF16 = torch.bfloat16


def _text():
    from wuxianhuabu_b200 import text
    return text


def _check_device():
    from wuxianhuabu_b200 import h3
    h3.context().check_device()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(BF16)


# ------------------------------------------------------------------------------- references
def ref_inv_freq(rot, base, scaling):
    inv = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling is None or scaling.kind == "none":
        return inv
    if scaling.kind == "linear":
        return [f / scaling.factor for f in inv]
    out = []
    for f in inv:
        turns = scaling.original_positions * f / (2 * math.pi)
        w = min(1.0, max(0.0, (turns - scaling.low) / (scaling.high - scaling.low)))
        out.append((1 - w) * f / scaling.factor + w * f)
    return out


def ref_rope(x, pos, inv, interleaved, magnitude=1.0):
    """x [T, H, D] in 64 bits."""
    rot = 2 * len(inv)
    ang = pos.to(F64)[:, None] * torch.tensor(inv, dtype=F64, device=x.device)[None]
    c, s = (ang.cos() * magnitude)[:, None], (ang.sin() * magnitude)[:, None]
    x = x.to(F64)
    y = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    mag = torch.zeros_like(x)
    mag[..., a] = mag[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, mag


def ref_attention(q, k, v, scale, causal, window):
    """One sequence, 64 bits: out, lse and sum w |v| (the scale of the rounding errors)."""
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    lq, hq, _ = q.shape
    lk, hkv, _ = k.shape
    grp = hq // hkv
    k, v = k.repeat_interleave(grp, 1), v.repeat_interleave(grp, 1)
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    i = torch.arange(lq, device=q.device)[:, None] + (lk - lq)
    j = torch.arange(lk, device=q.device)[None]
    see = torch.ones((lq, lk), dtype=torch.bool, device=q.device)
    if causal:
        see &= j <= i
    if window:
        see &= j > i - window
    s = s.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, -1) if lk else torch.full((hq, lq), -math.inf, dtype=F64, device=q.device)
    w = torch.where(see[None], (s - torch.where(lse.isinf(), torch.zeros_like(lse), lse)[..., None]).exp(),
                    torch.zeros((), dtype=F64, device=q.device))
    # keys that a row does not see do not count, whatever they hold
    if torch.isfinite(v).all():
        out, mag = torch.einsum("hij,jhd->ihd", w, v), torch.einsum("hij,jhd->ihd", w, v.abs())
    else:
        prod = torch.where(see[None, :, :, None], w[..., None] * v.permute(1, 0, 2)[:, None],
                           torch.zeros((), dtype=F64, device=q.device))
        out, mag = prod.sum(2).permute(1, 0, 2), prod.abs().sum(2).permute(1, 0, 2)
    return out, lse.T, mag


def assert_attention(out, lse, ref, rlse, mag, what=""):
    ok = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(out), ok), f"{what}: finite where it should not be, or the reverse"
    err = (out.to(F64) - ref).abs()
    tol = 2.0 ** -8 * (ref.abs() + mag) * (1 + 2.0 ** -7) + 2.0 ** -14 * mag
    over = (err > tol) & ok
    assert not over.any(), f"{what}: {int(over.sum())} outputs off, worst {float((err / (tol + 1e-30))[ok].max()):.2f}x"
    if lse is not None:
        empty = rlse == -math.inf
        assert torch.equal(lse == -math.inf, empty), f"{what}: empty rows"
        fin = torch.isfinite(rlse)
        e = (lse.to(F64) - rlse)[fin].abs()
        assert e.numel() == 0 or float((e - 2.0 ** -20 * rlse[fin].abs()).max()) < 2e-5, f"{what}: lse {float(e.max())}"


# ------------------------------------------------------------------------------------- rope
@pytest.mark.parametrize("tokens,heads,hd,rot,interleaved,scaling,first", [
    (1, 1, 128, 128, False, "none", 0),
    (7, 5, 64, 64, True, "none", 3),
    (33, 40, 128, 64, True, "by_parts", 100003),
    (129, 12, 128, 24, False, "linear", 65535),
    (50, 3, 64, 8, False, "by_parts", 131000),
    (2050, 9, 128, 128, False, "none", 1),
])
def test_rope(tokens, heads, hd, rot, interleaved, scaling, first):
    text = _text()
    sc = None if scaling == "none" else text.RopeScaling(scaling, 8.0, magnitude=1.25)
    tab = text.RopeTable(rot, first + tokens, base=500000.0, interleaved=interleaved, scaling=sc)
    g = _gen(tokens)
    packed = _randn(g, tokens, heads + 3, hd)
    x = packed[:, 2:2 + heads]  # a slice of a packed projection: the token stride exceeds heads * hd
    pos = torch.randperm(tokens, generator=g, device="cuda").to(torch.int32) + first
    y = tab.apply(x, pos)
    _check_device()
    inv = ref_inv_freq(rot, 500000.0, sc)
    assert np.allclose(tab.inv_freq, inv, rtol=1e-14, atol=0)
    ref, mag = ref_rope(x, pos, inv, interleaved, 1.25 if sc else 1.0)
    assert ((y.to(F64) - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -21 * mag * 1.25).all()
    assert torch.equal(y[..., rot:], x[..., rot:])
    before = packed.clone()
    assert tab.apply(x, pos, out=x) is x  # in place, through the slice
    assert torch.equal(x, y) and torch.equal(packed[:, :2], before[:, :2])
    assert torch.equal(packed[:, 2 + heads:], before[:, 2 + heads:])


def test_rope_position_outside_the_table_is_reported():
    text = _text()
    from wuxianhuabu_b200 import h3
    tab = text.RopeTable(64, 16)
    x = _randn(_gen(1), 3, 2, 64)
    out = torch.full_like(x, 7.0)
    tab.apply(x, torch.tensor([1, 16, -1], dtype=torch.int32, device="cuda"), out=out)
    with pytest.raises(h3.WxError):
        _check_device()
    assert (out[1:] == 7.0).all() and not (out[0] == 7.0).any()
    tab.apply(x, torch.tensor([1, 15, 0], dtype=torch.int32, device="cuda"))
    _check_device()


# ------------------------------------------------------------------------------------ cache
def _slots(g, n, pages, page):
    return torch.randperm(pages * page, generator=g, device="cuda")[:n].contiguous()


def _half_step(x, fmt):
    """Half a step of the format at x, in 64 bits, per element of a row [..., hd]."""
    amax = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        return (amax / 127 / 2).expand_as(x)
    scale = amax / 448
    e = torch.floor(torch.log2((x / torch.where(scale > 0, scale, torch.ones_like(scale))).abs().clamp(min=2.0 ** -9)))
    return scale * 2.0 ** (e.clamp(min=-6) - 3) / 2


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("tokens,kv_heads,hd,page,roped", [
    (1, 1, 128, 16, False), (1, 8, 64, 16, True), (19, 3, 64, 32, False), (200, 4, 128, 64, True),
    (333, 8, 128, 256, False), (1500, 2, 128, 128, True),
])
def test_cache_write_and_read(fmt, tokens, kv_heads, hd, page, roped):
    text = _text()
    pages = (tokens + page - 1) // page + 2
    cache = text.PagedKVCache(pages, page, kv_heads, hd, fmt)
    g = _gen(tokens + hd)
    hq = 2 * kv_heads + 1
    qkv = _randn(g, tokens, hq + 2 * kv_heads, hd)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + kv_heads], qkv[:, hq + kv_heads:]
    slots = _slots(g, tokens, pages, page)
    if roped:
        pos = torch.arange(tokens, dtype=torch.int32, device="cuda") + 11
        rot = hd // 2
        tab = text.RopeTable(rot, tokens + 11, interleaved=True)
        got_q = cache.append_roped(q, k, v, slots, tab, pos)
        assert torch.equal(got_q, tab.apply(q, pos))  # the same rotation, bit for bit
        k64, kmag = ref_rope(k, pos, ref_inv_freq(rot, 10000.0, None), True)
    else:
        cache.append(k, v, slots)
        k64, kmag = k.to(F64), torch.zeros((), dtype=F64, device="cuda")
    gk, gv = cache.read(slots)
    _check_device()
    for got, ref, extra in ((gk, k64, kmag), (gv, v.to(F64), 0.0)):
        tol = 2.0 ** -8 * ref.abs() + 2.0 ** -21 * extra
        if fmt != "bf16":
            half = _half_step(ref, fmt)
            tol = tol + half * (1 + 2.0 ** -8) + 2.0 ** -21 * ref.abs().amax(-1, keepdim=True)
        assert ((got.to(F64) - ref).abs() <= tol).all(), fmt
    if fmt == "bf16" and not roped:
        assert torch.equal(gk, k) and torch.equal(gv, v)
    # rows nobody wrote stay zero
    other = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    other[slots] = False
    rest = other.nonzero().flatten()
    assert (cache.read(rest)[0] == 0).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_cache_stored_values_are_the_definition(fmt):
    """Stored values and scales, bit for bit, with ties, tiny, zero and non-finite rows."""
    text = _text()
    g = _gen(5)
    x = _randn(g, 64, 2, 128)
    x[1] = 0
    x[2] *= 2.0 ** -110
    x[3, 0, 5] = math.inf
    x[4, 1, 7] = math.nan
    x[5] = torch.linspace(-254, 254, 128, device="cuda").to(BF16)  # ties at x = amax * (n + 1/2) / 127
    x[6, :, 1:] = x[6, :, :1] / 2
    x[7] *= 2.0 ** 100
    cache = text.PagedKVCache(4, 16, 2, 128, fmt)
    slots = torch.arange(64, device="cuda")
    cache.append(x, x, slots)
    top = 127.0 if fmt == "int8" else 448.0
    xf = x.float()
    amax = xf.abs().amax(-1)
    finite = torch.isfinite(xf).all(-1)
    live = finite & (amax >= 2.0 ** -100)
    tops = torch.full_like(amax, top)  # (torch multiplies by the reciprocal of a plain number)
    inv = torch.where(live, tops / amax, torch.zeros_like(amax))
    y = torch.where(live[..., None], xf * inv[..., None], torch.zeros_like(xf))
    want = y.round().to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn).view(torch.int8)
    scale = torch.where(live, amax / tops, torch.zeros_like(amax))
    scale = torch.where(finite, scale, torch.full_like(scale, math.nan))
    got = cache.k.view(torch.int8).permute(0, 2, 1, 3).reshape(64, 2, 128)
    gs = cache.k_scale.permute(0, 2, 1).reshape(64, 2)
    assert torch.equal(got, want)
    assert torch.equal(torch.nan_to_num(gs, nan=-1.0), torch.nan_to_num(scale, nan=-1.0))
    back, _ = cache.read(slots)
    assert torch.isnan(back[3, 0]).all() and torch.isnan(back[4, 1]).all() and torch.isfinite(back[3, 1]).all()
    assert (back[1] == 0).all() and (back[2] == 0).all()


def test_cache_skipped_and_wrong_slots():
    text = _text()
    from wuxianhuabu_b200 import h3
    cache = text.PagedKVCache(2, 16, 1, 64, "int8")
    x = _randn(_gen(2), 3, 1, 64)
    cache.append(x, x, torch.tensor([4, -1, 9], device="cuda"))
    _check_device()
    k, _ = cache.read(torch.tensor([4, -1, 9, 5], device="cuda"))
    _check_device()
    assert k[0].any() and not k[1].any() and k[2].any() and not k[3].any()
    cache.append(x, x, torch.tensor([5, 32, 6], device="cuda"))  # slot 32 is past the end: skipped, reported
    with pytest.raises(h3.WxError):
        _check_device()
    assert cache.read(torch.tensor([5, 6], device="cuda"))[0].any(-1).all()
    _check_device()


# --------------------------------------------------------------------------- prompt attention
def _cu(lens):
    return torch.tensor(np.cumsum([0] + list(lens)), dtype=torch.int32, device="cuda")


PROMPTS = [
    ([1], 4, 2, 128, True, 0),
    ([5, 0, 3], 6, 2, 64, True, 0),
    ([16, 17, 15], 7, 1, 128, True, 0),
    ([128, 129, 127, 1], 8, 8, 128, True, 0),
    ([300, 77], 8, 2, 128, True, 0),
    ([513], 28, 4, 128, True, 0),
    ([700, 33], 4, 4, 64, True, 0),
    ([640, 257], 8, 1, 64, True, 100),
    ([400, 1, 222], 6, 2, 128, True, 1),
    ([384, 90], 4, 1, 128, False, 0),
    ([1025, 260], 3, 3, 64, False, 0),
    ([900], 5, 1, 128, True, 333),
    ([140, 60], 40, 2, 64, True, 0),
    ([2300], 2, 1, 128, True, 0),
]


@pytest.mark.parametrize("lens,hq,hkv,hd,causal,window", PROMPTS)
def test_prompt_attention(lens, hq, hkv, hd, causal, window):
    text = _text()
    g = _gen(sum(lens) + hq)
    qkv = _randn(g, sum(lens), hq + 2 * hkv, hd)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    scale = 1.3 / math.sqrt(hd)
    out, lse = text.prompt_attention(q, k, v, _cu(lens), max(lens), scale=scale, causal=causal, window=window,
                                     return_lse=True)
    _check_device()
    a = 0
    for n in lens:
        if n:
            ref, rl, mag = ref_attention(q[a:a + n], k[a:a + n], v[a:a + n], scale, causal, window)
            assert_attention(out[a:a + n], lse[a:a + n], ref, rl, mag, f"len {n}")
        a += n


@pytest.mark.parametrize("lens_q,lens_k,hq,hkv,hd,causal,window", [
    ([5, 40, 9], [9, 7, 0], 4, 2, 128, True, 0),       # more queries than keys: rows that see nothing
    ([130, 1, 300], [20, 300, 300], 8, 1, 64, True, 0),
    ([64, 200], [500, 130], 6, 3, 128, True, 70),
    ([33, 1], [0, 0], 2, 2, 64, False, 0),
    ([70], [1000], 4, 4, 128, False, 0),
])
def test_prompt_attention_with_other_key_lengths(lens_q, lens_k, hq, hkv, hd, causal, window):
    text = _text()
    g = _gen(sum(lens_q) + sum(lens_k))
    q = _randn(g, sum(lens_q), hq, hd)
    k, v = _randn(g, sum(lens_k), hkv, hd), _randn(g, sum(lens_k), hkv, hd)
    out = torch.full_like(q, math.nan)
    out, lse = text.prompt_attention(q, k, v, _cu(lens_q), max(lens_q), causal=causal, window=window,
                                     cu_seqlens_k=_cu(lens_k), out=out, return_lse=True)
    _check_device()
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        ref, rl, mag = ref_attention(q[a:a + n], k[b:b + m], v[b:b + m], 1 / math.sqrt(hd), causal, window)
        assert_attention(out[a:a + n], lse[a:a + n], ref, rl, mag, f"{n} over {m}")
        a, b = a + n, b + m


@pytest.mark.parametrize("hd,lens,window", [(128, [200, 150], 0), (64, [150, 200], 0), (128, [300], 40)])
def test_prompt_attention_ignores_what_a_row_does_not_see(hd, lens, window):
    """NaN and infinity in the keys and values of later tokens, and of the neighbour sequence."""
    text = _text()
    g = _gen(hd)
    n = sum(lens)
    q, k, v = _randn(g, n, 4, hd), _randn(g, n, 2, hd), _randn(g, n, 2, hd)
    k[90, 0], k[120, 1, 3] = math.nan, math.inf
    v[100, 0, 5], v[101, 1, 63], v[140, 0, 0] = math.nan, -math.inf, math.inf
    v[n - 1] = math.nan
    out, lse = text.prompt_attention(q, k, v, _cu(lens), max(lens), causal=True, window=window, return_lse=True)
    _check_device()
    a = 0
    for m in lens:
        ref, rl, mag = ref_attention(q[a:a + m], k[a:a + m], v[a:a + m], 1 / math.sqrt(hd), True, window)
        assert_attention(out[a:a + m], None, ref, rl, mag, f"len {m}")
        a += m


def test_prompt_attention_large_scores():
    """Scores far apart: the running maximum moves by hundreds, most weights underflow to zero."""
    text = _text()
    g = _gen(9)
    q, k, v = _randn(g, 300, 2, 128) * 6, _randn(g, 300, 1, 128) * 6, _randn(g, 300, 1, 128)
    out, lse = text.prompt_attention(q, k, v, _cu([300]), 300, return_lse=True)
    _check_device()
    ref, rl, mag = ref_attention(q, k, v, 1 / math.sqrt(128), True, 0)
    # scores reach several hundred: 2^-24 of them, over 128 products, moves a weight by 2^-11
    err = (out.to(F64) - ref).abs()
    assert (err <= (2.0 ** -8 + 2.0 ** -10) * (ref.abs() + mag) * 1.01).all()
    assert float((lse.to(F64) - rl).abs().max()) < 1e-3


# ---------------------------------------------------------------------------- paged attention
def _paged(g, fmt, q_lens, kv_lens, hq, hkv, hd, page, spread=1.0):
    text = _text()
    need = [(n + page - 1) // page for n in kv_lens]
    pages = sum(need) + 2
    cache = text.PagedKVCache(pages, page, hkv, hd, fmt)
    order = torch.randperm(pages, generator=g, device="cuda")
    table = torch.full((len(kv_lens), max(need + [1])), -7, dtype=torch.int32, device="cuda")
    ks, vs, at = [], [], 0
    # what earlier sequences left behind: not zeros
    junk = _randn(g, pages * page, hkv, hd) * 50
    cache.append(junk, junk, torch.arange(pages * page, device="cuda"))
    for i, n in enumerate(kv_lens):
        mine = order[at:at + need[i]]
        at += need[i]
        table[i, :need[i]] = mine.to(torch.int32)
        j = torch.arange(n, device="cuda")
        slots = mine[j // page] * page + j % page
        k, v = _randn(g, n, hkv, hd), _randn(g, n, hkv, hd) * spread
        if n:
            cache.append(k, v, slots)
            if fmt != "bf16":  # what the cache holds, as fp32 value * scale in 64 bits
                pg, off = mine[j // page], j % page
                k = cache.k.view(torch.int8)[pg, :, off].view(cache.k.dtype).float().to(F64) * \
                    cache.k_scale[pg, :, off].to(F64)[..., None]
                v = cache.v.view(torch.int8)[pg, :, off].view(cache.v.dtype).float().to(F64) * \
                    cache.v_scale[pg, :, off].to(F64)[..., None]
        ks.append(k)
        vs.append(v)
    q = _randn(g, sum(q_lens), hq, hd)
    return cache, table, q, ks, vs


PAGED = [
    ([1], [1], 2, 1, 128, 16, 0),
    ([1], [0], 2, 1, 64, 16, 0),
    ([1, 1, 1], [17, 200, 33], 4, 4, 64, 16, 0),
    ([1, 1], [1000, 129], 8, 1, 128, 64, 0),
    ([1] * 9, [5, 700, 64, 63, 65, 1, 2000, 128, 300], 14, 2, 128, 32, 0),
    ([1, 1, 1], [3000, 100, 511], 6, 2, 64, 128, 100),
    ([3, 1, 5], [50, 400, 5], 7, 1, 128, 16, 0),
    ([4, 0, 8], [1500, 77, 140], 8, 2, 64, 64, 0),
    ([9, 30], [12, 20], 4, 2, 128, 32, 0),             # 30 queries, 20 keys: rows that see nothing
    ([100, 37], [400, 37], 8, 2, 128, 64, 0),
    ([260], [900], 4, 1, 64, 256, 0),
    ([130, 20], [300, 1000], 28, 4, 128, 16, 90),
    ([2], [9000], 16, 2, 128, 64, 0),
    ([40], [5000], 8, 1, 128, 64, 0),
]


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,hd,page,window", PAGED)
def test_paged_attention(fmt, q_lens, kv_lens, hq, hkv, hd, page, window):
    text = _text()
    g = _gen(sum(kv_lens) + hq)
    cache, table, q, ks, vs = _paged(g, fmt, q_lens, kv_lens, hq, hkv, hd, page, spread=3.0)
    lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    out, lse = text.paged_attention(q, cache, _cu(q_lens), lens, table, max(q_lens), window=window, return_lse=True)
    _check_device()
    a = 0
    for n, k, v in zip(q_lens, ks, vs):
        if n:
            ref, rl, mag = ref_attention(q[a:a + n], k, v, 1 / math.sqrt(hd), True, window)
            assert_attention(out[a:a + n], lse[a:a + n], ref, rl, mag, f"{n} over {k.shape[0]}")
        a += n


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("q_len", [1, 6, 90])
def test_paged_attention_ignores_unwritten_slots(fmt, q_len):
    """The rest of the last page holds NaN (in an 8-bit cache: NaN scales and codes)."""
    text = _text()
    g = _gen(q_len)
    n = 150
    cache, table, q, ks, vs = _paged(g, fmt, [q_len], [n], 8, 2, 128, 64)
    last = int(table[0, 2])
    for t in (cache.k, cache.v):
        if fmt == "bf16":
            t[last, :, n % 64:] = math.nan
        else:
            t.view(torch.int8)[last, :, n % 64:] = 0x7f
    if fmt != "bf16":
        cache.k_scale[last, :, n % 64:] = math.nan
        cache.v_scale[last, :, n % 64:] = math.nan
    out, lse = text.paged_attention(q, cache, _cu([q_len]), torch.tensor([n], dtype=torch.int32, device="cuda"),
                                    table, q_len, return_lse=True)
    _check_device()
    ref, rl, mag = ref_attention(q, ks[0], vs[0], 1 / math.sqrt(128), True, 0)
    assert_attention(out, lse, ref, rl, mag, fmt)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [3, 2, 1], [70, 5, 33]])
def test_paged_attention_is_deterministic_and_alone_or_in_a_batch(q_lens):
    """The same call twice gives the same bits, whichever CTA joins the pieces."""
    text = _text()
    g = _gen(77)
    kv = [4000, 900, 2222]
    cache, table, q, _, _ = _paged(g, "int8", q_lens, kv, 8, 2, 128, 64)
    lens = torch.tensor(kv, dtype=torch.int32, device="cuda")
    first = text.paged_attention(q, cache, _cu(q_lens), lens, table, max(q_lens), return_lse=True)
    for _ in range(10):
        again = text.paged_attention(q, cache, _cu(q_lens), lens, table, max(q_lens), return_lse=True)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    _check_device()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,hd,page,window", [
    ([90], [4100], 8, 2, 128, 64, 0),                      # one item, cut into pieces of its keys
    ([70, 0, 200, 66], [2049, 300, 1025, 0], 4, 1, 64, 16, 0),  # some cut, some not, one without keys
    ([130, 66], [6000, 2048], 4, 4, 128, 32, 2500),        # a window that pieces begin inside
    ([150], [2900], 1, 1, 64, 256, 0),
])
def test_paged_attention_few_rows_long_keys(fmt, q_lens, kv_lens, hq, hkv, hd, page, window):
    test_paged_attention(fmt, q_lens, kv_lens, hq, hkv, hd, page, window)


@pytest.mark.parametrize("hd,causal,window", [(128, True, 0), (64, False, 0), (128, True, 1700)])
def test_prompt_attention_few_rows_long_keys(hd, causal, window):
    test_prompt_attention_with_other_key_lengths([50, 3], [5003, 1024], 8, 2, hd, causal, window)


def test_pieces_of_long_keys_ignore_what_a_row_does_not_see():
    """NaN in the value of a key that only the last rows see, and past the end of the last page."""
    text = _text()
    g = _gen(12)
    n, nq = 3000, 80
    cache, table, q, ks, vs = _paged(g, "bf16", [nq], [n], 4, 1, 128, 64)
    page, off = int(table[0, (n - 20) // 64]), (n - 20) % 64
    cache.v[page, :, off, 5] = math.nan
    cache.v[int(table[0, n // 64]), :, n % 64:] = math.inf
    out = text.paged_attention(q, cache, _cu([nq]), torch.tensor([n], dtype=torch.int32, device="cuda"), table, nq)
    _check_device()
    sees = torch.arange(nq, device="cuda") + n - nq >= n - 20
    assert torch.isnan(out[sees][:, :, 5]).all()
    rest = torch.ones(128, dtype=torch.bool, device="cuda")
    rest[5] = False
    ref, rl, mag = ref_attention(q, ks[0], vs[0], 1 / math.sqrt(128), True, 0)
    assert_attention(out[~sees], None, ref[~sees], rl[~sees], mag[~sees], "rows before the key")
    assert_attention(out[sees][..., rest], None, ref[sees][..., rest], rl[sees], mag[sees][..., rest], "other columns")


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_pieces_are_joined_in_order(fmt):
    text = _text()
    g = _gen(78)
    kv, nq = [9000, 2500], [100, 77]
    cache, table, q, _, _ = _paged(g, fmt, nq, kv, 8, 2, 128, 64)
    lens = torch.tensor(kv, dtype=torch.int32, device="cuda")
    first = text.paged_attention(q, cache, _cu(nq), lens, table, max(nq), return_lse=True)
    for _ in range(10):
        again = text.paged_attention(q, cache, _cu(nq), lens, table, max(nq), return_lse=True)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    _check_device()


def test_paged_equals_prompt_attention():
    """A prompt written to a bf16 cache and attended as one chunk gives what the packed call gives."""
    text = _text()
    g = _gen(3)
    n, hq, hkv = 500, 8, 2
    q, k, v = _randn(g, n, hq, 128), _randn(g, n, hkv, 128), _randn(g, n, hkv, 128)
    cache = text.PagedKVCache(8, 64, hkv, 128)
    cache.append(k, v, torch.arange(n, device="cuda"))
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None].contiguous()
    a = text.prompt_attention(q, k, v, _cu([n]), n)
    b = text.paged_attention(q, cache, _cu([n]), torch.tensor([n], dtype=torch.int32, device="cuda"), table, n)
    _check_device()
    ref, rl, mag = ref_attention(q, k, v, 1 / math.sqrt(128), True, 0)
    assert_attention(a, None, ref, rl, mag, "packed")
    assert_attention(b, None, ref, rl, mag, "paged")


@pytest.mark.parametrize("fmt,pages", [("bf16", 9000), ("int8", 18000)])
@pytest.mark.parametrize("q_len", [1, 70])
def test_cache_beyond_32_bit_offsets(fmt, pages, q_len):
    """More than 2^32 bytes of keys: pages from the end, the middle and the start of the cache."""
    text = _text()
    g = _gen(q_len)
    hq, hkv, hd, page, n = 16, 8, 128, 256, 600
    cache = text.PagedKVCache(pages, page, hkv, hd, fmt)
    assert cache.k.numel() * cache.k.element_size() > 1 << 32
    table = torch.tensor([[pages - 1, pages // 2, 0]], dtype=torch.int32, device="cuda")
    j = torch.arange(n, device="cuda")
    slots = table[0].long()[j // page] * page + j % page
    k, v = _randn(g, n, hkv, hd), _randn(g, n, hkv, hd)
    cache.append(k, v, slots)
    ks, vs = cache.read(slots)
    if fmt == "bf16":
        assert torch.equal(ks, k) and torch.equal(vs, v)
    else:
        pg, off = table[0].long()[j // page], j % page
        ks = cache.k[pg, :, off].to(F64) * cache.k_scale[pg, :, off].to(F64)[..., None]
        vs = cache.v[pg, :, off].to(F64) * cache.v_scale[pg, :, off].to(F64)[..., None]
        assert ((ks - k.to(F64)).abs() <= 0.5001 * cache.k_scale[pg, :, off].to(F64)[..., None]).all()
    q = _randn(g, q_len, hq, hd)
    out, lse = text.paged_attention(q, cache, _cu([q_len]), torch.tensor([n], dtype=torch.int32, device="cuda"),
                                    table, q_len, return_lse=True)
    _check_device()
    ref, rl, mag = ref_attention(q, ks, vs, 1 / math.sqrt(hd), True, 0)
    assert_attention(out, lse, ref, rl, mag, fmt)


# ---------------------------------------------------------------------------------- refusals
def test_refusals():
    text = _text()
    from wuxianhuabu_b200 import _lib, h3
    g = _gen(1)
    q, k = _randn(g, 4, 4, 128), _randn(g, 4, 2, 128)
    cu = _cu([4])

    def refused(status, fn):
        with pytest.raises(h3.WxError) as e:
            fn()
        assert e.value.status == status, e.value

    bad, unsup = _lib.WX_ERR_INVALID, _lib.WX_ERR_UNSUPPORTED
    refused(bad, lambda: text.prompt_attention(q.float(), k, k, cu, 4))
    refused(bad, lambda: text.prompt_attention(q, _randn(g, 4, 3, 128), _randn(g, 4, 3, 128), cu, 4))
    refused(bad, lambda: text.prompt_attention(q, k, k[:3], cu, 4))
    refused(bad, lambda: text.prompt_attention(q, k[:3], k[:3], cu, 4))
    refused(bad, lambda: text.prompt_attention(q, k, k, cu.long(), 4))
    refused(bad, lambda: text.prompt_attention(q, k, k, cu, 4, scale=-1.0))
    refused(bad, lambda: text.prompt_attention(q, k, k, cu, 4, causal=False, window=8))
    refused(bad, lambda: text.prompt_attention(q, k, k, cu, 4, window=-1))
    refused(bad, lambda: text.prompt_attention(q.transpose(1, 2).contiguous().transpose(1, 2), k, k, cu, 4))
    refused(unsup, lambda: text.prompt_attention(_randn(g, 4, 4, 96), _randn(g, 4, 2, 96), _randn(g, 4, 2, 96), cu, 4))
    wide = _randn(g, 4, 260, 64)
    refused(unsup, lambda: text.prompt_attention(wide, _randn(g, 4, 1, 64), _randn(g, 4, 1, 64), cu, 4))
    off = torch.empty(4 * 4 * 128 + 1, dtype=BF16, device="cuda")[1:].view(4, 4, 128)  # not 16-byte aligned
    refused(bad, lambda: text.prompt_attention(off, k, k, cu, 4))
    refused(unsup, lambda: text.PagedKVCache(2, 24, 1, 64).append(k[:, :1, :64], k[:, :1, :64],
                                                                  torch.zeros(4, dtype=torch.int64, device="cuda")))
    cache = text.PagedKVCache(2, 16, 2, 128, "int8")
    lens = torch.tensor([4], dtype=torch.int32, device="cuda")
    table = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    refused(bad, lambda: text.paged_attention(_randn(g, 4, 3, 128), cache, cu, lens, table, 4))
    refused(bad, lambda: text.paged_attention(q, cache, cu, lens, table[0], 4))
    refused(bad, lambda: text.paged_attention(q, cache, cu, lens.long(), table, 4))
    refused(bad, lambda: text.paged_attention(_randn(g, 4, 4, 64), cache, cu, lens, table, 4))
    # one page named so often that the walk over it could not be counted in 32 bits
    deep = torch.zeros((64, 1 << 19), dtype=torch.int32, device="cuda")
    mqa = text.PagedKVCache(1, 256, 64, 64)
    refused(unsup, lambda: text.paged_attention(_randn(g, 64, 64, 64), mqa, _cu([1] * 64),
                                                torch.ones(64, dtype=torch.int32, device="cuda"), deep, 1))
    refused(bad, lambda: cache.append(k, k, torch.zeros(3, dtype=torch.int64, device="cuda")))
    refused(bad, lambda: cache.append(q, q, torch.zeros(4, dtype=torch.int64, device="cuda")))
    refused(bad, lambda: text.PagedKVCache(2, 16, 2, 128, "int4"))
    refused(bad, lambda: text.PagedKVCache.from_tensors(cache.k, cache.v))
    refused(bad, lambda: text.RopeTable(12, 16))
    refused(bad, lambda: text.RopeTable(64, 16, scaling=text.RopeScaling("other")))
    refused(bad, lambda: text.RopeTable(64, 16, scaling=text.RopeScaling("linear", 0.5)))
    tab = text.RopeTable(128, 16)
    refused(bad, lambda: tab.apply(_randn(g, 4, 2, 64), torch.zeros(4, dtype=torch.int32, device="cuda")))
    refused(bad, lambda: tab.apply(q, torch.zeros(4, dtype=torch.int64, device="cuda")))
    _check_device()


def test_wrong_device_arguments_are_reported_not_followed():
    """Lengths, offsets and block entries beyond the buffers: clamped by the kernels, reported."""
    text = _text()
    from wuxianhuabu_b200 import h3
    g = _gen(1)
    for q_len in (1, 60):
        q = _randn(g, q_len, 4, 128)
        cache = text.PagedKVCache(3, 16, 2, 128, "int8")
        kk = _randn(g, 48, 2, 128)
        cache.append(kk, kk, torch.arange(48, device="cuda"))
        i32 = dict(dtype=torch.int32, device="cuda")
        for cu, lens, table in (
                ([0, q_len], [100], [[0, 1]]),          # longer than its block row
                ([0, q_len], [32], [[0, 3]]),           # no such page
                ([0, q_len], [-5], [[0, 1]]),
                ([0, q_len + 9], [20], [[0, 1]]),       # more query rows than there are
                ([-3, q_len], [20], [[0, 1]])):
            text.paged_attention(q, cache, torch.tensor(cu, **i32), torch.tensor(lens, **i32),
                                 torch.tensor(table, **i32), q_len)
            with pytest.raises(h3.WxError):
                _check_device()
    _check_device()


def test_empty_calls():
    text = _text()
    e = torch.empty((0, 4, 128), dtype=BF16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    assert text.prompt_attention(e, e[:, :2], e[:, :2], torch.tensor([0], **i32), 0).shape == (0, 4, 128)
    assert text.prompt_attention(e, e[:, :2], e[:, :2], torch.tensor([0, 0, 0], **i32), 0).shape == (0, 4, 128)
    cache = text.PagedKVCache(1, 16, 4, 128)
    cache.append(e, e, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert cache.read(torch.empty(0, dtype=torch.int64, device="cuda"))[0].shape == (0, 4, 128)
    assert text.RopeTable(64, 4).apply(e, torch.empty(0, **i32)).shape == (0, 4, 128)
    _check_device()


def test_calls_on_two_streams_share_the_workspace_safely():
    """Split items leave partial sums in the context's workspace: calls on another stream wait."""
    text = _text()
    g = _gen(4)
    cache, table, q, _, _ = _paged(g, "bf16", [1], [6000], 8, 2, 128, 64)
    lens = torch.tensor([6000], dtype=torch.int32, device="cuda")
    want = text.paged_attention(q, cache, _cu([1]), lens, table, 1)
    cu = _cu([1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(20):
        if i % 2:
            with torch.cuda.stream(side):
                outs.append(text.paged_attention(q, cache, cu, lens, table, 1))
        else:
            outs.append(text.paged_attention(q, cache, cu, lens, table, 1))
    torch.cuda.synchronize()
    _check_device()
    assert all(torch.equal(o, want) for o in outs)


# The states are normalised and each of the 2 x 2 sublayers rounds its input, products and sum to
# bf16 (2^-9 rms of the value, some 6 roundings): sqrt(24) 2^-9 = 0.01 between two orders of the
# same arithmetic. An 8-bit cache adds at most half a step of the row's largest value to every K
# and V entry (1 / 254 of 2.5 to 3 standard deviations, e4m3 2^-4 of the entry: 0.036 rms); the
# largest of these reaches the states through the attention's share of them. Five times that.
@pytest.mark.parametrize("fmt,bound", [("bf16", 0.05), ("int8", 0.1), ("e4m3", 0.2)])
def test_example_runs_the_operators_together(fmt, bound):
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "examples" / "encode_prompt.py"
    spec = importlib.util.spec_from_file_location("encode_prompt", path)
    module = importlib.util.module_from_spec(spec)
    import sys
    sys.modules["encode_prompt"] = module  # (dataclasses look their module up)
    spec.loader.exec_module(module)
    r = module.main(["--cache", fmt, "--new", "5"])
    assert r["finite"] and r["tokens"] == [82, 26]
    assert r["conditions"] == [(82, 256), (26, 256)]
    assert r["stepwise"] < bound and r["chunked"] < bound, r
