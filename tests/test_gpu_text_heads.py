"""Head norms with rotary positions, over one and several position axes, against the formula in 64 bits.

Tolerances. The mean of the squares is a sum of at most 19 roundings deep (16 of a lane, 3 joins), each
2^-24: 2^-19.7 of the mean, half of that of its root; rsqrtf is within 2 ulp (2^-22), the products with the
root and the weight one rounding each: 2^-20 relative of a normalised value. The rotation adds 4 roundings
of 2^-24 on |a| + |b|, the tables 2^-24 each: 2^-19 (|a| + |b|) together, and the output's rounding to bf16
is 2^-8 of the value. 8-bit caches: half a step of the format as in test_gpu_text, the row's largest
magnitude (and so the step) being off by 2^-19 itself."""
import math

import pytest
import torch

from tests.test_gpu_text import (BF16, F64, _check_device, _gen, _half_step, _randn, _slots, _text, ref_inv_freq)

pytestmark = pytest.mark.gpu


def ref_heads(x, w, eps, pos, inv, axes, interleaved):
    """y (64 bits) and the magnitudes |a| + |b| that its pairs are made of."""
    x = x.to(F64)
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.to(F64)
    rot = 2 * len(inv)
    pos = pos.to(F64) if pos.dim() == 2 else pos.to(F64)[None]
    ang = torch.stack([pos[a] * f for a, f in zip(axes, inv)], -1)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y = x.clone()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    mag = x.abs().clone()
    mag[..., a] = mag[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, mag


CASES = [  # tokens, q heads, k heads, head_dim, rot, interleaved, shares of the axes (None: one axis), dealt, norms
    (1, 1, 1, 128, 128, False, (24, 20, 20), True, "qk"),
    (3, 5, 2, 64, 64, False, (12, 10, 10), False, "qk"),
    (130, 32, 8, 128, 128, False, (24, 20, 20), False, "qk"),
    (77, 28, 4, 128, 128, True, (24, 20, 20), True, "qk"),
    (50, 7, 1, 128, 64, False, (16, 16), True, "q"),
    (50, 9, 3, 64, 24, True, (3, 3, 3, 3), True, "k"),
    (41, 6, 2, 64, 8, False, (2, 1, 1), False, "qk"),
    (1, 16, 4, 128, 128, False, None, False, "qk"),
    (2100, 8, 2, 64, 32, False, None, False, "qk"),
    (65, 40, 8, 128, 128, False, (64,), False, ""),
    (19, 3, 3, 128, 104, False, (20, 16, 16), True, ""),
    # many tokens: persistent warps
    (1800, 32, 8, 128, 128, False, (24, 20, 20), True, "qk"),
    (2001, 13, 7, 128, 128, True, (24, 20, 20), False, "qk"),
    (1777, 29, 15, 64, 64, False, (12, 10, 10), True, "qk"),
    (3700, 14, 5, 128, 64, False, (16, 16), True, "q"),
    (2900, 31, 9, 64, 24, True, (3, 3, 3, 3), True, "k"),
    (1850, 40, 33, 64, 40, False, (10, 5, 5), False, "qk"),
    (4000, 11, 5, 128, 8, False, None, False, "qk"),
    (1776, 33, 17, 128, 120, False, None, False, ""),
    (5000, 3, 1, 128, 128, False, None, False, "qk"),  # (not for them: few heads)
]


def _inputs(i, case):
    tokens, hq, hk, hd, rot, interleaved, shares, dealt, norms = case
    text = _text()
    g = _gen(100 + i)
    qkv = _randn(g, tokens, hq + 2 * hk, hd)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    q_norm, k_norm = ((1 + 0.3 * torch.randn(hd, generator=g, device="cuda")).to(BF16) for _ in range(2))
    axes = None if shares is None else text.rope_axes(shares, dealt)
    n = 1 if shares is None else len(shares)
    pos = torch.randint(0, 4000, (n, tokens), generator=g, device="cuda", dtype=torch.int32)
    pos[:, ::3] = pos[:1, ::3]  # (text between pictures: the axes together)
    tab = text.RopeTable(rot, 4000, base=500000.0, interleaved=interleaved, axes=axes)
    return tab, q, k, v, pos if shares else pos[0], q_norm if "q" in norms else None, k_norm if "k" in norms else None


@pytest.mark.parametrize("i", range(len(CASES)))
def test_apply_qk(i):
    tokens, hq, hk, hd, rot, interleaved, shares, dealt, norms = CASES[i]
    tab, q, k, v, pos, qw, kw = _inputs(i, CASES[i])
    eps = 1e-6 if i % 2 else 1e-2
    got = tab.apply_qk(q, k, pos, q_norm=qw, k_norm=kw, eps=eps)
    _check_device()
    inv, axes = ref_inv_freq(rot, 500000.0, None), tab.axes or [0] * (rot // 2)
    for y, x, w in zip(got, (q, k), (qw, kw)):
        ref, mag = ref_heads(x, w, eps, pos, inv, axes, interleaved)
        err = (y.to(F64) - ref).abs()
        assert (err <= 2.0 ** -8 * ref.abs() + 2.0 ** -19 * mag).all(), float((err / (ref.abs() + mag)).max())
    # in place, into a larger buffer's slices, and each alone
    both = torch.cat([q, k], 1)
    tab.apply_qk(both[:, :hq], both[:, hq:], pos, q_norm=qw, k_norm=kw, eps=eps, q_out=both[:, :hq], k_out=both[:, hq:])
    assert torch.equal(both[:, :hq], got[0]) and torch.equal(both[:, hq:], got[1])
    assert torch.equal(tab.apply(q, pos, norm=qw, eps=eps), got[0])
    assert torch.equal(tab.apply(k, pos, norm=kw, eps=eps, out=torch.empty_like(k)), got[1])
    _check_device()


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_append_roped(i, fmt):
    tokens, hq, hk, hd, rot, interleaved, shares, dealt, norms = CASES[i]
    text = _text()
    tab, q, k, v, pos, qw, kw = _inputs(i, CASES[i])
    g = _gen(7)
    page = (16, 32, 64)[i % 3]
    pages = tokens // page + 3
    cache = text.PagedKVCache(pages, page, hk, hd, fmt)
    slots = _slots(g, tokens, pages, page)
    got_q = cache.append_roped(q, k, v, slots, tab, pos, q_norm=qw, k_norm=kw, eps=1e-5)
    gk, gv = cache.read(slots)
    want_q, want_k = tab.apply_qk(q, k, pos, q_norm=qw, k_norm=kw, eps=1e-5)
    _check_device()
    assert torch.equal(got_q, want_q)  # the same rows, bit for bit
    inv, axes = ref_inv_freq(rot, 500000.0, None), tab.axes or [0] * (rot // 2)
    ref, mag = ref_heads(k, kw, 1e-5, pos, inv, axes, interleaved)
    if fmt == "bf16":
        assert torch.equal(gk, want_k) and torch.equal(gv, v)
        return
    for got, r, m in ((gk, ref, mag), (gv, v.to(F64), torch.zeros_like(mag))):
        tol = 2.0 ** -8 * r.abs() + 2.0 ** -19 * m + _half_step(r, fmt) * (1 + 2.0 ** -8) + \
            2.0 ** -19 * r.abs().amax(-1, keepdim=True)
        assert ((got.to(F64) - r).abs() <= tol).all(), fmt


def test_axes_together_are_one_axis():
    """Text: every axis at the same position gives the plain rotation, whatever the pairs' axes."""
    text = _text()
    g = _gen(3)
    x = _randn(g, 40, 6, 128)
    pos = torch.arange(40, dtype=torch.int32, device="cuda") * 5
    plain = text.RopeTable(128, 200)
    for dealt in (False, True):
        tab = text.RopeTable.from_tables(plain.cos, plain.sin, axes=text.rope_axes((24, 20, 20), dealt))
        assert torch.equal(tab.apply(x, pos.expand(3, -1).contiguous()), plain.apply(x, pos))
    _check_device()


def test_rows_of_zeros_infinities_and_nan():
    text = _text()
    g = _gen(4)
    tab = text.RopeTable(64, 10, axes=text.rope_axes((16, 8, 8)))
    q, w = _randn(g, 5, 3, 64), torch.ones(64, dtype=BF16, device="cuda")
    k = _randn(g, 5, 2, 64)
    q[1] = 0
    q[2, 1, 5] = math.inf
    q[3, 0, 63] = math.nan
    pos = torch.arange(15, dtype=torch.int32, device="cuda").view(3, 5) % 10
    a, b = tab.apply_qk(q, k, pos, q_norm=w, k_norm=w)
    clean = q.clone()
    clean[2, 1], clean[3, 0] = 1.0, 1.0
    c, _ = tab.apply_qk(clean, k, pos, q_norm=w, k_norm=w)
    _check_device()
    assert not a[1].any() and torch.isfinite(b).all()
    assert torch.isnan(a[3, 0]).all() and torch.isnan(a[2, 1, 5]) and torch.isnan(a[2, 1, 37])  # inf / inf
    same = torch.ones(5, 3, dtype=torch.bool, device="cuda")
    same[2, 1] = same[3, 0] = False
    assert torch.equal(a[same], c[same])


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_many_tokens_with_wrong_positions_and_slots(fmt):
    """Tokens that are skipped or wrong, among thousands that are not: the others as without them."""
    text = _text()
    from wuxianhuabu_b200 import h3
    g = _gen(9)
    n = 2500
    tab = text.RopeTable(128, 500, axes=text.rope_axes((24, 20, 20), True))
    q, k, v = _randn(g, n, 14, 128), _randn(g, n, 7, 128), _randn(g, n, 7, 128)
    w = torch.ones(128, dtype=BF16, device="cuda")
    pos = torch.randint(0, 500, (3, n), generator=g, device="cuda", dtype=torch.int32)
    slots = torch.randperm(n + 12, generator=g, device="cuda")[:n]
    caches = [text.PagedKVCache((n + 31) // 16, 16, 7, 128, fmt) for _ in range(2)]
    want = caches[0].append_roped(q, k, v, slots, tab, pos, q_norm=w, k_norm=w)
    _check_device()
    some, skipped, wrong, far = (torch.arange(i, n, 97, device="cuda") for i in range(4))
    slots2, pos2 = slots.clone(), pos.clone()
    slots2[skipped] = -5
    slots2[far] = (n + 31) // 16 * 16
    pos2[2, wrong] = 500
    pos2[0, some[:3]] = -1
    out = torch.full_like(q, 9.0)
    caches[1].append_roped(q, k, v, slots2, tab, pos2, q_out=out, q_norm=w, k_norm=w)
    with pytest.raises(h3.WxError):
        _check_device()
    lost = torch.zeros(n, dtype=torch.bool, device="cuda")
    lost[wrong] = lost[some[:3]] = True
    assert (out[lost] == 9.0).all() and torch.equal(out[~lost], want[~lost])
    unwritten = lost.clone()
    unwritten[skipped] = unwritten[far] = True
    for a, b in zip(caches[0].read(slots), caches[1].read(slots)):
        assert not b[unwritten].any() and torch.equal(a[~unwritten], b[~unwritten])
    _check_device()


def test_positions_outside_the_table_and_skipped_slots():
    text = _text()
    from wuxianhuabu_b200 import h3
    g = _gen(5)
    tab = text.RopeTable(128, 50, axes=text.rope_axes((24, 20, 20), True))
    q, k, v = _randn(g, 4, 4, 128), _randn(g, 4, 2, 128), _randn(g, 4, 2, 128)
    w = torch.ones(128, dtype=BF16, device="cuda")
    pos = torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    cache = text.PagedKVCache(2, 16, 2, 128)
    slots = torch.tensor([3, -1, 5, 7], device="cuda")
    out = torch.full_like(q, 9.0)
    cache.append_roped(q, k, v, slots, tab, pos, q_out=out, q_norm=w, k_norm=w)
    _check_device()
    assert (out != 9.0).any(-1).all() and not cache.read(torch.tensor([4], device="cuda"))[0].any()
    for axis, at in ((0, 50), (2, -1)):
        wrong = pos.clone()
        wrong[axis, 2] = at
        out.fill_(9.0)
        cache = text.PagedKVCache(2, 16, 2, 128)
        cache.append_roped(q, k, v, slots, tab, wrong, q_out=out, q_norm=w, k_norm=w)
        with pytest.raises(h3.WxError):
            _check_device()
        assert (out[2] == 9.0).all() and (out[[0, 1, 3]] != 9.0).any(-1).all()
        assert not cache.read(slots[2:3])[0].any() and cache.read(slots[3:])[0].any()
        _check_device()


def test_strided_positions_and_copies():
    import copy
    import pickle
    text = _text()
    g = _gen(6)
    tab = text.RopeTable(64, 300, axes=text.rope_axes((12, 10, 10), True))
    q, k = _randn(g, 9, 3, 64), _randn(g, 9, 1, 64)
    wide = torch.randint(0, 300, (4, 40), generator=g, device="cuda", dtype=torch.int32)
    pos = wide[:3, 11:20]
    want = tab.apply_qk(q, k, pos.contiguous())
    for t in (tab, copy.copy(tab), copy.deepcopy(tab), pickle.loads(pickle.dumps(tab))):
        got = t.apply_qk(q, k, pos)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    empty = tab.apply_qk(q[:0], k[:0], pos[:, :0])
    assert empty[0].shape == (0, 3, 64) and empty[1].shape == (0, 1, 64)
    _check_device()


def test_refusals():
    text = _text()
    from wuxianhuabu_b200 import h3
    g = _gen(8)
    tab = text.RopeTable(64, 30, axes=text.rope_axes((12, 10, 10)))
    q, k, w = _randn(g, 5, 3, 64), _randn(g, 5, 1, 64), torch.ones(64, dtype=BF16, device="cuda")
    pos = torch.zeros((3, 5), dtype=torch.int32, device="cuda")
    for call in (lambda: tab.apply_qk(q, k, pos[0]), lambda: tab.apply_qk(q, k, pos[:2]),
                 lambda: tab.apply_qk(q, k, pos[:, :4]), lambda: tab.apply_qk(q, k, pos.long()),
                 lambda: tab.apply_qk(q, k, torch.zeros((5, 3), dtype=torch.int32, device="cuda").t()),
                 lambda: tab.apply_qk(q, k[:4], pos), lambda: tab.apply_qk(q, k[..., :32], pos),
                 lambda: tab.apply_qk(q, k, pos, q_norm=w[:32]), lambda: tab.apply_qk(q, k, pos, k_norm=w.float()),
                 lambda: tab.apply_qk(q, k, pos, q_norm=w, eps=0.0), lambda: tab.apply_qk(q, k, pos, q_norm=w, eps=math.nan),
                 lambda: tab.apply_qk(q, k, pos, q_norm=w.repeat(2)[4:68]),  # (not on a 16-byte boundary)
                 lambda: tab.apply(q, pos, norm=w[:8]), lambda: tab.apply(q, pos, norm=w, eps=-1.0),
                 lambda: tab.apply_qk(q, k, pos, q_out=q[:4]), lambda: tab.apply_qk(q.cpu(), k, pos),
                 lambda: text.RopeTable(64, 30, axes=(0, 1)), lambda: text.RopeTable(64, 30, axes=[4] * 32),
                 lambda: text.RopeTable(64, 30, axes=[-1] * 32), lambda: text.RopeTable(64, 30, axes=())):
        with pytest.raises(h3.WxError):
            call()
    _check_device()
