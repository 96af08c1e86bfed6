"""The text-side operators of this framework and the work they stand for.

A video is denoised under the hidden states of its prompts. A decoder-only text model makes
those states: its layers need rotary positions, a paged K/V cache, attention over whole
(packed, causal) prompts, and attention of new tokens over the cache when a prompt is
extended or rewritten token by token. ``listed`` gives calls over that range, ``draw`` more
of the same kind. Every operator exists here in a plain form (elementary torch operations in
fp32) and, with ``own`` set, as the call a user makes of this package.
"""
import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
# largest magnitude that a stored value of the format can hold
QMAX = {"int8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -100  # a row with no magnitude above this is stored as zeros


def _text(ns):
    return " ".join(str(n) for n in ns)


def _ints(text):
    return [int(n) for n in text.split()]


def listed():
    return [
        # q and k heads of one long prompt (or a packed batch), before they enter attention
        dict(name="rope_8k_half", op="rope", tokens=8192, hq=32, hkv=8, hd=128, rot=128, interleaved=False,
             scaling="none", factor=1.0, first=0),
        # a short continuation deep in a long context: part of the head, interleaved, scaled
        dict(name="rope_long_part", op="rope", tokens=333, hq=28, hkv=4, hd=128, rot=64, interleaved=True,
             scaling="by_parts", factor=8.0, first=100003),
        # one layer's entry of a long prompt into an 8-bit cache, rope fused with the write,
        # and the layer's K/V read back for a consumer that wants bf16
        dict(name="cache_prompt_int8", op="cache", tokens=4096, prefix=0, hq=32, hkv=8, hd=128, page=64, fmt="int8",
             roped=True),
        # a decoding batch of 24 writes one token each; one sequence's prefix is read back
        dict(name="cache_step_e4m3", op="cache", tokens=24, prefix=2011, hq=16, hkv=4, hd=64, page=16, fmt="e4m3",
             roped=False),
        # positive and negative prompt of one generation
        dict(name="prompt_pair", op="prompt", lens="512 77", hq=32, hkv=8, hd=128, causal=True, window=0),
        # long prompts packed with short ones
        dict(name="prompt_ragged_long", op="prompt", lens="9001 1 5003 2380", hq=32, hkv=8, hd=128, causal=True,
             window=0),
        # equal heads of width 64, sliding window
        dict(name="prompt_window_hd64", op="prompt", lens="4096 1117", hq=16, hkv=16, hd=64, causal=True,
             window=1024),
        # one token of one short sequence: latency
        dict(name="decode_tiny_bf16", op="paged", q_lens="1 1", kv_lens="203 64", hq=16, hkv=16, hd=64, page=16,
             fmt="bf16", window=0),
        # one token of one long sequence
        dict(name="decode_one_long_int8", op="paged", q_lens="1", kv_lens="65537", hq=64, hkv=8, hd=128, page=64,
             fmt="int8", window=0),
        # a serving batch, ragged
        dict(name="decode_batch_bf16", op="paged", q_lens=_text([1] * 64),
             kv_lens=_text(100 + (i * 2477) % 7919 for i in range(64)),
             hq=32, hkv=8, hd=128, page=64, fmt="bf16", window=0),
        # a few drafted tokens per sequence, group of 7
        dict(name="verify_int8", op="paged", q_lens=_text([5] * 16),
             kv_lens=_text(1000 + 211 * i for i in range(16)), hq=28, hkv=4, hd=128, page=16, fmt="int8", window=0),
        # a prompt's next chunk over what is cached already
        dict(name="chunk_e4m3", op="paged", q_lens="1024 300", kv_lens="16384 9999", hq=32, hkv=8, hd=128, page=64,
             fmt="e4m3", window=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "cache", "prompt", "prompt", "paged", "paged", "paged"])
    hq, hkv = rng.choice([(32, 8), (16, 16), (28, 4), (64, 8), (24, 8), (8, 1), (12, 4), (32, 4)])
    hd = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    if op == "rope":
        rot = rng.choice([hd, hd, hd // 2, hd // 4])
        scaling = rng.choice(["none", "linear", "by_parts"])
        return dict(op=op, tokens=_log_int(rng, 1, 8000 * 40 // (hq + hkv)), hq=hq, hkv=hkv, hd=hd, rot=rot,
                    interleaved=rng.random() < 0.5, scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
                    first=rng.choice([0, _log_int(rng, 1, 120000)]))
    if op == "cache":
        return dict(op=op, tokens=_log_int(rng, 1, 4000), prefix=rng.choice([0, _log_int(rng, 1, 4000)]), hq=hq,
                    hkv=hkv, hd=hd, page=page, fmt=rng.choice(["bf16", "int8", "e4m3"]), roped=rng.random() < 0.5)
    if op == "prompt":
        causal = hq > 32 or rng.random() < 0.8
        lens = [rng.choice([_log_int(rng, 1, 3600), _log_int(rng, 16, 1500)]) for _ in range(rng.randint(1, 4))]
        return dict(op=op, lens=_text(lens), hq=hq, hkv=hkv, hd=hd, causal=causal,
                    window=rng.choice([0, 0, _log_int(rng, 64, 2000)]) if causal else 0)
    kind = rng.choice(["decode", "decode", "verify", "chunk"])
    fmt = rng.choice(["bf16", "int8", "e4m3"])
    window = rng.choice([0, 0, 0, _log_int(rng, 128, 4000)])
    if kind == "decode":
        n = _log_int(rng, 1, 64)
        kv = [_log_int(rng, 1, 60000 if n <= 4 else 7000) for _ in range(n)]
        q = [1] * n
    elif kind == "verify":
        n = _log_int(rng, 1, 24)
        q = [rng.randint(2, 9) for _ in range(n)]
        kv = [a + _log_int(rng, 1, 6000) for a in q]
    else:
        n = rng.randint(1, 3)
        q = [_log_int(rng, 16, 600) for _ in range(n)]
        kv = [a + rng.choice([0, _log_int(rng, 1, 12000)]) for a in q]
    return dict(op="paged", q_lens=_text(q), kv_lens=_text(kv), hq=hq, hkv=hkv, hd=hd, page=page, fmt=fmt, window=window)


# ------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(BF16)


def _cu(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=DEV)


def _inv_freq(rot, scaling, factor, base=500000.0, original=8192.0, low=1.0, high=4.0):
    """The inverse frequencies of the rotated pairs, in 64 bits."""
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    if scaling == "linear":
        return inv / factor
    if scaling == "by_parts":
        turns = original * inv / (2.0 * math.pi)
        w = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return (1.0 - w) * inv / factor + w * inv
    return inv


def _tables(inv, n):
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv[None, :]
    return a.cos().float(), a.sin().float()


def _quantise(x, fmt):
    """bf16 or fp32 rows [..., hd] -> stored values and one fp32 scale per row."""
    xf = x.float()
    if fmt == "bf16":
        return xf.to(BF16), None
    amax = xf.abs().amax(-1)
    ok = torch.isfinite(amax)
    live = ok & (amax >= TINY)
    safe = torch.where(live, amax, torch.ones_like(amax))
    top = torch.full_like(amax, QMAX[fmt])  # (torch would multiply by the reciprocal of a plain number)
    y = torch.where(live[..., None], xf * (top / safe)[..., None], torch.zeros_like(xf))
    q = y.round().to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)
    scale = torch.where(live, amax / top, torch.zeros_like(amax))
    return q, torch.where(ok, scale, torch.full_like(scale, math.nan))


def _cache(g, pages, case):
    """A cache of `pages` pages holding quantised K/V, as earlier calls left it."""
    fmt = case["fmt"]
    out = []
    for _ in range(2):
        x = _randn(g, pages, case["hkv"], case["page"], case["hd"])
        out += list(_quantise(x, fmt))
    kq, ks, vq, vs = out
    return kq, vq, ks, vs


def prepare(case, seed):
    g = _gen(seed)
    op, hq, hkv, hd = case["op"], case["hq"], case["hkv"], case["hd"]
    st = dict(case=case, op=op)
    if op == "rope":
        n = case["tokens"]
        qkv = _randn(g, n, hq + 2 * hkv, hd)  # the projection's packed output: q heads | k heads | v heads
        st["x"] = qkv[:, :hq + hkv]
        st["pos"] = torch.arange(case["first"], case["first"] + n, dtype=torch.int32, device=DEV)
        st["cos"], st["sin"] = _tables(_inv_freq(case["rot"], case["scaling"], case["factor"]), case["first"] + n)
        if own:
            from wuxianhuabu_b200 import text
            st["table"] = text.RopeTable.from_tables(st["cos"], st["sin"], interleaved=case["interleaved"])
        return st
    if op == "cache":
        n, total = case["tokens"], case["tokens"] + case["prefix"]
        qkv = _randn(g, n, hq + 2 * hkv, hd)
        st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        pages = (total + case["page"] - 1) // case["page"] + 3
        st["cache"] = _cache(g, pages, case)
        table = torch.randperm(pages, generator=g, device=DEV)
        at = torch.arange(total, device=DEV)
        st["all_slots"] = table[at // case["page"]] * case["page"] + at % case["page"]
        st["slots"] = st["all_slots"][case["prefix"]:].contiguous()
        st["pos"] = torch.arange(case["prefix"], total, dtype=torch.int32, device=DEV)
        st["cos"], st["sin"] = _tables(_inv_freq(hd, "none", 1.0), total)
        if own:
            from wuxianhuabu_b200 import text
            st["table"] = text.RopeTable.from_tables(st["cos"], st["sin"], interleaved=False)
            st["paged"] = text.PagedKVCache.from_tensors(*st["cache"])
        return st
    st["scale"] = 1.0 / math.sqrt(hd)
    if op == "prompt":
        st["lens"] = _ints(case["lens"])
        st["cu"] = _cu(st["lens"])
        qkv = _randn(g, sum(st["lens"]), hq + 2 * hkv, hd)
        st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        return st
    st["q_lens"], st["lens"] = _ints(case["q_lens"]), _ints(case["kv_lens"])
    kv, page = st["lens"], case["page"]
    need = [(n + page - 1) // page for n in kv]
    pages = sum(need) + 3
    st["q"] = _randn(g, sum(st["q_lens"]), hq, hd)
    st["cu"] = _cu(st["q_lens"])
    st["kv_lens"] = torch.tensor(kv, dtype=torch.int32, device=DEV)
    st["cache"] = _cache(g, pages, case)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    st["blocks"] = torch.full((len(kv), max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        st["blocks"][i, :n] = order[at:at + n]
        at += n
    if own:
        from wuxianhuabu_b200 import text
        st["paged"] = text.PagedKVCache.from_tensors(*st["cache"])
    return st


# ------------------------------------------------------------------------------- plain forms
def _rotate(x, pos, cos, sin, interleaved):
    xf = x.float()
    c, s = cos[pos.long()][:, None, :], sin[pos.long()][:, None, :]
    half = c.shape[-1]
    rest = xf[..., 2 * half:]
    if interleaved:
        a, b = xf[..., 0:2 * half:2], xf[..., 1:2 * half:2]
        r = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = xf[..., :half], xf[..., half:2 * half]
        r = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([r, rest], -1)


def _attend(q, k, v, scale, causal, window, dtype):
    """One sequence: q [Lq, Hq, hd], k and v [Lk, Hkv, hd] -> out [Lq, Hq, hd], lse [Lq, Hq]."""
    lq, hq, hd = q.shape
    lk, hkv = k.shape[0], k.shape[1]
    q = q.to(dtype).view(lq, hkv, hq // hkv, hd).permute(1, 2, 0, 3)  # [Hkv, G, Lq, hd]
    kt = k.to(dtype).permute(1, 2, 0)[:, None]
    vv = v.to(dtype).permute(1, 0, 2)[:, None]
    out = torch.empty(hkv, hq // hkv, lq, hd, dtype=dtype, device=q.device)
    lse = torch.empty(hkv, hq // hkv, lq, dtype=dtype, device=q.device)
    col = torch.arange(lk, device=q.device)[None, :]
    step = max(1, int(2 ** 28 // max(1, hq * lk)))
    for a in range(0, lq, step):
        b = min(lq, a + step)
        s = torch.matmul(q[:, :, a:b], kt) * scale
        row = torch.arange(a, b, device=q.device)[:, None] + (lk - lq)
        if causal or window:
            off = torch.zeros(b - a, lk, dtype=torch.bool, device=q.device)
            if causal:
                off = off | (col > row)
            if window:
                off = off | (col <= row - window)
            s = s.masked_fill(off, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = (s - m).exp()
        den = p.sum(-1, keepdim=True)
        out[:, :, a:b] = torch.matmul(p, vv) / den
        lse[:, :, a:b] = (m + den.log()).squeeze(-1)
    return out.permute(2, 0, 1, 3).reshape(lq, hq, hd), lse.permute(2, 0, 1).reshape(lq, hq)


def _values(q, scale):
    return q.float() if scale is None else q.float() * scale[..., None]


def run(st):
    case, op = st["case"], st["op"]
    if op == "rope":
        if own:
            return st["table"].apply(st["x"], st["pos"])
        return _rotate(st["x"], st["pos"], st["cos"], st["sin"], case["interleaved"]).to(BF16)
    if op == "cache":
        if own:
            if case["roped"]:
                q = st["paged"].append_roped(st["q"], st["k"], st["v"], st["slots"], st["table"], st["pos"])
                return (q,) + st["paged"].read(st["all_slots"])
            st["paged"].append(st["k"], st["v"], st["slots"])
            return st["paged"].read(st["all_slots"])
        kc, vc, ks, vs = st["cache"]
        k, out = st["k"], ()
        if case["roped"]:
            out = (_rotate(st["q"], st["pos"], st["cos"], st["sin"], False).to(BF16),)
            k = _rotate(k, st["pos"], st["cos"], st["sin"], False)
        page = case["page"]
        for src, dst, sc in ((k, kc, ks), (st["v"], vc, vs)):
            q, s = _quantise(src, case["fmt"])
            at, inside = st["slots"] // page, st["slots"] % page
            raw = dst if case["fmt"] == "bf16" else dst.view(torch.int8)
            raw[at, :, inside] = q if case["fmt"] == "bf16" else q.view(torch.int8)
            if sc is not None:
                sc[at, :, inside] = s
        at, inside = st["all_slots"] // page, st["all_slots"] % page
        for src, sc in ((kc, ks), (vc, vs)):
            raw = src if case["fmt"] == "bf16" else src.view(torch.int8)
            rows = raw[at, :, inside]
            if case["fmt"] != "bf16":
                rows = rows.view(src.dtype)
            out += (_values(rows, None if sc is None else sc[at, :, inside]).to(BF16),)
        return out
    if op == "prompt":
        if own:
            from wuxianhuabu_b200 import text
            return text.prompt_attention(st["q"], st["k"], st["v"], st["cu"], max(st["lens"]), scale=st["scale"],
                                         causal=case["causal"], window=case["window"], return_lse=True)
        outs, a = [], 0
        for n in st["lens"]:
            outs.append(_attend(st["q"][a:a + n], st["k"][a:a + n], st["v"][a:a + n], st["scale"], case["causal"],
                                case["window"], torch.float32))
            a += n
        return torch.cat([o for o, _ in outs]).to(BF16), torch.cat([x for _, x in outs])
    if own:
        from wuxianhuabu_b200 import text
        return text.paged_attention(st["q"], st["paged"], st["cu"], st["kv_lens"], st["blocks"], max(st["q_lens"]),
                                    scale=st["scale"], causal=True, window=case["window"], return_lse=True)
    outs, a = [], 0
    for i, (n, m) in enumerate(zip(st["q_lens"], st["lens"])):
        k, v = _paged_rows(st, i, m)
        outs.append(_attend(st["q"][a:a + n], k, v, st["scale"], True, case["window"], torch.float32))
        a += n
    return torch.cat([o for o, _ in outs]).to(BF16), torch.cat([x for _, x in outs])


def _paged_rows(st, i, m):
    """The first m cached K and V rows of sequence i as fp32 [m, Hkv, hd]."""
    kc, vc, ks, vs = st["cache"]
    page = st["case"]["page"]
    at = st["blocks"][i, :(m + page - 1) // page].long()
    rows = []
    for c, s in ((kc, ks), (vc, vs)):
        raw = c if c.dtype == BF16 else c.view(torch.int8)
        x = _values(raw[at].view(c.dtype), None if s is None else s[at])  # [n, Hkv, page, hd]
        rows.append(x.permute(0, 2, 1, 3).flatten(0, 1)[:m])
    return rows


# -------------------------------------------------------------------------------- definitions
def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "rope":
        inv = _inv_freq(case["rot"], case["scaling"], case["factor"])
        return _turn64(st["x"].to(f64), st["pos"], inv, case["interleaved"])
    if case["op"] == "cache":
        out = []
        k, v = st["k"].to(f64), st["v"].to(f64)
        if case["roped"]:
            inv = _inv_freq(case["hd"], "none", 1.0)
            out.append(_turn64(st["q"].to(f64), st["pos"], inv, False))
            k = _turn64(k, st["pos"], inv, False)
        kc, vc, ks, vs = st["cache"]
        old = st["all_slots"][:case["prefix"]]
        at, inside = old // case["page"], old % case["page"]
        for new, c, s in ((k, kc, ks), (v, vc, vs)):
            if case["fmt"] == "bf16":
                before, after = c[at, :, inside].to(f64), new
            else:
                before = c.view(torch.int8)[at, :, inside].view(c.dtype).float().to(f64) * s[at, :, inside][..., None]
                step = new.abs().amax(-1, keepdim=True) / QMAX[case["fmt"]]
                y = new / step
                if case["fmt"] == "int8":
                    y = y.round()
                else:  # nearest value with 3 fraction bits, exponent not below -6
                    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0)
                    y = torch.round(y / 2.0 ** (e - 3)) * 2.0 ** (e - 3)
                after = y * step
            out.append(torch.cat([before, after]))
        return tuple(out)
    if case["op"] == "prompt":
        qs, ks = st["lens"], st["lens"]
    else:
        qs, ks = st["q_lens"], st["lens"]
    causal = case.get("causal", True)
    outs, lses, a = [], [], 0
    for i, (n, m) in enumerate(zip(qs, ks)):
        q = st["q"][a:a + n].to(f64)
        if case["op"] == "prompt":
            k, v = st["k"][a:a + n].to(f64), st["v"][a:a + n].to(f64)
        else:
            kc, vc, sk, sv = st["cache"]
            j = torch.arange(m, device=DEV)
            pg, inside = st["blocks"][i].long()[j // case["page"]], j % case["page"]
            k, v = (c.view(torch.int8 if c.dtype != BF16 else BF16)[pg, :, inside].view(c.dtype).float().to(f64)
                    for c in (kc, vc))
            if sk is not None:
                k, v = k * sk[pg, :, inside][..., None], v * sv[pg, :, inside][..., None]
        o = torch.empty(n, case["hq"], case["hd"], dtype=f64, device=DEV)
        z = torch.empty(n, case["hq"], dtype=f64, device=DEV)
        grp = case["hq"] // case["hkv"]
        for h in range(case["hq"]):
            kh, vh = k[:, h // grp], v[:, h // grp]
            for r0 in range(0, n, 4096):
                r1 = min(n, r0 + 4096)
                s = (q[r0:r1, h] @ kh.T) * st["scale"]
                i_, j_ = torch.arange(r0, r1, device=DEV)[:, None] + (m - n), torch.arange(m, device=DEV)[None, :]
                seen = (j_ <= i_) if causal else torch.ones_like(s, dtype=torch.bool)
                if case["window"]:
                    seen = seen & (j_ > i_ - case["window"])
                s = s.masked_fill(~seen, -math.inf)
                z[r0:r1, h] = torch.logsumexp(s, -1)
                o[r0:r1, h] = torch.softmax(s, -1) @ vh
        outs.append(o)
        lses.append(z)
        a += n
    return torch.cat(outs), torch.cat(lses)


def _turn64(x, pos, inv, interleaved):
    """The rotation as a complex product, in 64 bits."""
    ang = pos.to(torch.float64)[:, None] * inv[None, :]
    unit = torch.polar(torch.ones_like(ang), ang)[:, None, :]
    half = inv.numel()
    y = x.clone()
    if interleaved:
        z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * unit
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * unit
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


# ------------------------------------------------------------------------------------- work
def _pairs(n, m, causal, window):
    """Query/key pairs that the mask leaves, and keys that some query sees."""
    total = 0
    off = m - n
    for i in range(n):
        hi = min(m, i + off + 1) if causal else m
        lo = max(0, i + off - window + 1) if window else 0
        total += max(0, hi - lo)
    first = max(0, off - window + 1) if window else 0
    return total, m - first


def work(case):
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if case["op"] == "rope":
        n = case["tokens"]
        return {"bytes": n * (hq + hkv) * hd * 4 + n * case["rot"] * 4 + n * 4,
                "flops": 3 * n * (hq + hkv) * case["rot"]}
    if case["op"] == "cache":
        n, total = case["tokens"], case["tokens"] + case["prefix"]
        row = hd * 2 if case["fmt"] == "bf16" else hd + 4
        moved = 2 * hkv * (n * (2 * hd + row) + total * (row + 2 * hd)) + (n + total) * 8
        if case["roped"]:
            moved += n * hq * hd * 4 + n * hd * 4
        return {"bytes": moved, "flops": 2 * hkv * hd * (3 * n + total) + (3 * n * (hq + hkv) * hd if case["roped"] else 0)}
    if case["op"] == "prompt":
        pairs = sum(_pairs(n, n, case["causal"], case["window"])[0] for n in _ints(case["lens"]))
        n = sum(_ints(case["lens"]))
        return {"bytes": n * hd * 2 * (2 * hq + 2 * hkv) + n * hq * 4, "flops": 4 * hd * hq * pairs}
    row = hd * 2 if case["fmt"] == "bf16" else hd + 4
    pairs, keys = 0, 0
    for n, m in zip(_ints(case["q_lens"]), _ints(case["kv_lens"])):
        p, k = _pairs(n, m, True, case["window"])
        pairs, keys = pairs + p, keys + k
    n = sum(_ints(case["q_lens"]))
    return {"bytes": 2 * hkv * keys * row + n * hq * (4 * hd + 4), "flops": 4 * hd * hq * pairs}
