"""Further text-side operators of this framework and the work they stand for.

The prompts that condition a video come with pictures and clips in them, many at a time, and mostly
behind one long common text (the system prompt, the storyboard rules). Beside rotary positions, the
paged cache and its attention (perf/operators.py), serving them needs: block tables and slot maps of
a step made from the requests' lengths where they lie, on the device (``plan``); norms of the query
and key heads with rotary positions over time, height and width in the pass that also fills the
cache (``qk``); attention with a sliding window beside which the first tokens stay visible
(``sinks``); attention over a cached prefix that all sequences share, read once for all of them
(``prefix``). Every operator exists here in a plain form (elementary torch operations in fp32) and,
with ``own`` set, as the call a user makes of this package.
"""
import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
F64 = torch.float64
QMAX = {"int8": 127.0, "e4m3": 448.0}  # largest magnitude that a stored value of the format can hold
TINY = 2.0 ** -100                     # a row with no magnitude above this is stored as zeros
EPS = 1e-6                             # of the head norms
BASE = 500000.0                        # of the rotary frequencies


def _text(ns):
    return " ".join(str(n) for n in ns)


def _ints(text):
    return [int(n) for n in text.split()]


def listed():
    return [
        # a decoding step of a serving batch: one token a sequence, now and then a new page
        dict(name="plan_step", op="plan", batch=64, page=64, most=8000, kind="step", budget=64),
        # prompts that arrive among running sequences, some of which drop rejected drafts or end; a step
        # takes so many tokens at most, and its arrays have that many entries
        dict(name="plan_arrivals", op="plan", batch=300, page=16, most=3000, kind="mixed", budget=16384),
        # one layer's q, k and v of a decoding step into an 8-bit cache
        dict(name="qk_step_e4m3", op="qk", kind="step", tokens=24, hq=16, hkv=4, hd=64, axes=3, dealt=False,
             fmt="e4m3", page=16),
        # a clip of 16 frames within its prompt: q and k of one layer, positions over three axes
        dict(name="qk_clip", op="qk", kind="clip", lead=211, frames=16, rows=18, cols=27, tail=77, hq=32, hkv=8,
             hd=128, axes=3, dealt=True, fmt="none", page=64),
        # pictures' tokens into an int8 cache, and the layer's K/V read back for a consumer that wants bf16
        dict(name="qk_picture_int8", op="qk", kind="clip", lead=40, frames=1, rows=64, cols=61, tail=333, hq=32, hkv=8,
             hd=128, axes=3, dealt=False, fmt="int8", page=64),
        # long prompts under a window, their first tokens visible throughout
        dict(name="sinks_prompt", op="sinks", q_lens="9001 1 5003", kv_lens="", hq=32, hkv=8, hd=128, fmt="none",
             page=64, window=1024, sinks=4),
        # one token of two short sequences: latency
        dict(name="sinks_tiny_bf16", op="sinks", q_lens="1 1", kv_lens="203 64", hq=16, hkv=16, hd=64, fmt="bf16",
             page=16, window=64, sinks=4),
        # a decoding batch far past the window
        dict(name="sinks_decode_int8", op="sinks", q_lens=_text([1] * 48),
             kv_lens=_text(500 + (i * 7919) % 30011 for i in range(48)), hq=32, hkv=8, hd=128, fmt="int8", page=64,
             window=4096, sinks=64),
        # a few sequences behind a short common text: latency
        dict(name="prefix_tiny_bf16", op="prefix", prefix=333, q_lens="1 1 1", kv_lens="1 40 17", hq=16, hkv=16, hd=64,
             fmt="bf16", page=16),
        # a serving batch behind one system prompt
        dict(name="prefix_decode_bf16", op="prefix", prefix=8011, q_lens=_text([1] * 64),
             kv_lens=_text(1 + (i * 2477) % 701 for i in range(64)), hq=32, hkv=8, hd=128, fmt="bf16", page=64),
        # many continuations of one long document
        dict(name="prefix_decode_e4m3", op="prefix", prefix=40000, q_lens=_text([1] * 128),
             kv_lens=_text(20 + (i * 3571) % 1501 for i in range(128)), hq=64, hkv=8, hd=128, fmt="e4m3", page=64),
        # prompts that arrive behind the common text, all their tokens new
        dict(name="prefix_prompts_int8", op="prefix", prefix=6000, q_lens="77 512 130 33 256 201",
             kv_lens="77 512 130 33 256 201", hq=28, hkv=4, hd=128, fmt="int8", page=32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "qk", "qk", "sinks", "sinks", "prefix", "prefix"])
    hq, hkv = rng.choice([(32, 8), (16, 16), (28, 4), (64, 8), (24, 8), (8, 1), (12, 4), (32, 4)])
    hd = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    fmt = rng.choice(["bf16", "int8", "e4m3"])
    if op == "plan":
        batch, kind = _log_int(rng, 1, 500), rng.choice(["step", "mixed"])
        most = _log_int(rng, 40, 8000)
        return dict(op=op, batch=batch, page=page, most=most, kind=kind,
                    budget=batch + rng.choice([0, 1, 40]) if kind == "step" else _log_int(rng, 100, 40000))
    if op == "qk":
        if rng.random() < 0.4:
            return dict(op=op, kind="step", tokens=_log_int(rng, 1, 300), hq=hq, hkv=hkv, hd=hd,
                        axes=rng.choice([1, 3, 3]), dealt=rng.random() < 0.5, fmt=fmt, page=page)
        frames, rows = rng.choice([1, 1, rng.randint(2, 16)]), rng.randint(2, 30)
        cols = max(1, min(40, 6000 * 32 // (frames * rows * hq)))
        return dict(op=op, kind="clip", lead=_log_int(rng, 1, 900), frames=frames, rows=rows, cols=rng.randint(1, cols),
                    tail=_log_int(rng, 1, 300), hq=hq, hkv=hkv, hd=hd, axes=rng.choice([1, 3, 3, 3]),
                    dealt=rng.random() < 0.5, fmt=rng.choice(["none", fmt]), page=page)
    if op == "sinks":
        window, sinks = _log_int(rng, 32, 4096), rng.choice([1, 4, 4, 16, _log_int(rng, 1, 500)])
        kind = rng.choice(["prompt", "decode", "decode", "chunk"])
        if kind == "prompt":
            q, kv, fmt = [_log_int(rng, 1, 5000) for _ in range(rng.randint(1, 3))], [], "none"
        elif kind == "decode":
            n = _log_int(rng, 1, 64)
            q, kv = [1] * n, [_log_int(rng, 1, 20000) for _ in range(n)]
        else:
            q = [_log_int(rng, 2, 600) for _ in range(rng.randint(1, 4))]
            kv = [a + rng.choice([0, _log_int(rng, 1, 12000)]) for a in q]
        return dict(op=op, q_lens=_text(q), kv_lens=_text(kv), hq=hq, hkv=hkv, hd=hd, fmt=fmt, page=page, window=window,
                    sinks=sinks)
    kind = rng.choice(["decode", "decode", "drafts", "prompts"])
    if kind == "prompts":
        q = [_log_int(rng, 4, 600) for _ in range(rng.randint(2, 6))]
        kv = list(q)
    else:
        n = _log_int(rng, 2, 100)
        q = [1 if kind == "decode" else rng.randint(2, 6) for _ in range(n)]
        kv = [a - 1 + _log_int(rng, 1, 1200) for a in q]
    return dict(op=op, prefix=_log_int(rng, 20, 24000), q_lens=_text(q), kv_lens=_text(kv), hq=hq, hkv=hkv, hd=hd,
                fmt=fmt, page=page)


# ------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(BF16)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cu(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return _i32(c)


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
    out = []
    for _ in range(2):
        x = _randn(g, pages, case["hkv"], case["page"], case["hd"])
        out += list(_quantise(x, case["fmt"]))
    kq, ks, vq, vs = out
    return kq, vq, ks, vs


def _axis_of_pair(case):
    """The position axis that each of the hd / 2 pairs turns by: height and width have 5 of 16 pairs
    each, time the others; in runs, or dealt out in turn while an axis has pairs left."""
    pairs = case["hd"] // 2
    if case["axes"] == 1:
        return [0] * pairs
    share = [pairs - 2 * (pairs * 5 // 16), pairs * 5 // 16, pairs * 5 // 16]
    if not case["dealt"]:
        return [a for a in range(3) for _ in range(share[a])]
    out = []
    while len(out) < pairs:
        for a in range(3):
            if share[a]:
                share[a] -= 1
                out.append(a)
    return out


def _positions(case, g):
    """[3, tokens]: text counts all axes on together; a clip counts frames, rows and columns, and the
    text behind it goes on from the largest of them."""
    if case["kind"] == "step":
        p = torch.randint(0, 30000, (case["tokens"],), generator=g, device=DEV, dtype=torch.int32)
        return p.expand(3, -1).contiguous()
    f, r, c = case["frames"], case["rows"], case["cols"]
    lead = torch.arange(case["lead"], device=DEV).expand(3, -1)
    grid = torch.stack(torch.meshgrid(torch.arange(f, device=DEV), torch.arange(r, device=DEV),
                                      torch.arange(c, device=DEV), indexing="ij")).reshape(3, -1) + case["lead"]
    tail = torch.arange(case["tail"], device=DEV).expand(3, -1) + case["lead"] + max(f, r, c)
    return torch.cat([lead, grid, tail], 1).to(torch.int32)


def _requests(case, seed):
    """Cached, kept and new tokens of each request of a plan, from the seed alone."""
    g = torch.Generator()
    g.manual_seed(seed)
    n, most = case["batch"], case["most"]
    cached = torch.randint(0, most, (n,), generator=g)
    kept, new = cached.clone(), torch.ones(n, dtype=torch.int64)
    if case["kind"] == "mixed":
        dice = torch.rand(n, generator=g)
        arrives, rejects, idle = dice < 0.15, (dice >= 0.15) & (dice < 0.4), dice > 0.9
        kept = torch.where(arrives, 0, kept)  # an ended request's place is taken by a new prompt
        kept = torch.where(rejects, (kept - torch.randint(1, 6, (n,), generator=g)).clamp(min=0), kept)
        new = torch.where(arrives, torch.randint(1, max(2, min(most, 300000 // n)), (n,), generator=g), new)
        new = torch.where(rejects, torch.randint(1, 6, (n,), generator=g), new)
        new = torch.where(idle, 0, new)
    before = new.cumsum(0) - new
    return cached, kept, torch.minimum(new, (case["budget"] - before).clamp(min=0))


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    st = dict(case=case, op=op)
    if op == "plan":
        cached, kept, new = _requests(case, seed)
        page = case["page"]
        have = (cached + page - 1) // page
        want = (kept + new + page - 1) // page
        blocks = 2 * case["most"] // page + 2
        pages = case["batch"] * blocks
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        # the free list is a stack that grows downwards: its entries from `taken` on are free
        taken = int(have.sum())
        table = torch.full((case["batch"], blocks), -1, dtype=torch.int32)
        table[torch.arange(blocks)[None] < have[:, None]] = order[:taken].cpu()
        st.update(cached=cached.to(DEV, torch.int32), kept=kept.to(DEV, torch.int32), new=new.to(DEV, torch.int32),
                  table=table.to(DEV), free=order, taken=_i32([taken]), tokens=case["budget"])
        if own:
            from wuxianhuabu_b200 import text
            st["pool"] = text.PagePool.from_tensors(page, st["free"], st["taken"], st["cached"], st["table"])
        return st
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if op == "qk":
        pos = _positions(case, g)
        n = pos.shape[1]
        qkv = _randn(g, n, hq + 2 * hkv, hd)  # the projection's packed output: q heads | k heads | v heads
        st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        st["q_norm"], st["k_norm"] = ((1.0 + 0.1 * _randn(g, hd).float()).to(BF16) for _ in range(2))
        st["pos"] = pos if case["axes"] == 3 else pos[0].contiguous()
        st["axis"] = _axis_of_pair(case)
        angle = torch.arange(int(pos.max()) + 1, dtype=F64, device=DEV)[:, None] * _inv_freq(hd)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        if case["fmt"] != "none":
            pages = (n + case["page"] - 1) // case["page"] + 3
            st["cache"] = _cache(g, pages, case)
            st["slots"] = torch.randperm(pages * case["page"], generator=g, device=DEV)[:n].contiguous() \
                if case["kind"] == "step" else _paged_slots(g, pages, case["page"], n)
        if own:
            from wuxianhuabu_b200 import text
            st["rope"] = text.RopeTable.from_tables(st["cos"], st["sin"],
                                                    axes=st["axis"] if case["axes"] == 3 else None)
            if case["fmt"] != "none":
                st["paged"] = text.PagedKVCache.from_tensors(*st["cache"])
        return st
    st["scale"] = 1.0 / math.sqrt(hd)
    st["q_lens"], st["lens"] = _ints(case["q_lens"]), _ints(case["kv_lens"])
    st["cu"] = _cu(st["q_lens"])
    if op == "sinks" and case["fmt"] == "none":
        qkv = _randn(g, sum(st["q_lens"]), hq + 2 * hkv, hd)
        st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        return st
    page = case["page"]
    need = [(n + page - 1) // page for n in st["lens"]]
    shared = (case.get("prefix", 0) + page - 1) // page
    pages = sum(need) + shared + 3
    st["q"] = _randn(g, sum(st["q_lens"]), hq, hd)
    st["kv_lens"] = _i32(st["lens"])
    st["cache"] = _cache(g, pages, case)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    st["prefix_blocks"] = order[:shared].clone()
    st["blocks"] = torch.full((len(need), max(need)), -1, dtype=torch.int32, device=DEV)
    at = shared
    for i, n in enumerate(need):
        st["blocks"][i, :n] = order[at:at + n]
        at += n
    if own:
        from wuxianhuabu_b200 import text
        st["paged"] = text.PagedKVCache.from_tensors(*st["cache"])
    return st


def _paged_slots(g, pages, page, n):
    table = torch.randperm(pages, generator=g, device=DEV)
    at = torch.arange(n, device=DEV)
    return table[at // page] * page + at % page


def _inv_freq(hd):
    return BASE ** (-torch.arange(0, hd, 2, dtype=F64, device=DEV) / hd)


# ------------------------------------------------------------------------------- plain forms
def run(st):
    return {"plan": _run_plan, "qk": _run_qk, "sinks": _run_sinks, "prefix": _run_prefix}[st["op"]](st)


def _run_plan(st):
    page, tokens = st["case"]["page"], st["tokens"]
    if own:
        step = st["pool"].plan(st["new"], tokens, keep=st["kept"], commit=False)
        return step.positions, step.slots, step.cu_seqlens, step.kv_lens, step.taken, st["pool"].table, st["pool"].free
    cached, kept, new = (st[x].long() for x in ("cached", "kept", "new"))
    table, free, taken = st["table"].clone(), st["free"].clone(), st["taken"].long()
    have, want = (cached + page - 1) // page, (kept + new + page - 1) // page
    column = torch.arange(table.shape[1], device=DEV)[None, :]
    # pages that sequences give back go on top of the stack, in order, before any are taken
    given = table[(column >= want[:, None]) & (column < have[:, None])]
    top = taken - given.numel()
    free[top + torch.arange(given.numel(), device=DEV)] = given
    fresh = (column >= have[:, None]) & (column < want[:, None])
    count = fresh.sum()
    rank = fresh.flatten().cumsum(0).view_as(fresh) - 1
    table = torch.where(fresh, free[(top + rank).clamp(0, free.numel() - 1)], table)
    ends = new.cumsum(0)
    cu = torch.cat([ends.new_zeros(1), ends])
    row = torch.arange(tokens, device=DEV)
    seq = torch.searchsorted(ends, row, right=True).clamp(max=len(new) - 1)
    live = row < ends[-1]
    at = torch.where(live, row - cu[seq] + kept[seq], 0)
    slot = table[seq, at // page].long() * page + at % page
    return (at.to(torch.int32), torch.where(live, slot, -1), cu.to(torch.int32), (kept + new).to(torch.int32),
            (top + count).to(torch.int32), table, free)


def _norm(x, w):
    xf = x.float()
    return xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS) * w.float()


def _turn(x, st):
    """x [tokens, heads, hd] fp32: pair (i, i + hd / 2) turned by the position of its axis."""
    pos = st["pos"].long()
    pair = torch.arange(x.shape[-1] // 2, device=DEV)
    at = pos[torch.tensor(st["axis"], device=DEV)].T if pos.dim() == 2 else pos[:, None]  # [tokens, pairs]
    c, s = st["cos"][at, pair][:, None], st["sin"][at, pair][:, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _run_qk(st):
    case = st["case"]
    fmt = case["fmt"]
    if own:
        norms = dict(q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS)
        if fmt == "none":
            return st["rope"].apply_qk(st["q"], st["k"], st["pos"], **norms)
        q = st["paged"].append_roped(st["q"], st["k"], st["v"], st["slots"], st["rope"], st["pos"], **norms)
        return (q,) + ((st["paged"].k, st["paged"].v) if fmt == "bf16" else st["paged"].read(st["slots"]))
    q, k = _turn(_norm(st["q"], st["q_norm"]), st), _turn(_norm(st["k"], st["k_norm"]), st)
    if fmt == "none":
        return q.to(BF16), k.to(BF16)
    kc, vc, ks, vs = st["cache"]
    page = case["page"]
    at, inside = st["slots"] // page, st["slots"] % page
    out = [q.to(BF16)]
    for src, dst, sc in ((k, kc, ks), (st["v"], vc, vs)):
        x, s = _quantise(src, fmt)
        raw = dst if fmt == "bf16" else dst.view(torch.int8)
        raw[at, :, inside] = x if fmt == "bf16" else x.view(torch.int8)
        if fmt == "bf16":
            out.append(dst)
        else:
            sc[at, :, inside] = s
            out.append((raw[at, :, inside].view(dst.dtype).float() * sc[at, :, inside][..., None]).to(BF16))
    return tuple(out)


def _attend(q, k, v, scale, seen):
    """One sequence: q [Lq, Hq, hd], k and v [Lk, Hkv, hd]; ``seen(a, b)`` the mask of rows a..b, or
    None for all -> out [Lq, Hq, hd], lse [Lq, Hq]."""
    lq, hq, hd = q.shape
    lk, hkv = k.shape[0], k.shape[1]
    q = q.float().view(lq, hkv, hq // hkv, hd).permute(1, 2, 0, 3)  # [Hkv, G, Lq, hd]
    kt, vv = k.float().permute(1, 2, 0)[:, None], v.float().permute(1, 0, 2)[:, None]
    out = torch.empty(hkv, hq // hkv, lq, hd, device=DEV)
    lse = torch.empty(hkv, hq // hkv, lq, device=DEV)
    step = max(1, int(2 ** 28 // max(1, hq * lk)))
    for a in range(0, lq, step):
        b = min(lq, a + step)
        s = torch.matmul(q[:, :, a:b], kt) * scale
        s = s.masked_fill(~seen(a, b), -math.inf)
        m = s.amax(-1, keepdim=True)
        p = (s - m).exp()
        den = p.sum(-1, keepdim=True)
        out[:, :, a:b] = torch.matmul(p, vv) / den
        lse[:, :, a:b] = (m + den.log()).squeeze(-1)
    return out.permute(2, 0, 1, 3).reshape(lq, hq, hd), lse.permute(2, 0, 1).reshape(lq, hq)


def _rows(st, pages, m):
    """The first m cached K and V rows of these pages as fp32 [m, Hkv, hd]."""
    kc, vc, ks, vs = st["cache"]
    at = pages[:(m + st["case"]["page"] - 1) // st["case"]["page"]].long()
    rows = []
    for c, s in ((kc, ks), (vc, vs)):
        raw = c if c.dtype == BF16 else c.view(torch.int8)
        x = raw[at].view(c.dtype).float()  # [n, Hkv, page, hd]
        if s is not None:
            x = x * s[at][..., None]
        rows.append(x.permute(0, 2, 1, 3).flatten(0, 1)[:m])
    return rows


def _run_sinks(st):
    case = st["case"]
    window, sinks = case["window"], case["sinks"]
    packed = case["fmt"] == "none"
    if own:
        from wuxianhuabu_b200 import text
        how = dict(scale=st["scale"], window=window, sinks=sinks, return_lse=True)
        if packed:
            return text.prompt_attention(st["q"], st["k"], st["v"], st["cu"], max(st["q_lens"]), **how)
        return text.paged_attention(st["q"], st["paged"], st["cu"], st["kv_lens"], st["blocks"], max(st["q_lens"]),
                                    **how)
    outs, a = [], 0
    for i, n in enumerate(st["q_lens"]):
        m = n if packed else st["lens"][i]
        k, v = (st["k"][a:a + n], st["v"][a:a + n]) if packed else _rows(st, st["blocks"][i], m)
        col = torch.arange(m, device=DEV)[None, :]

        def seen(r0, r1, m=m, n=n, col=col):
            row = torch.arange(r0, r1, device=DEV)[:, None] + (m - n)
            return (col <= row) & ((col > row - window) | (col < sinks))

        outs.append(_attend(st["q"][a:a + n], k, v, st["scale"], seen))
        a += n
    return torch.cat([o for o, _ in outs]).to(BF16), torch.cat([x for _, x in outs])


def _run_prefix(st):
    p = st["case"]["prefix"]
    if own:
        from wuxianhuabu_b200 import text
        return text.prefix_attention(st["q"], st["paged"], st["prefix_blocks"], p, st["cu"], st["kv_lens"],
                                     st["blocks"], max(st["q_lens"]), scale=st["scale"], return_lse=True)
    pk, pv = _rows(st, st["prefix_blocks"], p)
    outs, a = [], 0
    for i, (n, m) in enumerate(zip(st["q_lens"], st["lens"])):
        k, v = _rows(st, st["blocks"][i], m)
        col = torch.arange(p + m, device=DEV)[None, :]

        def seen(r0, r1, m=m, n=n, col=col):
            return col <= torch.arange(r0, r1, device=DEV)[:, None] + (p + m - n)

        outs.append(_attend(st["q"][a:a + n], torch.cat([pk, k]), torch.cat([pv, v]), st["scale"], seen))
        a += n
    return torch.cat([o for o, _ in outs]).to(BF16), torch.cat([x for _, x in outs])


# -------------------------------------------------------------------------------- definitions
def exact(case, seed):
    st = prepare(case, seed)
    return {"plan": _exact_plan, "qk": _exact_qk, "sinks": _exact_attention, "prefix": _exact_attention}[case["op"]](st)


def _exact_plan(st):
    """Sequence by sequence, on the host."""
    page = st["case"]["page"]
    cached, kept, new = (st[x].tolist() for x in ("cached", "kept", "new"))
    table, free, taken = st["table"].tolist(), st["free"].tolist(), int(st["taken"])
    stack = free[:taken]
    for b, (a, k, n) in enumerate(zip(cached, kept, new)):
        gone = table[b][-(-(k + n) // page):-(-a // page)]
        stack = stack + gone  # (in order; moved below the top together)
    given = stack[taken:]
    taken -= len(given)
    free[taken:taken + len(given)] = given
    positions, slots, cu = [], [], [0]
    for b, (a, k, n) in enumerate(zip(cached, kept, new)):
        for j in range(-(-a // page), -(-(k + n) // page)):
            table[b][j] = free[taken]
            taken += 1
        for t in range(k, k + n):
            positions.append(t)
            slots.append(table[b][t // page] * page + t % page)
        cu.append(cu[-1] + n)
    rest = st["tokens"] - len(slots)
    return (_i32(positions + [0] * rest), torch.tensor(slots + [-1] * rest, dtype=torch.int64, device=DEV), _i32(cu),
            _i32([k + n for k, n in zip(kept, new)]), _i32([taken]), _i32(table), _i32(free))


def _stored64(x, fmt):
    """The values that stand for x [..., hd] after it was stored in an 8-bit format."""
    step = x.abs().amax(-1, keepdim=True) / QMAX[fmt]
    y = x / step
    if fmt == "int8":
        return y.round() * step
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0)  # 3 fraction bits
    return torch.round(y / 2.0 ** (e - 3)) * 2.0 ** (e - 3) * step


def _exact_qk(st):
    case = st["case"]
    hd, fmt = case["hd"], case["fmt"]
    pos = st["pos"].to(F64).reshape(-1, st["q"].shape[0])
    angle = torch.stack([pos[a] * f for a, f in zip(st["axis"], _inv_freq(hd))], -1)
    unit = torch.polar(torch.ones_like(angle), angle)[:, None, :]  # the rotation as a complex product

    def head(x, w):
        x = x.to(F64)
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + EPS) * w.to(F64)
        z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * unit
        return torch.cat([z.real, z.imag], -1)

    q, k = head(st["q"], st["q_norm"]), head(st["k"], st["k_norm"])
    if fmt == "none":
        return q, k
    v = st["v"].to(F64)
    if fmt != "bf16":
        return q, _stored64(k, fmt), _stored64(v, fmt)
    at, inside = st["slots"] // case["page"], st["slots"] % case["page"]
    out = [q]
    for x, c in ((k, st["cache"][0]), (v, st["cache"][1])):
        whole = c.to(F64)
        whole[at, :, inside] = x
        out.append(whole)
    return tuple(out)


def _exact_attention(st):
    case = st["case"]
    hq, hkv, hd, packed = case["hq"], case["hkv"], case["hd"], case["fmt"] == "none"
    prefix, window, sinks = case.get("prefix", 0), case.get("window", 0), case.get("sinks", 0)

    def stored(pages, count):
        j = torch.arange(count, device=DEV)
        pg, inside = pages.long()[j // case["page"]], j % case["page"]
        out = []
        for c, s in zip(st["cache"][:2], st["cache"][2:]):
            x = c.view(torch.int8 if c.dtype != BF16 else BF16)[pg, :, inside].view(c.dtype).float().to(F64)
            out.append(x if s is None else x * s[pg, :, inside].to(F64)[..., None])
        return out

    before = stored(st["prefix_blocks"], prefix) if prefix else None
    outs, lses, a = [], [], 0
    for i, n in enumerate(st["q_lens"]):
        if packed:
            k, v = st["k"][a:a + n].to(F64), st["v"][a:a + n].to(F64)
        else:
            k, v = stored(st["blocks"][i], st["lens"][i])
        own_keys = k.shape[0]
        q = st["q"][a:a + n].to(F64)
        o = torch.empty(n, hq, hd, dtype=F64, device=DEV)
        z = torch.empty(n, hq, dtype=F64, device=DEV)
        at = torch.arange(n, device=DEV)[:, None] + (own_keys - n)
        j = torch.arange(own_keys, device=DEV)[None, :]
        hidden = j > at
        if window:
            hidden = hidden | ((j <= at - window) & (j >= sinks))
        grp = hq // hkv
        for h in range(hkv):
            mine = q[:, h * grp:(h + 1) * grp]  # [n, grp, hd]
            for r0 in range(0, n, 1024):
                r1 = min(n, r0 + 1024)
                s = torch.einsum("igd,jd->igj", mine[r0:r1], k[:, h]) * st["scale"]
                s = s.masked_fill(hidden[r0:r1, None], -math.inf)
                vals = v[:, h]
                if prefix:
                    s = torch.cat([torch.einsum("igd,jd->igj", mine[r0:r1], before[0][:, h]) * st["scale"], s], -1)
                    vals = torch.cat([before[1][:, h], vals])
                z[r0:r1, h * grp:(h + 1) * grp] = torch.logsumexp(s, -1)
                o[r0:r1, h * grp:(h + 1) * grp] = torch.softmax(s, -1) @ vals
        outs.append(o)
        lses.append(z)
        a += n
    return torch.cat(outs), torch.cat(lses)


# ------------------------------------------------------------------------------------- work
def _pairs(n, m, window, sinks):
    """Query/key pairs that the mask leaves, and keys that some query sees."""
    total = 0
    for i in range(n):
        hi = max(0, i + m - n + 1)
        lo = max(0, hi - window) if window else 0
        total += hi - lo + min(lo, sinks)
    lo = max(0, m - n + 1 - window) if window else 0
    return total, m - lo + min(lo, sinks)


def work(case):
    if case["op"] == "plan":
        b = case["batch"]
        _, _, new = _requests(case, 0)
        n = int(new.sum())
        # lengths, one page number a sequence, and the step's arrays
        return {"bytes": case["budget"] * 12 + n // case["page"] * 8 + b * 24, "flops": 0}
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    row = hd * 2 if case["fmt"] in ("bf16", "none") else hd + 4
    if case["op"] == "qk":
        n = case["tokens"] if case["kind"] == "step" else \
            case["lead"] + case["frames"] * case["rows"] * case["cols"] + case["tail"]
        moved = n * (hq * 4 * hd + hkv * 2 * hd + hd * 4 + 4 * case["axes"])
        flops = n * (hq + hkv) * hd * 8
        if case["fmt"] == "none":
            return {"bytes": moved + n * hkv * 2 * hd, "flops": flops}
        moved += n * (hkv * (2 * hd + 2 * row) + 8)
        if case["fmt"] != "bf16":  # read back
            moved += 2 * n * hkv * (row + 2 * hd)
            flops += 4 * n * hkv * hd
        return {"bytes": moved, "flops": flops}
    q_lens, kv = _ints(case["q_lens"]), _ints(case["kv_lens"])
    n, pairs, keys = sum(q_lens), 0, case.get("prefix", 0)
    pairs = n * keys
    for a, m in zip(q_lens, kv if kv else q_lens):
        p, k = _pairs(a, m, case.get("window", 0), case.get("sinks", 0))
        pairs, keys = pairs + p, keys + k
    return {"bytes": 2 * hkv * keys * row + n * hq * (4 * hd + 4), "flops": 4 * hd * hq * pairs}
