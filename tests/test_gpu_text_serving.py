"""The operators of a serving step together: plan, head norms with positions and cache write, attention behind a
shared prefix or under a window with first tokens. Prompts arrive, continue, lose rejected drafts and end; captured
and direct steps; the bounds-checked build; memory beside the outputs; caches beyond 32-bit offsets."""
import os
import random
import subprocess
import sys
import tempfile
from pathlib import Path

import numpy as np
import pytest
import torch

from tests.test_gpu_text import BF16, F64, _check_device, _cu, _gen, _randn, _text, assert_attention, ref_inv_freq
from tests.test_gpu_text_checked import _frame_kept, _framed
from tests.test_gpu_text_heads import ref_heads
from tests.test_gpu_text_sinks import ref_seen, seen

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Server:
    """One layer of a model serving a batch: everything but its linears."""

    def __init__(self, fmt, batch, prefix, hq=8, hkv=2, hd=128, page=16, blocks=40, seed=1):
        self.text, self.g = _text(), _gen(seed)
        self.hq, self.hkv, self.hd, self.page, self.prefix, self.batch = hq, hkv, hd, page, prefix, batch
        front = -(-prefix // page)
        self.cache = self.text.PagedKVCache(front + batch * blocks, page, hkv, hd, fmt)
        self.pool = self.text.PagePool(front + batch * blocks, page, batch, blocks)
        self.front = self.pool.free[:front].clone()
        self.pool.taken.fill_(front)  # (the prefix holds the first pages)
        share = hd // 2 * 5 // 16
        self.axes = self.text.rope_axes((hd // 2 - 2 * share, share, share), True)
        self.rope = self.text.RopeTable(hd, 4096, base=500000.0, axes=self.axes)
        self.q_norm, self.k_norm = ((1 + 0.2 * torch.randn(hd, generator=self.g, device="cuda")).to(BF16) for _ in range(2))
        if prefix:
            j = torch.arange(prefix, device="cuda")
            slots = self.front.long()[j // page] * page + j % page
            q, k, v = self.rows(prefix)
            self.cache.append_roped(q, k, v, slots, self.rope, j.to(torch.int32).expand(3, -1).contiguous(),
                                    q_norm=self.q_norm, k_norm=self.k_norm)
            self.front_kv = self.stored(self.front, prefix)
        else:
            none = torch.zeros(0, hkv, hd, dtype=F64, device="cuda")
            self.front_kv = none, none

    def rows(self, n):
        x = _randn(self.g, n, self.hq + 2 * self.hkv, self.hd)
        return x[:, :self.hq], x[:, self.hq:self.hq + self.hkv], x[:, self.hq + self.hkv:]

    def stored(self, pages, n):
        """The first n keys and values of these pages, 64 bits."""
        j = torch.arange(n, device="cuda")
        pg, off = pages.long()[j // self.page], j % self.page
        out = []
        for c, s in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
            x = c.view(torch.int8 if c.dtype != BF16 else BF16)[pg, :, off].view(c.dtype).float().to(F64)
            out.append(x if s is None else x * s[pg, :, off].to(F64)[..., None])
        return out

    def step(self, new, tokens, longest, q, k, v, keep=None, window=0, sinks=0):
        plan = self.pool.plan(new, tokens, keep=keep, first_position=self.prefix)
        pos = plan.positions.expand(3, -1).contiguous()
        q = self.cache.append_roped(q, k, v, plan.slots, self.rope, pos, q_norm=self.q_norm, k_norm=self.k_norm)
        if window:
            out = self.text.paged_attention(q, self.cache, plan.cu_seqlens, plan.kv_lens, self.pool.table, longest,
                                            window=window, sinks=sinks, return_lse=True)
        else:
            out = self.text.prefix_attention(q, self.cache, self.front, self.prefix, plan.cu_seqlens, plan.kv_lens,
                                             self.pool.table, longest, return_lse=True)
        return plan, q, out

    def check(self, plan, raw_q, q, out, lse, window=0, sinks=0):
        cu, lens = plan.cu_seqlens.tolist(), plan.kv_lens.tolist()
        inv = ref_inv_freq(self.hd, 500000.0, None)
        n = cu[-1]
        want, mag = ref_heads(raw_q[:n], self.q_norm, 1e-6, plan.positions[:n].expand(3, -1), inv, self.axes, False)
        assert ((q[:n].to(F64) - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * mag).all()
        for b in range(self.batch):
            a, e, m = cu[b], cu[b + 1], lens[b]
            if a == e:
                continue
            k, v = self.stored(self.pool.table[b], m)
            p = 0 if window else self.prefix
            see = torch.ones((e - a, p + m), dtype=torch.bool, device="cuda")
            see[:, p:] = seen(e - a, m, window, sinks)
            if p:
                k, v = torch.cat([self.front_kv[0], k]), torch.cat([self.front_kv[1], v])
            ref, rl, mg = ref_seen(q[a:e], k, v, self.hd ** -0.5, see)
            assert_attention(out[a:e], lse[a:e], ref, rl, mg, f"sequence {b}")


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("batch,prefix,window,sinks,hd", [(5, 150, 0, 0, 128), (40, 600, 0, 0, 64), (6, 0, 48, 5, 128),
                                                         (3, 0, 0, 0, 64)])
def test_requests_come_and_go(fmt, batch, prefix, window, sinks, hd):
    s = Server(fmt, batch, prefix, hd=hd)
    rng = random.Random(batch)
    lens = [0] * batch
    for step in range(7):
        keep, new = list(lens), []
        for b in range(batch):
            kind = rng.random()
            if step == 0 or kind < 0.15:  # a prompt in a free or an ended request's place
                keep[b] = 0
                new.append(rng.randint(1, 120))
            elif kind < 0.35:  # drafts, of the last of which some were rejected
                keep[b] = max(0, lens[b] - rng.randint(0, 3))
                new.append(rng.randint(1, 4))
            else:
                new.append(0 if kind > 0.92 else 1)
            lens[b] = keep[b] + new[b]
        tokens = sum(new) + (step % 3) * 5  # (padded steps too)
        q, k, v = s.rows(tokens)
        plan, turned, (out, lse) = s.step(_i32(new), tokens, max(new), q, k, v, keep=_i32(keep), window=window, sinks=sinks)
        _check_device()
        assert plan.kv_lens.tolist() == lens
        s.check(plan, q, turned, out, lse, window, sinks)


@pytest.mark.parametrize("prefix,window", [(300, 0), (0, 40)])
def test_a_captured_step_serves_on(prefix, window):
    """The whole step in one graph, state in place: the same bits as direct steps of a twin."""
    a, b = (Server("int8", 24, prefix, seed=3) for _ in range(2))
    first = [1 + 7 * i % 90 for i in range(24)]
    q, k, v = a.rows(sum(first))
    for s in (a, b):
        s.step(_i32(first), sum(first), max(first), q, k, v, window=window, sinks=3)
    new = _i32([1] * 24)
    x = [t.contiguous() for t in a.rows(24)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, turned, (out, lse) = a.step(new, 24, 1, *x, window=window, sinks=3)
    for _ in range(20):
        for t, y in zip(x, b.rows(24)):
            t.copy_(y)
        graph.replay()
        plan_b, turned_b, (out_b, lse_b) = b.step(new, 24, 1, *x, window=window, sinks=3)
        assert torch.equal(out, out_b) and torch.equal(lse, lse_b) and torch.equal(turned, turned_b)
        assert torch.equal(plan.slots, plan_b.slots) and torch.equal(a.pool.lens, b.pool.lens)
    _check_device()
    a.check(plan, x[0], turned, out, lse, window, 3)


def test_two_streams_and_branches_of_a_capture():
    servers = [Server("bf16", 40, 900, seed=5), Server("e4m3", 7, 2000, seed=6), Server("bf16", 3, 100, seed=7)]
    calls = []
    for s in servers:
        n = [1 + 5 * i % 60 for i in range(s.batch)]
        q, k, v = s.rows(sum(n))
        plan, turned, _ = s.step(_i32(n), sum(n), max(n), q, k, v)
        q = turned[plan.cu_seqlens[1:].long() - 1].contiguous()
        cu, lens = _cu([1] * s.batch), plan.kv_lens.clone()
        calls.append(lambda s=s, q=q, cu=cu, lens=lens: s.text.prefix_attention(q, s.cache, s.front, s.prefix, cu, lens,
                                                                              s.pool.table, 1))
    wants = [c().clone() for c in calls]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        outs = []
        for c, side in zip(calls, sides):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                outs.append(c())
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        outs = []
        for c, side in zip(calls, sides):
            side.wait_stream(here)
            with torch.cuda.stream(side):
                outs.append(c())
        for side in sides:
            here.wait_stream(side)
    for _ in range(5):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants))
    _check_device()


def _call(server, n=1, seed=1):
    """A prefix call of n new rows a sequence over what the server holds, and the same rows as a slice."""
    s = server
    q = _randn(_gen(seed), n * s.batch, s.hq + 3, s.hd)[:, 1:1 + s.hq]
    cu = _cu([n] * s.batch)
    return lambda **how: s.text.prefix_attention(how.pop("q", q), s.cache, s.front, s.prefix, cu, s.pool.lens, s.pool.table,
                                                 n, **how), q


def _served(fmt, batch, prefix, seed):
    s = Server(fmt, batch, prefix, seed=seed)
    n = [5 + 3 * i % 40 for i in range(batch)]
    s.step(_i32(n), sum(n), max(n), *s.rows(sum(n)))
    return s


@pytest.mark.parametrize("batch,n", [(40, 1), (3, 1), (5, 40)])
def test_rows_of_a_packed_projection_in_and_out(batch, n):
    call, q = _call(_served("bf16", batch, 700, 11), n)
    want = call(q=q.contiguous())
    whole, out = _framed(n * batch, 8, 128)
    assert torch.equal(call(), want) and torch.equal(call(out=out), want)
    _check_device()
    assert torch.equal(out, want) and _frame_kept(whole, n * batch, 8)


def test_a_profiled_call_and_two_threads():
    """Events between the kernels of a call, and calls of two threads on streams of their own."""
    import ctypes
    import threading
    from wuxianhuabu_b200 import h3
    calls = [_call(_served("bf16", 40, 900, 12))[0], _call(_served("int8", 33, 1500, 13))[0]]
    wants = [c() for c in calls]
    ctx = h3.context()
    assert ctx.lib.wx_ctx_profile_enable(ctx.h, 1) == 0
    try:
        got = [c() for c in calls]
        ms, counts = (ctypes.c_double * 16)(), (ctypes.c_int64 * 16)()
        torch.cuda.synchronize()
        ctx.lib.wx_ctx_profile_read(ctx.h, ms, counts, 16)
    finally:
        assert ctx.lib.wx_ctx_profile_enable(ctx.h, 0) == 0
    assert all(torch.equal(a, b) for a, b in zip(got, wants))
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            outs = [calls[i]() for _ in range(30)]
            torch.cuda.current_stream().synchronize()
            wrong.extend(o for o in outs if not torch.equal(o, wants[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    _check_device()


def test_sequences_that_begin_behind_the_first_row():
    s = _served("e4m3", 20, 400, 14)
    q = _randn(_gen(3), 25, 8, 128)
    out = torch.full_like(q, 3.0)
    cu = torch.arange(21, dtype=torch.int32, device="cuda") + 4
    s.text.prefix_attention(q, s.cache, s.front, s.prefix, cu, s.pool.lens, s.pool.table, 1, out=out)
    _check_device()
    assert (out[:4] == 3.0).all() and (out[24:] == 3.0).all()
    for b, n in enumerate(s.pool.lens.tolist()):
        k, v = (torch.cat(x) for x in zip(s.front_kv, s.stored(s.pool.table[b], n)))
        ref, _, mag = ref_seen(q[4 + b:5 + b], k, v, 128 ** -0.5, torch.ones(1, 400 + n, dtype=torch.bool, device="cuda"))
        assert_attention(out[4 + b:5 + b], None, ref, None, mag, f"sequence {b}")


@pytest.mark.parametrize("fmt,pages", [("bf16", 9000), ("int8", 18000)])
@pytest.mark.parametrize("q_lens", [[1, 1], [1] * 40, [70, 3]])
def test_a_cache_beyond_32_bit_offsets(fmt, pages, q_lens):
    text, g = _text(), _gen(len(q_lens))
    hq, hkv, hd, page = 16, 8, 128, 256
    cache = text.PagedKVCache(pages, page, hkv, hd, fmt)
    assert cache.k.numel() * cache.k.element_size() > 1 << 32
    front = _i32([pages - 1, 1, pages // 2 + 3])
    table = _i32([[pages - 2 - i] for i in range(len(q_lens))])
    prefix, lens = 700, [n + 7 for n in q_lens]
    rope = text.RopeTable(hd, 1024)
    w = torch.ones(hd, dtype=BF16, device="cuda")
    kv = []
    for pg, n in [(front, prefix)] + [(table[b], n) for b, n in enumerate(lens)]:
        j = torch.arange(n, device="cuda")
        slots = pg.long()[j // page] * page + j % page
        q, k, v = _randn(g, n, hq, hd), _randn(g, n, hkv, hd), _randn(g, n, hkv, hd)
        cache.append_roped(q, k, v, slots, rope, j.to(torch.int32), k_norm=w)
        x = [c.view(torch.int8 if fmt != "bf16" else BF16)[pg.long()[j // page], :, j % page].view(c.dtype).to(F64)
             for c in (cache.k, cache.v)]
        if fmt != "bf16":
            x = [y * s[pg.long()[j // page], :, j % page].to(F64)[..., None] for y, s in zip(x, (cache.k_scale, cache.v_scale))]
        kv.append(x)
    q = _randn(g, sum(q_lens), hq, hd)
    out, lse = text.prefix_attention(q, cache, front, prefix, _cu(q_lens), _i32(lens), table, max(q_lens), return_lse=True)
    _check_device()
    a = 0
    for b, n in enumerate(q_lens):
        see = torch.ones((n, prefix + lens[b]), dtype=torch.bool, device="cuda")
        see[:, prefix:] = seen(n, lens[b], 0, 0)
        ref, rl, mag = ref_seen(q[a:a + n], torch.cat([kv[0][0], kv[1 + b][0]]), torch.cat([kv[0][1], kv[1 + b][1]]),
                                hd ** -0.5, see)
        assert_attention(out[a:a + n], lse[a:a + n], ref, rl, mag, fmt)
        a += n


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("q_lens", [[1, 2], [1] * 50, [90, 0, 33]])
def test_only_the_rows_are_written(fmt, q_lens):
    s = Server(fmt, len(q_lens), 200)
    n = sum(q_lens)
    plan = s.pool.plan(_i32(q_lens), n + 4)
    q, k, v = s.rows(n + 4)
    whole, turned = _framed(n + 4, 8, 128)
    s.cache.append_roped(q, k, v, plan.slots, s.rope, plan.positions.expand(3, -1).contiguous(), q_out=turned,
                         q_norm=s.q_norm, k_norm=s.k_norm)
    assert _frame_kept(whole, n + 4, 8)
    before = [t.clone() for t in (s.cache.k, s.cache.v, s.pool.table, s.front)]
    whole, out = _framed(n + 4, 8, 128)
    s.text.prefix_attention(turned, s.cache, s.front, 200, plan.cu_seqlens, plan.kv_lens, s.pool.table, max(q_lens), out=out)
    _check_device()
    assert _frame_kept(whole, n, 8)
    for x, y in zip((s.cache.k, s.cache.v, s.pool.table, s.front), before):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_many_tokens_write_only_their_rows():
    """The persistent kernel of the head norms: rows and slots beside its own keep what they held."""
    text, g = _text(), _gen(4)
    n, hq, hkv, hd, page = 2100, 14, 6, 128, 32
    tab = text.RopeTable(hd, 64)
    w = torch.ones(hd, dtype=BF16, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda") % 64
    x = _randn(g, n, hq + 2 * hkv, hd)
    wq, q_out = _framed(n, hq, hd)
    wk, k_out = _framed(n, hkv, hd)
    tab.apply_qk(x[:, :hq], x[:, hq:hq + hkv], pos, q_norm=w, k_norm=w, q_out=q_out, k_out=k_out)
    _check_device()
    assert _frame_kept(wq, n, hq) and _frame_kept(wk, n, hkv)
    for fmt in ("bf16", "int8", "e4m3"):
        pages = n // page + 3
        cache = text.PagedKVCache(pages, page, hkv, hd, fmt)
        junk = _randn(g, pages * page, hkv, hd)
        cache.append(junk, junk, torch.arange(pages * page, device="cuda"))
        held = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:n]
        wq, q_out = _framed(n, hq, hd)
        cache.append_roped(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], slots, tab, pos, q_out=q_out, q_norm=w, k_norm=w)
        _check_device()
        assert _frame_kept(wq, n, hq)
        other = torch.ones(pages * page, dtype=torch.bool, device="cuda")
        other[slots] = False
        now = [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
        for a, b in zip(now, held):
            a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b))
            a, b = (t.transpose(1, 2).reshape(pages * page, hkv, -1) for t in (a, b))
            assert torch.equal(a[other], b[other])


def test_the_example_shares_a_beginning():
    """Prompts behind one cached beginning give the states of the whole prompts, up to the roundings of bf16 between
    the layers, which are made at the same places in both."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("encode_prompt_shared", ROOT / "examples" / "encode_prompt.py")
    module = importlib.util.module_from_spec(spec)
    sys.modules["encode_prompt_shared"] = module
    spec.loader.exec_module(module)
    r = module.main(["--new", "2"])
    assert r["finite"] and r["shared"] < 0.02, r


CHILD = r'''
import sys
import numpy as np
sys.path.insert(0, sys.argv[1])
import torch
from tests.test_gpu_text import _cu, _gen, _paged, _randn, _text
from tests.test_gpu_text_heads import CASES as HEADS, _inputs
from tests.test_gpu_text_prefix import CASES as PREFIX, _behind
from tests.test_gpu_text_sinks import PAGED, PROMPTS
from wuxianhuabu_b200 import h3
text, outs = _text(), {}
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
def keep(name, *ts):
    for i, t in enumerate(ts):
        outs[f"{name}.{i}"] = t.contiguous().view(torch.uint8).cpu().numpy()
for i, (lens, hq, hkv, hd, window, sinks) in enumerate(PROMPTS):
    qkv = _randn(_gen(i), sum(lens), hq + 2 * hkv, hd)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    keep(f"prompt{i}", *text.prompt_attention(q, k, v, _cu(lens), max(lens), window=window, sinks=sinks, return_lse=True))
for fmt in ("bf16", "int8", "e4m3"):
    for i, (q_lens, kv_lens, hq, hkv, hd, page, window, sinks) in enumerate(PAGED):
        cache, table, q, _, _ = _paged(_gen(50 + i), fmt, q_lens, kv_lens, hq, hkv, hd, page)
        keep(f"{fmt}{i}", *text.paged_attention(q, cache, _cu(q_lens), i32(kv_lens), table, max(q_lens), window=window,
                                                sinks=sinks, return_lse=True))
    for i, (prefix, q_lens, kv_lens, hq, hkv, hd, page) in enumerate(PREFIX):
        cache, front, table, q, _, _ = _behind(_gen(70 + i), fmt, prefix, q_lens, kv_lens, hq, hkv, hd, page)
        keep(f"prefix{fmt}{i}", *text.prefix_attention(q, cache, front, prefix, _cu(q_lens), i32(kv_lens), table,
                                                       max(q_lens), return_lse=True))
    for i, case in enumerate(HEADS):
        tab, q, k, v, pos, qw, kw = _inputs(i, case)
        cache = text.PagedKVCache(q.shape[0] // 16 + 2, 16, k.shape[1], k.shape[2], fmt)
        slots = torch.arange(q.shape[0], device="cuda")
        keep(f"heads{fmt}{i}", cache.append_roped(q, k, v, slots, tab, pos, q_norm=qw, k_norm=kw), *cache.read(slots),
             *tab.apply_qk(q, k, pos, q_norm=qw, k_norm=kw))
pool = text.PagePool(400, 16, 30, 12)
g = torch.Generator().manual_seed(1)
for step in range(5):
    new = torch.randint(0, 30, (30,), generator=g)
    stay = (torch.rand(30, generator=g) < 0.7).to(torch.int32).cuda() * pool.lens
    plan = pool.plan(new.to(torch.int32).cuda(), 900, keep=stay)
    keep(f"plan{step}", plan.positions, plan.slots, plan.cu_seqlens, plan.kv_lens, plan.taken, pool.table, pool.free)
h3.context().check_device()  # raises on a recorded device error (bounds: code 8)
np.savez(sys.argv[2], **outs)
print("ok")
'''


def _run(variant, path):
    env = dict(os.environ)
    env.pop("WX_LIB_VARIANT", None)
    if variant:
        env["WX_LIB_VARIANT"] = variant
    r = subprocess.run([sys.executable, "-c", CHILD, str(ROOT), path], env=env, capture_output=True, text=True,
                       timeout=900, cwd=str(ROOT))
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout[-2000:] + r.stderr[-2000:]
    return np.load(path)


def test_the_checked_build_finds_nothing_and_gives_the_same_bits():
    if not (ROOT / "wuxianhuabu_b200" / "libwx_checked.so").exists():
        pytest.fail("libwx_checked.so is missing: __graft_entry__.build() builds it")
    with tempfile.TemporaryDirectory() as d:
        a, b = _run("checked", os.path.join(d, "checked.npz")), _run("", os.path.join(d, "normal.npz"))
        assert sorted(a.files) == sorted(b.files)
        for k in a.files:
            assert np.array_equal(a[k], b[k]), k
