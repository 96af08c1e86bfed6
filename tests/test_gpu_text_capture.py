"""Text-side calls captured in CUDA graphs. The captured work has scratch of its own that lives as long as the
context: a larger direct call does not take it away, and replays run beside direct calls. Replays give the
bits of the direct call on the same inputs."""
import pytest
import torch

from tests.test_gpu_text import BF16, _check_device, _cu, _gen, _paged, _randn, _text

pytestmark = pytest.mark.gpu


def _i32(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


class Step:
    """One layer's share of a decoding step: rope and cache write, attention over the cache, reading back."""

    def __init__(self, fmt, kv_len, new, seed, hq=8, hkv=2, hd=128, page=64):
        self.text, g = _text(), _gen(seed)
        self.cache, self.table, self.q, _, _ = _paged(g, fmt, [new], [kv_len], hq, hkv, hd, page)
        self.cu, self.lens, self.new = _cu([new]), _i32(kv_len), new
        self.rope = self.text.RopeTable(hd, kv_len + 1)
        self.pos = torch.arange(kv_len - new, kv_len, dtype=torch.int32, device="cuda")
        j = self.pos.long()
        self.slots = self.table[0].long()[j // page] * page + j % page
        self.k, self.v = _randn(g, new, hkv, hd), _randn(g, new, hkv, hd)

    def refresh(self, seed):
        g = _gen(seed)
        for t in (self.q, self.k, self.v):
            t.copy_(_randn(g, *t.shape))

    def run(self):
        q = self.cache.append_roped(self.q, self.k, self.v, self.slots, self.rope, self.pos)
        out, lse = self.text.paged_attention(q, self.cache, self.cu, self.lens, self.table, self.new, return_lse=True)
        return (out, lse) + self.cache.read(self.slots)


def _capture(run):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    return g, out


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def _clone(out):
    return [x.clone() for x in out]


# few rows: pieces joined by the last arrival; many: items cut up and joined by a second kernel
@pytest.mark.parametrize("fmt,kv_len,new", [("int8", 9000, 1), ("bf16", 5000, 3), ("e4m3", 4100, 90), ("bf16", 600, 200)])
def test_replays_after_a_larger_direct_call(fmt, kv_len, new):
    step = Step(fmt, kv_len, new, 1)
    step.run()
    graph, out = _capture(step.run)
    wide = Step(fmt, 9000, 130, 2, hq=64, hkv=16, hd=128)  # more partial sums and items than all calls before
    many = Step(fmt, 300, 1, 3)
    text = _text()
    for seed in range(3):
        step.refresh(10 + seed)
        graph.replay()
        got = _clone(out)
        wide.run()
        n = 30000  # as many items: more arrival counters
        q = many.q.expand(n, -1, -1).contiguous()
        text.paged_attention(q, many.cache, torch.arange(n + 1, dtype=torch.int32, device="cuda"), many.lens.expand(n).contiguous(),
                             many.table.expand(n, -1).contiguous(), 1)
        junk = [torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda") for _ in range(40)]
        graph.replay()
        again = _clone(out)
        del junk
        want = _clone(step.run())
        assert _same(got, want) and _same(again, want)
    _check_device()


def test_captures_need_no_call_before_them_and_may_grow():
    """A context that has no scratch yet, captured calls of growing size in one graph and in the next."""
    from wuxianhuabu_b200 import h3
    small, large = Step("bf16", 3000, 1, 4), Step("bf16", 9000, 130, 5, hq=64, hkv=16)
    want = _clone(small.run()), _clone(large.run())  # (the kernels are loaded, on the usual context)
    _check_device()
    dev = torch.cuda.current_device()
    usual = h3._contexts[dev]
    h3._contexts[dev] = h3.Context(dev)
    try:
        both, outs = _capture(lambda: (small.run(), large.run()))
        ctx = h3.context()
        held = ctx.lib.wx_ctx_workspace_bytes(ctx.h)
        assert held > 0
        second, out2 = _capture(large.run)
        for _ in range(3):
            both.replay()
            assert _same(outs[0], want[0]) and _same(outs[1], want[1])
            second.replay()
            assert _same(out2, want[1])
        direct = _clone(small.run())
        assert _same(direct, want[0])
        both.replay()
        assert _same(outs[0], want[0]) and _same(outs[1], want[1])
        h3.context().check_device()
        torch.cuda.synchronize()
        del both, second
        h3.context().close()
    finally:
        h3._contexts[dev] = usual


def test_replays_beside_direct_calls():
    """Other inputs on another stream at the same time: neither reaches the other's partial sums."""
    a, b = Step("bf16", 9000, 1, 6), Step("bf16", 8000, 2, 7)
    c, d = Step("int8", 6000, 100, 8), Step("int8", 7000, 80, 9)
    wants = [_clone(s.run()) for s in (a, b, c, d)]
    graph, outs = _capture(lambda: (a.run(), c.run()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    replayed, direct = [], []
    for i in range(20):
        with torch.cuda.stream(side):
            graph.replay()
            replayed.append((_clone(outs[0]), _clone(outs[1])))
        direct.append((b.run(), d.run()))
    torch.cuda.synchronize()
    _check_device()
    for x, y in replayed:
        assert _same(x, wants[0]) and _same(y, wants[2])
    for x, y in direct:
        assert _same(x, wants[1]) and _same(y, wants[3])
    assert wants[0][0].dtype == BF16
