"""Plans of paged steps against the same made request by request on the host: whole numbers, equal."""
import random

import pytest
import torch

from tests.test_gpu_text import _check_device, _text

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class HostPool:
    """The definition, request by request."""

    def __init__(self, free, page, batch, blocks):
        self.free, self.page, self.taken = list(free), page, 0
        self.lens, self.table = [0] * batch, [[-1] * blocks for _ in range(batch)]

    def pages(self, n):
        return -(-n // self.page)

    def plan(self, new, tokens, keep=None, first=0):
        keep = list(self.lens) if keep is None else keep
        back = []
        for b, n in enumerate(self.lens):
            back += self.table[b][self.pages(keep[b] + new[b]):self.pages(n)]
        self.taken -= len(back)
        self.free[self.taken:self.taken + len(back)] = back
        pos, slots, cu = [], [], [0]
        for b, n in enumerate(self.lens):
            for j in range(self.pages(n), self.pages(keep[b] + new[b])):
                self.table[b][j] = self.free[self.taken]
                self.taken += 1
            for i in range(keep[b], keep[b] + new[b]):
                pos.append(first + i)
                slots.append(self.table[b][i // self.page] * self.page + i % self.page)
            cu.append(cu[-1] + new[b])
            self.lens[b] = keep[b] + new[b]
        rest = tokens - len(pos)
        return pos + [0] * rest, slots + [-1] * rest, cu


def _same(plan, pool, want, host):
    pos, slots, cu = want
    assert plan.positions.tolist() == pos
    assert plan.slots.tolist() == slots
    assert plan.cu_seqlens.tolist() == cu
    assert plan.kv_lens.tolist() == host.lens
    assert plan.taken.tolist() == [host.taken]
    assert pool.table.tolist() == host.table
    assert pool.free.tolist() == host.free


@pytest.mark.parametrize("batch,page,most,padding", [
    (1, 16, 40, 0), (3, 16, 100, 5), (64, 64, 700, 0), (513, 32, 60, 100), (1100, 16, 30, 1), (2, 256, 3000, 700),
    (8192, 16, 4, 0),
])
def test_steps_in_a_row(batch, page, most, padding):
    """Prompts, single tokens, rejected drafts, ended and idle sequences, in place."""
    text = _text()
    rng = random.Random(batch * 31 + page)
    blocks = -(-3 * most // page) + 1
    order = list(range(batch * blocks))
    rng.shuffle(order)
    pool = text.PagePool(batch * blocks, page, batch, blocks)
    pool.free = _i32(order)
    host = HostPool(order, page, batch, blocks)
    for step in range(6):
        keep, new = [], []
        for b in range(batch):
            n, kind = host.lens[b], rng.random()
            k = 0 if kind < 0.2 else max(0, n - rng.randint(1, 20)) if kind < 0.4 else n
            room = blocks * page - k
            keep.append(k)
            new.append(0 if kind > 0.9 else min(room, rng.randint(1, most)) if kind < 0.2 or step == 0 else min(room, 1))
        tokens = sum(new) + padding
        plan = pool.plan(_i32(new), tokens, keep=None if step in (0, 3) else _i32(keep), first_position=7 * step)
        if step in (0, 3):
            keep = None
        _same(plan, pool, host.plan(new, tokens, keep, 7 * step), host)
        _check_device()
    assert plan.kv_lens is pool.lens


def test_a_step_is_planned_again():
    """Without commit nothing but table entries behind the lengths changes; then with."""
    text = _text()
    pool = text.PagePool(40, 16, 4, 8)
    host = HostPool(range(40), 16, 4, 8)
    first = [33, 1, 16, 0]
    _same(pool.plan(_i32(first), 50), pool, host.plan(first, 50), host)
    lens, taken = pool.lens.clone(), pool.taken.clone()
    tries = [pool.plan(_i32([20, 0, 1, 5]), 26, keep=_i32([2, 0, 16, 0]), commit=False) for _ in range(3)]
    assert torch.equal(pool.lens, lens) and torch.equal(pool.taken, taken)
    for t in tries[1:]:
        for a, b in zip(vars(t).values(), vars(tries[0]).values()):
            assert torch.equal(a, b)
    want = host.plan([20, 0, 1, 5], 26, [2, 0, 16, 0])
    _same(tries[0], pool, want, host)
    again = pool.plan(_i32([20, 0, 1, 5]), 26, keep=_i32([2, 0, 16, 0]))
    _same(again, pool, want, host)
    assert torch.equal(again.kv_lens, tries[0].kv_lens)
    _check_device()


def test_all_pages_out_and_back():
    text = _text()
    pool = text.PagePool(6, 16, 2, 6)
    host = HostPool(range(6), 16, 2, 6)
    for new, keep in (([96, 0], None), ([0, 96], [0, 0]), ([80, 16], [0, 0]), ([0, 0], [0, 0])):
        tokens = sum(new)
        _same(pool.plan(_i32(new), tokens, keep=None if keep is None else _i32(keep)), pool,
              host.plan(new, tokens, keep), host)
    assert host.taken == 0 and sorted(pool.free.tolist()) == list(range(6))
    _check_device()


def test_empty_batch_and_no_tokens():
    text = _text()
    pool = text.PagePool(4, 16, 0, 2)
    plan = pool.plan(_i32([]), 3)
    assert plan.positions.tolist() == [0, 0, 0] and plan.slots.tolist() == [-1, -1, -1]
    assert plan.cu_seqlens.tolist() == [0] and plan.taken.tolist() == [0]
    pool = text.PagePool(4, 16, 2, 2)
    plan = pool.plan(_i32([0, 0]), 0)
    assert plan.cu_seqlens.tolist() == [0, 0, 0] and plan.positions.numel() == 0
    _check_device()


@pytest.mark.parametrize("new,keep,tokens,first", [
    ([5, 3], None, 7, 0),             # more new tokens than the step has entries
    ([49, 0], None, 60, 0),           # more blocks than the table has
    ([30, 46], None, 80, 0),          # more pages than are free
    ([-1, 0], None, 5, 0), ([1, 0], [-1, 0], 5, 0),
    ([1, 0], [21, 0], 5, 0),          # more kept than there are
    ([1, 0], None, 5, 2 ** 31 - 20),  # a position beyond 32 bits
    ([2 ** 31 - 1, 2 ** 31 - 1], None, 5, 0),
])
def test_a_step_that_does_not_fit_changes_nothing(new, keep, tokens, first):
    text = _text()
    from wuxianhuabu_b200 import h3
    pool = text.PagePool(5, 16, 2, 4)
    pool.plan(_i32([20, 2]), 22)
    _check_device()
    before = [t.clone() for t in (pool.free, pool.taken, pool.lens, pool.table)]
    plan = pool.plan(_i32(new), tokens, keep=None if keep is None else _i32(keep), first_position=first)
    with pytest.raises(h3.WxError):
        _check_device()
    for a, b in zip(before, (pool.free, pool.taken, pool.lens, pool.table)):
        assert torch.equal(a, b)
    assert plan.cu_seqlens.tolist() == [0, 0, 0]
    assert plan.slots.tolist() == [-1] * tokens and plan.positions.tolist() == [0] * tokens
    pool.plan(_i32([1, 1]), 2)  # the next step that fits goes through
    _check_device()
    assert pool.lens.tolist() == [21, 3]


def test_pages_that_are_none_are_reported():
    text = _text()
    from wuxianhuabu_b200 import h3
    pool = text.PagePool(4, 16, 1, 4)
    pool.free = _i32([0, 9, -3, 2])
    plan = pool.plan(_i32([40]), 40)
    with pytest.raises(h3.WxError):
        _check_device()
    assert plan.slots.tolist() == list(range(16)) + [-1] * 24


def test_captured_steps_count_on():
    """A captured plan updates lengths and pages in place: every replay is the next step."""
    text = _text()
    pool, host = text.PagePool(64, 16, 3, 16), HostPool(range(64), 16, 3, 16)
    new = _i32([1, 2, 0])
    pool.plan(_i32([30, 5, 90]), 125)
    host.plan([30, 5, 90], 125)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = pool.plan(new, 700)  # (two CTAs: the counter of arrivals is the captured one)
    for _ in range(20):
        graph.replay()
        torch.cuda.synchronize()
        _same(plan, pool, host.plan([1, 2, 0], 700), host)
    new.copy_(_i32([0, 0, 100]))
    graph.replay()
    _same(plan, pool, host.plan([0, 0, 100], 700), host)
    _check_device()


def test_refusals():
    text = _text()
    from wuxianhuabu_b200 import h3
    pool = text.PagePool(8, 16, 2, 4)
    one = _i32([1, 1])
    for call in (lambda: pool.plan(_i32([1]), 4), lambda: pool.plan(one.long(), 4), lambda: pool.plan(one, -1),
                 lambda: pool.plan(one, 2 ** 31), lambda: pool.plan(one, 4, keep=one.long()),
                 lambda: pool.plan(one, 4, first_position=-1), lambda: pool.plan(one.cpu(), 4),
                 lambda: text.PagePool(8, 24, 2, 4).plan(one, 4), lambda: text.PagePool(0, 16, 2, 4),
                 lambda: text.PagePool(8, 16, 2, 0), lambda: text.PagePool(8, 16, 8193, 1).plan(_i32([1] * 8193), 4),
                 lambda: text.PagePool.from_tensors(16, pool.free, pool.taken, pool.lens, pool.table[:1]),
                 lambda: text.PagePool.from_tensors(16, pool.free, pool.lens, pool.lens, pool.table)):
        with pytest.raises(h3.WxError):
            call()
    _check_device()
    assert pool.lens.tolist() == [0, 0]
