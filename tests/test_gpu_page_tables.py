"""Block tables resized and slots mapped on the GPU against the oracle's lists: whole numbers, so everything is equal."""

import random

import pytest
import torch

from conftest import announce
from oracle import page_tables as ora

pytestmark = pytest.mark.gpu


def _state(rng, slots, most, total):
    """Tables of random fillings over ``total`` pages, and the free ones in some order."""
    order = list(range(total))
    rng.shuffle(order)
    pages = [0] * slots
    table = [[-9] * most for _ in range(slots)]
    for s in range(slots):
        n = rng.randint(0, min(most, len(order) // 2))
        pages[s] = n
        table[s][:n] = [order.pop() for _ in range(n)]
    return table, pages, order


class Held:
    """The same state on the GPU and as lists."""

    def __init__(self, dev, table, pages, stack, capacity, stride=0):
        self.table, self.pages, self.stack, self.capacity = [list(t) for t in table], list(pages), list(stack), capacity
        most = len(table[0])
        self.store = torch.full((len(table), most + stride), -5, dtype=torch.int32, device=dev)
        self.t = self.store[:, :most]
        self.t.copy_(torch.tensor(table, dtype=torch.int32))
        self.p = torch.tensor(pages, dtype=torch.int32, device=dev)
        self.f = torch.full((capacity,), -3, dtype=torch.int32, device=dev)
        self.f[: len(stack)] = torch.tensor(stack, dtype=torch.int32)
        self.n = torch.tensor([len(stack)], dtype=torch.int32, device=dev)

    def resize(self, dev, idx, lens, page, index=torch.int32):
        from eagle_harness.vllm.page_tables import resize_tables

        resize_tables(self.t, self.p, torch.tensor(idx, dtype=index, device=dev), torch.tensor(lens, dtype=index, device=dev), self.f,
                      self.n, page)
        torch.cuda.synchronize()
        ora.resized(self.table, self.pages, idx, lens, self.stack, self.capacity, page)

    def check(self):
        assert self.p.tolist() == self.pages and self.n.tolist() == [len(self.stack)]
        assert self.f[: len(self.stack)].tolist() == self.stack
        got = self.t.tolist()
        assert [g[:n] for g, n in zip(got, self.pages)] == [t[:n] for t, n in zip(self.table, self.pages)]
        assert (self.store[:, self.t.shape[1]:] == -5).all()


@pytest.mark.parametrize("page", [1, 16, 24, 100])
@pytest.mark.parametrize("slots,most,stride", [(1, 1, 0), (7, 9, 3), (40, 300, 0), (1100, 5, 1), (2500, 3, 0)])
def test_tables_follow_lengths(dev, slots, most, stride, page):
    announce(f"resize tables slots={slots} most={most} page={page}")
    rng = random.Random(slots * 31 + page)
    total = slots * most
    h = Held(dev, *_state(rng, slots, most, total), total, stride)
    h.check()
    for step in range(5):
        idx = rng.sample(range(slots), rng.randint(1, slots))
        lens = [rng.choice((0, 1, page, page + 1, rng.randint(0, most * page), most * page, most * page + 1)) for _ in idx]
        for at in range(len(idx)):
            if rng.random() < 0.05:
                idx[at] = rng.choice((-1, slots, slots + 5))
        h.resize(dev, idx, lens, page, index=torch.int64 if step % 2 else torch.int32)
        h.check()


def test_too_few_pages_serve_the_first_requests(dev):
    announce("resize tables: too few pages")
    h = Held(dev, [[0, 0, 0, 0] for _ in range(6)], [0] * 6, [10, 11, 12, 13, 14], 9)
    h.table[5][:2], h.pages[5] = [20, 21], 2
    h.t[5, :2] = torch.tensor([20, 21], dtype=torch.int32)
    h.p[5] = 2
    h.resize(dev, [0, 1, 5, 2, 3, 4], [2, 4, 0, 3, 1, 1], 1)
    h.check()
    assert h.pages == [2, 4, 0, 0, 0, 0]  # 7 pages: 2 and 4 fit, then 3 does not, nor what follows
    h.resize(dev, [0, 1, 2, 3, 4, 5], [0, 0, 4, 3, 0, 0], 1)
    h.check()
    assert h.pages == [0, 0, 4, 3, 0, 0]


def test_giving_back_undoes_taking(dev):
    announce("resize tables: undone")
    rng = random.Random(4)
    h = Held(dev, *_state(rng, 200, 40, 9000), 9000)
    idx = rng.sample(range(200), 150)
    old = [h.pages[s] * 16 for s in idx]
    stack = list(h.stack)
    h.resize(dev, idx, [n + rng.randint(0, 60) for n in old], 16)
    h.check()
    h.resize(dev, idx, old, 16)
    h.check()
    assert h.stack == stack


def test_a_stack_that_cannot_hold_its_pages_changes_nothing(dev):
    announce("resize tables: no such stack")
    h = Held(dev, [[4, 5, 6]], [3], [1, 2], 3)
    h.resize(dev, [0], [0], 1)
    h.check()
    assert h.pages == [3]
    h.n.fill_(-1)
    from eagle_harness.vllm.page_tables import resize_tables

    one = torch.zeros(1, dtype=torch.int32, device=dev)
    resize_tables(h.t, h.p, one, one, h.f, h.n, 1)
    assert h.n.tolist() == [-1] and h.p.tolist() == [3]


@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("slots,most,requests,rows,extra", [(1, 1, 1, 1, 0), (9, 33, 6, 40, 7), (70, 600, 64, 17, 0), (4, 2000, 2, 9000, 11),
                                                             (300, 20, 257, 5, 100)])
def test_slots_of_rows(dev, slots, most, requests, rows, extra, page):
    from eagle_harness.vllm.page_tables import slot_maps

    announce(f"slot maps slots={slots} most={most} requests={requests} page={page}")
    rng = random.Random(most + page)
    table, pages, _ = _state(rng, slots, most, slots * most * 2 + 10)
    idx = rng.sample(range(slots), requests)
    counts = [rng.choice((0, 1, rng.randint(0, rows), rows)) for _ in idx]
    context = [rng.choice((0, rng.randint(0, most * page), max(0, pages[s] * page - n))) for s, n in zip(idx, counts)]
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    if requests > 3:
        idx[2], idx[3] = -1, slots  # padded requests
    t = lambda x, d=torch.int32: torch.tensor(x, dtype=d, device=dev)  # noqa: E731
    out = torch.full((starts[-1] + extra,), 99, dtype=torch.int64, device=dev)
    batch = torch.full((requests + 2, most), 77, dtype=torch.int32, device=dev)
    a, b = slot_maps(t(table), t(pages), t(idx), t(context, torch.int64), t(starts), page, slots=out, batch_table=batch)
    torch.cuda.synchronize()
    assert a is out and b is batch
    want = [ora.slot_of(table, pages, s, c + j, page) for s, c, n in zip(idx, context, counts) for j in range(n)]
    assert out.tolist() == want + [-1] * extra
    for r, s in enumerate(idx):
        held = pages[s] if 0 <= s < slots else 0
        assert batch[r].tolist() == (table[s][:held] if held else []) + [0] * (most - held)
    assert (batch[requests:] == 77).all()


def test_slots_without_requests_and_far_positions(dev):
    from eagle_harness.vllm.page_tables import slot_maps

    announce("slot maps: no requests, far positions")
    i32 = dict(dtype=torch.int32, device=dev)
    table, pages = torch.tensor([[(1 << 31) - 1, 5]], **i32), torch.tensor([2], **i32)
    out = torch.zeros(4, dtype=torch.int64, device=dev)
    slot_maps(table, pages, torch.zeros(0, **i32), torch.zeros(0, **i32), torch.zeros(1, **i32), 16, slots=out)
    assert out.tolist() == [-1] * 4
    page = 1 << 30
    context = torch.tensor([page - 1], dtype=torch.int64, device=dev)
    slot_maps(table, pages, torch.zeros(1, **i32), context, torch.tensor([0, 3], **i32), page, slots=out)
    assert out.tolist() == [((1 << 31) - 1) * page + page - 1, 5 * page, 5 * page + 1, -1]
    context.fill_(2 * page - 1)  # the table's last place, past 31 bits, then nothing
    slot_maps(table, pages, torch.zeros(1, **i32), context, torch.tensor([0, 3], **i32), page, slots=out)
    assert out.tolist() == [5 * page + page - 1, -1, -1, -1]


def test_captured_and_replayed(dev):
    from eagle_harness.vllm.page_tables import resize_tables, slot_maps

    announce("page tables captured")
    rng = random.Random(8)
    h = Held(dev, *_state(rng, 12, 30, 400), 400)
    idx = rng.sample(range(12), 9)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    idx_t, lens, context, starts = t(idx), t([0] * 9), t([0] * 9), t(list(range(0, 37, 4)))
    out, batch = torch.zeros(40, dtype=torch.int64, device=dev), torch.zeros(9, 30, dtype=torch.int32, device=dev)
    slot_maps(h.t, h.p, idx_t, context, starts, 16, slots=out, batch_table=batch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        resize_tables(h.t, h.p, idx_t, lens, h.f, h.n, 16)
        slot_maps(h.t, h.p, idx_t, context, starts, 16, slots=out, batch_table=batch)
    for _ in range(4):
        new = [rng.randint(4, 400) for _ in idx]
        lens.copy_(t(new))
        context.copy_(t([n - 4 for n in new]))
        graph.replay()
        torch.cuda.synchronize()
        ora.resized(h.table, h.pages, idx, new, h.stack, h.capacity, 16)
        h.check()
        assert out.tolist() == [ora.slot_of(h.table, h.pages, s, n - 4 + j, 16) for s, n in zip(idx, new) for j in range(4)] + [-1] * 4
