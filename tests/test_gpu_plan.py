"""The step plan against the allocator's own rules, request by request."""

from __future__ import annotations

import pytest
import torch

from conftest import gpu

pytestmark = gpu


class Alloc:
    """Allocator state on the GPU and a Python twin that pops one block at a time."""

    def __init__(self, rows, width, blocks, bs, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.bs, self.width = bs, width
        self.free = torch.randperm(blocks, generator=g).int().cuda()
        self.stack = self.free.tolist()
        self.top = torch.tensor([blocks], dtype=torch.int32, device="cuda")
        self.tables = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        self.tl = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.sl = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.py_tables, self.py_len = [[] for _ in range(rows)], [0] * rows

    def call(self, rows, new, cap=None):
        import cloverinfer_b200 as cb
        n = len(rows)
        cap = sum(max(0, x) for r, x in zip(rows, new) if r >= 0) if cap is None else cap
        qsl = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda")
        ctx = torch.full((cap,), -7, dtype=torch.int32, device="cuda")
        slots = torch.full((cap,), -7, dtype=torch.int64, device="cuda")
        cb.plan_step(self.free, self.top, self.tables, self.tl, self.sl,
                     torch.tensor(rows, dtype=torch.int32, device="cuda"),
                     torch.tensor(new, dtype=torch.int32, device="cuda"), self.bs, qsl, ctx, slots, self.status)
        torch.cuda.synchronize()
        return qsl.tolist(), ctx.tolist(), slots.tolist()

    def expect(self, rows, new, cap=None):
        qsl, ctx, slots = [0], [], []
        for r, k in zip(rows, new):
            k = k if r >= 0 else 0
            for pos in range(self.py_len[r], self.py_len[r] + k):
                while len(self.py_tables[r]) * self.bs <= pos:
                    self.py_tables[r].append(self.stack.pop())
                slots.append(self.py_tables[r][pos // self.bs] * self.bs + pos % self.bs)
                ctx.append(pos + 1)
            if r >= 0:
                self.py_len[r] += k
            qsl.append(qsl[-1] + k)
        pad = (cap or len(ctx)) - len(ctx)
        return qsl, ctx + [0] * pad, slots + [-1] * pad

    def same_state(self):
        assert int(self.status.item()) == 0
        assert int(self.top.item()) == len(self.stack)
        assert self.sl.tolist() == self.py_len
        assert self.tl.tolist() == [len(t) for t in self.py_tables]
        want = torch.full(self.tables.shape, -1, dtype=torch.int32)
        for i, t in enumerate(self.py_tables):
            want[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        assert torch.equal(self.tables.cpu(), want)


@pytest.mark.parametrize("n,rows,bs,hi", [(1, 1, 16, 1), (8, 11, 16, 1), (256, 256, 32, 4), (700, 900, 16, 9),
                                          (5, 9, 1, 3), (40, 50, 48, 3000), (3, 4, 7, 9000)])
def test_steps_match_the_allocator(n, rows, bs, hi):
    g = torch.Generator().manual_seed(n + hi)
    a = Alloc(rows, 4 * (hi // bs + 2), 4 * rows * (hi // bs + 2), bs, seed=hi)
    for step in range(4):
        r = torch.randperm(rows, generator=g)[:n].tolist()
        new = torch.randint(0, hi + 1, (n,), generator=g).tolist()
        if step == 2:
            r[n // 2] = -1  # padding
        cap = sum(new) + 5 if step % 2 else None
        got = a.call(r, new, cap if cap else sum(k for x, k in zip(r, new) if x >= 0))
        want = a.expect(r, new, cap if cap else None)
        assert got == want
        a.same_state()


def test_matches_reserve_and_slots():
    """The same pops and slots as block_reserve + compute_slots."""
    from cloverinfer_b200 import _lib
    a = Alloc(20, 64, 600, 16, seed=3)
    free, top, tables, tl = a.free.clone(), a.top.clone(), a.tables.clone(), a.tl.clone()
    rows, held = [4, 0, 19, 7], [0, 0, 0, 0]
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    for new in ([100, 1, 17, 16], [1, 1, 1, 1], [4, 60, 0, 2]):
        qsl, ctx, slots = a.call(rows, new)
        rd = torch.tensor(rows, dtype=torch.int32, device="cuda")
        target = torch.tensor([h + k for h, k in zip(held, new)], dtype=torch.int32, device="cuda")
        _lib.block_reserve(free, top, tables, tl, rd, target, 16, st)
        out = torch.empty(sum(new), dtype=torch.int64, device="cuda")
        _lib.compute_slots(tables, rd, torch.tensor(held, dtype=torch.int32, device="cuda"),
                           torch.tensor(qsl, dtype=torch.int32, device="cuda"), 16, 600, out, st)
        assert out.tolist() == slots
        held = [h + k for h, k in zip(held, new)]
        assert torch.equal(tables, a.tables) and torch.equal(tl, a.tl) and int(top) == int(a.top)
    assert int(st.item()) == 0


def test_steps_that_do_not_fit_change_nothing():
    from cloverinfer_b200 import _lib
    a = Alloc(6, 8, 20, 16, seed=1)
    a.call([0, 1, 2], [100, 16, 17])
    a.expect([0, 1, 2], [100, 16, 17])
    a.same_state()
    empty = lambda n, cap: ([0] * (n + 1), [0] * cap, [-1] * cap)  # noqa: E731
    for rows, new, cap, bit in [
            ([3, 4], [128, 100], 228, _lib.DEV_OOM),
            ([0, 1], [29, 1], 30, _lib.DEV_TABLE_FULL),
            ([0, 0], [1, 1], 2, _lib.DEV_BAD_PLAN),
            ([0, 6], [1, 1], 2, _lib.DEV_BAD_PLAN),
            ([0, 1], [-1, 1], 2, _lib.DEV_BAD_PLAN),
            ([0, 1], [3, 2], 4, _lib.DEV_BAD_PLAN),
            ([0, 1], [2 ** 31 - 1, 2 ** 31 - 1], 4, _lib.DEV_BAD_PLAN)]:
        assert a.call(rows, new, cap) == empty(len(rows), cap), (rows, new)
        assert int(a.status.item()) == bit, (rows, new)
        a.status.zero_()
        a.same_state()
    # and the state still works
    assert a.call([5, 0], [3, 20]) == a.expect([5, 0], [3, 20])
    a.same_state()


def test_sizes_of_zero():
    a = Alloc(3, 4, 8, 16)
    assert a.call([], [], 3) == ([0], [0] * 3, [-1] * 3)
    assert a.call([1, -1], [0, 5], 0) == ([0, 0, 0], [], [])
    a.same_state()


def test_captured_plan_advances():
    """One captured plan, replayed: every replay is the next step."""
    import cloverinfer_b200 as cb
    a = Alloc(8, 16, 100, 16, seed=5)
    rows = torch.tensor([2, 5, 7], dtype=torch.int32, device="cuda")
    new = torch.tensor([1, 3, 2], dtype=torch.int32, device="cuda")
    qsl = torch.zeros(4, dtype=torch.int32, device="cuda")
    ctx = torch.zeros(6, dtype=torch.int32, device="cuda")
    slots = torch.zeros(6, dtype=torch.int64, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cb.plan_step(a.free, a.top, a.tables, a.tl, a.sl, rows, new, 16, qsl, ctx, slots, a.status)
    for _ in range(40):
        g.replay()
        torch.cuda.synchronize()
        want = a.expect([2, 5, 7], [1, 3, 2])
        assert (qsl.tolist(), ctx.tolist(), slots.tolist()) == want
    a.same_state()
