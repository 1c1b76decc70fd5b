"""Planned steps and plans on the GPU whose requests change, pad or repeat between
the plan and the layers that run it."""

from __future__ import annotations

import pytest
import torch

from conftest import gpu

pytestmark = gpu


def make(hkv=2, D=64, L=2, **kw):
    from cloverinfer_b200 import B200AttentionBackend
    be = B200AttentionBackend(num_blocks=64, num_kv_heads=hkv, max_seqs=4, device="cuda", **kw)
    g = torch.Generator().manual_seed(3)
    for rid, n in (("a", 40), ("b", 17)):
        be.init_request(rid, [{"key": torch.randn(n, hkv, D, generator=g).bfloat16(),
                               "value": torch.randn(n, hkv, D, generator=g).bfloat16()} for _ in range(L)])
    return be, g


@pytest.mark.parametrize("kw", [{}, {"kv_dtype": torch.int8}], ids=["plain", "int8"])
@pytest.mark.parametrize("reused", [False, True])
def test_a_request_freed_inside_a_step(kw, reused):
    """The step is refused before it touches the cache; the request that is left
    finishes its layers by itself."""
    be, g = make(**kw)
    hq, hkv, D = 4, 2, 64
    rnd = lambda n, h: torch.randn(n, h, D, generator=g).bfloat16().cuda()  # noqa: E731
    step = be.begin_step(["a", "b"])
    be.decode_planned(step, 0, rnd(2, hq), rnd(2, hkv), rnd(2, hkv), 0.1)
    be.free_request("a")
    if reused:  # the row and its blocks go to a request of the same length
        be.init_request("c", [{"key": torch.ones(40, hkv, D), "value": torch.ones(40, hkv, D)}] * 2)
    torch.cuda.synchronize()
    held = [be.pool.k.clone(), be.pool.v.clone(), be.pool.tables.clone()]
    with pytest.raises(KeyError):
        be.decode_planned(step, 1, rnd(2, hq), rnd(2, hkv), rnd(2, hkv), 0.1)
    torch.cuda.synchronize()
    for was, now in zip(held, (be.pool.k, be.pool.v, be.pool.tables)):
        assert torch.equal(was.view(torch.uint8), now.view(torch.uint8))
    be.decode_batch(["b"], 1, rnd(1, hq), rnd(1, hkv), rnd(1, hkv), 0.1)
    assert be.get_context_len("b") == 18
    be.pool.check_status()


def test_a_step_without_requests_or_tokens():
    be, _ = make()
    e = torch.zeros(0, 4, 64, device="cuda").bfloat16()
    kv = torch.zeros(0, 2, 64, device="cuda").bfloat16()
    for ids, n_new in (([], None), (["a", "b"], [0, 0])):
        step = be.begin_step(ids, n_new)
        assert be.decode_planned(step, 0, e, kv, kv).shape == (0, 4, 64)
    assert be.get_context_len("a") == 40
    be.pool.check_status()


def test_plans_of_different_sizes_from_two_threads():
    """The kernel's shared-memory limit is the process's: a call of one size must not
    lower it under another's launch."""
    import threading

    import cloverinfer_b200 as cb
    i32 = dict(dtype=torch.int32, device="cuda")

    def state(items, rows):
        return (torch.arange(64, **i32), torch.tensor([64], **i32), torch.full((rows, 2), -1, **i32),
                torch.zeros(rows, **i32), torch.zeros(rows, **i32), torch.arange(items, **i32),
                torch.zeros(items, **i32), 16, torch.zeros(items + 1, **i32), torch.zeros(1, **i32),
                torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, **i32))

    states, failed = [state(8192, 1 << 18), state(2048, 4096)], []
    torch.cuda.synchronize()

    def run(s):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(1500):
                    cb.plan_step(*s)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(s,)) for s in states]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed[0]
    assert all(int(s[-1].item()) == 0 for s in states)


@pytest.mark.parametrize("D", [64, 48])  # the tensor-core kernel, the other one
def test_padding_and_one_row_per_sequence(D):
    """max_q = 1 with as many rows as sequences takes row b for sequence b: padding
    behind the last row is fine, padding before one is flagged (D = 48 reads the rows'
    offsets and answers it), and max_q = 2 answers either.  Padding's own output rows
    stay as they were."""
    from cloverinfer_b200 import PagedKVPool, _lib
    hq, hkv = 4, 2
    pool = PagedKVPool(32, 16, hkv, D, max_seqs=4, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    rnd = lambda n, h: torch.randn(n, h, D, generator=g).bfloat16().cuda()  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    p = pool.plan_step(i32([0, 1, 2]), i32([30, 9, 50]), 89)
    pool.append(0, rnd(89, hkv), rnd(89, hkv), p.slots)
    q = rnd(3, hq)
    for rows, good in (([2, 0, -1], True), ([-1, 2, 0], False), ([2, -1, 0], False), ([-1, 2], False), ([1, -1], True),
                       ([-1, -1], True)):
        n = len(rows)
        p = pool.plan_step(i32(rows), i32([1] * n), n)
        new = rnd(n, hkv)
        pool.append(0, new, new, p.slots)
        want = pool.decode(0, q[:n], p.query_start_loc, p.ctx_lens, p.rows, 2, 64, 0.2, out=torch.zeros_like(q[:n]))
        pool.check_status()
        got = pool.decode(0, q[:n], p.query_start_loc, p.ctx_lens, p.rows, 1, 64, 0.2, out=torch.zeros_like(q[:n]))
        torch.cuda.synchronize()
        code = int(pool.status.item())
        pool.status.zero_()
        if good or D == 48:
            assert code == 0 and torch.equal(got, want), rows
        else:
            assert code == _lib.DEV_BAD_PLAN, rows


def test_the_largest_plan():
    """8192 items over 262144 rows and a cluster of the most CTAs."""
    import cloverinfer_b200 as cb
    i32 = dict(dtype=torch.int32, device="cuda")
    n, rows, m = 8192, 1 << 18, 8192 * 9
    g = torch.Generator().manual_seed(2)
    at = torch.randperm(rows, generator=g)[:n].int().cuda()
    new = torch.randint(0, 10, (n,), generator=g).int().cuda()
    top, qsl = torch.tensor([n], **i32), torch.zeros(n + 1, **i32)
    ctx, slots = torch.zeros(m, **i32), torch.zeros(m, dtype=torch.int64, device="cuda")
    tables, tl, sl, st = torch.full((rows, 1), -1, **i32), torch.zeros(rows, **i32), torch.zeros(rows, **i32), torch.zeros(1, **i32)
    cb.plan_step(torch.arange(n, **i32), top, tables, tl, sl, at, new, 16, qsl, ctx, slots, st)
    assert int(st.item()) == 0
    off = torch.nn.functional.pad(new.cumsum(0), (1, 0)).int()
    assert torch.equal(qsl, off) and torch.equal(sl[at.long()], new)
    used = new > 0
    assert torch.equal(tables[at.long(), 0][used], n - used.int().cumsum(0)[used].int())
    item = torch.repeat_interleave(torch.arange(n, device="cuda"), new.long())
    total = item.numel()
    pos = torch.arange(total, device="cuda") - off[item]
    assert torch.equal(ctx[:total].long(), pos + 1) and bool((ctx[total:] == 0).all())
    assert torch.equal(slots[:total], tables[at.long(), 0][item].long() * 16 + pos)
    assert bool((slots[total:] == -1).all())
