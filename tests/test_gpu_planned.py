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
