"""A head-sharded backend over a scaled cache with differential layers, on CPU
ranks (gloo): each rank hands its own heads of queries, keys, values and lambdas
to the decode, and every rank ends with all heads in order.  The decode itself is
a stand-in that marks what it was given."""

from __future__ import annotations

import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_sharded_cpu import _free_port


class Pool:
    """Stands in for the pool: out = q * lam + the KV head's k - 2 v."""
    scaled = True

    def new_dtype(self, *dtypes):
        return torch.float32

    def attend(self, layer, q, qsl, ctx, rows, max_q, max_ctx, scale, *, k_new, v_new, diff, out=None):
        group = q.shape[1] // k_new.shape[1]
        kv = (k_new - 2 * v_new).repeat_interleave(group, 1)
        res = q * diff.lam[None, :, None] * scale + kv
        return res if out is None else out.copy_(res)


def _worker(rank, world, port, hkv, group, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from cloverinfer_b200 import B200AttentionBackend, DiffAttention, HeadShardGroup
        from cloverinfer_b200.backend import PlannedStep, _Request, _Stats
        be = B200AttentionBackend.__new__(B200AttentionBackend)
        T, D, hq = 3, 4, hkv * group
        be.shard, be.pool, be.device, be.head_dim = HeadShardGroup(), Pool(), torch.device("cpu"), D
        be.num_layers, be.num_kv_heads, be.kv_range = 2, hkv, be.shard.kv_range(hkv)
        be.gather_mode, be.partition_tokens, be._peer, be._pending_ingest = "peer", 0, None, []
        be.max_rows_per_call, be._kv_esz, be.stats, be.kv_dtype = 64, 1, _Stats(), torch.int8
        lam = torch.arange(1, 1 + hq).float()
        be.differential, be._diff = [DiffAttention(lam), DiffAttention(-lam)], []
        be._reqs = {"a": _Request(0, [7, 7], 7)}
        e = torch.zeros(0, dtype=torch.int32)
        step = PlannedStep(["a"], [be._reqs["a"]], [T], [7 + T], e, e, e, e)
        g = torch.Generator().manual_seed(1)
        ok = True
        for layer in range(2):
            x, k, v = (torch.randn(T, h, D, generator=g) for h in (hq, hkv, hkv))
            want = x * be.differential[layer].lam[None, :, None] * 0.5 + (k - 2 * v).repeat_interleave(group, 1)
            got = be.decode_planned(step, layer, x, k, v, 0.5)
            ok = ok and torch.equal(got, want) and be._reqs["a"].layer_len[layer] == 7 + T
        q.put((rank, ok and be.get_context_len("a") == 7 + T))
    except Exception as err:  # report instead of leaving the parent waiting
        q.put((rank, repr(err)))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("hkv,group,world", [(4, 2, 2), (3, 4, 2), (5, 1, 3)])
def test_planned_steps_of_a_sharded_backend(hkv, group, world):
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, hkv, group, q)) for r in range(world)]
    for p in procs:
        p.start()
    res = sorted((q.get(timeout=120) for _ in procs), key=lambda r: r[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert all(r[1] is True for r in res), res
