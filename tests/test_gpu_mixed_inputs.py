"""Scaled caches filled from tensors of mixed types: what is quantised are the
values that were given."""

from __future__ import annotations

import pytest
import torch

from conftest import gpu
from test_gpu_attend import F8, I8, quantise

pytestmark = gpu

BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16


def held(codes, scales, table, n):
    """Codes and scales of a sequence's first n tokens, [n, H, D] and [n, H]."""
    ids = torch.tensor(table, device="cuda")
    c = codes[ids].flatten(0, 1)[:n]
    return c.cpu(), scales[ids].transpose(1, 2).flatten(0, 1)[:n].cpu()


def same(got, x, kv):
    code, s = quantise(x, kv)
    return torch.equal(got[0].view(torch.uint8), code.view(torch.uint8)) and torch.equal(got[1], s)


@pytest.mark.parametrize("kv", [I8, F8])
@pytest.mark.parametrize("host", [True, False])
def test_init_request_of_mixed_types(kv, host):
    from cloverinfer_b200 import B200AttentionBackend
    H, D, n = 2, 64, 37
    g = torch.Generator().manual_seed(1)
    rnd = lambda dt: torch.randn(n, H, D, generator=g).to(dt)  # noqa: E731
    be = B200AttentionBackend(num_blocks=16, num_kv_heads=H, kv_dtype=kv, kv_scales=True, max_seqs=2, device="cuda")
    layers = [{"key": rnd(BF16), "value": rnd(F32)}, {"key": rnd(F32), "value": rnd(F16)}, {"key": rnd(BF16), "value": rnd(BF16)}]
    be.init_request("a", layers if host else [{k: v.cuda() for k, v in x.items()} for x in layers])
    torch.cuda.synchronize()
    p = be.pool
    for i, layer in enumerate(layers):
        assert same(held(p.k[i], p.k_scale[i], p.row_table(0), n), layer["key"], kv), i
        assert same(held(p.v[i], p.v_scale[i], p.row_table(0), n), layer["value"], kv), i


def test_manager_of_mixed_types():
    from cloverinfer_b200 import KVCacheManager
    H, D = 2, 64
    g = torch.Generator().manual_seed(2)
    m = KVCacheManager(8, 16, H, D, dtype=I8)
    k, v = torch.randn(20, H, D, generator=g).bfloat16(), torch.randn(20, H, D, generator=g)
    m.load_initial_kv("r", k[:19], v[:19])
    m.write_new_kv("r", k[19], v[19])
    torch.cuda.synchronize()
    table, p = m.block_tables["r"], m.pool
    assert same(held(p.k[0], p.k_scale[0], table, 20), k, I8)
    assert same(held(p.v[0], p.v_scale[0], table, 20), v, I8)
