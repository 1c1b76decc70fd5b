"""DiffAttention and a backend's share of its heads: host logic, no GPU."""

from __future__ import annotations

import pytest
import torch

from cloverinfer_b200 import B200AttentionBackend, DiffAttention
from cloverinfer_b200.head_groups import kv_head_shards


def test_heads_makes_what_the_kernel_takes():
    """float32 and contiguous, whatever the model's parameters are, all heads or some."""
    lam = torch.rand(2, 8)[0].bfloat16()
    w = torch.rand(64, 2)[:, 0].bfloat16()
    for lo, hi in ((0, 8), (2, 6)):
        for d in (DiffAttention(lam, w), DiffAttention(lam.float(), w), DiffAttention(lam, w.float().contiguous()),
                  DiffAttention(lam.float().repeat(2)[::2], None)):
            got = d.heads(lo, hi, "cpu")
            assert got.lam.dtype == torch.float32 and got.lam.is_contiguous()
            assert torch.equal(got.lam, d.lam[lo:hi].float())
            assert (got.norm_weight is None) == (d.norm_weight is None)
            if got.norm_weight is not None:
                assert got.norm_weight.dtype == torch.float32 and got.norm_weight.is_contiguous()
                assert torch.equal(got.norm_weight, d.norm_weight.float())
            assert (got.eps, got.out_scale) == (d.eps, d.out_scale)
    fits = DiffAttention(torch.rand(8), torch.rand(64))
    assert fits.heads(0, 8, "cpu") is fits


def test_from_vectors():
    g = torch.Generator().manual_seed(0)
    q1, k1, q2, k2 = (torch.randn(4, 32, generator=g) * 0.1 for _ in range(4))
    w = torch.rand(64, generator=g)
    d = DiffAttention.from_vectors(q1, k1, q2, k2, 0.2, 4, w)
    want = torch.exp((q1.double() * k1.double()).sum(1)) - torch.exp((q2.double() * k2.double()).sum(1)) + 0.2
    assert (d.lam.double() - want).abs().max() <= want.abs().max() * 2.0 ** -24
    assert d.out_scale == 1 - 0.2 and d.norm_weight is w
    # without a norm the output has no place for 1 - lambda_init
    with pytest.raises(ValueError):
        DiffAttention.from_vectors(q1, k1, q2, k2, 0.2, 4)


@pytest.mark.parametrize("world", [1, 2, 3, 4, 8])
def test_every_rank_has_the_lambdas_of_its_heads(world):
    """The shards' query heads, rank by rank, are all heads in order."""
    hkv, group = 8, 4
    lam = torch.arange(hkv * group).float()
    w = torch.rand(128)
    got = []
    for lo, hi in kv_head_shards(hkv, world):
        be = B200AttentionBackend.__new__(B200AttentionBackend)
        be.differential, be._diff = [DiffAttention(lam, w), DiffAttention(-lam, None)], []
        be.kv_range, be.num_kv_heads, be.device = (lo, hi), hkv, torch.device("cpu")
        d = be._diff_layer(1, hkv * group)
        assert d.norm_weight is None and be._diff_layer(0, hkv * group).norm_weight is w or world > 1
        got.append(-d.lam)
        assert got[-1].numel() == (hi - lo) * group
        with pytest.raises(ValueError):
            be._diff = []
            be._diff_layer(0, hkv)
    assert torch.equal(torch.cat(got), lam)
