"""Calls of the step plan, the quantising append and the decodes over scaled and
differential caches that are damaged, unusual or at the border of what the
arguments allow.  Attention is held to the bound of test_gpu_attend."""

from __future__ import annotations

import pytest
import torch

from conftest import gpu
from test_gpu_attend import BF16, F16, F32, F8, I8, Case

pytestmark = gpu


def same_bytes(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ---------------------------------------------------------------- bad pages under an append
@pytest.mark.parametrize("kv,maps,D", [(I8, 1, 128), (F8, 1, 64), (I8, 1, 256), (I8, 1, 40), (BF16, 2, 128), (F16, 2, 64),
                                       (F32, 2, 64)])
@pytest.mark.parametrize("bad", [-1, "past the cache"])
def test_an_append_to_a_bad_page_writes_nothing(kv, maps, D, bad):
    """The new tokens of a bad page are skipped; every other slot of the caches
    keeps or gets what it should, block 0 (another request's) among them."""
    from cloverinfer_b200 import _lib
    for lens, new in (([60, 47], [1, 1]), ([600, 530, 33], [1, 1, 1]), ([50, 66, 9], [4, 4, 2]),
                      ([900, 66, 450], [4, 4, 2])):
        c = Case(lens, new, hq=4, hkv=2, D=D, kv=kv, q_dt=F32 if kv == F32 else F16 if kv == F16 else BF16,
                 maps=maps, seed=31)
        kc, vc, ks, vs = c.append_reference()
        # the page of request 0's last token: what it would get stays as it was
        page = int(c.tables[0, (lens[0] - 1) // c.bs])
        for pos in range(lens[0] - new[0], lens[0]):
            if pos // c.bs == (lens[0] - 1) // c.bs:
                for want, have in ((kc, c.kc), (vc, c.vc)):
                    want[page, pos % c.bs] = have[page, pos % c.bs]
                if ks is not None:
                    ks[page, :, pos % c.bs] = c.ks[page, :, pos % c.bs]
                    vs[page, :, pos % c.bs] = c.vs[page, :, pos % c.bs]
        c.tables[0, (lens[0] - 1) // c.bs] = c.nb + 5 if bad == "past the cache" else bad
        out = c.run(step=True)
        torch.cuda.synchronize()
        assert int(c.status.item()) == _lib.DEV_BAD_BLOCK
        assert same_bytes(c.kc, kc) and same_bytes(c.vc, vc), (lens, new)
        if ks is not None:
            assert torch.equal(c.ks, ks) and torch.equal(c.vs, vs), (lens, new)
        assert bool(torch.isfinite(out[new[0]:c.T]).all())


# ---------------------------------------------------------------- queries far from zero mean
@pytest.mark.parametrize("q_dt", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("maps", [1, 2])
def test_int8_scores_of_queries_with_a_mean(D, maps, q_dt):
    """Queries around 8, keys with one dim each: the products that a score sums are
    one large value and zeros, whose sum rounds (and so may the bound) by next to
    nothing, while the sum of the query over all dims is D times as large."""
    c = Case([5] * 24 + [200], hq=16, hkv=4, D=D, kv=I8, q_dt=q_dt, maps=maps, seed=41, norm=False)
    g = torch.Generator().manual_seed(42)
    c.q = (8 + 0.02 * torch.randn(c.q.shape, generator=g)).to(q_dt).cuda()
    # token t of a block: code 127 at a dim of its own (in each half for two maps)
    codes = torch.zeros(c.nb, c.bs, c.hkv, D, dtype=I8)
    at = torch.randint(0, D // maps, (c.nb, c.bs, c.hkv), generator=g)
    for m in range(maps):
        codes.scatter_(3, (at + m * (D // 2))[..., None], 127)
    c.kc = codes.cuda()
    c.ks.fill_(1 / 127)
    c.vs.fill_(1 / 127)
    c.scale = 120.0  # scores near 960, which rounding may move by (D + 8) 2^-24 of that
    c.check(c.run(), f"D{D} {q_dt}")
