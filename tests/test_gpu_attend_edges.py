"""Calls of the step plan, the quantising append and the decodes over scaled and
differential caches that are damaged, unusual or at the border of what the
arguments allow.  Attention is held to the bound of test_gpu_attend."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import gpu
from test_gpu_attend import BF16, F16, F32, F8, I8, Case, quantise

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


# ---------------------------------------------------------------- weights of very different size
def repeated(c, times):
    """The one-request case as a batch of equal requests over the same blocks: enough
    work that a worker's piece of a context is thousands of tokens long.  (c.reference
    stays that of one.)"""
    n = c.lens[0]
    c.q = c.q[:1].repeat(times, 1, 1)
    c.tables = c.tables[:1].repeat(times, 1)
    c.qsl = torch.arange(times + 1, dtype=torch.int32, device="cuda")
    c.ctx = torch.full((times,), n, dtype=torch.int32, device="cuda")
    return c


SPIKE_KINDS = [(F16, 2), (I8, 1), (F8, 1), (I8, 2), (BF16, 2)]


@pytest.mark.parametrize("kv,maps", SPIKE_KINDS)
@pytest.mark.parametrize("bits", [12.3, 19.6, 26.1])
def test_many_small_weights_beside_a_large_one(kv, maps, bits):
    """One token 2^bits above 40000 equal ones: its V row has dim 0 alone, theirs the
    other dims, so those hold nothing but the small weights.  (192 such requests: the
    token's piece holds about a tenth of them.)  Bound, relative: an fp16
    weight is held to 2^-22, or by half of fp16's least step, 2^-25, where the largest
    weight is at least 2^12; the score, the base-2 exponential and the sums as in
    test_gpu_attend."""
    n, D, at = 40000, 128, 777
    c = Case([n], hq=8, hkv=1, D=D, kv=kv, q_dt=F32, maps=maps, seed=51, norm=False)
    w = D // maps
    half = torch.zeros(D, dtype=torch.float64)
    half[::w] = 1.0  # one dim of each map carries the score
    c.q = torch.zeros_like(c.q)
    c.q[..., ::w] = 1.0
    c.scale = 1.0
    nats = bits * math.log(2.0)
    k, v = torch.zeros(n, D), torch.ones(n, D)
    v[:, 0] = 0
    k[at] = half.float() * nats
    v[at] = 0
    v[at, 0] = 1.0
    g = torch.Generator().manual_seed(52)
    k[:, 3] = torch.rand(n, generator=g) - 0.5  # (rows without a score; q is 0 there)
    blocks = c.tables[0, :-(-n // c.bs)].long()
    pad = lambda x: torch.cat([x, torch.zeros(len(blocks) * c.bs - n, D)]).view(-1, c.bs, 1, D)  # noqa: E731
    for cache, scales, x in ((c.kc, c.ks, pad(k)), (c.vc, c.vs, pad(v))):
        if scales is None:
            cache[blocks] = x.to(kv).cuda()
        else:
            code, s = quantise(x, kv)
            cache.view(torch.uint8)[blocks] = code.view(torch.uint8).cuda()
            scales[blocks] = s.transpose(1, 2).cuda()
    c.lam.zero_()
    out = repeated(c, 192).run().double()
    torch.cuda.synchronize()
    assert int(c.status.item()) == 0
    ref, _ = c.reference()
    delta = (D + 8) * 2.0 ** -24 * nats
    small = 2.0 ** -bits * 2.0 ** 12
    rel = 2 * delta + 2.0 ** -20 + (n + 64) * 2.0 ** -24 + max(2.0 ** -22, 2.0 ** -25 / small)
    err = ((out - ref).abs() / ref.abs())[..., 1:].max()
    assert float(err) <= rel, f"{kv} {bits}: {float(err):.3g} of the small weights' sum, bound {rel:.3g}"
    assert float(((out - ref).abs() / ref.abs())[..., 0].max()) <= rel


@pytest.mark.parametrize("kv", [I8, F8])
@pytest.mark.parametrize("q_dt", [F32, BF16])
def test_zero_and_tiny_value_rows(kv, q_dt):
    """Thousands of zero V rows before the others; V rows so small, or so large, that
    a weight times their scale is far outside fp16."""
    c = Case([6000, 40, 3000], hq=8, hkv=2, kv=kv, q_dt=q_dt, seed=61, spread=False)
    ids = c.tables[0, :300].long()  # 4800 tokens
    c.vc.view(torch.uint8)[ids] = 0
    c.vs[ids] = 0
    c.check(c.run(), "zeros first")
    one = Case([6000], hq=8, hkv=2, kv=kv, q_dt=q_dt, seed=61, spread=False)
    one.vc.view(torch.uint8)[one.tables[0, :300].long()] = 0
    one.vs[one.tables[0, :300].long()] = 0
    one.check(repeated(one, 1200).run()[-1:], "zeros first, pieces of whole contexts")
    c.vc.view(torch.uint8)[c.tables[2, :188].long()] = 0
    c.vs[c.tables[2, :188].long()] = 0
    out = c.run()
    c.check(out, "nothing but zeros")
    assert bool((out[2] == 0).all())
    for e in (-40, -84, 115):
        c = Case([700, 40, 100], hq=8, hkv=2, kv=kv, q_dt=q_dt, seed=62, spread=False)
        c.vs *= 2.0 ** e
        c.check(c.run(), f"V of 2^{e}")
        c.vs[c.tables[0, 7]] *= 2.0 ** (60 if e < 0 else -60)  # a block of a far other size among them
        c.check(c.run(), f"V of 2^{e} beside others")


# ---------------------------------------------------------------- contexts past the tables
@pytest.mark.parametrize("kv,maps,D,new", [(I8, 1, 128, 1), (I8, 1, 128, 40), (F8, 1, 40, 1), (F16, 2, 128, 1), (F32, 2, 64, 1)])
def test_contexts_past_the_table_columns(kv, maps, D, new):
    """A view of some columns of wider tables: a longer context is cut off and
    flagged, its new token written nowhere, and the other request is answered."""
    from cloverinfer_b200 import _lib
    for blocks in (3, 60):
        n = 16 * blocks
        c = Case([n + 5, n - 3], [1, min(new, n // 2)], hq=4, hkv=2, D=D, kv=kv, q_dt=F32 if kv != F16 else F16, maps=maps,
                 seed=71)
        kc, vc, ks, vs = c.append_reference()
        page = int(c.tables[0, blocks])
        for want, have in ((kc, c.kc), (vc, c.vc)) + (((ks.transpose(1, 2), c.ks.transpose(1, 2)),
                                                       (vs.transpose(1, 2), c.vs.transpose(1, 2))) if ks is not None else ()):
            want[page, 4] = have[page, 4]
        wide = torch.full((2, blocks + 9), -1, dtype=torch.int32, device="cuda")
        wide[:, 7:7 + blocks + 1] = c.tables[:, :blocks + 1]
        full, c.tables = c.tables, wide[:, 7:7 + blocks]
        out = c.run(step=True)
        torch.cuda.synchronize()
        assert int(c.status.item()) == _lib.DEV_CTX_RANGE
        assert same_bytes(c.kc, kc) and same_bytes(c.vc, vc)
        if ks is not None:
            assert torch.equal(c.ks, ks) and torch.equal(c.vs, vs)
        # the second request alone, over the full tables
        c.tables, c.status = full, torch.zeros_like(c.status)
        ref, tol = c.reference()
        assert bool(((out.double() - ref).abs() <= tol)[1:c.T].all())


# ---------------------------------------------------------------- rows without tokens under a norm
@pytest.mark.parametrize("kv,D", [(F32, 64), (BF16, 128), (F16, 64), (I8, 128), (I8, 40)])
@pytest.mark.parametrize("longest", [40, 900])
def test_rows_without_tokens_are_zero_under_any_norm(kv, D, longest):
    """Alone, and as the first row of several; eps = 0 makes their norm 0 / 0."""
    import cloverinfer_b200 as cb
    c = Case([0, 3, longest], [1, 4, 1], hq=4, hkv=2, D=D, kv=kv, q_dt=F32, maps=2, seed=81)
    assert c.ctx_list == [0, 0, 1, 2, 3, longest]
    for eps in (0.0, 1e-5):
        out = torch.full_like(c.q, float("nan"))
        cb.diff_decode(out, c.q, c.kc, c.vc, c.lam, c.tables, c.qsl, c.ctx, max_queries_per_seq=c.max_q,
                       max_ctx_len=c.max_ctx, score_scale=c.scale, norm_weight=c.w, eps=eps, out_scale=0.6,
                       k_scales=c.ks, v_scales=c.vs, status=c.status)
        torch.cuda.synchronize()
        assert bool((out[:2] == 0).all()), eps
        assert bool(torch.isfinite(out).all())
    c.check(out, "eps 1e-5")
