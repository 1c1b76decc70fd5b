"""Decode over an 8-bit cache with scales, differential decode and the
quantising append against their definitions in 64 bits.

Tolerance (``bound``), from the arithmetic, per case:
  * a score is a sum of D products in fp32 (plus the scale): off by at most
    delta = (D + 8) * 2^-24 * S, S the largest sum of |q_d k_d| * scale;
  * softmax weights are then off by a factor within e^(2 delta), and by the
    base-2 exponential's few 2^-22; splitting a weight into two 16-bit terms
    leaves 2^-16 of it (bf16; 2^-21 for fp16), into three 2^-23;
  * the weighted sum adds n + 64 roundings of 2^-24 (n tokens, the join of the
    pieces), each of at most max|v|;
  * a 16-bit output rounds by half a step.
Differential maps add up with factor 1 + |lambda|; the norm divides that by the
rms and moves the rms itself, so a value o/rms moves by at most
(1 + |o| / rms) times it.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import gpu

pytestmark = gpu

I8, F8 = torch.int8, torch.float8_e4m3fn
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TOP = {I8: 127.0, F8: 448.0}
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def quantise(x, kv):
    """The stored codes and scales of rows x [..., D], in fp32 as defined."""
    x = x.float()
    a = x.abs().amax(-1)
    fine, zero = a.isfinite() & (a >= 2.0 ** -100), torch.zeros_like(a)
    s = torch.where(fine, a / torch.full_like(a, TOP[kv]), zero)
    f = torch.where(fine, a.reciprocal() * TOP[kv], zero)
    y = torch.where(fine[..., None], x * f[..., None], torch.zeros_like(x))
    code = y.round().clamp(-127, 127).to(I8) if kv == I8 else y.to(F8)
    return code, torch.where(a.isfinite(), s, torch.full_like(a, float("nan")))


class Case:
    """Random paged caches, tables and queries of one call."""

    def __init__(self, lens, n_new=None, *, hq=8, hkv=2, D=128, bs=16, kv=I8, q_dt=F32, maps=1, seed=0,
                 tables_rows=0, extra_rows=0, norm=True, new_dt=None, spread=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hq, self.hkv, self.D, self.bs, self.kv, self.maps = list(lens), hq, hkv, D, bs, kv, maps
        B = len(lens)
        self.n_new = [1] * B if n_new is None else list(n_new)
        self.T = sum(self.n_new)
        nblk = [max(1, -(-n // bs)) for n in lens]
        self.nb = sum(nblk) + 3
        perm = torch.randperm(self.nb, generator=g)
        rows = B + tables_rows
        self.seq_rows = torch.randperm(rows, generator=g)[:B] if tables_rows else torch.arange(B)
        tables = torch.full((rows, max(nblk) + 1), -1, dtype=torch.int32)
        o = 0
        for i, k in enumerate(nblk):
            tables[self.seq_rows[i], :k] = perm[o:o + k].to(torch.int32)
            o += k
        qsl, ctx = [0], []
        for n, k in zip(lens, self.n_new):
            qsl.append(qsl[-1] + k)
            ctx += [max(0, n - k + 1 + j) for j in range(k)]
        self.ctx_list, self.qsl_list = ctx, qsl
        R = self.T + extra_rows
        self.q = torch.randn(R, hq, D, generator=g).to(q_dt).cuda()
        kc = torch.randn(self.nb, bs, hkv, D, generator=g)
        vc = torch.randn(self.nb, bs, hkv, D, generator=g)
        if spread:  # rows of very different magnitude, for the scales
            vc *= torch.exp(torch.randn(self.nb, bs, hkv, 1, generator=g))
        self.ks = self.vs = None
        if kv in TOP:
            (kc, ks), (vc, vs) = quantise(kc, kv), quantise(vc, kv)
            self.ks, self.vs = (s.transpose(1, 2).contiguous().cuda() for s in (ks, vs))
        self.kc, self.vc = kc.to(kv).cuda(), vc.to(kv).cuda()
        dt = new_dt or (q_dt if kv in TOP else kv)
        self.kn = torch.randn(R, hkv, D, generator=g).to(dt).cuda()
        self.vn = torch.randn(R, hkv, D, generator=g).to(dt).cuda()
        self.lam = (torch.rand(hq, generator=g) * 0.6 + 0.2).cuda()
        self.w = (1 + 0.1 * torch.randn(D, generator=g)).cuda() if norm else None
        self.tables = tables.cuda()
        self.qsl = torch.tensor(qsl, dtype=torch.int32).cuda()
        self.ctx = torch.tensor(ctx + [0] * extra_rows, dtype=torch.int32).cuda()
        self.rows_d = self.seq_rows.int().cuda() if tables_rows else None
        self.scale = 1 / math.sqrt(D // maps)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.max_q, self.max_ctx = max(self.n_new + [1]), max(self.lens + [0])

    def run(self, step=False, out=None, **kw):
        import cloverinfer_b200 as cb
        if out is None:
            out = torch.full_like(self.q, float("nan"))
        args = dict(max_queries_per_seq=self.max_q, max_ctx_len=self.max_ctx, score_scale=self.scale,
                    seq_rows=self.rows_d, status=self.status)
        if step:
            args.update(k_new=self.kn, v_new=self.vn)
        args.update(kw)
        if self.maps == 1:
            cb.scaled_decode(out, self.q, self.kc, self.vc, self.ks, self.vs, self.tables, self.qsl, self.ctx,
                             **args)
        else:
            cb.diff_decode(out, self.q, self.kc, self.vc, self.lam, self.tables, self.qsl, self.ctx,
                           norm_weight=self.w, eps=1e-5, out_scale=0.6, k_scales=self.ks, v_scales=self.vs,
                           **args)
        return out

    def append_reference(self):
        """What the caches hold after the step's append."""
        kc, vc = self.kc.clone(), self.vc.clone()
        ks, vs = (None, None) if self.ks is None else (self.ks.clone(), self.vs.clone())
        r = 0
        for b, k in enumerate(self.n_new):
            for _ in range(k):
                pos = self.ctx_list[r] - 1
                if pos >= 0:
                    blk = int(self.tables[self.seq_rows[b], pos // self.bs])
                    for c, s, x in ((kc, ks, self.kn[r]), (vc, vs, self.vn[r])):
                        if s is None:
                            c[blk, pos % self.bs] = x
                        else:
                            code, sc = quantise(x, self.kv)
                            c.view(torch.uint8)[blk, pos % self.bs] = code.view(torch.uint8)
                            s[blk, :, pos % self.bs] = sc
                r += 1
        return kc, vc, ks, vs

    def reference(self):
        """(out, bound) in 64 bits from what the caches hold now."""
        f = torch.float64
        hq, hkv, D = self.hq, self.hkv, self.D
        g = hq // hkv
        out = torch.zeros(self.T, hq, D, dtype=f, device="cuda")
        tol = torch.zeros_like(out)
        w = D // self.maps
        terms = 2.0 ** -16 if self.kv == BF16 and self.q.dtype == BF16 else 2.0 ** -21
        r = 0
        for b, k in enumerate(self.n_new):
            n = max([self.ctx_list[r + j] for j in range(k)] + [0])
            ids = self.tables[self.seq_rows[b], :-(-n // self.bs)].long()
            K, V = (c[ids].to(f) for c in (self.kc, self.vc))
            if self.ks is not None:
                K = K * self.ks[ids].to(f).permute(0, 2, 1)[..., None]
                V = V * self.vs[ids].to(f).permute(0, 2, 1)[..., None]
            K, V = K.reshape(-1, hkv, D), V.reshape(-1, hkv, D)
            for _ in range(k):
                m = self.ctx_list[r]
                for h in range(hkv if m else 0):
                    heads = slice(h * g, (h + 1) * g)
                    q, v = self.q[r, heads].to(f), V[:m, h]
                    o = torch.zeros(g, D, dtype=f, device="cuda")
                    e = torch.zeros(g, 1, dtype=f, device="cuda")
                    for mp in range(self.maps):
                        qm, km = q[:, mp * w:(mp + 1) * w], K[:m, h, mp * w:(mp + 1) * w]
                        p = torch.softmax(qm @ km.T * self.scale, -1)
                        s = (qm.abs() @ km.abs().T).amax(-1, keepdim=True) * self.scale
                        delta = (D + 8) * 2.0 ** -24 * s
                        # weights times |v|: what any relative error of the weights is taken of
                        mass = (p @ v.abs()).amax(-1, keepdim=True)
                        err = mass * (2 * delta + terms + 2.0 ** -20 + (m + 64) * 2.0 ** -24)
                        sign = 1.0 if mp == 0 else -self.lam[heads].to(f)[:, None]
                        o = o + sign * (p @ v)
                        e = e + (1.0 if mp == 0 else sign.abs()) * err
                    e = e.expand(g, D)
                    if self.maps == 2 and self.w is not None:
                        rms = torch.sqrt((o * o).mean(-1, keepdim=True) + 1e-5)
                        y = o / rms
                        c = (self.w.to(f) * 0.6).abs()
                        e = e / rms * (1 + y.abs()) * c + y.abs() * c * 2.0 ** -20
                        o = y * self.w.to(f) * 0.6
                    out[r, heads] = o
                    tol[r, heads] = e
                r += 1
        return out, tol + out.abs() * HALF[self.q.dtype] * 1.01

    def check(self, out, what=""):
        torch.cuda.synchronize()
        assert int(self.status.item()) == 0, what
        ref, tol = self.reference()
        got = out[:self.T].double()
        assert torch.isfinite(got).all(), what
        bad = (got - ref).abs() > tol
        worst = ((got - ref).abs() / tol.clamp_min(1e-300)).max() if got.numel() else 0
        assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float(worst):.3g} of the bound"


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 511, 4097]
SHORT = [0, 1, 2, 16, 31, 100, 256]


# ---------------------------------------------------------------- scaled decode
@pytest.mark.parametrize("lens", [LENS, SHORT], ids=["long", "short"])
@pytest.mark.parametrize("kv,q_dt", [(I8, F32), (I8, BF16), (F8, F16), (F8, BF16), (F8, F32)])
@pytest.mark.parametrize("D,bs,hq,hkv", [(64, 16, 12, 12), (128, 16, 28, 4), (128, 32, 32, 8), (256, 48, 8, 1),
                                         (96, 16, 6, 3), (33, 5, 4, 2)])
def test_scaled_decode(D, bs, hq, hkv, kv, q_dt, lens):
    c = Case(lens, hq=hq, hkv=hkv, D=D, bs=bs, kv=kv, q_dt=q_dt, seed=D + bs)
    out = c.run()
    c.check(out, f"D{D} bs{bs} {hq}/{hkv} {kv} {q_dt}")
    assert bool((out[0] == 0).all())  # an empty context


@pytest.mark.parametrize("kv", [I8, F8])
@pytest.mark.parametrize("D,bs,hq,hkv", [(128, 32, 32, 8), (128, 16, 8, 1), (64, 16, 6, 2), (256, 16, 8, 2), (40, 8, 4, 4)])
@pytest.mark.parametrize("step", [False, True])
def test_scaled_multi_token_rows(D, bs, hq, hkv, kv, step):
    lens, new = [1, 2, 5, 17, 33, 64, 900, 0, 2048, 40], [1, 2, 4, 3, 4, 4, 2, 0, 4, 21]
    c = Case(lens, new, hq=hq, hkv=hkv, D=D, bs=bs, kv=kv, q_dt=BF16, seed=7, tables_rows=3, extra_rows=2)
    want = c.append_reference()
    mark = torch.full_like(c.q, 7.0)
    out = c.run(step=step, out=mark)
    if step:
        torch.cuda.synchronize()
        for got, ref in zip((c.kc, c.vc), want[:2]):
            assert torch.equal(got.view(torch.uint8), ref.view(torch.uint8))
        assert torch.equal(c.ks, want[2]) and torch.equal(c.vs, want[3])
    c.check(out, f"step {step}")
    assert bool((out[c.T:] == 7).all())  # rows behind the last sequence


def test_scaled_strides_and_new_types():
    for new_dt in (F32, F16, BF16):
        c = Case([300, 17, 40], hq=8, hkv=2, kv=I8, q_dt=F16, new_dt=new_dt, seed=3)
        wide = torch.zeros(3, 3, 8, 128, dtype=F16, device="cuda")
        wide[:, 1] = c.q
        c.q = wide[:, 1]
        both = torch.stack([c.kn, c.vn], 1).contiguous()  # K and V interleaved per token
        c.kn, c.vn = both[:, 0], both[:, 1]
        want = c.append_reference()
        o = torch.zeros(3, 2, 8, 128, dtype=F16, device="cuda")
        c.run(step=True, out=o[:, 1])
        assert torch.equal(c.kc, want[0]) and torch.equal(c.vs, want[3])
        c.check(o[:, 1], str(new_dt))
        assert bool((o[:, 0] == 0).all())


def test_single_rows_and_heads_of_any_stride():
    """One row, one head: the strides of axes of length one say nothing."""
    for maps, kv in ((1, I8), (2, F16)):
        c = Case([90], hq=1, hkv=1, kv=kv, q_dt=F16, maps=maps, seed=6)
        c.q, c.kn, c.vn = (x.as_strided(x.shape, (0, 7, 1)) for x in (c.q, c.kn, c.vn))
        want = c.append_reference()
        out = c.run(step=True)
        assert torch.equal(c.kc.view(torch.uint8), want[0].view(torch.uint8))
        c.check(out, "one row")


# ---------------------------------------------------------------- differential decode
@pytest.mark.parametrize("lens", [LENS, SHORT], ids=["long", "short"])
@pytest.mark.parametrize("kv,q_dt", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32), (I8, BF16), (F8, F32)])
@pytest.mark.parametrize("D,bs,hq,hkv", [(64, 16, 12, 12), (128, 16, 28, 4), (128, 32, 8, 1), (256, 16, 8, 2), (34, 7, 4, 2)])
def test_diff_decode(D, bs, hq, hkv, kv, q_dt, lens):
    c = Case(lens, hq=hq, hkv=hkv, D=D, bs=bs, kv=kv, q_dt=q_dt, maps=2, seed=D + bs)
    out = c.run()
    c.check(out, f"D{D} bs{bs} {hq}/{hkv} {kv} {q_dt}")
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("kv,q_dt", [(BF16, BF16), (F16, F32), (F32, F32), (I8, F16)])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("step", [False, True])
def test_diff_multi_token_rows(kv, q_dt, norm, step):
    lens, new = [1, 2, 5, 17, 33, 64, 900, 0, 2048, 40], [1, 2, 4, 3, 4, 4, 2, 0, 4, 21]
    c = Case(lens, new, hq=8, hkv=2, kv=kv, q_dt=q_dt, maps=2, seed=9, tables_rows=2, extra_rows=1, norm=norm)
    want = c.append_reference()
    mark = torch.full_like(c.q, 7.0)
    out = c.run(step=step, out=mark)
    if step:
        assert torch.equal(c.kc.view(torch.uint8), want[0].view(torch.uint8))
        assert torch.equal(c.vc.view(torch.uint8), want[1].view(torch.uint8))
    c.check(out, f"{kv} norm {norm} step {step}")
    assert bool((out[c.T:] == 7).all())


def test_diff_of_equal_maps_and_zero_lambda():
    """Equal halves: o = (1 - lambda) of either map; lambda 0: map 1 alone."""
    c = Case([5, 700], hq=4, hkv=2, kv=F32, q_dt=F32, maps=2, norm=False)
    c.kc[..., 64:] = c.kc[..., :64]
    c.q[..., 64:] = c.q[..., :64]
    c.check(c.run(), "equal maps")
    c.lam.zero_()
    c.check(c.run(), "lambda 0")


# ---------------------------------------------------------------- shapes of the batch
KINDS = [(I8, BF16, 1, 128), (F8, F32, 1, 64), (F16, F16, 2, 128), (F32, F32, 2, 48)]


@pytest.mark.parametrize("kv,q_dt,maps,D", KINDS)
def test_batches_of_many_sizes(kv, q_dt, maps, D):
    """No context at all; more sequences than threads of a CTA; one long request; a
    batch whose requests are mostly short beside a long one."""
    g = torch.Generator().manual_seed(D)
    many = torch.randint(0, 60, (900,), generator=g).tolist()
    for lens in ([0, 0, 0], many + [700], [70001], [3] * 40 + [20000], [256] * 5, [257] * 5):
        c = Case(lens, hq=2, hkv=1, D=D, kv=kv, q_dt=q_dt, maps=maps, seed=len(lens))
        c.check(c.run(), f"{len(lens)} requests, longest {max(lens)}")


@pytest.mark.parametrize("kv,q_dt,maps,D", KINDS)
def test_a_prompt_of_new_rows(kv, q_dt, maps, D):
    """Hundreds of causal rows of one request: many column chunks of one context."""
    c = Case([330, 40], [300, 1], hq=4, hkv=2, D=D, kv=kv, q_dt=q_dt, maps=maps, seed=8)
    want = c.append_reference()
    out = c.run(step=True)
    assert torch.equal(c.kc.view(torch.uint8), want[0].view(torch.uint8))
    c.check(out, "300 rows")


def test_the_bound_of_contexts_may_be_loose():
    for maps, kv in ((1, I8), (2, F16)):
        c = Case([100, 1, 3000], hq=8, hkv=2, kv=kv, q_dt=F16, maps=maps, seed=12)
        c.max_ctx = 131072
        c.check(c.run(), "loose")


def test_zero_and_negative_score_scales():
    for scale in (0.0, -0.2):
        for maps, kv in ((1, F8), (2, BF16), (2, F32)):
            c = Case([100, 17], hq=4, hkv=2, kv=kv, q_dt=F32, maps=maps, seed=13, norm=False)
            c.scale = scale
            out = c.run()
            c.scale = scale
            ref, tol = c.reference()
            # (the bound's S is of |scale|)
            c.scale = abs(scale)
            tol = torch.maximum(tol, c.reference()[1])
            assert bool(((out.double() - ref).abs() <= tol).all()), (scale, maps, kv)


# ---------------------------------------------------------------- masked places
@pytest.mark.parametrize("kv,maps", [(BF16, 2), (F16, 2), (F32, 2), (I8, 1), (F8, 1), (F8, 2)])
@pytest.mark.parametrize("D", [128, 48])
def test_nothing_leaks_from_masked_places(kv, maps, D):
    """Free slots, foreign blocks and later tokens hold NaN and infinities."""
    lens, new = [1, 37, 130, 600], [1, 3, 4, 2]
    c = Case(lens, new, hq=4, hkv=2, D=D, kv=kv, q_dt=F32, maps=maps, seed=21)
    used = torch.zeros(c.nb, c.bs, dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(n):
            used[int(c.tables[b, p // c.bs]), p % c.bs] = True
    free = ~used.cuda()
    if kv in TOP:
        c.ks.transpose(1, 2)[free] = float("nan")
        c.vs.transpose(1, 2)[free] = float("inf")
        c.kc.view(torch.uint8)[free] = 0x7F
        c.vc.view(torch.uint8)[free] = 0xFF  # e4m3: NaN
    else:
        c.kc[free] = float("nan")
        c.vc[free] = float("inf")
    c.check(c.run(), "free slots")
    # the last token of the 130-token sequence: only its last row may see it
    blk, off = int(c.tables[2, 129 // c.bs]), 129 % c.bs
    if kv in TOP:
        c.ks[blk, :, off] = float("nan")
        c.vs[blk, :, off] = float("nan")
    else:
        c.kc[blk, off] = float("-inf")
        c.vc[blk, off] = float("nan")
    out = c.run()
    torch.cuda.synchronize()
    row = c.qsl_list[3] - 1
    assert bool(torch.isnan(out[row]).all())
    keep = [i for i in range(c.T) if i != row]
    assert bool(torch.isfinite(out[keep]).all())


def test_scores_of_one_sign_and_large_values():
    """Scores far from zero (either side) and a V row that dwarfs the others."""
    for kv, maps in ((I8, 1), (F8, 2), (BF16, 2), (F32, 2)):
        c = Case([257, 1000, 3], hq=8, hkv=2, kv=kv, q_dt=F32, maps=maps, seed=5, norm=False)
        c.q = c.q.abs() * 3
        neg = -1.0 if maps == 1 else 1.0
        c.q *= neg
        if kv == I8:
            c.kc = c.kc.abs()
            c.vs[int(c.tables[0, 3]), :, 2] = 4096.0
        c.check(c.run(), str(kv))


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("kv", [I8, F8])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("n,h,D,bs", [(1, 1, 1, 1), (20, 8, 128, 16), (333, 4, 80, 32), (7, 3, 33, 5), (64, 1, 256, 16), (9, 2, 520, 16)])
def test_append_is_exact(n, h, D, bs, dt, kv):
    import cloverinfer_b200 as cb
    g = torch.Generator().manual_seed(n + D)
    nb = -(-n // bs) + 2
    new = (torch.randn(2, n, h, D, generator=g) * torch.exp(3 * torch.randn(2, n, h, 1, generator=g))).to(dt)
    new[0, 0, 0] = 0.0
    slots = torch.randperm(nb * bs, generator=g)[:n]
    if n > 3:
        slots[1] = -1
    kc = torch.full((nb, bs, h, D), 3, dtype=torch.uint8, device="cuda").view(kv)
    vc = kc.clone()
    ks = torch.full((nb, h, bs), -1.0, device="cuda")
    vs = ks.clone()
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = new.cuda()
    cb.kv_append_scaled(kc, vc, ks, vs, d[0], d[1], slots.cuda(), st)
    for c, s, x in ((kc, ks, new[0]), (vc, vs, new[1])):
        code, sc = quantise(x, kv)
        want_c = torch.full((nb * bs, h, D), 3, dtype=torch.uint8)
        want_s = torch.full((nb * bs, h), -1.0)
        keep = slots >= 0
        want_c[slots[keep]] = code.view(torch.uint8)[keep]
        want_s[slots[keep]] = sc[keep]
        assert torch.equal(c.view(torch.uint8).reshape(nb * bs, h, D).cpu(), want_c)
        got_s = s.transpose(1, 2).reshape(nb * bs, h).cpu()
        assert torch.equal(got_s.isnan(), want_s.isnan())  # a row with an infinity
        assert torch.equal(got_s.nan_to_num(0.0), want_s.nan_to_num(0.0))
    assert int(st.item()) == 0


def test_append_edges():
    """Slots past the cache, rows too small for a scale, infinities and NaN."""
    import cloverinfer_b200 as cb
    from cloverinfer_b200 import _lib
    nb, bs, h, D = 2, 16, 2, 64
    for kv in (I8, F8):
        kc = torch.zeros(nb, bs, h, D, dtype=torch.uint8, device="cuda").view(kv)
        vc = kc.clone()
        ks = torch.zeros(nb, h, bs, device="cuda")
        vs = ks.clone()
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        x = torch.ones(5, h, D, device="cuda")
        x[0, 0, 3] = float("inf")
        x[0, 1, 3] = float("nan")
        x[1] = 2.0 ** -101
        x[2] = -1e38
        cb.kv_append_scaled(kc, vc, ks, vs, x, x, torch.tensor([0, 1, 2, 3, nb * bs], device="cuda"), st)
        assert int(st.item()) == _lib.DEV_BAD_SLOT
        assert bool(torch.isnan(ks[0, :, 0]).all()) and bool((kc.view(torch.uint8)[0, 0] == 0).all())
        assert bool((ks[0, :, 1] == 0).all()) and bool((vc.view(torch.uint8)[0, 1] == 0).all())
        assert bool((kc[0, 2].float() == -TOP[kv]).all())
        assert bool((kc[0, 3].float() == TOP[kv]).all())


def test_append_layers():
    import cloverinfer_b200 as cb
    L, n, h, D, nb, bs = 3, 10, 2, 64, 4, 16
    x = torch.randn(L, 2, n, h, D, device="cuda").bfloat16()
    kc = torch.zeros(L, nb, bs, h, D, dtype=I8, device="cuda")
    vc = torch.zeros_like(kc)
    ks = torch.zeros(L, nb, h, bs, device="cuda")
    vs = torch.zeros_like(ks)
    slots = torch.randperm(nb * bs)[:n].cuda()
    cb.kv_append_scaled(kc, vc, ks, vs, x[:, 0], x[:, 1], slots, None)
    for layer in range(L):
        one = [t[layer].clone().zero_() for t in (kc, vc, ks, vs)]
        cb.kv_append_scaled(*one, x[layer, 0], x[layer, 1], slots, None)
        for got, ref in zip((kc, vc, ks, vs), one):
            assert torch.equal(got[layer], ref)


# ---------------------------------------------------------------- offsets, streams, graphs
def test_cache_past_2_31_elements():
    for kv, maps in ((I8, 1), (F16, 2)):
        nb, bs, h, D = 140000, 16, 8, 128
        kc = torch.zeros(nb, bs, h, D, dtype=kv, device="cuda")
        vc = torch.zeros_like(kc)
        c = Case([400], hq=8, hkv=8, kv=kv, q_dt=F16, maps=maps, seed=2)
        hi = torch.arange(nb - 30, nb, device="cuda")[:c.nb]
        kc[hi], vc[hi] = c.kc, c.vc
        if c.ks is not None:
            ks = torch.zeros(nb, h, bs, device="cuda")
            vs = torch.zeros_like(ks)
            ks[hi], vs[hi] = c.ks, c.vs
            c.ks, c.vs = ks, vs
        c.tables = torch.where(c.tables >= 0, c.tables + (nb - 30), c.tables)
        c.kc, c.vc = kc, vc
        want = c.append_reference()
        out = c.run(step=True)
        assert torch.equal(c.kc.view(torch.uint8), want[0].view(torch.uint8))
        c.check(out, "high blocks")


@pytest.mark.parametrize("maps,kv", [(1, I8), (2, BF16)])
def test_streams_and_graphs(maps, kv):
    """A side stream, and two captured graphs replayed at once on two streams."""
    cs = [Case([3000, 17, 900], hq=8, hkv=2, kv=kv, q_dt=BF16, maps=maps, seed=s) for s in (1, 2)]
    want = [c.run() for c in cs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = cs[0].run()
    side.synchronize()
    assert torch.equal(got, want[0])
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for c in cs:
        o = torch.zeros_like(c.q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run(out=o)
        graphs.append(g)
        outs.append(o)
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_sequences_may_share_blocks():
    """Two sequences on one table row (a shared prefix), and a row order of its own."""
    c = Case([900, 900], hq=8, hkv=2, kv=I8, q_dt=F32, tables_rows=1, seed=4)
    c.seq_rows[1] = c.seq_rows[0]
    c.rows_d = c.seq_rows.int().cuda()
    c.check(c.run(), "shared row")


def test_bad_pages_are_flagged():
    from cloverinfer_b200 import _lib
    for kv, maps, D in ((I8, 1, 128), (I8, 1, 40), (F16, 2, 128), (F32, 2, 64)):
        for lens in ([600, 600], [60, 60]):
            c = Case(lens, hq=4, hkv=2, D=D, kv=kv, q_dt=F32, maps=maps)
            c.tables[0, 2] = c.nb + 5
            c.tables[0, 1] = -1
            good = c.run()
            torch.cuda.synchronize()
            assert int(c.status.item()) == _lib.DEV_BAD_BLOCK
            assert bool(torch.isfinite(good[1]).all())
            c.status.zero_()
            c.max_ctx = lens[0] // 2
            c.run()
            assert int(c.status.item()) & _lib.DEV_CTX_RANGE
