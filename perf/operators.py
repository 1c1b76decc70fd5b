"""The step plan, the 8-bit KV append, the decode over an 8-bit cache with scales and
differential decode attention: real calls over their real range, each with its plain form.

``own`` is set by whoever measures: False computes the plain form (elementary torch
operations in 32 bits), True calls the framework.
"""

import math

import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": F8}
TOP = {torch.int8: 127.0, F8: 448.0}  # the largest code of an 8-bit cache
EPS = 1e-5


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of a small batch: the plan of 8 requests, a token each.
        plan("plan-decode-8", 8, 64, 2048, 1, 1, 16),
        # Mixed continuous batching: 256 requests, 1-4 new tokens, block 32.
        plan("plan-mixed-256", 256, 16, 16384, 1, 4, 32),
        # Admission of 48 ragged prompts at once: thousands of slots and new blocks each.
        plan("plan-prompts-48", 48, 0, 512, 1021, 8192, 16),
        # The new tokens of a 32-request decode step, Qwen2.5-7B heads.
        append("append-step-32", 32, 4, 128, 16, "bf16", "i8"),
        # A long prompt's K/V of one layer, Llama-3-8B heads, an odd length.
        append("append-prompt-16381", 16381, 8, 128, 16, "f16", "e4m3"),
        # One short request, OPT-125m heads, fp32 queries: latency.
        decode("scaled-one-37", 1, 37, 37, 1, 1, 12, 12, 64, 16, "f32", "i8", step=True),
        # Qwen2.5-7B heads, 32 ragged requests: append and attend.
        decode("scaled-ragged-32", 32, 1024, 4096, 1, 1, 28, 4, 128, 16, "bf16", "i8", step=True),
        # Llama-3-8B heads, 8 requests of 32k tokens: the bandwidth of a long cache.
        decode("scaled-long-8", 8, 32768, 32768, 1, 1, 32, 8, 128, 16, "bf16", "e4m3"),
        # Mixed continuous batching, 1-4 causal rows a request, block 32.
        decode("scaled-mixed-64", 64, 16, 16384, 1, 4, 32, 8, 128, 32, "f16", "i8"),
        # OPT-125m heads, fp32 cache, differential maps of 32 dims: append and attend.
        diff("diff-small-4", 4, 128, 512, 1, 1, 12, 12, 64, 16, "f32", "f32", step=True),
        # Qwen2.5-7B heads, 32 ragged requests.
        diff("diff-ragged-32", 32, 1024, 4096, 1, 1, 28, 4, 128, 16, "bf16", "bf16"),
        # Llama-3-8B heads, 8 requests of 32k tokens.
        diff("diff-long-8", 8, 32768, 32768, 1, 1, 32, 8, 128, 16, "f16", "f16"),
    ]


def plan(name, batch, lo, hi, new_lo, new_hi, block):
    return {"name": name, "op": "plan", "batch": batch, "len_lo": lo, "len_hi": hi, "new_lo": new_lo,
            "new_hi": new_hi, "block": block}


def append(name, tokens, heads, dim, block, new, kv):
    return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "dim": dim, "block": block,
            "new": new, "kv": kv}


def decode(name, batch, lo, hi, new_lo, new_hi, hq, hkv, dim, block, q, kv, step=False):
    return {"name": name, "op": "scaled", "batch": batch, "len_lo": lo, "len_hi": hi, "new_lo": new_lo,
            "new_hi": new_hi, "hq": hq, "hkv": hkv, "dim": dim, "block": block, "q": q, "kv": kv, "step": step}


def diff(*a, **k):
    return dict(decode(*a, **k), op="diff")


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["plan", "append", "scaled", "scaled", "diff", "diff"])
    block = rng.choice([16, 16, 32])
    if op == "plan":
        if rng.random() < 0.3:
            c = plan("", log(1, 48), 0, log(1, 512), 1, log(64, 8192), block)
        else:
            c = plan("", log(1, 1024), 1, log(64, 16384), rng.choice([0, 1]), rng.choice([1, 2, 4]), block)
    elif op == "append":
        c = append("", log(1, 16384), rng.choice([1, 2, 4, 8, 12]), rng.choice([64, 80, 128, 256]), block,
                   rng.choice(["f32", "f16", "bf16"]), rng.choice(["i8", "e4m3"]))
    else:
        hkv, group, dim = rng.choice([(12, 1, 64), (4, 7, 128), (8, 4, 128), (1, 8, 128), (2, 3, 64), (2, 4, 256),
                                      (3, 2, 96)])
        batch = log(1, 128)
        # the padded size of the whole batch stays under the largest listed case's
        hi = min(32768, max(1, int(240e6) // (batch * hkv * dim)))
        hi = log(1, hi)
        lo = rng.choice([1, max(1, hi // 4), hi])
        new = rng.choice([1, 1, 1, 2, 4]) if hi < 8192 else 1
        if op == "scaled":
            q, kv = rng.choice(["f32", "f16", "bf16"]), rng.choice(["i8", "e4m3"])
        else:
            q, kv = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("f32", "f16"), ("f32", "bf16"),
                                ("f32", "f32"), ("bf16", "i8")])
        step = batch * hi * hkv * dim < 4e6 and rng.random() < 0.5
        c = decode("", batch, lo, hi, 1, new, hkv * group, hkv, dim, block, q, kv, step)
        c["op"] = op
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def lengths(case, seed):
    """Per request: tokens held before the call (plan) or attended by its last row
    (decode), log-uniform as in continuous batching, and new tokens.  The case gives the
    lengths, the seed their order."""
    b = case["batch"]
    g = torch.Generator().manual_seed(b * 7919 + case["len_hi"] * 31 + case["new_hi"])
    lo, hi = case["len_lo"], case["len_hi"]
    u = torch.rand(b, generator=g, dtype=torch.float64)
    held = torch.exp(math.log(lo + 1) + (math.log(hi + 1) - math.log(lo + 1)) * u) - 1
    held = held.round().long().clamp(lo, hi)
    if case["op"] != "plan" and lo < hi:
        held[int(torch.randint(b, (1,), generator=g))] = hi  # the longest the caller allows
    new = torch.randint(case["new_lo"], case["new_hi"] + 1, (b,), generator=g)
    if case["op"] != "plan":
        new = torch.minimum(new, held.clamp(min=1))
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(b, generator=g)
    return held[order], new[order], g


def quantised(x, kv):
    """8-bit codes and scales of rows x [..., dim]."""
    top = TOP[kv]
    a = x.abs().amax(-1, keepdim=True)
    y = x * torch.where(a > 0, top / a, torch.zeros_like(a))
    code = y.round().clamp(-top, top).to(torch.int8) if kv == torch.int8 else y.to(kv)
    return code, (a / top).squeeze(-1)


def cache(nb, bs, h, d, kv, g):
    """A filled cache [nb, bs, h, d] (N(0, 1)) and, for 8 bits, its scales [nb, h, bs]."""
    out = torch.empty((nb, bs, h, d), dtype=kv, device="cuda")
    scales = torch.empty((nb, h, bs), dtype=torch.float32, device="cuda") if kv in TOP else None
    per = max(1, (1 << 27) // (bs * h * d))
    for i in range(0, nb, per):
        x = torch.randn((min(per, nb - i), bs, h, d), generator=g, device="cuda")
        if scales is None:
            out[i:i + per] = x
        else:
            out[i:i + per], s = quantised(x, kv)
            scales[i:i + per] = s.transpose(1, 2)
    return out, scales


def prepare(case, seed):
    gd = torch.Generator(device="cuda").manual_seed(seed + 1)
    s = {"case": case}
    if case["op"] == "append":
        n, h, d, bs = case["tokens"], case["heads"], case["dim"], case["block"]
        kv, nb = TYPES[case["kv"]], -(-n // bs) + 3
        slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(seed))[:n]
        s["slots"] = slots.cuda()
        s["new"] = torch.randn((2, n, h, d), generator=gd, device="cuda").to(TYPES[case["new"]])
        s["kc"] = torch.zeros((nb, bs, h, d), dtype=torch.uint8, device="cuda").view(kv)
        s["vc"] = torch.zeros((nb, bs, h, d), dtype=torch.uint8, device="cuda").view(kv)
        s["ks"] = torch.zeros((nb, h, bs), device="cuda")
        s["vs"] = torch.zeros((nb, h, bs), device="cuda")
        s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        return s
    held, new, g = lengths(case, seed)
    b, bs = case["batch"], case["block"]
    if case["op"] == "plan":
        # allocator state in one buffer: [free_top | table_len | seq_lens | tables]
        rows = torch.randperm(b + 3, generator=g)[:b]
        have = torch.maximum(-(-held // bs), torch.ones_like(held))
        width = int((-(-(held + new) // bs)).max()) + 2
        nb = int(torch.maximum(have, -(-(held + new) // bs)).sum()) + 17
        perm = torch.randperm(nb, generator=g).int()
        tables = torch.full((b + 3, width), -1, dtype=torch.int32)
        tl = torch.zeros(b + 3, dtype=torch.int32)
        sl = torch.zeros(b + 3, dtype=torch.int32)
        at = nb
        for i in range(b):
            r, k = int(rows[i]), int(have[i])
            tables[r, :k] = perm[at - k:at].flip(0)
            at, tl[r], sl[r] = at - k, k, int(held[i])
        saved = torch.cat([torch.tensor([at], dtype=torch.int32), tl, sl, tables.reshape(-1)]).cuda()
        live = saved.clone()
        n, m = b + 3, int(new.sum())
        s.update(saved=saved, live=live, free=perm.cuda(), top=live[:1], tl=live[1:1 + n],
                 sl=live[1 + n:1 + 2 * n], tables=live[1 + 2 * n:].view(n, width),
                 rows=rows.int().cuda(), n_new=new.int().cuda(), m=m, bs=bs,
                 qsl=torch.empty(b + 1, dtype=torch.int32, device="cuda"),
                 ctx=torch.empty(m, dtype=torch.int32, device="cuda"),
                 slots=torch.empty(m, dtype=torch.int64, device="cuda"),
                 status=torch.zeros(1, dtype=torch.int32, device="cuda"))
        return s
    hkv, hq, d = case["hkv"], case["hq"], case["dim"]
    kv, qt = TYPES[case["kv"]], TYPES[case["q"]]
    blocks = -(-held // bs)
    nb = int(blocks.sum()) + 5
    perm = torch.randperm(nb, generator=g).int()
    tables = torch.full((b, int(blocks.max()) + 1), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(blocks.tolist()):
        tables[i, :k] = perm[at:at + k]
        at += k
    t = int(new.sum())
    qsl = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)])
    seq = torch.repeat_interleave(torch.arange(b), new)
    ctx = held[seq] - new[seq] + 1 + torch.arange(t) - qsl[seq]
    s["kc"], s["ks"] = cache(nb, bs, hkv, d, kv, gd)
    s["vc"], s["vs"] = cache(nb, bs, hkv, d, kv, gd)
    s["q"] = torch.randn((t, hq, d), generator=gd, device="cuda").to(qt)
    s["new"] = torch.randn((2, t, hkv, d), generator=gd, device="cuda").to(qt if kv in TOP else kv)
    s["lam"] = torch.rand(hq, generator=gd, device="cuda") * 0.6 + 0.2
    s["w"] = 1 + 0.1 * torch.randn(d, generator=gd, device="cuda")
    s["max_q"], s["max_ctx"] = int(new.max()), int(held.max())
    s["scale"] = 1 / math.sqrt(d // 2 if case["op"] == "diff" else d)
    s.update(tables=tables.cuda(), qsl=qsl.int().cuda(), ctx=ctx.int().cuda(), seq=seq.cuda(),
             out=torch.empty((t, hq, d), dtype=qt, device="cuda"),
             status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    return s


# ------------------------------------------------------------------ plain forms
def plain_plan(s):
    bs, tl, sl, tables = s["bs"], s["tl"], s["sl"], s["tables"]
    rows, n_new = s["rows"].long(), s["n_new"]
    held, have = sl[rows], tl[rows]
    grow = (torch.div(held + n_new + bs - 1, bs, rounding_mode="floor") - have).clamp(min=0)
    first = grow.cumsum(0) - grow
    qsl = torch.nn.functional.pad(n_new.cumsum(0), (1, 0)).int()
    j = torch.arange(tables.shape[1], device=rows.device)
    fresh = (j >= have[:, None]) & (j < (have + grow)[:, None])
    pick = s["top"].long() - 1 - (first[:, None] + j - have[:, None])
    got = torch.where(fresh, s["free"][pick.clamp(0, s["free"].numel() - 1)], tables[rows])
    tables[rows] = got
    tok = torch.arange(s["m"], device=rows.device)
    item = torch.searchsorted(qsl[1:].long(), tok, right=True)
    pos = held[item] + (tok - qsl[item])
    s["slots"].copy_(got[item, torch.div(pos, bs, rounding_mode="floor").long()].long() * bs + pos % bs)
    s["ctx"].copy_(pos + 1)
    s["qsl"].copy_(qsl)
    tl[rows] = (have + grow).int()
    sl[rows] = (held + n_new).int()
    s["top"].sub_(grow.sum())


def plain_append(kc, vc, ks, vs, new, blk, off):
    for c, sc, x in ((kc, ks, new[0]), (vc, vs, new[1])):
        if sc is None:
            c[blk, off] = x.to(c.dtype)
        else:
            code, scale = quantised(x.float(), c.dtype)
            c.view(torch.uint8)[blk, off] = code.view(torch.uint8)
            sc[blk, :, off] = scale


def plain_rows(s):
    """Attention of every row over its request's padded context: maps [T, M, Hq, L]
    applied to V, and how the heads' dims split over the maps."""
    case, tab = s["case"], s["tables"].clamp(min=0)[:, :-1].long()
    b, bs, hkv, hq, d = case["batch"], case["block"], case["hkv"], case["hq"], case["dim"]
    maps = 2 if case["op"] == "diff" else 1

    def rows_of(c, sc):
        x = c[tab].float()
        if sc is not None:
            x = x * sc[tab].transpose(2, 3)[..., None]
        return x.reshape(b, -1, hkv, d)

    # queries padded to [B, max_q]
    slot = torch.arange(s["q"].shape[0], device="cuda") - s["qsl"][s["seq"]]
    q = torch.zeros((b, s["max_q"], hkv, hq // hkv, maps, d // maps), device="cuda")
    q[s["seq"], slot] = s["q"].float().view(-1, hkv, hq // hkv, maps, d // maps)
    lim = torch.zeros((b, s["max_q"]), dtype=torch.int32, device="cuda")
    lim[s["seq"], slot] = s["ctx"]
    k = rows_of(s["kc"], s["ks"])
    k = k.view(b, -1, hkv, maps, d // maps)
    sc = torch.einsum("bqhgmd,blhmd->bhmqgl", q, k) * s["scale"]
    del k
    seen = torch.arange(sc.shape[-1], device="cuda") < lim[:, None, None, :, None, None]
    sc.masked_fill_(~seen, -math.inf)
    top = sc.amax(-1, keepdim=True).nan_to_num_(neginf=0.0)
    sc = sc.sub_(top).exp_()
    tot = sc.sum(-1)
    o = torch.einsum("bhmqgl,blhd->bqhgmd", sc, rows_of(s["vc"], s["vs"]))
    o = o / tot.permute(0, 3, 1, 4, 2)[..., None]
    return o[s["seq"], slot].reshape(-1, hq, maps, d)


def plain_decode(s):
    if s["case"]["step"]:
        pos = s["ctx"].long() - 1
        blk = s["tables"][s["seq"], torch.div(pos, s["case"]["block"], rounding_mode="floor")].long()
        plain_append(s["kc"], s["vc"], s["ks"], s["vs"], s["new"], blk, pos % s["case"]["block"])
    o = plain_rows(s)
    if s["case"]["op"] == "diff":
        o = o[:, :, 0] - s["lam"][:, None] * o[:, :, 1]
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS) * s["w"] * 0.5
    else:
        o = o[:, :, 0]
    s["out"].copy_(o)


# ------------------------------------------------------------------ a pass
def run(s):
    op = s["case"]["op"]
    if op == "plan":
        s["live"].copy_(s["saved"])  # every pass plans the same step of the same requests
        if own:
            import cloverinfer_b200 as cb
            cb.plan_step(s["free"], s["top"], s["tables"], s["tl"], s["sl"], s["rows"], s["n_new"], s["bs"],
                         s["qsl"], s["ctx"], s["slots"], s["status"])
        else:
            plain_plan(s)
        return {"qsl": s["qsl"], "ctx": s["ctx"], "slots": s["slots"], "live": s["live"]}
    if op == "append":
        if own:
            import cloverinfer_b200 as cb
            cb.kv_append_scaled(s["kc"], s["vc"], s["ks"], s["vs"], s["new"][0], s["new"][1], s["slots"], s["status"])
        else:
            bs = s["case"]["block"]
            plain_append(s["kc"], s["vc"], s["ks"], s["vs"], s["new"],
                         torch.div(s["slots"], bs, rounding_mode="floor"), s["slots"] % bs)
        return {"kc": s["kc"], "vc": s["vc"], "ks": s["ks"], "vs": s["vs"]}
    step = s["case"]["step"]
    if own:
        import cloverinfer_b200 as cb
        kw = dict(max_queries_per_seq=s["max_q"], max_ctx_len=s["max_ctx"], score_scale=s["scale"],
                  status=s["status"])
        if step:
            kw.update(k_new=s["new"][0], v_new=s["new"][1])
        if op == "scaled":
            cb.scaled_decode(s["out"], s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["tables"], s["qsl"],
                             s["ctx"], **kw)
        else:
            cb.diff_decode(s["out"], s["q"], s["kc"], s["vc"], s["lam"], s["tables"], s["qsl"], s["ctx"],
                           norm_weight=s["w"], eps=EPS, out_scale=0.5, k_scales=s["ks"], v_scales=s["vs"], **kw)
    else:
        plain_decode(s)
    r = {"out": s["out"]}
    if step:
        r.update(kc=s["kc"], vc=s["vc"])
        if s["ks"] is not None:
            r.update(ks=s["ks"], vs=s["vs"])
    return r


# ------------------------------------------------------------------ the definitions in 64 bits
def exact_plan(s):
    """Request by request, pop by pop."""
    bs, free = s["bs"], s["free"].tolist()
    n = s["tl"].numel()
    top, tl, sl = int(s["top"]), s["tl"].tolist(), s["sl"].tolist()
    tables, qsl, ctx, slots = s["tables"].tolist(), [0], [], []
    for r, new in zip(s["rows"].tolist(), s["n_new"].tolist()):
        for pos in range(sl[r], sl[r] + new):
            while tl[r] * bs <= pos:
                top -= 1
                tables[r][tl[r]] = free[top]
                tl[r] += 1
            slots.append(tables[r][pos // bs] * bs + pos % bs)
            ctx.append(pos + 1)
        sl[r] += new
        qsl.append(qsl[-1] + new)
    live = torch.tensor([top] + tl + sl + sum(tables, []), dtype=torch.int32)
    assert live.numel() == 1 + 2 * n + s["tables"].numel()
    return {"qsl": torch.tensor(qsl, dtype=torch.int32), "ctx": torch.tensor(ctx, dtype=torch.int32),
            "slots": torch.tensor(slots), "live": live}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return exact_plan(s)
    f = torch.float64

    def code64(x, kv):
        a = x.abs().amax(-1)
        return a / TOP[kv]

    if case["op"] == "append":
        r = {"kc": None, "vc": None}
        bs = case["block"]
        for name, x in (("ks", s["new"][0]), ("vs", s["new"][1])):
            sc = torch.zeros_like(s[name], dtype=f)
            sc[s["slots"] // bs, :, s["slots"] % bs] = code64(x.to(f), s["kc"].dtype)
            r[name] = sc
        return r
    hq, hkv, d, bs = case["hq"], case["hkv"], case["dim"], case["block"]
    g = hq // hkv
    out = torch.zeros((s["q"].shape[0], hq, d), dtype=f, device="cuda")
    qsl, ctx, tables = s["qsl"].tolist(), s["ctx"].tolist(), s["tables"].long()
    kept = {"kc": None, "vc": None}
    if case["step"]:
        kept = {n: s[n].clone() for n in ("kc", "vc")}
        if s["ks"] is not None:
            kept.update(ks=s["ks"].to(f), vs=s["vs"].to(f))
        for b in range(case["batch"]):
            for r in range(qsl[b], qsl[b + 1]):
                blk, off = int(tables[b, (ctx[r] - 1) // bs]), (ctx[r] - 1) % bs
                for n, x in (("k", s["new"][0][r]), ("v", s["new"][1][r])):
                    if s["ks"] is None:
                        kept[n + "c"][blk, off] = x
                    else:
                        kept[n + "c"][blk, off] = quantised(x.float(), s["kc"].dtype)[0]
                        kept[n + "s"][blk, :, off] = code64(x.to(f), s["kc"].dtype)
    for b in range(case["batch"]):
        if qsl[b + 1] == qsl[b]:
            continue
        n = max(ctx[qsl[b]:qsl[b + 1]])
        ids = tables[b, :-(-n // bs)]
        side = []
        for name in ("k", "v"):
            c, sc = (kept[name + "c"], kept.get(name + "s")) if case["step"] else (s[name + "c"], s[name + "s"])
            x = c[ids].to(f)
            if sc is not None:
                x = x * sc[ids].to(f).permute(0, 2, 1).unsqueeze(-1)
            side.append(x.reshape(-1, hkv, d))
        k, v = side
        for r in range(qsl[b], qsl[b + 1]):
            m = ctx[r]
            for h in range(hkv):
                q = s["q"][r, h * g:(h + 1) * g].to(f)
                if case["op"] == "scaled":
                    o = torch.softmax(q @ k[:m, h].T * s["scale"], -1) @ v[:m, h]
                else:
                    w = d // 2
                    p1 = torch.softmax(q[:, :w] @ k[:m, h, :w].T * s["scale"], -1)
                    p2 = torch.softmax(q[:, w:] @ k[:m, h, w:].T * s["scale"], -1)
                    o = (p1 - s["lam"][h * g:(h + 1) * g, None].to(f) * p2) @ v[:m, h]
                    o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * s["w"].to(f) * 0.5
                out[r, h * g:(h + 1) * g] = o
    r = {"out": out}
    if case["step"]:
        r.update(kc=None, vc=None)
        if s["ks"] is not None:
            r.update(ks=kept["ks"], vs=kept["vs"])
    return r


# ------------------------------------------------------------------ bytes and operations
def work(case):
    if case["op"] == "append":
        n, h, d = case["tokens"], case["heads"], case["dim"]
        e = torch.empty((), dtype=TYPES[case["new"]]).element_size()
        return {"bytes": 2 * n * h * (d * (e + 1) + 4) + 8 * n, "flops": 4 * n * h * d}
    held, new, _ = lengths(case, 0)
    t, b, bs = int(new.sum()), case["batch"], case["block"]
    if case["op"] == "plan":
        grow = int(((-(-(held + new) // bs)) - (-(-held // bs)).clamp(min=1)).clamp(min=0).sum())
        return {"bytes": 12 * t + 4 * (6 * b + 3) + 8 * grow, "flops": t}
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    kv, e = TYPES[case["kv"]], torch.empty((), dtype=TYPES[case["q"]]).element_size()
    row = 2 * d * torch.empty((), dtype=kv).element_size() + (8 if kv in TOP else 0)
    rows = int((held * new).sum())
    pv = 2 if case["op"] == "diff" else 1
    return {"bytes": int(held.sum()) * hkv * row + 2 * t * hq * d * e + t * hkv * row * (2 if case["step"] else 0),
            "flops": rows * hq * d * 2 * (1 + pv)}
