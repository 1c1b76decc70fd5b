"""The step plan, the quantising append, the decode over an 8-bit cache and
differential decode as the framework's own paths run them: the pool with
device-resident lengths (eager and captured), the backend's interface and its
planned steps, and the manager.  Tolerances: the caches hold what the formulas
give exactly; attention as in conftest.assert_attn_close against fp32 oracles
fed the very values the cache stands for."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import assert_attn_close, gpu
from oracle import attend, repeat_kv
from test_gpu_attend import F8, I8, quantise

pytestmark = gpu


def held(x, kv):
    """What a cache of type kv holds for rows x, as fp32."""
    if kv in (I8, F8):
        code, scale = quantise(x, kv)
        return code.float() * scale[..., None]
    return x.to(kv).float()


def diff_ref(q, k, v, scale, d):
    """Differential attention of one row, fp32: q [Hq, D], k/v [L, Hq, D]."""
    h = q.shape[1] // 2
    one = attend(torch.cat([q[:, :h], 0 * q[:, h:]], 1), k, v, scale)
    two = attend(torch.cat([0 * q[:, :h], q[:, h:]], 1), k, v, scale)
    o = one - d.lam.cpu()[:, None] * two
    if d.norm_weight is not None:
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + d.eps) * d.norm_weight.cpu() * d.out_scale
    return o


def layers_of_diff(n, hq, D, seed):
    from cloverinfer_b200 import DiffAttention
    g = torch.Generator().manual_seed(seed)
    v = lambda: torch.randn(D // 2, generator=g) * 0.1  # noqa: E731
    return [DiffAttention.from_vectors(v(), v(), v(), v(), 0.8 - 0.6 * math.exp(-0.3 * i), hq,
                                       1 + 0.1 * torch.randn(D, generator=g)) for i in range(n)]


@pytest.mark.parametrize("kv,maps", [(I8, 1), (F8, 1), (torch.bfloat16, 2), (I8, 2)])
@pytest.mark.parametrize("captured", [False, True])
def test_pool_steps_from_lengths_on_the_gpu(kv, maps, captured):
    """plan + append + decode of growing sequences, with no host bookkeeping between
    steps; captured, one graph replayed step after step."""
    from cloverinfer_b200 import PagedKVPool
    B, hq, hkv, D, bs, steps = 3, 8, 2, 128, 16, 20
    pool = PagedKVPool(64, bs, hkv, D, num_layers=2, dtype=kv, max_seqs=5, max_blocks_per_seq=16,
                       scaled=kv in (I8, F8))
    pool.shuffle_free_stack(3)
    diffs = [d.heads(0, hq, "cuda") for d in layers_of_diff(2, hq, D, 1)] if maps == 2 else [None, None]
    g = torch.Generator().manual_seed(9)
    rows = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    n_new = torch.tensor([1, 2, 1], dtype=torch.int32, device="cuda")
    T, scale = 4, 1 / math.sqrt(D // maps)
    dt = torch.bfloat16
    x = [torch.zeros(2, T, h, D, dtype=dt, device="cuda") for h in (hq, hkv, hkv)]
    out = torch.zeros(2, T, hq, D, dtype=dt, device="cuda")

    def step():
        p = pool.plan_step(rows, n_new, T)
        for layer in range(2):
            if pool.scaled or maps == 2:
                pool.append(layer, x[1][layer], x[2][layer], p.slots)
                pool.attend(layer, x[0][layer], p.query_start_loc, p.ctx_lens, p.rows, 2, 256, scale,
                            diff=diffs[layer], out=out[layer])

    graph = None
    if captured:
        side = torch.cuda.Stream()  # one-time set-up outside the capture, on a copy of the state
        saved = [t.clone() for t in (pool.free_top, pool.tables, pool.table_len, pool.seq_lens)]
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        for t, s in zip((pool.free_top, pool.tables, pool.table_len, pool.seq_lens), saved):
            t.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    keys = [[[] for _ in range(B)] for _ in range(2)]
    vals = [[[] for _ in range(B)] for _ in range(2)]
    for _ in range(steps):
        host = [torch.randn(t.shape, generator=g).to(dt) for t in x]
        for t, h in zip(x, host):
            t.copy_(h)
        graph.replay() if captured else step()
        torch.cuda.synchronize()
        off = 0
        for b, n in enumerate((1, 2, 1)):
            for j in range(n):
                for layer in range(2):
                    keys[layer][b].append(held(host[1][layer, off + j], kv))
                    vals[layer][b].append(held(host[2][layer, off + j], kv))
                    k, v = torch.stack(keys[layer][b]), torch.stack(vals[layer][b])
                    k, v = repeat_kv(k, hq // hkv), repeat_kv(v, hq // hkv)
                    q = host[0][layer, off + j].float()
                    ref = attend(q, k, v, scale) if maps == 1 else diff_ref(q, k, v, scale, diffs[layer])
                    assert_attn_close(out[layer, off + j], ref, out_dtype=dt, what=f"{kv} b{b} layer {layer}")
            off += n
    pool.check_status()
    pool.refresh_host()
    assert pool.seq_lens.tolist() == [2 * steps, 0, steps, 0, steps]
    assert pool.row_blocks == [-(-n // bs) for n in pool.seq_lens.tolist()]
    pool.release([4, 0, 2])
    assert pool.free_count == pool.num_blocks and int(pool.free_top.item()) == pool.num_blocks


BACKENDS = {
    "int8": dict(kv_dtype=I8),
    "e4m3 scaled": dict(kv_dtype=F8, kv_scales=True),
    "diff bf16": dict(kv_dtype=torch.bfloat16, diff=True),
    "diff fp32": dict(kv_dtype=torch.float32, diff=True),
    "diff int8": dict(kv_dtype=I8, diff=True),
}


def _backend(name, L, hq, hkv, D, **kw):
    from cloverinfer_b200 import B200AttentionBackend
    cfg = dict(BACKENDS[name])
    diffs = layers_of_diff(L, hq, D, 5) if cfg.pop("diff", False) else None
    be = B200AttentionBackend(num_blocks=256, num_kv_heads=hkv, max_seqs=6, shuffle_seed=1, differential=diffs,
                              device="cuda", **cfg, **kw)
    return be, diffs, cfg["kv_dtype"]


class Mirror:
    """The caches' content and the reference of every call."""

    def __init__(self, diffs, kv, rep, scale):
        self.diffs, self.kv, self.rep, self.scale, self.k, self.v = diffs, kv, rep, scale, {}, {}

    def init(self, rid, layers):
        self.k[rid] = [list(held(x["key"], self.kv)) for x in layers]
        self.v[rid] = [list(held(x["value"], self.kv)) for x in layers]

    def step(self, rid, layer, q, k, v):
        self.k[rid][layer].append(held(k, self.kv))
        self.v[rid][layer].append(held(v, self.kv))
        k = repeat_kv(torch.stack(self.k[rid][layer]), self.rep)
        v = repeat_kv(torch.stack(self.v[rid][layer]), self.rep)
        if self.diffs is None:
            return attend(q.float(), k, v, self.scale)
        return diff_ref(q.float(), k, v, self.scale, self.diffs[layer])


@pytest.mark.parametrize("name", list(BACKENDS))
@pytest.mark.parametrize("graphs", [True, False])
def test_backend_interface(name, graphs):
    """init_request, decode_layer_batch on host items (eager, then captured) and device
    items, decode_batch with several tokens and a consumer's buffer."""
    L, hq, hkv, D = 2, 8, 2, 64
    be, diffs, kv = _backend(name, L, hq, hkv, D, cuda_graphs=graphs)
    scale = 1 / math.sqrt(D)
    g = torch.Generator().manual_seed(2)
    mirror = Mirror(diffs, kv, hq // hkv, scale)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    new_dt = torch.float32 if kv == torch.float32 else torch.bfloat16
    for rid, n in (("a", 300), ("b", 15), ("c", 1)):
        layers = [{"key": rnd(n, hkv, D).to(new_dt), "value": rnd(n, hkv, D).to(new_dt)} for _ in range(L)]
        assert be.init_request(rid, layers) == n
        mirror.init(rid, layers)
    for step in range(4):
        for layer in range(L):
            items = [{"request_id": r, "layer_idx": layer, "score_scale": scale, "query": rnd(hq, D),
                      "key": rnd(hkv, D).to(new_dt), "value": rnd(hkv, D).to(new_dt)} for r in "abc"]
            dev = step == 3
            sent = [{k: v.cuda() if dev and torch.is_tensor(v) else v for k, v in it.items()} for it in items]
            for it, o in zip(items, be.decode_layer_batch(sent)):
                ref = mirror.step(it["request_id"], layer, it["query"], it["key"], it["value"])
                assert_attn_close(o[0], ref, kv_dtype=torch.bfloat16, what=f"{name} step {step} layer {layer}")
    n_new = [2, 1, 3]
    for layer in range(L):
        q, k, v = rnd(6, hq, D), rnd(6, hkv, D).to(new_dt), rnd(6, hkv, D).to(new_dt)
        buf = torch.zeros(6, hq * D, dtype=torch.bfloat16, device="cuda")
        res = be.decode_batch(list("abc"), layer, q.cuda(), k.cuda(), v.cuda(), scale, n_new=n_new, out=buf)
        assert res.data_ptr() == buf.data_ptr()
        off = 0
        for r, n in zip("abc", n_new):
            for j in range(n):
                ref = mirror.step(r, layer, q[off + j], k[off + j], v[off + j])
                assert_attn_close(res[off + j], ref, out_dtype=torch.bfloat16, what=f"{name} batch")
            off += n
    assert be.get_context_len("a") == 306
    info = be.get_debug_info()
    assert info["kv_scaled"] == (kv in (I8, F8)) and info["differential"] == (diffs is not None)
    for r in "abc":
        be.free_request(r)
    assert be.pool.free_count == be.pool.num_blocks


@pytest.mark.parametrize("name", ["int8", "diff bf16", "plain"])
def test_backend_planned_steps(name):
    """begin_step once, every layer of it: the same outputs and state as decode_batch."""
    from cloverinfer_b200 import B200AttentionBackend
    L, hq, hkv, D = 3, 8, 2, 128
    make = (lambda: B200AttentionBackend(num_blocks=256, num_kv_heads=hkv, max_seqs=6, shuffle_seed=1,
                                         device="cuda")) if name == "plain" else (lambda: _backend(name, L, hq, hkv, D)[0])
    one, two = make(), make()
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16()  # noqa: E731
    for rid, n in (("a", 40), ("b", 16), ("c", 700)):
        layers = [{"key": rnd(n, hkv, D), "value": rnd(n, hkv, D)} for _ in range(L)]
        assert one.init_request(rid, layers) == two.init_request(rid, layers) == n
    for n_new in ([1, 1, 1], [3, 1, 2], [0, 40, 1], [1, 1, 1]):
        ids = list("cab")
        step = two.begin_step(ids, n_new)
        T = sum(n_new)
        for layer in range(L):
            q, k, v = rnd(T, hq, D).cuda(), rnd(T, hkv, D).cuda(), rnd(T, hkv, D).cuda()
            want = one.decode_batch([r for r, n in zip(ids, n_new) if n], layer, q, k, v, 0.1,
                                    n_new=[n for n in n_new if n])
            got = two.decode_planned(step, layer, q, k, v, 0.1)
            # A request without new tokens changes how the step is split, so the fp32 results
            # differ by rounding; each side then rounds to bf16 by at most 2^-8 of its value,
            # and two values on either side of a tie end a whole step, 2 * 2^-8, apart.
            err = (got.float() - want.float()).abs()
            assert bool((err <= 2e-3 + 2 * 2.0 ** -8 * want.float().abs()).all()), f"{name} {n_new} layer {layer}"
        with pytest.raises(RuntimeError):
            two.decode_planned(step, 0, q, k, v)  # that layer went on
    assert torch.equal(one.pool.tables, two.pool.tables) and torch.equal(one.pool.free_top, two.pool.free_top)
    assert one.pool.free_count == two.pool.free_count and one.pool.row_blocks == two.pool.row_blocks
    one.pool.check_status()
    two.pool.check_status()
    with pytest.raises(KeyError):
        two.begin_step(["nobody"])
    with pytest.raises(ValueError):
        two.begin_step(["a", "a"])
    with pytest.raises(ValueError):
        two.begin_step(["a"], [-1])
    with pytest.raises(RuntimeError):
        two.begin_step(["a"], [256 * 16])
    assert int(two.pool.free_top.item()) == two.pool.free_count


def test_manager_with_an_8_bit_cache():
    from cloverinfer_b200 import KVCacheManager
    h, D = 4, 64
    m = KVCacheManager(64, 16, h, D, dtype=I8)
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(90, h, D, generator=g), torch.randn(90, h, D, generator=g)
    m.load_initial_kv("r", k[:89], v[:89])
    m.write_new_kv("r", k[89], v[89])
    q = torch.randn(1, h, D, generator=g)
    out = m.attention(q.cuda(), ["r"])
    assert_attn_close(out[0], attend(q[0], held(k, I8), held(v, I8), 1 / math.sqrt(D)), what="manager int8")
    m.free("r")
    assert len(m.free_blocks) == 64


def test_refusals_of_pool_and_backend():
    from cloverinfer_b200 import B200AttentionBackend, DiffAttention, PagedKVPool
    with pytest.raises(TypeError):
        PagedKVPool(4, 16, 2, 64, dtype=torch.bfloat16, scaled=True)
    with pytest.raises(TypeError):
        PagedKVPool(4, 16, 2, 64, dtype=I8, scaled=False)
    kv = lambda D, n=3: [{"key": torch.zeros(n, 2, D), "value": torch.zeros(n, 2, D)}]  # noqa: E731
    with pytest.raises(TypeError):
        B200AttentionBackend(num_blocks=8, kv_scales=True, device="cuda").init_request("a", kv(64))
    lam = DiffAttention(torch.zeros(4))
    with pytest.raises(ValueError):
        B200AttentionBackend(num_blocks=8, differential=[lam, lam], device="cuda").init_request("a", kv(64))
    with pytest.raises(ValueError):
        B200AttentionBackend(num_blocks=8, differential=[lam], device="cuda").init_request("a", kv(33))
    with pytest.raises(TypeError):
        B200AttentionBackend(num_blocks=8, differential=[lam], kv_dtype=F8, device="cuda").init_request("a", kv(64))
    be = B200AttentionBackend(num_blocks=8, differential=[lam], device="cuda")
    be.init_request("a", kv(64))
    with pytest.raises(ValueError):  # lam of 4 heads, 8 query heads
        be.decode_batch(["a"], 0, torch.zeros(1, 8, 64).cuda(), torch.zeros(1, 2, 64).cuda(),
                        torch.zeros(1, 2, 64).cuda())
