"""Refusals of the step plan, the quantising append and the decodes over them:
answered with error codes or exceptions before any GPU work."""

from __future__ import annotations

import pytest
import torch

from cloverinfer_b200 import _lib


def _plan(n=1, rows=4, width=8, bs=16, cap=4, blocks=8, ptr=4096):
    return _lib.lib().clover_b200_plan_step(ptr, ptr, blocks, ptr, width, ptr, ptr, rows, ptr, ptr, n, bs, ptr,
                                            ptr, ptr, cap, None, None)


def test_plan_step_refusals():
    for kw in (dict(n=-1), dict(bs=0), dict(width=0), dict(rows=0), dict(cap=-1), dict(blocks=-1),
               dict(width=1 << 28, bs=16), dict(ptr=None)):
        assert _plan(**kw) == _lib.ERR_INVALID_ARG, kw
    for kw in (dict(n=8193), dict(rows=(1 << 18) + 1)):
        assert _plan(**kw) == _lib.ERR_UNSUPPORTED, kw


def _append(kv=_lib.INT8, new=_lib.BF16, n=4, layers=1, h=2, d=64, bs=16, nb=4, tok=None, cl=0, sl=0, ptr=4096):
    return _lib.lib().clover_b200_kv_append_scaled(
        ptr, ptr, ptr, ptr, kv, cl, sl, ptr, ptr, new, 0, h * d if tok is None else tok, ptr, n, layers, h, d, bs,
        nb, None, None)


def test_append_scaled_refusals():
    for kw in (dict(n=-1), dict(h=0), dict(d=0), dict(bs=0), dict(tok=1), dict(ptr=None),
               dict(layers=2, cl=1, sl=1 << 20), dict(layers=2, cl=1 << 20, sl=1), dict(layers=65536)):
        assert _append(**kw) == _lib.ERR_INVALID_ARG, kw
    for kw in (dict(kv=_lib.BF16), dict(new=_lib.INT8), dict(new=9)):
        assert _append(**kw) == _lib.ERR_UNSUPPORTED, kw
    assert _append(n=0, ptr=None) == 0 and _append(layers=0, ptr=None) == 0


def _decode(maps, kv, q=_lib.F32, scales=4096, hq=8, hkv=2, d=128, bs=16, nb=8, new=None, new_dt=_lib.BF16,
            stride=None, ws=None, wsb=0, max_ctx=4096, tables=1, lam=4096, ptr=4096, n=1):
    stride = hq * d if stride is None else stride
    head = (ptr, stride, ptr, stride, q, ptr, ptr, scales, scales, kv, nb, bs, new, new, hkv * d, new_dt, ptr,
            tables, None, ptr, ptr, n, n, 1, max_ctx, hq, hkv, d, 1.0)
    tail = (ws, wsb, None, None)
    if maps == 1:
        return _lib.lib().clover_b200_scaled_decode(*head, *tail)
    return _lib.lib().clover_b200_diff_decode(*head, lam, None, 1e-5, 1.0, *tail)


@pytest.mark.parametrize("maps", [1, 2])
def test_decode_refusals(maps):
    i8 = _lib.INT8
    for kw in (dict(hq=7), dict(d=0), dict(bs=0), dict(nb=0), dict(stride=8), dict(scales=None), dict(ptr=None),
               dict(tables=0)):
        assert _decode(maps, i8, **kw) == _lib.ERR_INVALID_ARG, kw
    for kw in (dict(d=258), dict(q=i8), dict(nb=1 << 28), dict(new=4096, new_dt=i8)):
        assert _decode(maps, i8, **kw) == _lib.ERR_UNSUPPORTED, kw
    assert _decode(maps, i8) == _lib.ERR_WORKSPACE
    assert _decode(maps, i8, ws=4100, wsb=1 << 40) == _lib.ERR_WORKSPACE  # not 16-byte aligned
    assert _decode(maps, 9) == _lib.ERR_UNSUPPORTED
    assert _decode(maps, i8, n=0, ptr=None, scales=None) == 0


def test_decode_kinds():
    assert _decode(1, _lib.BF16) == _lib.ERR_UNSUPPORTED          # scaled_decode: 8-bit caches
    assert _decode(2, _lib.BF16) == _lib.ERR_INVALID_ARG          # scales without an 8-bit cache
    assert _decode(2, _lib.BF16, q=_lib.F16, scales=None) == _lib.ERR_UNSUPPORTED
    assert _decode(2, _lib.INT8, d=33, hq=2) == _lib.ERR_INVALID_ARG   # no halves
    assert _decode(2, _lib.INT8, lam=None) == _lib.ERR_INVALID_ARG
    assert _decode(2, _lib.BF16, scales=None, new=4096, new_dt=_lib.F32) == _lib.ERR_UNSUPPORTED


def test_workspace_query():
    f = _lib.lib().clover_b200_attend_workspace_bytes
    short = f(8, 8, 1, 100, 32, 8, 128, 16, _lib.INT8, _lib.F32, 0)
    assert short == 0
    one = f(8, 8, 1, 32768, 32, 8, 128, 16, _lib.INT8, _lib.F32, 0)
    many = f(512, 512, 1, 32768, 32, 8, 128, 16, _lib.INT8, _lib.F32, 0)
    assert 0 < one <= many < one + (1 << 20)  # the partials do not grow with the batch
    assert f(8, 8, 1, 32768, 30, 8, 128, 16, _lib.INT8, _lib.F32, 0) == -1
    assert f(1 << 20, 1, 1, 1 << 20, 32, 8, 128, 16, _lib.INT8, _lib.F32, 0) == -1


def test_wrappers_refuse_host_tensors_and_shapes():
    import cloverinfer_b200 as cb
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        cb.plan_step(i32, i32, i32.view(1, 1), i32, i32, i32, i32, 16, i32, i32, i32.long(), i32)
    c8, sc = torch.zeros(2, 16, 2, 64, dtype=torch.int8), torch.zeros(2, 2, 16)
    x = torch.zeros(1, 2, 64)
    with pytest.raises(ValueError):
        cb.kv_append_scaled(c8, c8, sc, sc, x, x, torch.zeros(1, dtype=torch.int64), None)
    with pytest.raises(ValueError):
        cb.scaled_decode(x, x, c8, c8, sc, sc, i32.view(1, 1), i32, i32, max_queries_per_seq=1, max_ctx_len=1,
                         score_scale=1.0)
    with pytest.raises(ValueError):
        cb.diff_decode(x, x, c8, c8, None, i32.view(1, 1), i32, i32, max_queries_per_seq=1, max_ctx_len=1,
                       score_scale=1.0)
