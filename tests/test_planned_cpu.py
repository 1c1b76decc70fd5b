"""Host rules of the backend's planned steps and of differential layers, on a
backend object without a GPU: nothing below launches anything."""

from __future__ import annotations

import pytest
import torch

from cloverinfer_b200 import B200AttentionBackend
from cloverinfer_b200.backend import PlannedStep, _Request


def bare(layers=2, hkv=2, D=64):
    """A backend's host state: requests "a" and "b" with 5 and 9 tokens, and a
    launch that only says that it was reached."""
    be = B200AttentionBackend.__new__(B200AttentionBackend)
    be.num_layers, be.num_kv_heads, be.head_dim, be.device = layers, hkv, D, torch.device("cpu")
    be._pending_ingest, be._peer = [], None
    be._reqs = {"a": _Request(0, [5] * layers, 5), "b": _Request(1, [9] * layers, 9)}

    def launch(reqs, layer, n_new, targets, query, *rest, **kw):
        for r, n in zip(reqs, n_new):
            r.layer_len[layer] += n
        return query

    be._launch = launch
    return be


def planned(be):
    ids = list(be._reqs)
    reqs = [be._reqs[r] for r in ids]
    n = [1] * len(ids)
    e = torch.zeros(0, dtype=torch.int32)
    return PlannedStep(request_ids=ids, reqs=reqs, n_new=n, targets=[r.layer_len[0] + 1 for r in reqs], rows=e,
                       query_start_loc=e, ctx_lens=e, slots=e)


def test_a_planned_step_refuses_requests_that_left():
    x, kv = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64)
    for again in (False, True):
        be = bare()
        step = planned(be)
        assert be.decode_planned(step, 0, x, kv, kv).shape == x.shape
        gone = be._reqs.pop("a")  # freed between two layers of the step
        if again:  # and its id taken by another request of the same length
            be._reqs["a"] = _Request(gone.row, list(gone.layer_len), gone.ctx)
        held = {r: list(q.layer_len) for r, q in be._reqs.items()}
        with pytest.raises(KeyError):
            be.decode_planned(step, 1, x, kv, kv)
        assert {r: q.layer_len for r, q in be._reqs.items()} == held


def test_lengths_of_padding_rows_are_skipped():
    """The rows of a plan may hold padding; out of the pool they index nothing."""
    from cloverinfer_b200 import PagedKVPool
    pool = PagedKVPool.__new__(PagedKVPool)
    pool.max_seqs, pool._seq_lens = 4, torch.zeros(5, dtype=torch.int32)
    pool.seq_lens = pool._seq_lens[:4]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    pool.set_seq_lens(i32([2, -1, 0, 9, -7]), i32([5, 6, 7, 8, 9]))
    assert pool.seq_lens.tolist() == [7, 0, 5, 0]
    pool.set_seq_lens(i32([]), i32([]))
    pool.set_seq_lens(i32([3]), i32([1]))
    assert pool.seq_lens.tolist() == [7, 0, 5, 1]


def _attend_args(monkeypatch, tables, max_ctx, rows=1, **kw):
    """What a scaled_decode of host tensors would hand to the library."""
    from cloverinfer_b200 import _lib
    seen = {}
    monkeypatch.setattr(_lib, "_one_device", lambda what, *ts: 0)
    monkeypatch.setattr(_lib, "_call_on", lambda dev, fn, *args: seen.update(args=args) or 0)
    c8, sc = torch.zeros(8, 16, 2, 64, dtype=torch.int8), torch.zeros(8, 2, 16)
    x = torch.zeros(rows, 4, 64)
    _lib.scaled_decode(x, x, c8, c8, sc, sc, tables, torch.arange(rows + 1, dtype=torch.int32),
                       torch.ones(rows, dtype=torch.int32), max_queries_per_seq=1, max_ctx_len=max_ctx,
                       score_scale=1.0, workspace=torch.zeros(1, dtype=torch.uint8), **kw)
    return seen["args"][17], seen["args"][24]  # table stride, longest context


def test_block_tables_of_one_row_and_of_some_columns(monkeypatch):
    t = torch.zeros(3, 8, dtype=torch.int32)
    assert _attend_args(monkeypatch, t, 100, 3) == (8, 100)
    # one row: its stride says nothing (here 1 and 0)
    col = torch.zeros(8, 1, dtype=torch.int32).t()
    assert col.stride() == (1, 1) and _attend_args(monkeypatch, col, 100) == (8, 100)
    assert _attend_args(monkeypatch, t[0].expand(1, 8), 128) == (8, 128)
    # no columns (a batch without tokens)
    assert _attend_args(monkeypatch, t[:1, :0], 0)[0] >= 1
    # some columns: no context reaches past them into the next row's, or past the last row's end
    assert _attend_args(monkeypatch, t[:, 6:], 100, 3) == (8, 32)
    assert _attend_args(monkeypatch, t[1:2, 2:5], 100) == (3, 48)


def test_one_layer_of_any_layer_stride(monkeypatch):
    """The axis of a single layer: its stride says nothing."""
    from cloverinfer_b200 import _lib
    seen = {}
    monkeypatch.setattr(_lib, "_one_device", lambda what, *ts: 0)
    monkeypatch.setattr(_lib, "_call_on", lambda dev, fn, *args: seen.update(args=args) or 0)
    c8, sc = torch.zeros(1, 4, 16, 2, 64, dtype=torch.int8), torch.zeros(1, 4, 2, 16)
    x = torch.zeros(3, 2, 64)
    _lib.kv_append_scaled(c8, c8, sc, sc, x[None], x.as_strided((1, 3, 2, 64), (7, 128, 64, 1)),
                          torch.arange(3), None)
    assert seen["args"][13:15] == (3, 1)  # tokens, layers
    none = c8[:0], c8[:0], sc[:0], sc[:0], x[None][:0], x[None][:0]
    assert _lib.kv_append_scaled(*none, torch.arange(3), None) is None
    two = torch.zeros(2, 3, 2, 64)
    with pytest.raises(ValueError):
        _lib.kv_append_scaled(c8.repeat(2, 1, 1, 1, 1), c8.repeat(2, 1, 1, 1, 1), sc.repeat(2, 1, 1, 1),
                              sc.repeat(2, 1, 1, 1), two, torch.zeros(4, 3, 2, 64)[::2], torch.arange(3), None)
