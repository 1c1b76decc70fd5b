"""Device-resident paged KV cache: block pool, LIFO allocator and block tables.

``PagedKVPool`` owns, in HBM:

* per-layer caches ``k[layer]``/``v[layer]`` of shape
  ``[num_blocks, block_size, num_kv_heads, head_dim]`` — the layout of
  ``KVCacheManager`` (src/core/memory_manager.py:35-46), zero-initialised;
* the free-block stack ``free_stack[num_blocks]`` + ``free_top`` (LIFO, the
  upstream ``list(range(num_blocks))`` with ``pop()``/``append``, :49);
* block tables ``tables[max_seqs, max_blocks_per_seq]`` (-1 padded, :167) and
  ``table_len[max_seqs]``, shared by every layer (all layers of a sequence
  hold the same number of tokens).

The host keeps only counters (free blocks, blocks per row) so it can raise the
upstream errors (``RuntimeError`` on exhaustion, :64-65, :108-109) before any
kernel runs; block ids never leave the GPU on the hot path.

An 8-bit pool (``dtype=torch.int8``, or ``torch.float8_e4m3fn`` with
``scaled=True``) also holds one fp32 scale per (token, KV head) for K and for V,
``k_scale``/``v_scale`` ``[layers, num_blocks, num_kv_heads, block_size]``; new
tokens come in f32, f16 or bf16 and are quantised by the append.

``plan_step`` plans a step from lengths on the GPU (``seq_lens``), with no host
bookkeeping: a captured plan + append + decode can be replayed step after step.

``KVCacheManager`` is the drop-in for the upstream class of the same name:
same constructor, methods, return values and errors, backed by the pool.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib


def to_device_i32(values: Sequence[int], device: torch.device) -> torch.Tensor:
    """One pinned, stream-ordered H2D copy of a small int32 array."""
    h = torch.tensor(list(values), dtype=torch.int32)
    if device.type != "cuda":
        return h
    return h.pin_memory().to(device, non_blocking=True)


def auto_partition(contexts: Sequence[int], max_q: int, sharded: bool = False) -> int:
    """The split for a batch whose caller left it to the library (0): the
    balanced split (``_lib.PARTITION_BALANCED``) for ragged batches of
    single-token rows — the longest context at least 1.25x the mean, where
    fixed partitions sized for the longest leave most CTAs short or empty —
    else 0 (fixed partitions chosen by the library from the longest context).
    Sharded steps keep 0."""
    n = len(contexts)
    if sharded or max_q != 1 or n == 0 or n > 1024:
        return 0
    longest = max(contexts)
    return _lib.PARTITION_BALANCED if longest * n >= 1.25 * sum(contexts) and longest > 0 else 0


_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


@dataclass(frozen=True)
class DiffAttention:
    """One layer's differential attention: per query head ``lam`` (float32 [Hq]), and
    the norm of its output (``norm_weight`` float32 [head_dim] or None, ``eps``,
    ``out_scale``): out = norm(softmax_1 V - lam * softmax_2 V)."""
    lam: torch.Tensor
    norm_weight: Optional[torch.Tensor] = None
    eps: float = 1e-5
    out_scale: float = 1.0

    @classmethod
    def from_vectors(cls, q1: torch.Tensor, k1: torch.Tensor, q2: torch.Tensor, k2: torch.Tensor,
                     lambda_init: float, num_heads: int, norm_weight: Optional[torch.Tensor] = None,
                     eps: float = 1e-5) -> "DiffAttention":
        """From the learned vectors ([d], or [num_heads, d]): lam = exp(q1 . k1) -
        exp(q2 . k2) + lambda_init, computed once in 64 bits; the norm's output is
        scaled by 1 - lambda_init.  ``norm_weight`` is needed (ones for a norm without
        weights): only a norm's output takes that factor."""
        if norm_weight is None:
            raise ValueError("from_vectors: norm_weight is needed (ones for a norm without weights); for the bare "
                             "difference of the maps construct DiffAttention(lam)")
        lam = (q1.double() * k1.double()).sum(-1).exp() - (q2.double() * k2.double()).sum(-1).exp() + lambda_init
        return cls(lam.float().expand(num_heads).contiguous(), norm_weight, eps, 1.0 - float(lambda_init))

    def heads(self, lo: int, hi: int, device) -> "DiffAttention":
        """The query heads [lo, hi) as the decode takes them: on ``device``, float32 and
        contiguous (this object if it is all of that already)."""
        ready = lambda x: x.to(device=torch.device(device), dtype=torch.float32).contiguous()  # noqa: E731
        lam = ready(self.lam if (lo, hi) == (0, self.lam.numel()) else self.lam[lo:hi])
        w = None if self.norm_weight is None else ready(self.norm_weight)
        if lam is self.lam and w is self.norm_weight:
            return self
        return DiffAttention(lam, w, self.eps, self.out_scale)


@dataclass
class StepPlan:
    """What :meth:`PagedKVPool.plan_step` made of one step, on the GPU."""
    rows: torch.Tensor             # [B] table rows
    query_start_loc: torch.Tensor  # [B + 1]
    ctx_lens: torch.Tensor         # [max_tokens]
    slots: torch.Tensor            # [max_tokens], -1 past the last token


class PagedKVPool:
    def __init__(self, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, *,
                 num_layers: int = 1, dtype: torch.dtype = torch.bfloat16,
                 device="cuda", max_seqs: int = 256, max_blocks_per_seq: Optional[int] = None,
                 scaled: Optional[bool] = None) -> None:
        self.scaled = dtype == torch.int8 if scaled is None else bool(scaled)
        if self.scaled != (dtype == torch.int8) and dtype != torch.float8_e4m3fn:
            raise TypeError(f"PagedKVPool: a {dtype} cache {'has no' if self.scaled else 'needs'} scales")
        if num_blocks <= 0 or block_size <= 0 or num_kv_heads <= 0 or head_dim <= 0:
            raise ValueError("PagedKVPool: sizes must be positive")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("PagedKVPool lives in GPU memory; a CUDA device is required")
        _lib.lib()  # fail loudly now if the CUDA library is missing
        self.num_blocks = int(num_blocks)
        self.block_size = int(block_size)
        self.num_kv_heads = int(num_kv_heads)
        self.head_dim = int(head_dim)
        self.num_layers = int(num_layers)
        self.dtype = dtype
        self.max_seqs = int(max_seqs)
        width = max_blocks_per_seq if max_blocks_per_seq is not None else min(num_blocks, 8192)
        self.max_blocks_per_seq = int(width)
        shape = (self.num_layers, self.num_blocks, self.block_size, self.num_kv_heads, self.head_dim)
        dev = self.device
        self.k = torch.zeros(shape, dtype=dtype, device=dev)
        self.v = torch.zeros(shape, dtype=dtype, device=dev)
        self.k_scale = self.v_scale = None
        if self.scaled:
            sshape = (self.num_layers, self.num_blocks, self.num_kv_heads, self.block_size)
            self.k_scale = torch.zeros(sshape, dtype=torch.float32, device=dev)
            self.v_scale = torch.zeros(sshape, dtype=torch.float32, device=dev)
        self.free_stack = torch.arange(self.num_blocks, dtype=torch.int32, device=dev)
        self.free_top = torch.tensor([self.num_blocks], dtype=torch.int32, device=dev)
        self.tables = torch.full((self.max_seqs, self.max_blocks_per_seq), -1, dtype=torch.int32, device=dev)
        self.table_len = torch.zeros(self.max_seqs, dtype=torch.int32, device=dev)
        # tokens held per row, for plan_step (the host paths do not use it), and a
        # place for those of rows outside the pool
        self._seq_lens = torch.zeros(self.max_seqs + 1, dtype=torch.int32, device=dev)
        self.seq_lens = self._seq_lens[:self.max_seqs]
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        # host mirror: counters only
        self.free_count = self.num_blocks
        self.row_blocks = [0] * self.max_seqs
        self._free_rows = list(range(self.max_seqs - 1, -1, -1))
        self._workspace: Optional[torch.Tensor] = None

    def shuffle_free_stack(self, seed: int) -> None:
        """Permute the initial free stack (a workload knob: random,
        non-contiguous block tables).  Only valid while no block is in use."""
        if self.free_count != self.num_blocks:
            raise RuntimeError("shuffle_free_stack: blocks are in use")
        g = torch.Generator().manual_seed(seed)
        perm = torch.randperm(self.num_blocks, generator=g).to(torch.int32)
        self.free_stack.copy_(perm.to(self.device))

    # ------------------------------------------------------------ rows
    def acquire_row(self) -> int:
        if not self._free_rows:
            raise RuntimeError(f"PagedKVPool: more than max_seqs={self.max_seqs} live sequences")
        return self._free_rows.pop()

    def release_row(self, row: int) -> None:
        self.release([row])
        self._free_rows.append(row)

    # ------------------------------------------------------------ allocator
    def blocks_for(self, tokens: int) -> int:
        return 0 if tokens <= 0 else -(-tokens // self.block_size)

    def demand(self, rows: Sequence[int], targets: Sequence[int]) -> int:
        need = 0
        for r, t in zip(rows, targets):
            want = self.blocks_for(t)
            if want > self.max_blocks_per_seq:
                raise RuntimeError(
                    f"sequence needs {want} blocks > max_blocks_per_seq={self.max_blocks_per_seq}")
            need += max(0, want - self.row_blocks[r])
        return need

    def reserve(self, rows: Sequence[int], targets: Sequence[int], oom_message: str = "OOM: Not enough blocks") -> int:
        """Grow each row to hold ``targets[i]`` tokens (item order = pop order)."""
        if len(set(rows)) != len(rows):
            raise ValueError("reserve: duplicate rows in one batch")
        need = self.demand(rows, targets)
        if need > self.free_count:
            raise RuntimeError(oom_message)
        if need == 0:
            return 0
        self.commit_reserve(rows, targets, need, to_device_i32(rows, self.device),
                            to_device_i32(targets, self.device))
        return need

    def commit_reserve(self, rows: Sequence[int], targets: Sequence[int], need: int,
                       rows_d: torch.Tensor, targets_d: torch.Tensor) -> None:
        """The reserve kernel for a batch already checked with ``demand`` (``need``
        blocks, at most ``free_count``), reading rows and targets from device
        int32 tensors the caller staged; then the host counters."""
        _lib.block_reserve(self.free_stack, self.free_top, self.tables, self.table_len, rows_d,
                           targets_d, self.block_size, self.status)
        for r, t in zip(rows, targets):
            self.row_blocks[r] = max(self.row_blocks[r], self.blocks_for(t))
        self.free_count -= need

    def release(self, rows: Sequence[int]) -> None:
        rows = [r for r in rows if self.row_blocks[r] > 0]
        if not rows:
            return
        if len(set(rows)) != len(rows):
            raise ValueError("release: duplicate rows in one batch")
        rd = to_device_i32(rows, self.device)
        _lib.block_free(self.free_stack, self.free_top, self.tables, self.table_len, rd, self.status)
        for r in rows:
            self.free_count += self.row_blocks[r]
            self.row_blocks[r] = 0

    def slots(self, rows_d: torch.Tensor, positions_d: torch.Tensor, offsets_d: torch.Tensor,
              n_tokens: int) -> torch.Tensor:
        out = torch.empty(n_tokens, dtype=torch.int64, device=self.device)
        _lib.compute_slots(self.tables, rows_d, positions_d, offsets_d, self.block_size,
                           self.num_blocks, out, self.status)
        return out

    # ------------------------------------------------------------ plan on the GPU
    def set_seq_lens(self, rows: torch.Tensor, lens: torch.Tensor) -> None:
        """Tell ``plan_step`` how many tokens rows hold (device int32 tensors): once per
        sequence, and again when its row goes to another one.  Rows outside the pool
        (a plan's padding) are skipped."""
        at = torch.where((rows >= 0) & (rows < self.max_seqs), rows, self.max_seqs)
        self._seq_lens.index_copy_(0, at.long(), lens)

    def plan_step(self, rows: torch.Tensor, n_new: torch.Tensor, max_tokens: int) -> StepPlan:
        """Plan one step from ``seq_lens`` on the GPU: grow the tables of ``rows`` (device
        int32; negative: padding) for ``n_new`` (device int32) more tokens each, at most
        ``max_tokens`` in all, and advance ``seq_lens``.  No host sync and no host
        bookkeeping: ``refresh_host`` brings the host counters in line before host paths
        (``reserve``, ``release``, ...) touch the pool again.  A step that does not fit
        changes nothing, plans nothing and raises a bit in ``status``.  With padding or
        zero counts inside the batch, pass the decodes ``max_q`` >= 2 unless they are the
        scaled or differential ones (with max_q = 1 the others take row b for sequence b)."""
        dev = self.device
        qsl = torch.empty(rows.numel() + 1, dtype=torch.int32, device=dev)
        ctx = torch.empty(int(max_tokens), dtype=torch.int32, device=dev)
        slots = torch.empty(int(max_tokens), dtype=torch.int64, device=dev)
        _lib.plan_step(self.free_stack, self.free_top, self.tables, self.table_len, self.seq_lens, rows, n_new,
                       self.block_size, qsl, ctx, slots, self.status)
        return StepPlan(rows, qsl, ctx, slots)

    def refresh_host(self) -> None:
        """Host counters from the device state (synchronises)."""
        self.free_count = int(self.free_top.item())
        self.row_blocks = self.table_len.tolist()

    # ------------------------------------------------------------ data path
    def new_dtype(self, *dtypes: torch.dtype) -> torch.dtype:
        """The dtype new K/V of these dtypes are handed to one append in: the cache's, or
        for a scaled cache their own float type (float32 where they differ)."""
        if not self.scaled:
            return self.dtype
        return dtypes[0] if len(set(dtypes)) == 1 and dtypes[0] in _FLOATS else torch.float32

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, slots: torch.Tensor) -> None:
        if self.scaled:
            _lib.kv_append_scaled(self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], k_new,
                                  v_new, slots, self.status)
        else:
            _lib.kv_append(self.k[layer], self.v[layer], k_new, v_new, slots, self.status)

    def append_layers(self, k_new: torch.Tensor, v_new: torch.Tensor, slots: torch.Tensor) -> None:
        """Every layer's new tokens [L, n, H, D] in one launch."""
        if self.scaled:
            _lib.kv_append_scaled(self.k, self.v, self.k_scale, self.v_scale, k_new, v_new, slots, self.status)
        else:
            _lib.kv_append_layers(self.k, self.v, k_new, v_new, slots, self.status)

    def scales(self, layer: int):
        """(k_scale, v_scale) of a layer, (None, None) without scales."""
        return (self.k_scale[layer], self.v_scale[layer]) if self.scaled else (None, None)

    def attend(self, layer: int, q: torch.Tensor, query_start_loc: torch.Tensor, ctx_lens: torch.Tensor,
               seq_rows: Optional[torch.Tensor], max_q: int, max_ctx: int, score_scale: float, *,
               k_new: Optional[torch.Tensor] = None, v_new: Optional[torch.Tensor] = None,
               diff: Optional[DiffAttention] = None, out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The decodes over a scaled cache, and differential ones (``diff``) over any:
        append k_new/v_new at ctx - 1 if given, then attend."""
        if out is None:
            out = torch.empty_like(q)
        ks, vs = self.scales(layer)
        kw = dict(max_queries_per_seq=max_q, max_ctx_len=max_ctx, score_scale=score_scale, k_new=k_new,
                  v_new=v_new, seq_rows=seq_rows, workspace=workspace,
                  status=self.status if status is None else status)
        if diff is not None:
            _lib.diff_decode(out, q, self.k[layer], self.v[layer], diff.lam, self.tables, query_start_loc,
                             ctx_lens, norm_weight=diff.norm_weight, eps=diff.eps, out_scale=diff.out_scale,
                             k_scales=ks, v_scales=vs, **kw)
        else:
            _lib.scaled_decode(out, q, self.k[layer], self.v[layer], ks, vs, self.tables, query_start_loc,
                               ctx_lens, **kw)
        return out

    def workspace(self, nbytes: int) -> Optional[torch.Tensor]:
        """A reusable device workspace of at least ``nbytes`` (grown, never shrunk)."""
        if nbytes <= 0:
            return None
        if self._workspace is None or self._workspace.numel() < nbytes:
            self._workspace = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=self.device)
        return self._workspace

    def decode(self, layer: int, q: torch.Tensor, query_start_loc: torch.Tensor, ctx_lens: torch.Tensor,
               seq_rows: Optional[torch.Tensor], max_q: int, max_ctx: int, score_scale: float,
               out: Optional[torch.Tensor] = None, partition_tokens: int = 0) -> torch.Tensor:
        if self.scaled:  # (splits by itself: partition_tokens does not apply)
            return self.attend(layer, q, query_start_loc, ctx_lens, seq_rows, max_q, max_ctx, score_scale, out=out)
        if out is None:
            out = torch.empty_like(q)
        n_seqs = query_start_loc.numel() - 1
        nbytes = _lib.decode_workspace_bytes(n_seqs, q.shape[0], max_q, max_ctx, q.shape[1],
                                             self.num_kv_heads, self.head_dim, self.block_size,
                                             self.dtype, q.dtype, partition_tokens)
        _lib.paged_decode(out, q, self.k[layer], self.v[layer], self.tables, query_start_loc,
                          ctx_lens, max_queries_per_seq=max_q, max_ctx_len=max_ctx,
                          score_scale=score_scale, seq_rows=seq_rows,
                          partition_tokens=partition_tokens, workspace=self.workspace(nbytes),
                          status=self.status)
        return out

    def decode_step(self, layer: int, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                    query_start_loc: torch.Tensor, ctx_lens: torch.Tensor,
                    seq_rows: Optional[torch.Tensor], max_q: int, max_ctx: int, score_scale: float,
                    out: Optional[torch.Tensor] = None, partition_tokens: int = 0,
                    check: bool = True) -> torch.Tensor:
        """Append every query row's new token at ctx - 1 and attend (one fused
        launch for a plain decode step).  Capacity must be reserved first."""
        if self.scaled:
            return self.attend(layer, q, query_start_loc, ctx_lens, seq_rows, max_q, max_ctx, score_scale,
                               k_new=k_new, v_new=v_new, out=out)
        if out is None:
            out = torch.empty_like(q)
        n_seqs = query_start_loc.numel() - 1
        nbytes = _lib.decode_workspace_bytes(n_seqs, q.shape[0], max_q, max_ctx, q.shape[1],
                                             self.num_kv_heads, self.head_dim, self.block_size,
                                             self.dtype, q.dtype, partition_tokens)
        _lib.decode_step(out, q, self.k[layer], self.v[layer], k_new, v_new, self.tables,
                         query_start_loc, ctx_lens, max_queries_per_seq=max_q, max_ctx_len=max_ctx,
                         score_scale=score_scale, seq_rows=seq_rows,
                         partition_tokens=partition_tokens, workspace=self.workspace(nbytes),
                         status=self.status, check=check)
        return out

    def decode_step_gather(self, layer: int, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                           query_start_loc: torch.Tensor, ctx_lens: torch.Tensor,
                           seq_rows: Optional[torch.Tensor], max_q: int, max_ctx: int,
                           score_scale: float, gather, partition_tokens: int = 0,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """decode_step for a head-sharded group: the all-gathered output of
        every rank lands in ``out`` ([rows, Hq_total, D] view of a consumer
        buffer, any f32/f16/bf16) or in ``gather.out`` (returned view, valid
        until the next call).  Not for scaled caches."""
        if self.scaled:
            raise TypeError("decode_step_gather: a scaled cache has no fused gather")
        n_seqs = query_start_loc.numel() - 1
        nbytes = _lib.decode_gather_workspace_bytes(n_seqs, q.shape[0], max_q, max_ctx, q.shape[1],
                                                    self.num_kv_heads, self.head_dim,
                                                    self.block_size, self.dtype, q.dtype,
                                                    partition_tokens)
        _lib.decode_step_gather(q, self.k[layer], self.v[layer], k_new, v_new, self.tables,
                                query_start_loc, ctx_lens, gather, max_queries_per_seq=max_q,
                                max_ctx_len=max_ctx, score_scale=score_scale, seq_rows=seq_rows,
                                partition_tokens=partition_tokens, workspace=self.workspace(nbytes),
                                status=self.status, out=out)
        return gather.out[:q.shape[0]] if out is None else out

    # ------------------------------------------------------------ checks / views
    def check_status(self) -> None:
        """Raise if any kernel flagged a bad index since the last check (syncs)."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            self.raise_status(code)

    @staticmethod
    def raise_status(code: int) -> None:
        """Raise the RuntimeError that names the CLOVER_B200_DEV_* bits of ``code``."""
        names = [n for n, bit in [("bad slot", _lib.DEV_BAD_SLOT), ("bad block id", _lib.DEV_BAD_BLOCK),
                                  ("table full", _lib.DEV_TABLE_FULL), ("out of blocks", _lib.DEV_OOM),
                                  ("wait timeout", _lib.DEV_TIMEOUT), ("context > max_ctx_len", _lib.DEV_CTX_RANGE),
                                  ("bad step plan", _lib.DEV_BAD_PLAN)]
                 if code & bit]
        raise RuntimeError(f"libclover_b200 device status 0x{code:x}: {', '.join(names)}")

    def row_table(self, row: int) -> List[int]:
        n = self.row_blocks[row]
        return self.tables[row, :n].tolist() if n else []

    def free_list(self) -> List[int]:
        top = int(self.free_top.item())
        return self.free_stack[:top].tolist()


class KVCacheManager:
    """Drop-in for CloverInfer's ``KVCacheManager`` (src/core/memory_manager.py:18-239)
    with the block pool, free stack and block tables in GPU memory and the
    paged attention on the sm_100a kernel.

    Differences, all deliberate: ``attention`` computes in fp32 and returns
    q's dtype (the upstream CUDA op accumulated the output in fp16,
    attention.cu:101-106); bf16 is supported; there is no CPU path — the
    manager requires a CUDA device.
    """

    def __init__(self, num_blocks: int, block_size: int, num_heads: int, head_dim: int,
                 dtype=torch.float32, device="cuda", max_seqs: int = 256,
                 max_blocks_per_seq: Optional[int] = None) -> None:
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.device = device
        self.pool = PagedKVPool(num_blocks, block_size, num_heads, head_dim, num_layers=1,
                                dtype=dtype, device=device, max_seqs=max_seqs,
                                max_blocks_per_seq=max_blocks_per_seq)
        self.k_cache = self.pool.k[0]
        self.v_cache = self.pool.v[0]
        self.context_lens: Dict[str, int] = {}
        self._rows: Dict[str, int] = {}

    # memory_manager.py:55-72
    def allocate(self, request_id: str, seq_len: int = 0) -> None:
        if request_id in self._rows:
            raise ValueError(f"Request {request_id} already exists")
        row = self.pool.acquire_row()
        try:
            self.pool.reserve([row], [max(seq_len + 1, 1)], "OOM: Not enough blocks")
        except Exception:
            self.pool._free_rows.append(row)
            raise
        self._rows[request_id] = row
        self.context_lens[request_id] = seq_len

    # memory_manager.py:74-93
    def load_initial_kv(self, request_id: str, k_data: torch.Tensor, v_data: torch.Tensor) -> None:
        n = int(k_data.shape[0])
        if request_id not in self._rows:
            self.allocate(request_id, n)
        row = self._rows[request_id]
        if n > 0:
            dev = self.pool.device
            rd = to_device_i32([row], dev)
            pd = to_device_i32([0], dev)
            od = to_device_i32([0, n], dev)
            slots = self.pool.slots(rd, pd, od, n)
            dt = self.pool.new_dtype(k_data.dtype, v_data.dtype)
            k = k_data.to(device=dev, dtype=dt).contiguous()
            v = v_data.to(device=dev, dtype=dt).contiguous()
            self.pool.append(0, k, v, slots)
        self.context_lens[request_id] = n

    # memory_manager.py:95-121
    def _grow_for_append(self, request_id: str) -> int:
        cur = self.context_lens[request_id]
        row = self._rows[request_id]
        self.pool.reserve([row], [cur + 1], "OOM during append")
        self.context_lens[request_id] = cur + 1
        return cur

    def append_slot(self, request_id: str) -> Tuple[int, int]:
        pos = self._grow_for_append(request_id)
        blk = int(self.pool.tables[self._rows[request_id], pos // self.block_size].item())
        return blk, pos % self.block_size

    # memory_manager.py:123-132
    def write_new_kv(self, request_id: str, k: torch.Tensor, v: torch.Tensor) -> None:
        k = k.squeeze(0) if k.dim() == 3 else k
        v = v.squeeze(0) if v.dim() == 3 else v
        pos = self._grow_for_append(request_id)
        dev = self.pool.device
        row = self._rows[request_id]
        slots = self.pool.slots(to_device_i32([row], dev), to_device_i32([pos], dev),
                                to_device_i32([0, 1], dev), 1)
        dt = self.pool.new_dtype(k.dtype, v.dtype)
        self.pool.append(0, k.to(device=dev, dtype=dt).reshape(1, self.num_heads, self.head_dim).contiguous(),
                         v.to(device=dev, dtype=dt).reshape(1, self.num_heads, self.head_dim).contiguous(),
                         slots)

    # memory_manager.py:134-143
    def free(self, request_id: str) -> None:
        if request_id not in self._rows:
            return
        row = self._rows.pop(request_id)
        self.pool.release_row(row)
        del self.context_lens[request_id]

    @property
    def block_tables(self) -> Dict[str, List[int]]:
        return {rid: self.pool.row_table(row) for rid, row in self._rows.items()}

    @property
    def free_blocks(self) -> List[int]:
        return self.pool.free_list()

    # memory_manager.py:145-173
    def get_kernel_inputs(self, request_ids: List[str]):
        rows = [self._rows[r] for r in request_ids]
        width = max((self.pool.row_blocks[r] for r in rows), default=0)
        idx = torch.tensor(rows, dtype=torch.long, device=self.pool.device)
        tables = self.pool.tables.index_select(0, idx)[:, :width].contiguous()
        lens = [self.context_lens[r] for r in request_ids]
        return tables, torch.tensor(lens, dtype=torch.int32, device=self.pool.device), max(lens, default=0)

    # memory_manager.py:175-190 (scale fixed at 1/sqrt(D), memory_manager.py:199)
    def attention(self, q: torch.Tensor, request_ids: List[str]) -> torch.Tensor:
        dev = self.pool.device
        qd = q.to(dev)
        if qd.dtype not in (torch.float32, self.dtype):
            qd = qd.to(torch.float32)
        qd = qd.contiguous()
        n = len(request_ids)
        lens = [self.context_lens[r] for r in request_ids]
        rows = to_device_i32([self._rows[r] for r in request_ids], dev)
        qsl = to_device_i32(list(range(n + 1)), dev)
        ctx = to_device_i32(lens, dev)
        out = self.pool.decode(0, qd, qsl, ctx, rows, 1, max(lens, default=0),
                               1.0 / math.sqrt(self.head_dim))
        return out.to(q.dtype) if out.dtype != q.dtype else out
