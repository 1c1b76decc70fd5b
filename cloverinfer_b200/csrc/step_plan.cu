// Step plan on the GPU: block tables, slot map and query layout of one step,
// built from the requests' lengths in one launch.
//
// For item i (table row rows[i], len_i = seq_lens[row] tokens held, n_i new):
//     grow_i = max(0, ceil((len_i + n_i) / bs) - table_len[row])
//     query_start_loc[i] = sum of n over the items before i
//     token j of item i: pos = len_i + j, ctx = pos + 1,
//         slot = block(pos / bs) * bs + pos % bs
// where block(k) is the table's entry for k < table_len[row] and otherwise the
// popped block free_stack[top - 1 - (growth of the items before i + k - table_len[row])]:
// the pops of clover_b200_block_reserve (KVCacheManager.allocate / append_slot,
// src/core/memory_manager.py:55-72, :95-121) in the same order, so a token's
// slot needs no wait for the table to be written.  A block id outside the cache
// (a damaged table or stack) raises BAD_BLOCK and gives its tokens slot -1; the
// state is committed all the same.
//
// Bound: launch latency and three dependent loads (rows, lengths, block ids)
// for a decode step; for admissions of whole prompts the 12 bytes written per
// token (228k tokens, 48 requests: 35 us from 8 CTAs of 512 threads, a round of
// dependent loads per 16k tokens; 16 from 16 CTAs of 1024 threads).  One thread-block
// cluster: every CTA scans all items by itself (into
// shared memory) and takes its share of the tokens, and the state that the
// scans read (lengths, table lengths, stack top) is committed after the
// cluster barrier, so no global counter or scratch memory is needed.
#include <mutex>

#include <cooperative_groups.h>

#include "common.cuh"

namespace clover {

namespace cg = cooperative_groups;

constexpr int kPlanSmall = 256, kPlanLarge = 1024;  // threads: decode steps, admissions
constexpr int kPlanMaxItems = 8192;
constexpr int kPlanMaxRows = 1 << 18;
constexpr int kPlanGroup = 4;  // consecutive tokens of one thread

struct PlanArgs {
  int32_t* free_stack;
  int32_t* free_top;
  int32_t num_blocks;
  int32_t* tables;
  int32_t stride;
  int32_t* table_len;
  int32_t* seq_lens;
  int32_t num_rows;
  const int32_t* rows;
  const int32_t* n_new;
  int32_t n;
  int32_t bs;
  int32_t* qsl;
  int32_t* ctx;
  int64_t* slots;
  int32_t max_tokens;
  int32_t vec;  // ctx and slots are 16-byte aligned
  int32_t* status;
};

// Last i in [0, n) with off[i] <= k (off ascending, off[0] = 0).
__device__ __forceinline__ int plan_find(const int32_t* off, int n, int32_t k) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (off[mid] <= k) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <int kPlanThreads>
__global__ void __launch_bounds__(kPlanThreads)
plan_step_kernel(const PlanArgs a) {
  constexpr int NW = kPlanThreads / 32;
  __shared__ int64_t s_sum[2][NW];
  __shared__ int32_t s_bad;
  extern __shared__ int32_t s_dyn[];
  int32_t* s_tok = s_dyn;            // [n + 1] first token
  int32_t* s_pop = s_tok + a.n + 1;  // [n + 1] first popped block
  int32_t* s_row = s_pop + a.n + 1;  // [n] table row (-1: padding)
  int32_t* s_len = s_row + a.n;      // [n] tokens held
  int32_t* s_have = s_len + a.n;     // [n] blocks held
  uint32_t* s_seen = reinterpret_cast<uint32_t*>(s_have + a.n);  // rows bitmap
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  for (int i = tid; i < (a.num_rows + 31) / 32; i += kPlanThreads) s_seen[i] = 0;
  if (tid == 0) s_bad = 0;
  __syncthreads();

  // ---- scan the items: tokens in the low word, popped blocks in the high one
  const int32_t top = *a.free_top;
  int64_t run_tok = 0, run_pop = 0;
  for (int base = 0; base < a.n; base += kPlanThreads) {
    const int i = base + tid;
    int32_t row = -1, len = 0, have = 0, bad = 0;
    int64_t tok = 0, pop = 0;
    if (i < a.n) {
      row = a.rows[i];
      const int32_t fresh = a.n_new[i];
      if (row >= a.num_rows || (row >= 0 && (fresh < 0 || fresh > a.max_tokens))) {
        bad = CLOVER_B200_DEV_BAD_PLAN;
        row = -1;
      } else if (row >= 0) {
        if (atomicOr(&s_seen[row >> 5], 1u << (row & 31)) >> (row & 31) & 1u)
          bad = CLOVER_B200_DEV_BAD_PLAN;  // the row stands in the batch twice
        len = a.seq_lens[row];
        have = a.table_len[row];
        tok = fresh;
        const int64_t want = ((int64_t)len + fresh + a.bs - 1) / a.bs;
        if (len < 0 || have < 0 || have > a.stride) bad |= CLOVER_B200_DEV_BAD_PLAN;
        else if (want > a.stride) bad |= CLOVER_B200_DEV_TABLE_FULL;
        else if (fresh > 0 && want > have) pop = want - have;
      }
      s_row[i] = row;
      s_len[i] = len;
      s_have[i] = have;
    }
    if (bad) atomicOr(&s_bad, bad);
    // exclusive sums over the CTA (64 bits: an unacceptable plan may overflow 32)
    int64_t in_t = tok, in_p = pop;
    const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, in_t, off), z = __shfl_up_sync(0xffffffffu, in_p, off);
      if (lane >= off) {
        in_t += y;
        in_p += z;
      }
    }
    if (lane == 31) {
      s_sum[0][warp] = in_t;
      s_sum[1][warp] = in_p;
    }
    __syncthreads();
    int64_t off_t = in_t - tok, off_p = in_p - pop, tot_t = 0, tot_p = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) {
        off_t += s_sum[0][w];
        off_p += s_sum[1][w];
      }
      tot_t += s_sum[0][w];
      tot_p += s_sum[1][w];
    }
    __syncthreads();
    if (i < a.n) {
      s_tok[i] = (int32_t)(run_tok + off_t);
      s_pop[i] = (int32_t)(run_pop + off_p);
    }
    run_tok += tot_t;
    run_pop += tot_p;
  }
  if (tid == 0) {
    s_tok[a.n] = (int32_t)run_tok;
    s_pop[a.n] = (int32_t)run_pop;
    if (run_tok > a.max_tokens || top > a.num_blocks || top < 0) s_bad |= CLOVER_B200_DEV_BAD_PLAN;
    if (!s_bad && run_pop > top) s_bad = CLOVER_B200_DEV_OOM;
  }
  __syncthreads();
  const bool bad = s_bad != 0;
  // Every CTA has read the lengths and the stack top: rank 0 may commit them
  // once all have arrived.
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

  const int32_t total = bad ? 0 : s_tok[a.n];
  const int step = ctas * kPlanThreads;
  for (int i = rank * kPlanThreads + tid; i <= a.n; i += step) a.qsl[i] = bad ? 0 : s_tok[i];
  if (!bad) {
    // table entries of the popped blocks (none of them is read here)
    for (int k = rank * kPlanThreads + tid; k < s_pop[a.n]; k += step) {
      const int it = plan_find(s_pop, a.n, k);
      const int32_t blk = a.free_stack[top - 1 - k];
      a.tables[(int64_t)s_row[it] * a.stride + s_have[it] + (k - s_pop[it])] = blk;
    }
  }
  // tokens: kPlanGroup consecutive ones per thread, one search each
  for (int64_t t0 = (int64_t)(rank * kPlanThreads + tid) * kPlanGroup; t0 < a.max_tokens;
       t0 += (int64_t)step * kPlanGroup) {
    int it = t0 < total ? plan_find(s_tok, a.n, (int32_t)t0) : 0;
    int32_t last_b = -1, blk = -1;
    int32_t ctx[kPlanGroup];
    int64_t slot[kPlanGroup];
#pragma unroll
    for (int j = 0; j < kPlanGroup; ++j) {
      const int64_t t = t0 + j;
      ctx[j] = 0;
      slot[j] = -1;
      if (t < total) {
        while (t >= s_tok[it + 1]) {
          ++it;
          last_b = -1;
        }
        const int32_t pos = s_len[it] + (int32_t)(t - s_tok[it]);
        const int32_t b = pos / a.bs;
        if (b != last_b) {
          last_b = b;
          blk = b < s_have[it] ? a.tables[(int64_t)s_row[it] * a.stride + b]
                               : a.free_stack[top - 1 - (s_pop[it] + b - s_have[it])];
          if (blk < 0 || blk >= a.num_blocks) raise_status(a.status, CLOVER_B200_DEV_BAD_BLOCK);
        }
        ctx[j] = pos + 1;
        if (blk >= 0 && blk < a.num_blocks) slot[j] = (int64_t)blk * a.bs + (pos - b * a.bs);
      }
    }
    if (a.vec && t0 + kPlanGroup <= a.max_tokens) {
      *reinterpret_cast<int4*>(a.ctx + t0) = make_int4(ctx[0], ctx[1], ctx[2], ctx[3]);
      longlong2* out = reinterpret_cast<longlong2*>(a.slots + t0);
      out[0] = make_longlong2(slot[0], slot[1]);
      out[1] = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int j = 0; j < kPlanGroup; ++j) {
        if (t0 + j < a.max_tokens) {
          a.ctx[t0 + j] = ctx[j];
          a.slots[t0 + j] = slot[j];
        }
      }
    }
  }

  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0) {
    if (bad) {
      if (tid == 0) raise_status(a.status, s_bad);
    } else {
      for (int i = tid; i < a.n; i += kPlanThreads) {
        const int32_t row = s_row[i];
        if (row < 0) continue;
        a.seq_lens[row] = s_len[i] + (s_tok[i + 1] - s_tok[i]);
        a.table_len[row] = s_have[i] + (s_pop[i + 1] - s_pop[i]);
      }
      if (tid == 0) *a.free_top = top - s_pop[a.n];
    }
  }
  // A decode launched right behind reads its layout before it waits for this
  // kernel's completion (it may start when the last CTA ends): every write is
  // performed by then.
  __threadfence();
}

// ------------------------------------------------------------------ host side
// Shared memory of a plan: five words per item and two more, a bit per row.
static size_t plan_smem(int64_t items, int64_t rows) {
  return (size_t)(2 * (items + 1) + 3 * items + (rows + 31) / 32) * 4;
}

// Lets the kernel have what the largest plan takes.  These limits are the
// process's, not a call's, so they are set once per device and never lowered
// under another thread's launch.
template <int kPlanThreads>
static int plan_configure() {
  static std::mutex mu;
  static uint64_t done = 0;  // one bit per device ordinal
  int dev = 0;
  int rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 64 && (done >> dev & 1)) return CLOVER_B200_OK;
  rc = check_cuda(cudaFuncSetAttribute(plan_step_kernel<kPlanThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)plan_smem(kPlanMaxItems, kPlanMaxRows)),
                  "plan_step shared memory");
  if (!rc)
    rc = check_cuda(cudaFuncSetAttribute(plan_step_kernel<kPlanThreads>,
                                         cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                    "plan_step cluster size");
  if (!rc && dev < 64) done |= 1ull << dev;
  return rc;
}

}  // namespace clover

using namespace clover;

extern "C" int clover_b200_plan_step(int32_t* free_stack, int32_t* free_top, int32_t num_blocks,
                                     int32_t* block_tables, int32_t table_stride,
                                     int32_t* table_len, int32_t* seq_lens, int32_t num_rows,
                                     const int32_t* rows, const int32_t* n_new, int32_t n_items,
                                     int32_t block_size, int32_t* query_start_loc,
                                     int32_t* ctx_lens, int64_t* slot_mapping, int32_t max_tokens,
                                     int32_t* dev_status, void* stream) {
  if (n_items < 0 || block_size <= 0 || table_stride <= 0 || num_blocks < 0 || num_rows <= 0 ||
      max_tokens < 0 || (int64_t)table_stride * block_size > INT32_MAX)
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "plan_step: bad sizes");
  if (n_items > kPlanMaxItems || num_rows > kPlanMaxRows)
    return set_error(CLOVER_B200_ERR_UNSUPPORTED, "plan_step: more than %d items or %d rows",
                     kPlanMaxItems, kPlanMaxRows);
  if (!query_start_loc || (max_tokens > 0 && (!ctx_lens || !slot_mapping)) ||
      (n_items > 0 && (!free_stack || !free_top || !block_tables || !table_len || !seq_lens ||
                       !rows || !n_new)))
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "plan_step: null pointer");
  if (n_items == 0) {
    // nothing to plan: an empty layout and no slots
    cudaStream_t s = (cudaStream_t)stream;
    int rc = check_cuda(cudaMemsetAsync(query_start_loc, 0, 4, s), "plan_step");
    if (!rc && max_tokens > 0)
      rc = check_cuda(cudaMemsetAsync(ctx_lens, 0, (size_t)max_tokens * 4, s), "plan_step");
    if (!rc && max_tokens > 0)
      rc = check_cuda(cudaMemsetAsync(slot_mapping, 0xff, (size_t)max_tokens * 8, s), "plan_step");
    return rc;
  }
  PlanArgs a{free_stack, free_top, num_blocks, block_tables, table_stride, table_len, seq_lens,
             num_rows, rows, n_new, n_items, block_size, query_start_loc, ctx_lens, slot_mapping,
             max_tokens,
             ((reinterpret_cast<uintptr_t>(ctx_lens) | reinterpret_cast<uintptr_t>(slot_mapping)) & 15) == 0,
             dev_status};
  const size_t smem = plan_smem(n_items, num_rows);
  // One small CTA covers a decode step; admissions take up to 16 large ones.
  const bool small = max_tokens <= 4 * kPlanSmall * kPlanGroup && n_items <= 4 * kPlanSmall;
  const int threads = small ? kPlanSmall : kPlanLarge;
  int ctas = 1;
  while (!small && ctas < 16 && (int64_t)ctas * threads * kPlanGroup < max_tokens) ctas *= 2;
  void (*kern)(PlanArgs) = small ? plan_step_kernel<kPlanSmall> : plan_step_kernel<kPlanLarge>;
  if (smem > 40 * 1024 || ctas > 8) {  // beyond what every kernel may have
    const int rc = small ? plan_configure<kPlanSmall>() : plan_configure<kPlanLarge>();
    if (rc) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a), "plan_step launch");
}
