// Decode attention over a 16/32-bit cache or an 8-bit cache with scales, with
// one softmax map per head or two (differential attention): arguments, the
// split of a step's work over its workers, and how a worker's result leaves it.
//
// Work: a unit is 16 or 32 consecutive tokens (the kernel's choice) of one
// segment; a segment is (sequence b, KV head, column chunk) and holds
// n = ceil(ctx_b / unit) units, ctx_b the context of the sequence's last row (rows are in causal
// order).  A column is one (query row, query head of the KV head's group,
// map), so a KV tile is read once for all heads of a group, all new tokens and
// both maps.  A worker is one warp.
//   * split launches: units are numbered sequence-major, then segment, then
//     along the context, and worker w takes [w per, (w + 1) per), so ragged
//     batches leave no worker idle.  A worker's range meets at most two
//     segments it does not hold whole: its first (a piece that starts inside
//     the segment, partial slot 2w) and its last (a piece with the segment's
//     first unit, slot 2w + 1).  The workspace is therefore 2 slots per worker
//     whatever the batch, and the pieces of a segment are slot 2w + 1 of its
//     first worker and slots 2(w + 1), 2(w + 2), ... of the following ones.
//   * whole launches (short contexts): worker w takes segments w, w + W, ...
//     and writes their outputs; no second kernel runs.
#pragma once

#include <math.h>

#include "decode_common.cuh"
#include "quantise.cuh"

namespace clover {

constexpr int kUnitTok = 16;     // a unit is a multiple of this
constexpr int kAttendWarps = 4;  // workers of a CTA
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kAttendMinTok = 128;  // a worker's least range
constexpr int kAttendMaxPerSm = 16; // workers per SM the workspace allows for

struct AttendArgs {
  void* out;
  int64_t out_stride;
  const void* q;
  int64_t q_stride;
  int32_t q_dtype;
  const void* kc;
  const void* vc;
  const float* ks;  // [num_blocks, num_kv_heads, block_size]; null: no scales
  const float* vs;
  const int32_t* tables;
  int32_t table_stride;
  const int32_t* seq_rows;
  const int32_t* qsl;
  const int32_t* ctx;
  int32_t n_seqs, n_rows, max_ctx;
  int32_t unit_log2;  // log2 of a unit's tokens
  int32_t hq, hkv, group, maps;  // maps: 1, or 2 for differential attention
  int32_t D, bs;
  int64_t num_blocks;
  float scale_log2;
  int32_t cols;    // columns per chunk
  int32_t chunks;  // chunks of the sequence with the most rows
  int32_t whole;   // whole launch
  int32_t workers;
  // workspace of split launches
  float* part;    // [2 workers][cols][D]: unnormalised outputs
  float2* part_ml;  // [2 workers][cols]: running maximum (base 2) and sum
  int2* seg;      // [n_seqs][hkv][chunks]: first worker and number of pieces
  // differential attention
  const float* lam;
  const float* norm_w;
  float eps, out_scale;
  // fused append (tensor-core path): row r's new K/V at position ctx[r] - 1
  const void* k_new;
  const void* v_new;
  int64_t new_stride;
  int32_t new_dtype;
  int32_t* status;
  uint64_t wait_ns;
};

struct AttendCol {
  int32_t row, head, map, lim;
  bool valid;
};

// Column c of (query rows row0 .. row0 + nq - 1, KV head kvh).
__device__ __forceinline__ AttendCol attend_col(const AttendArgs& a, int row0, int nq, int kvh, int c) {
  AttendCol r{0, 0, 0, 0, false};
  const int per = a.group * a.maps;
  const int j = c / per;
  if (j < nq) {
    const int k = c - j * per;
    r.row = row0 + j;
    r.head = kvh * a.group + (a.maps == 2 ? k >> 1 : k);
    r.map = a.maps == 2 ? k & 1 : 0;
    r.lim = min(__ldg(a.ctx + r.row), a.max_ctx);
    r.valid = true;
  }
  return r;
}

__device__ __forceinline__ float attend_load_q(const AttendArgs& a, int64_t i) {
  switch (a.q_dtype) {
    case CLOVER_B200_F32: return static_cast<const float*>(a.q)[i];
    case CLOVER_B200_F16: return __half2float(static_cast<const __half*>(a.q)[i]);
    default: return __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[i]);
  }
}

__device__ __forceinline__ void attend_store(const AttendArgs& a, int64_t i, float v) {
  switch (a.q_dtype) {
    case CLOVER_B200_F32: static_cast<float*>(a.out)[i] = v; break;
    case CLOVER_B200_F16: static_cast<__half*>(a.out)[i] = __float2half_rn(v); break;
    default: static_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16_rn(v); break;
  }
}

// 1 / L of a column that attends to lim tokens: 0 without any (its output is
// zero), NaN when every score was -inf (as the softmax of such a row is).
__device__ __forceinline__ float attend_inv(float l, int lim) {
  if (lim <= 0) return 0.f;
  return l == 0.f ? __int_as_float(0x7fc00000) : 1.f / l;
}

// ------------------------------------------------------------------ cursor
// One sequence of the batch as the cursor sees it.
struct SeqInfo {
  int row0, nq, ctx, n, hc;  // first row, rows, longest context, units per segment, segments
};

__device__ __forceinline__ SeqInfo seq_info(const AttendArgs& a, int b) {
  SeqInfo s;
  s.row0 = __ldg(a.qsl + b);
  s.nq = min(__ldg(a.qsl + b + 1), a.n_rows) - s.row0;
  s.n = 0;
  s.hc = 0;
  s.ctx = 0;
  if (s.nq <= 0 || s.row0 < 0) {
    s.nq = 0;
    return s;
  }
  s.ctx = max(0, min(__ldg(a.ctx + s.row0 + s.nq - 1), a.max_ctx));
  s.n = (s.ctx + (1 << a.unit_log2) - 1) >> a.unit_log2;
  const int ch = (s.nq * a.group * a.maps + a.cols - 1) / a.cols;
  s.hc = a.hkv * (ch < a.chunks ? ch : a.chunks);
  return s;
}

// Flags a sequence longer than max_ctx or with more rows than the caller's bound.
__device__ __forceinline__ void attend_check_seq(const AttendArgs& a, const SeqInfo& s) {
  if (s.nq > 0 && (__ldg(a.ctx + s.row0 + s.nq - 1) > a.max_ctx ||
                   (int64_t)s.nq * a.group * a.maps > (int64_t)a.chunks * a.cols))
    raise_status(a.status, CLOVER_B200_DEV_CTX_RANGE);
}

// A worker's position: unit jj of segment h (of s.hc) of sequence b; seg0 is the
// flat number of the segment's first unit.  Split launches end after `left`
// units, whole launches at the last segment.
struct Cursor {
  int b, h, jj, left, seg0;
  SeqInfo s;

  // The first unit of a worker (b, offset of its first unit within b).
  __device__ __forceinline__ void start(const AttendArgs& a, int b0, int off, int base, int units) {
    b = b0;
    s = seq_info(a, b);
    h = off / s.n;
    jj = off - h * s.n;
    seg0 = base + h * s.n;
    left = units;
  }
  // Whole launches: the first segment with units among sg, sg + workers, ...
  __device__ __forceinline__ bool seek(const AttendArgs& a, int64_t sg) {
    const int hcmax = a.hkv * a.chunks;
    for (; sg < (int64_t)a.n_seqs * hcmax; sg += a.workers) {
      b = (int)sg / hcmax;
      h = (int)sg - b * hcmax;
      s = seq_info(a, b);
      if (h < s.hc && s.n > 0) {
        jj = 0;
        seg0 = (int)sg;
        return true;
      }
    }
    return false;
  }
  // Next unit; false at the end.
  __device__ __forceinline__ bool next(const AttendArgs& a) {
    if (a.whole) return ++jj < s.n || seek(a, (int64_t)seg0 + a.workers);
    if (--left <= 0) return false;
    if (++jj < s.n) return true;
    jj = 0;
    seg0 += s.n;
    if (++h < s.hc) return true;
    h = 0;
    do {
      if (++b >= a.n_seqs) {
        left = 0;
        return false;
      }
      s = seq_info(a, b);
    } while (s.n * s.hc == 0);
    return true;
  }
};

// Shared memory of the plan.
struct AttendPlan {
  int warp_sum[kAttendWarps];
  int start[kAttendWarps][3];  // sequence, offset in it, flat number of its first unit
};

// Every CTA counts the step's units by itself (thread i takes sequences
// [i c, (i + 1) c)) and finds where its workers start.  Returns the units per
// worker; all threads call it.
__device__ __forceinline__ int attend_plan(const AttendArgs& a, AttendPlan& p, int& total) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c = (a.n_seqs + kAttendThreads - 1) / kAttendThreads;
  const int b0 = tid * c, b1 = min(a.n_seqs, b0 + c);
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    const SeqInfo s = seq_info(a, b);
    if (blockIdx.x == 0) attend_check_seq(a, s);
    mine += s.n * s.hc;
  }
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += y;
  }
  if (lane == 31) p.warp_sum[warp] = incl;
  if (tid < kAttendWarps) p.start[tid][0] = -1;
  __syncthreads();
  int before = incl - mine;
  total = 0;
#pragma unroll
  for (int w = 0; w < kAttendWarps; ++w) {
    if (w < warp) before += p.warp_sum[w];
    total += p.warp_sum[w];
  }
  int per = (total + a.workers - 1) / a.workers;
  per = max(per, kAttendMinTok >> a.unit_log2);
#pragma unroll
  for (int k = 0; k < kAttendWarps; ++k) {
    const int64_t u0 = (int64_t)(blockIdx.x * kAttendWarps + k) * per;
    if (u0 >= before && u0 < before + mine) {
      int at = before;
      for (int b = b0; b < b1; ++b) {
        const SeqInfo s = seq_info(a, b);
        const int u = s.n * s.hc;
        if (u0 < at + u) {
          p.start[k][0] = b;
          p.start[k][1] = (int)(u0 - at);
          p.start[k][2] = at;
          break;
        }
        at += u;
      }
    }
  }
  __syncthreads();
  return per;
}

// ------------------------------------------------------------------ results
// Final value of one dim from the maps' normalised outputs.
__device__ __forceinline__ float diff_value(float o1, float o2, float lam) { return fmaf(-lam, o2, o1); }

// Host side (paged_attend_mma.cu): the tensor-core kernel for these types and
// shape; cols 8 or 16.  a == null only reports its resident CTAs in *grid.
bool attend_mma_supported(int kv_dtype, int q_dtype, int D, int bs);
int attend_mma_unit_log2(int kv_dtype, int D);
int attend_mma(int kv_dtype, int q_dtype, int cols, const AttendArgs* a, int D, cudaStream_t s, int* grid);

}  // namespace clover
