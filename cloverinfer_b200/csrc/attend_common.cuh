// Decode attention over a 16/32-bit cache or an 8-bit cache with scales, with
// one softmax map per head or two (differential attention): arguments, the
// split of a step's work over its workers, and how a worker's result leaves it.
//
// Work: a unit is 16 or 32 consecutive tokens (the kernel's choice) of one
// segment; a segment is (sequence b, KV head, column chunk) and holds
// n = ceil(ctx_b / unit) units, ctx_b the context of the sequence's last row (rows are in causal
// order).  A column is one (query row, query head of the KV head's group,
// map), so a KV tile is read once for all heads of a group, all new tokens and
// both maps.  A worker is one warp (generic kernel) or one ring of stages with
// its warps (tensor-core kernel).
//   * aligned launches: a segment is cut into ceil(n / per) equal pieces, per
//     the least range for which the step has at most as many pieces as there
//     are workers; pieces are numbered sequence-major, then along the context,
//     then by segment, and worker w takes piece w (partial slot w).  The heads of
//     a KV block then stream at the same time, so DRAM serves whole blocks
//     instead of one head's 128 or 256 bytes here and there.
//   * ranged launches, where aligned pieces would leave workers idle (more
//     than a sixth longer than an even share: many segments, or very ragged
//     ones): units are numbered sequence-major, then segment, then along the
//     context, with the segment's cost in empty numbers before its first unit (a
//     worker with many short segments else takes far longer than one inside a
//     long one), and worker w takes [w per, (w + 1) per).  A range meets at most
//     two segments it does not hold whole: its first (a piece that starts inside
//     the segment, partial slot 2w) and its last (a piece with the segment's
//     first unit, slot 2w + 1).  The workspace is 2 slots per worker whatever
//     the batch, and the pieces of a segment are slot 2w + 1 of its first worker
//     and slots 2(w + 1), 2(w + 2), ... of the following ones.
//   * whole launches (short contexts): worker w takes segments w, w + W, ...
//     and writes their outputs; no second kernel runs.
#pragma once

#include <math.h>

#include "decode_common.cuh"
#include "quantise.cuh"

namespace clover {

constexpr int kUnitTok = 16;     // a unit is a multiple of this
constexpr int kAttendWarps = 4;  // workers of a generic CTA
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kAttendMinTok = 64;   // a worker's least range (measured: 32 requests of 300 tokens, 19.2 us at 128)
constexpr int kSegCostTok = 128;    // what a segment costs beside its units (queries, output), as tokens
constexpr int kAttendMaxPerSm = 16; // generic workers per SM

struct AttendArgs {
  void* out;
  int64_t out_stride;
  const void* q;
  int64_t q_stride;
  int32_t q_dtype;
  int32_t q_vec;  // query rows are 16-byte aligned
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
  int32_t seg_cost;   // of a segment, in units
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
  // [n_seqs][hkv][chunks]: the segment's pieces are slots x, y + z, y + 2z, ...
  // (w of them; <= 1: written by its worker)
  int4* seg;
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
// flat number of the segment's first unit (ranged launches) or the segment
// (whole ones).  Aligned and ranged launches end after `left` units, whole ones
// at the last segment.
struct Cursor {
  int b, h, jj, left, seg0;
  SeqInfo s;

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
    if ((left -= a.seg_cost) <= 0) return false;
    jj = 0;
    seg0 += s.n + a.seg_cost;
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

// Shared memory of the plan of a CTA with NW warps and R workers.
constexpr int kAlignTries = 6;  // aligned ranges up to 5/32 longer than an even share
template <int NW, int R>
struct AttendPlan {
  int sum[NW][kAlignTries + 2];  // per warp: numbers, pieces at each range tried, units
  int start[R][4];               // sequence, segment, first unit, units (ranged: flat number of the segment)
  int seg0[R];
};

// What all workers of a launch share: units per worker, and whether the pieces
// are aligned.
struct AttendSplit {
  int per, total;
  int quota;  // workers of a CTA that have work
  bool aligned;
};

// Worker r of this CTA: the CTA's workers are consecutive, so every SM has the
// same share of the step; r >= quota has no work.
__device__ __forceinline__ int attend_worker(const AttendSplit& sp, int r) { return blockIdx.x * sp.quota + r; }

// Range k of those tried for aligned pieces.
__device__ __forceinline__ int attend_try(int even, int k) { return even + (even * k + 31) / 32; }

// Every CTA counts the step's units by itself (thread i takes sequences
// [i c, (i + 1) c)) and finds where its workers start; all threads call it.
template <int NW, int R>
__device__ __forceinline__ AttendSplit attend_plan(const AttendArgs& a, AttendPlan<NW, R>& p) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c = (a.n_seqs + NW * 32 - 1) / (NW * 32);
  const int b0 = min(a.n_seqs, tid * c), b1 = min(a.n_seqs, b0 + c);
  SeqInfo kept{0, 0, 0, 0, 0};  // of the one sequence of a thread (c = 1)
  auto info = [&](int b) { return c == 1 ? kept : seq_info(a, b); };
  // numbers of a sequence in a ranged launch
  auto numbers = [&](const SeqInfo& s) { return s.n > 0 ? s.hc * (s.n + a.seg_cost) : 0; };
  int mine = 0, units = 0;
  for (int b = b0; b < b1; ++b) {
    kept = seq_info(a, b);
    if (blockIdx.x == 0) attend_check_seq(a, kept);
    mine += numbers(kept);
    units += kept.n * kept.hc;
  }
  int x = __reduce_add_sync(0xffffffffu, mine);
  units = __reduce_add_sync(0xffffffffu, units);
  if (lane == 0) {
    p.sum[warp][0] = x;
    p.sum[warp][kAlignTries + 1] = units;
  }
  if (tid < R) p.start[tid][0] = -1;
  __syncthreads();
  AttendSplit sp{0, 0, R, false};
  int all_units = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    sp.total += p.sum[w][0];
    all_units += p.sum[w][kAlignTries + 1];
  }
  // even shares: of the numbers (a range has to hold more than a segment's
  // cost), and of the units for aligned pieces
  const int least = kAttendMinTok >> a.unit_log2;
  const int even = max((sp.total + a.workers - 1) / a.workers, a.seg_cost + least);
  const int even_units = max((all_units + a.workers - 1) / a.workers, least);
  int pieces[kAlignTries];
#pragma unroll
  for (int k = 0; k < kAlignTries; ++k) pieces[k] = 0;
  for (int b = b0; b < b1; ++b) {
    const SeqInfo s = info(b);
#pragma unroll
    for (int k = 0; k < kAlignTries; ++k) {
      const int per = attend_try(even_units, k);
      pieces[k] += s.hc * ((s.n + per - 1) / per);
    }
  }
#pragma unroll
  for (int k = 0; k < kAlignTries; ++k) {
    x = __reduce_add_sync(0xffffffffu, pieces[k]);
    if (lane == 0) p.sum[warp][k + 1] = x;
  }
  __syncthreads();
  int col = 0;  // of p.sum: what is numbered
  int used = (sp.total + even - 1) / even;  // workers
  sp.per = even;
#pragma unroll
  for (int k = 0; k < kAlignTries; ++k) {
    int all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) all += p.sum[w][k + 1];
    if (!sp.aligned && all <= a.workers) {
      sp.aligned = true;
      sp.per = attend_try(even_units, k);
      mine = pieces[k];
      col = k + 1;
      used = all;
    }
  }
  sp.quota = min(R, max(1, (used + (int)gridDim.x - 1) / (int)gridDim.x));
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += y;
  }
  int before = incl - mine;
  for (int w = 0; w < warp; ++w) before += p.sum[w][col];
  for (int k = 0; k < sp.quota; ++k) {
    const int wid = attend_worker(sp, k);
    const int64_t u0 = sp.aligned ? wid : (int64_t)wid * sp.per;
    if (u0 < before || u0 >= before + mine) continue;
    int at = before;
    for (int b = b0; b < b1; ++b) {
      const SeqInfo s = info(b);
      const int kp = (s.n + sp.per - 1) / sp.per;
      const int u = sp.aligned ? s.hc * kp : numbers(s);
      if (u0 < at + u) {
        const int off = (int)(u0 - at);
        p.start[k][0] = b;
        if (sp.aligned) {
          const int i = off / s.hc, len = (s.n + kp - 1) / kp;
          p.start[k][1] = off - i * s.hc;
          p.start[k][2] = i * len;
          p.start[k][3] = min(len, s.n - i * len);
          p.seg0[k] = 0;
          if (i * len >= s.n) p.start[k][0] = -1;  // (rounding left the last piece empty)
        } else {
          const int h = off / (s.n + a.seg_cost), in = off - h * (s.n + a.seg_cost);
          p.start[k][1] = h;
          p.start[k][2] = max(0, in - a.seg_cost);
          p.start[k][3] = (int)min((int64_t)sp.per, sp.total - u0) - max(0, a.seg_cost - in);
          p.seg0[k] = at + h * (s.n + a.seg_cost);
          if (p.start[k][3] <= 0) p.start[k][0] = -1;  // (the batch ends before a unit)
        }
        break;
      }
      at += u;
    }
  }
  __syncthreads();
  return sp;
}

// Worker r's first unit; false without one.
template <int NW, int R>
__device__ __forceinline__ bool attend_start(const AttendArgs& a, const AttendPlan<NW, R>& p, int r, Cursor& cur) {
  if (p.start[r][0] < 0) return false;
  cur.b = p.start[r][0];
  cur.s = seq_info(a, cur.b);
  cur.h = p.start[r][1];
  cur.jj = p.start[r][2];
  cur.left = p.start[r][3];
  cur.seg0 = p.seg0[r];
  return true;
}

// The partial slot of a worker's piece, and (from the piece with the segment's
// first unit) the segment's entry for the join.
__device__ __forceinline__ int64_t attend_slot(const AttendSplit& sp, int wid, int first_jj) {
  return sp.aligned ? wid : 2 * (int64_t)wid + (first_jj == 0 ? 1 : 0);
}
__device__ __forceinline__ void attend_record(const AttendArgs& a, const AttendSplit& sp, int b, int h, int seg0,
                                              const SeqInfo& s, int wid) {
  int4 e;
  if (sp.aligned) {
    const int kp = (s.n + sp.per - 1) / sp.per, len = (s.n + kp - 1) / kp;
    e = make_int4(wid, wid, s.hc, (s.n + len - 1) / len);
  } else {
    const int first = seg0 + a.seg_cost, fw = first / sp.per;
    e = make_int4(2 * fw + 1, 2 * fw, 2, (first + s.n - 1) / sp.per - fw + 1);
  }
  a.seg[(int64_t)b * (a.hkv * a.chunks) + h] = e;
}

// ------------------------------------------------------------------ results
// Final value of one dim from the maps' normalised outputs.
__device__ __forceinline__ float diff_value(float o1, float o2, float lam) { return fmaf(-lam, o2, o1); }

// Host side (paged_attend_mma.cu): the tensor-core kernel for these types and
// shape; cols 8 or 16.  a == null only reports the workers of a CTA (one CTA per
// SM).
bool attend_mma_supported(int kv_dtype, int q_dtype, int D, int bs);
int attend_mma_unit_log2(int kv_dtype, int D);
int attend_mma(int kv_dtype, int q_dtype, int cols, const AttendArgs* a, int D, cudaStream_t s, int* rings);

}  // namespace clover
