// Decode over an 8-bit cache with scales, and differential decode attention:
// the kernel for every type, head_dim and block size, the join of split
// segments, and the C entries.
//
//     s_m,t = scale * ks_t * (q_m . kc_t),   p_m = softmax_t(s_m)
//     o_m   = sum_t p_m,t vs_t vc_t
// over the tokens a row may see; ks = vs = 1 without scales.  One map:
// out = o_1 (the attention of CpuAttentionBackend.decode_layer,
// src/core/attention_backend.py:113-118).  Two maps (differential attention):
// q = [q_1 | q_2] and k = [k_1 | k_2] are the halves of head_dim, v is whole;
//     o = o_1 - lambda_h o_2;   with a norm weight w:
//     out = o rsqrt(mean_d o_d^2 + eps) w_d out_scale.
// A column of map m is a query whose other half is zero, so both maps are
// columns of the same product with the K tile.  Sums, maxima and the norm are
// in fp32; the result is rounded once, to the query's type.  attend_common.cuh
// has the split over workers.
#include "attend_common.cuh"

#include <mutex>

namespace clover {

template <typename KT>
__device__ __forceinline__ float load_cache(const KT* p) { return load_f<KT>(p); }
template <>
__device__ __forceinline__ float load_cache<int8_t>(const int8_t* p) { return (float)*p; }
template <>
__device__ __forceinline__ float load_cache<__nv_fp8_e4m3>(const __nv_fp8_e4m3* p) { return float(*p); }

// ------------------------------------------------------------------ generic kernel
// Lane l holds dims l, l + 32, ... of NC columns.  Four tokens' rows are
// loaded at a time; a score is a warp sum.  Bound by the warp sums (5 shuffles
// per token and column), not by memory: the shapes the tensor-core kernel
// does not take (fp32 caches, other head_dims and blocks).
template <typename KT, int EPL, int NC>
__global__ void __launch_bounds__(kAttendThreads)
attend_generic_kernel(const AttendArgs a) {
  __shared__ AttendPlan<kAttendWarps, kAttendWarps> plan;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int wid = warp * gridDim.x + blockIdx.x;
  pdl_wait();
  AttendSplit sp{1, 0, 0, false};
  Cursor cur;
  int seg = 0;  // whole launches: the worker's segment (empty ones too: their zeros)
  const int hcmax = a.hkv * a.chunks;
  if (!a.whole) {
    sp = attend_plan<kAttendWarps, kAttendWarps>(a, plan);
    pdl_trigger();
    if (!attend_start(a, plan, warp, cur)) return;
    wid = attend_worker(sp, warp);
  } else {
    seg = wid - a.workers;
  }

  float qv[NC][EPL], acc[NC][EPL], m[NC], l[NC];
  int lim[NC];
  for (;;) {
    // ---- the next segment's piece
    int first_jj, chunk, kvh;
    if (a.whole) {
      bool found = false;
      for (seg += a.workers; seg < a.n_seqs * hcmax; seg += a.workers) {
        cur.b = seg / hcmax;
        cur.h = seg - cur.b * hcmax;
        cur.s = seq_info(a, cur.b);
        if (cur.h == 0 && lane == 0) attend_check_seq(a, cur.s);
        if (cur.h < cur.s.hc) {
          found = true;
          break;
        }
      }
      if (!found) break;
      cur.jj = 0;
      cur.left = cur.s.n;
    }
    first_jj = cur.jj;
    const int nch = cur.s.hc / a.hkv;
    kvh = cur.h / nch;
    chunk = cur.h - kvh * nch;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const AttendCol ci = attend_col(a, cur.s.row0, cur.s.nq, kvh, chunk * NC + c);
      lim[c] = ci.lim;
      if (lim[c] > cur.s.n * kUnitTok) {  // a row past its sequence's last row
        if (lane == 0) raise_status(a.status, CLOVER_B200_DEV_CTX_RANGE);
        lim[c] = cur.s.n * kUnitTok;
      }
      const int64_t qb = (int64_t)ci.row * a.q_stride + (int64_t)ci.head * a.D;
      const int half = a.D / 2;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const int d = lane + 32 * e;
        const bool in = ci.valid && d < a.D && (a.maps == 1 || (d >= half) == (ci.map == 1));
        qv[c][e] = in ? attend_load_q(a, qb + d) * a.scale_log2 : 0.f;
        acc[c][e] = 0.f;
      }
      m[c] = -INFINITY;
      l[c] = 0.f;
    }
    const int trow = a.seq_rows ? __ldg(a.seq_rows + cur.b) : cur.b;
    const int32_t* tab = a.tables + (int64_t)trow * a.table_stride;
    const int ctx_end = min(__ldg(a.ctx + cur.s.row0 + cur.s.nq - 1), a.max_ctx);
    const SeqInfo seq = cur.s;
    const int b = cur.b, h = cur.h, n = seq.n, seg0 = cur.seg0, row0 = seq.row0, nq = seq.nq;
    int last_jj = -1;
    bool more = true;
    while (cur.left > 0 && more && cur.b == b && cur.h == h) {
      last_jj = cur.jj;
      const int tok0 = cur.jj * kUnitTok;
      const int nt = min(kUnitTok, ctx_end - tok0);
      // lane t: the cache slot of token tok0 + t
      int64_t slot = 0, sidx = 0;
      if (lane < nt) {
        const int bi = (tok0 + lane) / a.bs, off = tok0 + lane - bi * a.bs;
        int blk = bi < a.table_stride ? __ldg(tab + bi) : -1;
        if (blk < 0 || blk >= a.num_blocks) {
          raise_status(a.status, CLOVER_B200_DEV_BAD_BLOCK);
          blk = 0;
        }
        slot = ((int64_t)blk * a.bs + off) * a.hkv + kvh;
        sidx = ((int64_t)blk * a.hkv + kvh) * a.bs + off;
      }
      float ksc = 1.f, vsc = 1.f;
      if (a.ks != nullptr && lane < nt) {
        ksc = a.ks[sidx];
        vsc = a.vs[sidx];
      }
      for (int t0 = 0; t0 < nt; t0 += 4) {
        float kx[4][EPL], vx[4][EPL], s[4][NC];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = min(t0 + i, nt - 1);
          const int64_t base = __shfl_sync(0xffffffffu, slot, t) * a.D;
#pragma unroll
          for (int e = 0; e < EPL; ++e) {
            const int d = lane + 32 * e;
            kx[i][e] = d < a.D ? load_cache(static_cast<const KT*>(a.kc) + base + d) : 0.f;
            vx[i][e] = d < a.D ? load_cache(static_cast<const KT*>(a.vc) + base + d) : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            float x = 0.f;
#pragma unroll
            for (int e = 0; e < EPL; ++e) x = fmaf(qv[c][e], kx[i][e], x);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
            s[i][c] = x;
          }
          const float kk = __shfl_sync(0xffffffffu, ksc, min(t0 + i, nt - 1));
#pragma unroll
          for (int c = 0; c < NC; ++c)
            s[i][c] = t0 + i < nt && tok0 + t0 + i < lim[c] ? s[i][c] * kk : -INFINITY;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float nm = fmaxf(m[c], fmaxf(fmaxf(s[0][c], s[1][c]), fmaxf(s[2][c], s[3][c])));
          const float u = nm == -INFINITY ? 0.f : nm;
          const float al = fast_exp2(m[c] - u);
          m[c] = nm;
          l[c] *= al;
#pragma unroll
          for (int e = 0; e < EPL; ++e) acc[c][e] *= al;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float vv = __shfl_sync(0xffffffffu, vsc, min(t0 + i, nt - 1));
            // a masked token adds nothing, whatever its V row holds
            if (t0 + i < nt && tok0 + t0 + i < lim[c]) {
              const float p = fast_exp2(s[i][c] - u);
              l[c] += p;
#pragma unroll
              for (int e = 0; e < EPL; ++e) acc[c][e] = fmaf(p * vv, vx[i][e], acc[c][e]);
            }
          }
        }
      }
      if (a.whole) {
        --cur.left;
        ++cur.jj;
      } else {
        more = cur.next(a);
      }
    }

    // ---- the piece is done: the output, or a partial
    const bool is_whole = a.whole || (first_jj == 0 && last_jj == n - 1);
    if (!is_whole) {
      const int64_t slot = attend_slot(sp, wid, first_jj);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          if (lane + 32 * e < a.D) a.part[(slot * NC + c) * a.D + lane + 32 * e] = acc[c][e];
        if (lane == 0) a.part_ml[slot * NC + c] = make_float2(m[c], l[c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const AttendCol ci = attend_col(a, row0, nq, kvh, chunk * NC + c);
        if (!ci.valid || ci.map == 1) continue;
        const float inv = attend_inv(l[c], lim[c]);
        const int64_t ob = (int64_t)ci.row * a.out_stride + (int64_t)ci.head * a.D;
        float o[EPL];
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[e] = lim[c] > 0 ? acc[c][e] * inv : 0.f;
        if (a.maps == 2) {
          const int c2 = c + 1 < NC ? c + 1 : c;  // map 2 of the head (NC = 1 has one map)
          const float lam = a.lam[ci.head], inv2 = attend_inv(l[c2], lim[c2]);
          float sq = 0.f;
#pragma unroll
          for (int e = 0; e < EPL; ++e) {
            o[e] = lim[c] > 0 ? diff_value(o[e], acc[c2][e] * inv2, lam) : 0.f;
            sq = fmaf(o[e], o[e], sq);
          }
          if (a.norm_w != nullptr && lim[c] > 0) {
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
            const float r = rsqrtf(sq / a.D + a.eps) * a.out_scale;
#pragma unroll
            for (int e = 0; e < EPL; ++e)
              if (lane + 32 * e < a.D) o[e] *= r * a.norm_w[lane + 32 * e];
          }
        }
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          if (lane + 32 * e < a.D) attend_store(a, ob + lane + 32 * e, o[e]);
      }
    }
    if (!a.whole && first_jj == 0 && lane == 0) attend_record(a, sp, b, h, seg0, seq, wid);
    if (!a.whole && (!more || cur.left <= 0)) break;
  }
}

// ------------------------------------------------------------------ join
// A CTA of 8 warps takes outputs of one segment (a column, or the pair of maps
// of a head), wpo warps each: 1 where there are outputs enough to fill the GPU,
// up to 8 where a few columns have hundreds of pieces.  A warp takes every
// wpo-th piece, kJoinFlight of them in flight; lane l holds dims l, l + 32, ...
constexpr int kJoinWarps = 8;
constexpr int kJoinThreads = kJoinWarps * 32;
constexpr int kJoinFlight = 4;

template <int EPL, int MAPS>
__global__ void __launch_bounds__(kJoinThreads)
attend_join_kernel(const AttendArgs a, int wpo) {
  __shared__ float s_o[MAPS][kJoinWarps][32 * EPL];
  __shared__ float2 s_ml[MAPS][kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int hcmax = a.hkv * a.chunks;
  const int outs = kJoinWarps / wpo;  // of a CTA
  const int64_t seg = blockIdx.x;
  const int b = (int)(seg / hcmax), h = (int)(seg - (int64_t)b * hcmax);
  const int out = blockIdx.y * outs + warp / wpo, part = warp % wpo;
  const int c0 = out * MAPS;
  // the step's layout is final before the attention kernel ran
  const SeqInfo s = seq_info(a, b);
  AttendCol ci{0, 0, 0, 0, false};
  if (h < s.hc && c0 < a.cols) {
    const int nch = s.hc / a.hkv, kvh = h / nch;
    ci = attend_col(a, s.row0, s.nq, kvh, (h - kvh * nch) * a.cols + c0);
  }
  pdl_wait();
  pdl_trigger();
  if (h >= s.hc) return;
  const int64_t ob = (int64_t)ci.row * a.out_stride + (int64_t)ci.head * a.D;
  if (s.n == 0) {  // an empty sequence has no worker
    if (ci.valid && part == 0)
      for (int d = lane; d < a.D; d += 32) attend_store(a, ob + d, 0.f);
    return;
  }
  const int4 sg = a.seg[seg];
  if (sg.w <= 1) return;  // written by its worker
  // (a worker that gave up waiting leaves its segment's entry unwritten)
  const int64_t last = sg.y + (int64_t)(sg.w - 1) * sg.z;
  if (sg.x < 0 || sg.y < 0 || sg.z <= 0 || sg.x >= 2 * a.workers || last >= 2 * a.workers) return;
  float o[MAPS][EPL], m[MAPS], l[MAPS];
#pragma unroll
  for (int mp = 0; mp < MAPS; ++mp) {
    m[mp] = -INFINITY;
    l[mp] = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[mp][e] = 0.f;
  }
  if (ci.valid) {
    for (int i0 = part; i0 < sg.w; i0 += wpo * kJoinFlight) {
#pragma unroll
      for (int mp = 0; mp < MAPS; ++mp) {
        float2 ml[kJoinFlight];
        float x[kJoinFlight][EPL];
#pragma unroll
        for (int f = 0; f < kJoinFlight; ++f) {
          const int i = i0 + f * wpo;
          const bool ok = i < sg.w;
          const int64_t slot = i == 0 ? sg.x : sg.y + (int64_t)i * sg.z;
          const int64_t at = ok ? slot * a.cols + c0 + mp : 0;
          ml[f] = ok ? __ldcg(a.part_ml + at) : make_float2(-INFINITY, 0.f);
#pragma unroll
          for (int e = 0; e < EPL; ++e)
            x[f][e] = ok && lane + 32 * e < a.D ? __ldcg(a.part + at * a.D + lane + 32 * e) : 0.f;
        }
        float nm = m[mp];
#pragma unroll
        for (int f = 0; f < kJoinFlight; ++f) nm = fmaxf(nm, ml[f].x);
        const float u = nm == -INFINITY ? 0.f : nm;
        const float f0 = fast_exp2(m[mp] - u);
        m[mp] = nm;
        l[mp] *= f0;
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[mp][e] *= f0;
#pragma unroll
        for (int f = 0; f < kJoinFlight; ++f) {
          const float fw = fast_exp2(ml[f].x - u);
          l[mp] = fmaf(ml[f].y, fw, l[mp]);
#pragma unroll
          for (int e = 0; e < EPL; ++e) o[mp][e] = fmaf(x[f][e], fw, o[mp][e]);
        }
      }
    }
  }
  if (wpo > 1) {
#pragma unroll
    for (int mp = 0; mp < MAPS; ++mp) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) s_o[mp][warp][lane + 32 * e] = o[mp][e];
      if (lane == 0) s_ml[mp][warp] = make_float2(m[mp], l[mp]);
    }
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int mp = 0; mp < MAPS; ++mp) {
      for (int k = 1; k < wpo; ++k) {
        const float2 ml = s_ml[mp][warp + k];
        const float nm = fmaxf(m[mp], ml.x), u = nm == -INFINITY ? 0.f : nm;
        const float f0 = fast_exp2(m[mp] - u), f1 = fast_exp2(ml.x - u);
        m[mp] = nm;
        l[mp] = fmaf(ml.y, f1, l[mp] * f0);
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[mp][e] = fmaf(s_o[mp][warp + k][lane + 32 * e], f1, o[mp][e] * f0);
      }
    }
  }
  if (!ci.valid) return;
  const bool any = ci.lim > 0;
#pragma unroll
  for (int mp = 0; mp < MAPS; ++mp) {
    const float inv = attend_inv(l[mp], ci.lim);
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[mp][e] = any ? o[mp][e] * inv : 0.f;
  }
  if (MAPS == 2) {
    const float lam = a.lam[ci.head];
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      o[0][e] = diff_value(o[0][e], o[MAPS - 1][e], lam);
      sq = fmaf(o[0][e], o[0][e], sq);
    }
    if (a.norm_w != nullptr && any) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
      const float r = rsqrtf(sq / a.D + a.eps) * a.out_scale;
#pragma unroll
      for (int e = 0; e < EPL; ++e)
        if (lane + 32 * e < a.D) o[0][e] *= r * a.norm_w[lane + 32 * e];
    }
  }
#pragma unroll
  for (int e = 0; e < EPL; ++e)
    if (lane + 32 * e < a.D) attend_store(a, ob + lane + 32 * e, o[0][e]);
}

template <int MAPS>
static cudaError_t launch_join(const AttendArgs& a, int sms, cudaStream_t s) {
  const int64_t segs = (int64_t)a.n_seqs * a.hkv * a.chunks;
  const int outs = (a.cols + MAPS - 1) / MAPS;  // of a segment
  int wpo = 1;
  while (wpo < kJoinWarps && segs * outs * wpo < (int64_t)sms * kJoinWarps * 2) wpo *= 2;
  const dim3 grid((unsigned)segs, (unsigned)((outs * wpo + kJoinWarps - 1) / kJoinWarps)), block(kJoinThreads);
  if (a.D <= 64) return launch_pdl(attend_join_kernel<2, MAPS>, grid, block, 0, s, a, wpo);
  if (a.D <= 128) return launch_pdl(attend_join_kernel<4, MAPS>, grid, block, 0, s, a, wpo);
  return launch_pdl(attend_join_kernel<8, MAPS>, grid, block, 0, s, a, wpo);
}

// ------------------------------------------------------------------ append
// Row r's new token at position ctx[r] - 1 of its sequence, before the
// attention of the same step: one warp per (row, K or V, head).
struct AppendRowsArgs {
  AttendArgs a;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  const void* kn;
  const void* vn;
  int64_t new_stride;
  int32_t new_dtype, kv_dtype, n_rows;
};

__global__ void __launch_bounds__(256) attend_append_kernel(const AppendRowsArgs p) {
  const AttendArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t work = (int64_t)p.n_rows * 2 * a.hkv;
  const int rows_end = __ldg(a.qsl + a.n_seqs);
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < work; w += (int64_t)gridDim.x * 8) {
    const int r = (int)(w / (2 * a.hkv));
    const int rest = (int)(w - (int64_t)r * 2 * a.hkv);
    const bool is_v = rest >= a.hkv;
    const int h = is_v ? rest - a.hkv : rest;
    if (r >= rows_end) continue;  // behind the last sequence
    int lo = 0, hi = a.n_seqs - 1;  // the last sequence that starts at or before r
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(a.qsl + mid) <= r) lo = mid; else hi = mid - 1;
    }
    const int pos = __ldg(a.ctx + r) - 1;
    if (pos < 0) continue;
    if (pos >= a.max_ctx) {  // past what the attention covers
      if (lane == 0) raise_status(a.status, CLOVER_B200_DEV_CTX_RANGE);
      continue;
    }
    const int trow = a.seq_rows ? __ldg(a.seq_rows + lo) : lo;
    const int bi = pos / a.bs, off = pos - bi * a.bs;
    const int blk = bi < a.table_stride ? __ldg(a.tables + (int64_t)trow * a.table_stride + bi) : -1;
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0) raise_status(a.status, CLOVER_B200_DEV_BAD_BLOCK);
      continue;
    }
    const int64_t row = (((int64_t)blk * a.bs + off) * a.hkv + h) * a.D;
    const int64_t at = (int64_t)r * p.new_stride + (int64_t)h * a.D;
    const void* src = is_v ? p.vn : p.kn;
    uint8_t* dst = is_v ? p.vc : p.kc;
    if (p.ks != nullptr) {
      const float s = p.kv_dtype == CLOVER_B200_INT8
                          ? encode_row_any<false>(p.new_dtype, src, at, dst + row, a.D, lane)
                          : encode_row_any<true>(p.new_dtype, src, at, dst + row, a.D, lane);
      if (lane == 0) (is_v ? p.vs : p.ks)[((int64_t)blk * a.hkv + h) * a.bs + off] = s;
    } else if (p.kv_dtype == CLOVER_B200_F32) {
      for (int d = lane; d < a.D; d += 32)
        reinterpret_cast<uint32_t*>(dst)[row + d] = static_cast<const uint32_t*>(src)[at + d];
    } else {
      for (int d = lane; d < a.D; d += 32)
        reinterpret_cast<uint16_t*>(dst)[row + d] = static_cast<const uint16_t*>(src)[at + d];
    }
  }
}

// ------------------------------------------------------------------ host side
template <typename KT, int EPL, int NC>
static int generic_grid(int sms) {
  static int cached = 0;
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  if (cached == 0) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attend_generic_kernel<KT, EPL, NC>,
                                                      kAttendThreads, 0) != cudaSuccess || n < 1)
      return sms;
    cached = n > kAttendMaxPerSm / kAttendWarps ? kAttendMaxPerSm / kAttendWarps : n;
  }
  return cached * sms;
}

template <typename KT, int EPL, int NC>
static int generic_launch(const AttendArgs* a, cudaStream_t s, int sms, int* grid) {
  if (a == nullptr) {
    *grid = generic_grid<KT, EPL, NC>(sms);
    return CLOVER_B200_OK;
  }
  return check_cuda(launch_pdl(attend_generic_kernel<KT, EPL, NC>, dim3(a->workers / kAttendWarps),
                               dim3(kAttendThreads), 0, s, *a),
                    "attend_generic launch");
}

template <typename KT, int EPL>
static int generic_nc(int cols, const AttendArgs* a, cudaStream_t s, int sms, int* grid) {
  switch (cols) {
    case 1: return generic_launch<KT, EPL, 1>(a, s, sms, grid);
    case 2: return generic_launch<KT, EPL, 2>(a, s, sms, grid);
    case 4: return generic_launch<KT, EPL, 4>(a, s, sms, grid);
    default: return generic_launch<KT, EPL, 8>(a, s, sms, grid);
  }
}

template <typename KT>
static int generic_epl(int D, int cols, const AttendArgs* a, cudaStream_t s, int sms, int* grid) {
  if (D <= 32) return generic_nc<KT, 1>(cols, a, s, sms, grid);
  if (D <= 64) return generic_nc<KT, 2>(cols, a, s, sms, grid);
  if (D <= 128) return generic_nc<KT, 4>(cols, a, s, sms, grid);
  return generic_nc<KT, 8>(cols, a, s, sms, grid);
}

static int attend_generic(int kv_dtype, int D, int cols, const AttendArgs* a, cudaStream_t s, int sms,
                          int* grid) {
  switch (kv_dtype) {
    case CLOVER_B200_F32: return generic_epl<float>(D, cols, a, s, sms, grid);
    case CLOVER_B200_F16: return generic_epl<__half>(D, cols, a, s, sms, grid);
    case CLOVER_B200_BF16: return generic_epl<__nv_bfloat16>(D, cols, a, s, sms, grid);
    case CLOVER_B200_INT8: return generic_epl<int8_t>(D, cols, a, s, sms, grid);
    default: return generic_epl<__nv_fp8_e4m3>(D, cols, a, s, sms, grid);
  }
}

struct AttendShape {
  bool mma, whole;
  int cols, chunks, workers, sms, unit_log2;
  int64_t part_bytes, ml_bytes, seg_bytes, bytes;
};

static int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

// The launch shape of one call, shared with the workspace query.
static int attend_shape(int n_seqs, int n_rows, int max_q, int max_ctx, int hq, int hkv, int D, int bs,
                        int kv_dtype, int q_dtype, int maps, AttendShape* p) {
  if (n_seqs < 0 || n_rows < 0 || max_q < 0 || max_ctx < 0 || hq <= 0 || hkv <= 0 || D <= 0 || bs <= 0)
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "attend: bad sizes");
  if (hq % hkv != 0)
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "attend: num_q_heads %% num_kv_heads != 0");
  if (D > 256) return set_error(CLOVER_B200_ERR_UNSUPPORTED, "attend: head_dim %d > 256", D);
  if (maps == 2 && (D & 1))
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "diff_decode: head_dim %d has no halves", D);
  if (q_dtype != CLOVER_B200_F32 && q_dtype != CLOVER_B200_F16 && q_dtype != CLOVER_B200_BF16)
    return set_error(CLOVER_B200_ERR_UNSUPPORTED, "attend: q dtype %d", q_dtype);
  const bool scaled = kv_dtype == CLOVER_B200_INT8 || kv_dtype == CLOVER_B200_FP8_E4M3;
  if (!scaled && kv_dtype != CLOVER_B200_F32 && kv_dtype != CLOVER_B200_F16 && kv_dtype != CLOVER_B200_BF16)
    return set_error(CLOVER_B200_ERR_UNSUPPORTED, "attend: kv dtype %d", kv_dtype);
  if (!scaled && q_dtype != CLOVER_B200_F32 && q_dtype != kv_dtype)
    return set_error(CLOVER_B200_ERR_UNSUPPORTED, "attend: queries are fp32 or of the cache's type");
  if (max_q == 0) max_q = 1;
  int dev = 0;
  p->sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t cols = (int64_t)max_q * (hq / hkv) * maps;
  p->mma = attend_mma_supported(kv_dtype, q_dtype, D, bs);
  p->cols = p->mma ? (cols > kMmaCols ? 2 * kMmaCols : kMmaCols)
                   : cols >= 8 ? 8 : cols >= 4 ? 4 : cols >= 2 ? 2 : 1;
  const int64_t chunks = (cols + p->cols - 1) / p->cols;
  p->unit_log2 = p->mma ? attend_mma_unit_log2(kv_dtype, D) : 4;
  const int64_t units = ((int64_t)max_ctx + (1 << p->unit_log2) - 1) >> p->unit_log2;
  const int64_t least = kAttendMinTok >> p->unit_log2;  // units of a worker's least range
  if (chunks > 65535 || (int64_t)n_seqs * hkv * chunks > INT32_MAX / 64 ||
      (int64_t)n_seqs * hkv * chunks * (units + kSegCostTok) > INT32_MAX)
    return set_error(CLOVER_B200_ERR_UNSUPPORTED, "attend: batch too large");
  p->chunks = (int)chunks;
  // Short contexts: a segment is at most two ranges' least work; splitting it
  // would cost the second launch more than it gains.
  p->whole = units <= 2 * least;
  int grid = p->sms, rings = kAttendWarps;
  const int rc = p->mma ? attend_mma(kv_dtype, q_dtype, p->cols, nullptr, D, nullptr, &rings)
                        : attend_generic(kv_dtype, D, p->cols, nullptr, nullptr, p->sms, &grid);
  if (rc) return rc;
  const int64_t segs = (int64_t)n_seqs * hkv * chunks;
  const int64_t want = p->whole ? segs : (segs * units + least - 1) / least;
  // one CTA per worker until every CTA has one: few workers spread over the SMs
  const int64_t ctas = want < 1 ? 1 : want < grid ? want : grid;
  p->workers = (int)ctas * rings;
  p->part_bytes = p->ml_bytes = p->seg_bytes = 0;
  if (!p->whole) {
    p->part_bytes = round256(2ll * p->workers * p->cols * D * 4);
    p->ml_bytes = round256(2ll * p->workers * p->cols * 8);
    p->seg_bytes = round256(segs * 16);
  }
  p->bytes = p->part_bytes + p->ml_bytes + p->seg_bytes;
  return CLOVER_B200_OK;
}

static int attend_impl(const char* what, void* out, int64_t out_row_stride, const void* q,
                       int64_t q_row_stride, int32_t q_dtype, void* k_cache, void* v_cache,
                       float* k_scales, float* v_scales, int32_t kv_dtype, int64_t num_blocks,
                       int32_t block_size, const void* k_new, const void* v_new,
                       int64_t new_token_stride, int32_t new_dtype, const int32_t* block_tables,
                       int32_t table_stride, const int32_t* seq_rows, const int32_t* query_start_loc,
                       const int32_t* ctx_lens, int32_t n_seqs, int32_t n_query_rows,
                       int32_t max_queries_per_seq, int32_t max_ctx_len, int32_t num_q_heads,
                       int32_t num_kv_heads, int32_t head_dim, float score_scale, int32_t maps,
                       const float* lam, const float* norm_weight, float eps, float out_scale,
                       void* workspace, int64_t workspace_bytes, int32_t* dev_status, void* stream) {
  AttendShape sh;
  int rc = attend_shape(n_seqs, n_query_rows, max_queries_per_seq, max_ctx_len, num_q_heads,
                        num_kv_heads, head_dim, block_size, kv_dtype, q_dtype, maps, &sh);
  if (rc) return rc;
  if (table_stride <= 0 || num_blocks <= 0)
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (n_seqs == 0 || n_query_rows == 0) return CLOVER_B200_OK;
  if (!out || !q || !k_cache || !v_cache || !block_tables || !query_start_loc || !ctx_lens ||
      (maps == 2 && !lam))
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "%s: null pointer", what);
  const bool eight = kv_dtype == CLOVER_B200_INT8 || kv_dtype == CLOVER_B200_FP8_E4M3;
  if (eight != (k_scales != nullptr) || eight != (v_scales != nullptr))
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "%s: an 8-bit cache has scales, another none", what);
  if (q_row_stride < (int64_t)num_q_heads * head_dim || out_row_stride < (int64_t)num_q_heads * head_dim)
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "%s: row stride < heads*head_dim", what);
  if ((k_new == nullptr) != (v_new == nullptr))
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "%s: new K without new V", what);
  if (k_new) {
    if (new_token_stride < (int64_t)num_kv_heads * head_dim)
      return set_error(CLOVER_B200_ERR_INVALID_ARG, "%s: token stride < heads*head_dim", what);
    if (eight ? (new_dtype != CLOVER_B200_F32 && new_dtype != CLOVER_B200_F16 && new_dtype != CLOVER_B200_BF16)
              : new_dtype != kv_dtype)
      return set_error(CLOVER_B200_ERR_UNSUPPORTED, "%s: new K/V dtype %d", what, new_dtype);
  }
  if (sh.mma && ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
                  reinterpret_cast<uintptr_t>(k_scales) | reinterpret_cast<uintptr_t>(v_scales)) & 15))
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "%s: cache or scales not 16-byte aligned", what);
  if (num_blocks * (int64_t)block_size > INT32_MAX)
    return set_error(CLOVER_B200_ERR_UNSUPPORTED, "%s: cache exceeds 2^31 slots", what);
  if (sh.bytes > 0 && (workspace == nullptr || workspace_bytes < sh.bytes ||
                       (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return set_error(CLOVER_B200_ERR_WORKSPACE, "%s: workspace needs %lld bytes, 16-byte aligned", what,
                     (long long)sh.bytes);

  AttendArgs a = {};
  a.out = out;
  a.out_stride = out_row_stride;
  a.q = q;
  a.q_stride = q_row_stride;
  a.q_dtype = q_dtype;
  a.kc = k_cache;
  a.vc = v_cache;
  a.ks = k_scales;
  a.vs = v_scales;
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.seq_rows = seq_rows;
  a.qsl = query_start_loc;
  a.ctx = ctx_lens;
  a.n_seqs = n_seqs;
  a.n_rows = n_query_rows;
  a.max_ctx = max_ctx_len;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.maps = maps;
  a.D = head_dim;
  a.q_vec = ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(q_row_stride * (q_dtype == CLOVER_B200_F32 ? 4 : 2))) & 15) == 0;
  a.bs = block_size;
  a.num_blocks = num_blocks;
  a.scale_log2 = score_scale * 1.4426950408889634f;
  a.unit_log2 = sh.unit_log2;
  a.seg_cost = kSegCostTok >> sh.unit_log2;
  a.cols = sh.cols;
  a.chunks = sh.chunks;
  a.whole = sh.whole;
  a.workers = sh.workers;
  char* ws = static_cast<char*>(workspace);
  if (!sh.whole) {
    a.part = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + sh.part_bytes);
    a.seg = reinterpret_cast<int4*>(ws + sh.part_bytes + sh.ml_bytes);
  }
  a.lam = lam;
  a.norm_w = norm_weight;
  a.eps = eps;
  a.out_scale = out_scale;
  a.status = dev_status;
  a.wait_ns = wait_limit_ns();
  cudaStream_t s = (cudaStream_t)stream;
  // With one chunk per (sequence, KV head) the worker that owns a new token's
  // unit writes it before its copy; several chunks would read what one writes.
  if (k_new && sh.mma && sh.chunks == 1) {
    a.k_new = k_new;
    a.v_new = v_new;
    a.new_stride = new_token_stride;
    a.new_dtype = new_dtype;
  } else if (k_new) {
    AppendRowsArgs p{a, (uint8_t*)k_cache, (uint8_t*)v_cache, k_scales, v_scales, k_new, v_new,
                     new_token_stride, new_dtype, kv_dtype, n_query_rows};
    const int64_t want = ((int64_t)n_query_rows * 2 * num_kv_heads + 7) / 8;
    const int64_t cap = (int64_t)sh.sms * 8;
    attend_append_kernel<<<(unsigned)(want < cap ? want : cap), 256, 0, s>>>(p);
    rc = check_cuda(cudaGetLastError(), "attend_append launch");
    if (rc) return rc;
  }
  rc = sh.mma ? attend_mma(kv_dtype, q_dtype, sh.cols, &a, head_dim, s, nullptr)
              : attend_generic(kv_dtype, head_dim, sh.cols, &a, s, sh.sms, nullptr);
  if (rc || sh.whole) return rc;
  const cudaError_t e = maps == 2 ? launch_join<2>(a, sh.sms, s) : launch_join<1>(a, sh.sms, s);
  return check_cuda(e, "attend_join launch");
}

}  // namespace clover

using namespace clover;

extern "C" int64_t clover_b200_attend_workspace_bytes(
    int32_t n_seqs, int32_t n_query_rows, int32_t max_queries_per_seq, int32_t max_ctx_len,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
    int32_t kv_dtype, int32_t q_dtype, int32_t differential) {
  AttendShape sh;
  if (attend_shape(n_seqs, n_query_rows, max_queries_per_seq, max_ctx_len, num_q_heads, num_kv_heads,
                   head_dim, block_size, kv_dtype, q_dtype, differential ? 2 : 1, &sh) != CLOVER_B200_OK)
    return -1;
  return sh.bytes;
}

extern "C" int clover_b200_scaled_decode(
    void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride, int32_t q_dtype,
    void* k_cache, void* v_cache, float* k_scales, float* v_scales, int32_t kv_dtype,
    int64_t num_blocks, int32_t block_size, const void* k_new, const void* v_new,
    int64_t new_token_stride, int32_t new_dtype, const int32_t* block_tables, int32_t table_stride,
    const int32_t* seq_rows, const int32_t* query_start_loc, const int32_t* ctx_lens, int32_t n_seqs,
    int32_t n_query_rows, int32_t max_queries_per_seq, int32_t max_ctx_len, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, float score_scale, void* workspace,
    int64_t workspace_bytes, int32_t* dev_status, void* stream) {
  if (kv_dtype != CLOVER_B200_INT8 && kv_dtype != CLOVER_B200_FP8_E4M3)
    return set_error(CLOVER_B200_ERR_UNSUPPORTED, "scaled_decode: cache dtype %d is not 8-bit", kv_dtype);
  return attend_impl("scaled_decode", out, out_row_stride, q, q_row_stride, q_dtype, k_cache, v_cache,
                     k_scales, v_scales, kv_dtype, num_blocks, block_size, k_new, v_new,
                     new_token_stride, new_dtype, block_tables, table_stride, seq_rows,
                     query_start_loc, ctx_lens, n_seqs, n_query_rows, max_queries_per_seq, max_ctx_len,
                     num_q_heads, num_kv_heads, head_dim, score_scale, 1, nullptr, nullptr, 0.f, 1.f,
                     workspace, workspace_bytes, dev_status, stream);
}

extern "C" int clover_b200_diff_decode(
    void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride, int32_t q_dtype,
    void* k_cache, void* v_cache, float* k_scales, float* v_scales, int32_t kv_dtype,
    int64_t num_blocks, int32_t block_size, const void* k_new, const void* v_new,
    int64_t new_token_stride, int32_t new_dtype, const int32_t* block_tables, int32_t table_stride,
    const int32_t* seq_rows, const int32_t* query_start_loc, const int32_t* ctx_lens, int32_t n_seqs,
    int32_t n_query_rows, int32_t max_queries_per_seq, int32_t max_ctx_len, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, float score_scale, const float* lambda,
    const float* norm_weight, float eps, float out_scale, void* workspace, int64_t workspace_bytes,
    int32_t* dev_status, void* stream) {
  return attend_impl("diff_decode", out, out_row_stride, q, q_row_stride, q_dtype, k_cache, v_cache,
                     k_scales, v_scales, kv_dtype, num_blocks, block_size, k_new, v_new,
                     new_token_stride, new_dtype, block_tables, table_stride, seq_rows,
                     query_start_loc, ctx_lens, n_seqs, n_query_rows, max_queries_per_seq, max_ctx_len,
                     num_q_heads, num_kv_heads, head_dim, score_scale, 2, lambda, norm_weight, eps,
                     out_scale, workspace, workspace_bytes, dev_status, stream);
}
