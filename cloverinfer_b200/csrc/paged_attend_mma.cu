// Tensor-core decode over a 16-bit cache (differential) or an 8-bit cache with
// scales: head_dim 64, 128 or 256, block sizes that are multiples of 16.
//
// Each warp owns a ring of stages; a stage is one unit, 16 tokens of one KV
// head (32 where a token row is at most 128 bytes): the K and V tiles (TMA
// boxes of 16 tokens, 128- or 64-byte swizzle) and, for 8 bits, their K and V
// scales (64-byte bulk copies), one mbarrier for all.  Per 16 tokens (tokens =
// M, columns = N = 8 per n-tile):
//     S[16 x 8] = K . Q^T,  O^T[D x 8] += V^T . P^T     (mma.sync m16n8k16)
// tcgen05 would need 64 or 128 rows of M per instruction: a decode column tile
// has 8 or 16 columns and every product here waits for memory, so the warp
// instruction on fragments in registers is the right size.
//
// 8-bit codes become fp16 in registers, exactly, between ldmatrix and the
// product (no staging pass):
//   * K: ldmatrix moves byte pairs, so thread (g, t) of a 16-byte chunk holds
//     dims 4t .. 4t + 3 of rows g and g + 8.  The order of a dot product's dims
//     is free: the query fragments take the same order.
//   * V: the transposing ldmatrix gives tokens (2t, 2t + 1) x dims (2g, 2g + 1)
//     in one word; the conversion picks the bytes of one dim, so M row g is dim
//     2g and row g + 8 dim 2g + 1.
//   * int8: byte ^ 0x80 under 0x64 is the fp16 1024 + 128 + x; subtract 1152.
//     e4m3: the conversion instruction.
// K's scale multiplies the score; V's scale multiplies the softmax weight.  The
// weights' reference is the running maximum of score + e, 2^e >= V's scale: a
// weight times its scale is then at most 1, so fp16 holds it whatever the
// scales are, and only one exponential is needed.  Weights are split into hi +
// lo 16-bit terms (2^-16 of the weight in bf16, 2^-22 in fp16; three terms,
// 2^-24, for fp32 queries over bf16).  fp32 queries are split the same way;
// columns of fp16 products are first scaled by a power of two so that their
// largest value is in [2^14, 2^15).
//
// The reference moves only when a stage's maximum exceeds it by more than 8
// (weights then reach at most 2^8, far inside fp16 and fp32): with the running
// maximum itself about half of the stages of a worker rescaled the
// accumulators.
#include <mutex>

#include <cudaTypedefs.h>

#include "attend_common.cuh"

namespace clover {

enum { KV_BF16 = 0, KV_F16 = 1, KV_I8 = 2, KV_E4M3 = 3 };

template <int KV> struct KvMma { using T = __half; };
template <> struct KvMma<KV_BF16> { using T = __nv_bfloat16; };

template <int KV, bool QF32, int D, int NT>
struct AttendGeom {
  static constexpr bool kEight = KV >= KV_I8;
  static constexpr int kEsz = kEight ? 1 : 2;
  static constexpr int kRow = D * kEsz;                  // bytes of a token row
  static constexpr int kSwz = kRow < 128 ? kRow : 128;   // bytes of a swizzled row
  static constexpr int kChunks = kRow / kSwz;            // TMA boxes per tile
  static constexpr int kTok = kRow <= 128 ? 32 : 16;     // tokens of a unit
  static constexpr int kTile = kTok * kRow;
  static constexpr int kTiles = 2 * kTile;               // K, V
  static constexpr int kScales = kEight ? 2 * kTok * 4 : 0;
  static constexpr int kQTerms = !QF32 ? 1 : KV == KV_BF16 ? 3 : 2;
  static constexpr int kPTerms = KV == KV_BF16 && QF32 ? 3 : 2;
  // Accumulators and query fragments decide how many warps an SM's registers
  // hold (4, 3 or 2 CTAs of 4 warps); the ring takes what shared memory that
  // leaves, at least two stages where they fit.
  static constexpr int kRegs = D / 16 * NT * (4 + 2 * kQTerms) + 64;
  static constexpr int kWantCtas = kRegs <= 128 ? 4 : kRegs <= 168 ? 3 : 2;
  static constexpr int kBudget = 216 * 1024;
  static constexpr int kStageB = kTiles + kScales;
  static constexpr int kCtas =
      kWantCtas == 4 && 4 * (kAttendWarps * 2 * kStageB + 1024) > kBudget ? 3 : kWantCtas;
  static constexpr int kFit = (kBudget / kCtas - 1024) / (kAttendWarps * kStageB);
  static constexpr int kStages = kFit < 1 ? 1 : kFit > 8 ? 8 : kFit;
  static constexpr int kWarpTiles = kStages * kTiles;
  static constexpr int kSmem = kAttendWarps * kStages * kStageB + 1024;
};

// Byte offset of 16-byte chunk c of tile row r (kSwz-byte rows, chunk groups
// of kSwz bytes one after the other).
template <int SWZ, int TOK>
__device__ __forceinline__ uint32_t attend_swz(int r, int c) {
  if (SWZ == 128) return (uint32_t)((c >> 3) * TOK * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
  return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
  return d;
}
__device__ __forceinline__ uint32_t hsub2_u(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t x) {
  uint32_t d;
  asm("{\n\t.reg .b16 l;\n\tcvt.u16.u32 l, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(d) : "r"(x));
  return d;
}

// Two fp16 pairs from four codes: bytes (0, 1), (2, 3), or with SPLIT the even
// and the odd bytes (0, 2), (1, 3).
template <int KV, bool SPLIT>
__device__ __forceinline__ void codes_to_f16(uint32_t x, uint32_t& lo, uint32_t& hi) {
  if (KV == KV_I8) {
    const uint32_t u = x ^ 0x80808080u;
    lo = hsub2_u(prmt(u, 0x64646464u, SPLIT ? 0x4240u : 0x4140u), 0x64806480u);
    hi = hsub2_u(prmt(u, 0x64646464u, SPLIT ? 0x4341u : 0x4342u), 0x64806480u);
  } else {
    const uint32_t y = SPLIT ? prmt(x, 0u, 0x3120u) : x;
    lo = e4m3x2_to_f16x2(y);
    hi = e4m3x2_to_f16x2(y >> 16);
  }
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
      : "memory");
}

// x0, x1 as TERMS 16-bit pairs whose sum is x to TERMS * 8 (bf16) or 11 bits.
template <typename T, int TERMS>
__device__ __forceinline__ void split_terms(float x0, float x1, uint32_t (&out)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    out[i] = Pack<T>::pack(x0, x1);
    const float2 h = Pack<T>::unpack(out[i]);
    x0 -= h.x;
    x1 -= h.y;
  }
}

// Columns of a warp: query fragments, accumulators, softmax state.  Lane
// (g, t) = (lane / 4, lane % 4) holds the query of column g of each n-tile and
// the accumulators of columns 2t and 2t + 1.
template <int KV, bool QF32, int D, int NT>
struct AttendCols {
  using G = AttendGeom<KV, QF32, D, NT>;
  uint32_t q[NT][D / 16][2][G::kQTerms];
  float acc[NT][D / 16][4];
  float m[NT][2], l[NT][2], sc[NT][2];  // sc: score scale in base 2
  int lim[NT][2];
  int min_lim;  // least limit of the chunk's columns
};

template <int KV, bool QF32, int D, int NT>
__device__ __forceinline__ void load_columns(const AttendArgs& a, const Cursor& cur, int kvh, int chunk,
                                             AttendCols<KV, QF32, D, NT>& c, int lane) {
  using G = AttendGeom<KV, QF32, D, NT>;
  using T = typename KvMma<KV>::T;
  constexpr bool kNorm = G::kEight || (KV == KV_F16 && QF32);
  const int half = D / 2;
  const int cap = cur.s.ctx;
  int least = cap;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const AttendCol ci =
        attend_col(a, cur.s.row0, cur.s.nq, kvh, chunk * (8 * NT) + nt * 8 + (lane >> 2));
    const int64_t qb = (int64_t)ci.row * a.q_stride + (int64_t)ci.head * D;
    float x[D / 16][4];
    uint32_t big = 0;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = G::kEight ? kk * 16 + (lane & 3) * 4 + i
                                : kk * 16 + (lane & 3) * 2 + (i & 1) + (i >> 1) * 8;
        const bool in = ci.valid && (a.maps == 1 || (d >= half) == (ci.map == 1));
        x[kk][i] = in ? attend_load_q(a, qb + d) : 0.f;
        big = max(big, abs_bits(x[kk][i]));
      }
    }
    float inv = 1.f;
    if (kNorm) {
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const int e = (int)(big >> 23);
      const int fe = e == 0 || e == 255 ? 127 : min(268 - e, 253);  // zero, Inf and NaN stay as they are
      const float f = __uint_as_float((uint32_t)fe << 23);
      inv = __uint_as_float((uint32_t)(254 - fe) << 23);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[kk][i] *= f;
    }
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      split_terms<T, G::kQTerms>(x[kk][0], x[kk][1], c.q[nt][kk][0]);
      split_terms<T, G::kQTerms>(x[kk][2], x[kk][3], c.q[nt][kk][1]);
    }
    // limits and score scales of columns 2t, 2t + 1 from the lanes that hold them
    int lim = ci.valid ? ci.lim : 0;
    if (lim > cap) {  // a row past its sequence's last row
      raise_status(a.status, CLOVER_B200_DEV_CTX_RANGE);
      lim = cap;
    }
    if (ci.valid) least = min(least, lim);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int src = ((lane & 3) * 2 + e) * 4;
      c.lim[nt][e] = __shfl_sync(0xffffffffu, lim, src);
      c.sc[nt][e] = a.scale_log2 * __shfl_sync(0xffffffffu, inv, src);
      c.m[nt][e] = -INFINITY;
      c.l[nt][e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      c.acc[nt][i][0] = c.acc[nt][i][1] = c.acc[nt][i][2] = c.acc[nt][i][3] = 0.f;
  }
  c.min_lim = __reduce_min_sync(0xffffffffu, least);
}

// Fragments of V^T, tokens 16 mt .. 16 mt + 15, for dims 16 i .. 16 i + 15 (8
// bits: 32 i .. 32 i + 31, two M tiles).
template <int KV, int SWZ, int TOK>
struct VFrag {
  static constexpr int kPer = KV >= KV_I8 ? 2 : 1;
  uint32_t a[kPer][4];
  __device__ __forceinline__ void load(uint32_t vs, int mt, int i, int lane) {
    const int grp = lane >> 3;
    if (KV >= KV_I8) {
      const int r = mt * 16 + (lane & 7) + (grp & 1) * 8;
      uint32_t x[4];
      ldsm_x4_trans(vs + attend_swz<SWZ, TOK>(r, 2 * i + (grp >> 1)), x[0], x[1], x[2], x[3]);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        codes_to_f16<KV, true>(x[2 * k], a[k][0], a[k][1]);
        codes_to_f16<KV, true>(x[2 * k + 1], a[k][2], a[k][3]);
      }
    } else {
      const int r = mt * 16 + (lane & 7) + (grp >> 1) * 8;
      ldsm_x4_trans(vs + attend_swz<SWZ, TOK>(r, 2 * i + (grp & 1)), a[0][0], a[0][1], a[0][2], a[0][3]);
    }
  }
};

// Zero V rows [r0, TOK) of a stage.
template <int ROW, int SWZ, int TOK>
__device__ __forceinline__ void zero_rows(uint8_t* v, int r0, int lane) {
  constexpr int kC = ROW / 16;
  for (int i = lane; i < (TOK - r0) * kC; i += 32)
    *reinterpret_cast<uint4*>(v + attend_swz<SWZ, TOK>(r0 + i / kC, i % kC)) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();  // before the next copy into this slot
  __syncwarp();
}

// Whether rows [r0, r1) of a V tile hold an infinity or NaN (codes: e4m3 NaN).
template <int KV, int ROW, int SWZ, int TOK>
__device__ __forceinline__ bool rows_nonfinite(const uint8_t* v, int r0, int r1, int lane) {
  constexpr int kC = ROW / 16;
  bool bad = false;
  for (int i = lane; i < (r1 - r0) * kC; i += 32) {
    const uint4 x = *reinterpret_cast<const uint4*>(v + attend_swz<SWZ, TOK>(r0 + i / kC, i % kC));
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (KV == KV_E4M3) {
#pragma unroll
        for (int s = 0; s < 32; s += 8) bad |= ((w[k] >> s) & 0x7fu) == 0x7fu;
      } else {
        const uint32_t e = KV == KV_BF16 ? 0x7f80u : 0x7c00u;
        bad |= (w[k] & e) == e || ((w[k] >> 16) & e) == e;
      }
    }
  }
  return __any_sync(0xffffffffu, bad);
}

// One stage of one warp.
template <int KV, bool QF32, int D, int NT>
__device__ __forceinline__ void attend_stage(uint32_t ks, uint32_t vs, uint8_t* vgen, const float* scales,
                                             int tok0, int nvalid, AttendCols<KV, QF32, D, NT>& c, int lane) {
  using G = AttendGeom<KV, QF32, D, NT>;
  using T = typename KvMma<KV>::T;
  using VF = VFrag<KV, G::kSwz, G::kTok>;
  constexpr int KK = D / 16, QT = G::kQTerms, PT = G::kPTerms, MT = G::kTok / 16;
  constexpr int CH = MT * NT == 1 ? 2 : 1;  // independent chains per score tile
  const int g = lane >> 2;

  // ---- S = K . Q^T, in base 2 with the scales, masked
  float s[MT][NT][4];
  float mx[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) mx[nt][0] = mx[nt][1] = -INFINITY;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float ch[NT][CH][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < CH; ++k) ch[nt][k][0] = ch[nt][k][1] = ch[nt][k][2] = ch[nt][k][3] = 0.f;
    const int r = mt * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
    if (G::kEight) {
#pragma unroll
      for (int i = 0; i < KK / 2; ++i) {
        uint32_t x[4];
        ldsm_x4(ks + attend_swz<G::kSwz, G::kTok>(r, 2 * i + (lane >> 4)), x[0], x[1], x[2], x[3]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t a0, a1, a2, a3;
          codes_to_f16<KV, false>(x[2 * k], a0, a2);
          codes_to_f16<KV, false>(x[2 * k + 1], a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < QT; ++q)
              MmaOp<T>::run(ch[nt][k % CH], a0, a1, a2, a3, c.q[nt][2 * i + k][0][q], c.q[nt][2 * i + k][1][q]);
        }
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        uint32_t a0, a1, a2, a3;
        ldsm_x4(ks + attend_swz<G::kSwz, G::kTok>(r, kk * 2 + (lane >> 4)), a0, a1, a2, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int q = 0; q < QT; ++q)
            MmaOp<T>::run(ch[nt][kk % CH], a0, a1, a2, a3, c.q[nt][kk][0][q], c.q[nt][kk][1][q]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = mt * 16 + g + 8 * h, t = tok0 + row;
      float ksc = 1.f, ve = 0.f;
      if (G::kEight) {
        ksc = scales[row];
        // 2^ve >= V's scale; scales below 2^-110 count as that (2^-107 is the least stored)
        ve = fmaxf((float)((int)(__float_as_uint(scales[G::kTok + row]) >> 23 & 255u) - 126), -110.f);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float raw = ch[nt][0][2 * h + e];
          if (CH == 2) raw += ch[nt][CH - 1][2 * h + e];
          raw *= c.sc[nt][e];
          const float x = t < c.lim[nt][e] ? (G::kEight ? raw * ksc : raw) : -INFINITY;
          s[mt][nt][2 * h + e] = x;
          mx[nt][e] = fmaxf(mx[nt][e], G::kEight ? x + ve : x);
        }
    }
  }

  // ---- the reference: move it when a column outgrows it
  bool moved = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1)
        mx[nt][e] = fmaxf(mx[nt][e], __shfl_xor_sync(0xffffffffu, mx[nt][e], off));
      moved |= mx[nt][e] > c.m[nt][e] + 8.f;
    }
  if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float nm = fmaxf(c.m[nt][e], mx[nt][e]);
        const float al = fast_exp2(c.m[nt][e] - (nm == -INFINITY ? 0.f : nm));
        c.m[nt][e] = nm;
        c.l[nt][e] *= al;
#pragma unroll
        for (int i = 0; i < KK; ++i) {
          c.acc[nt][i][e] *= al;
          c.acc[nt][i][2 + e] *= al;
        }
      }
  }

  // Rows that some column does not see: past the context they are zeroed; a
  // later token's infinity or NaN must not meet the zero weight of an earlier
  // row (multi-token rows), so such a stage takes its columns limit by limit,
  // zeroing rows as it goes.
  bool plain = true;
  if (KV != KV_I8 && tok0 + G::kTok > c.min_lim) {
    if (nvalid < G::kTok) zero_rows<G::kRow, G::kSwz, G::kTok>(vgen, nvalid, lane);
    const int lo = max(0, c.min_lim - tok0), hi = min(nvalid, G::kTok);
    if (lo < hi && rows_nonfinite<KV, G::kRow, G::kSwz, G::kTok>(vgen, lo, hi, lane)) plain = false;
  }

  // ---- weights, split and transposed; O^T += V^T . P^T
  uint32_t pt[MT][NT][2][PT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = mt * 16 + g + 8 * h, t = tok0 + row;
      const float vsc = G::kEight ? scales[G::kTok + row] : 1.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p0 = fast_exp2(s[mt][nt][2 * h] - (c.m[nt][0] == -INFINITY ? 0.f : c.m[nt][0]));
        float p1 = fast_exp2(s[mt][nt][2 * h + 1] - (c.m[nt][1] == -INFINITY ? 0.f : c.m[nt][1]));
        c.l[nt][0] += p0;
        c.l[nt][1] += p1;
        if (G::kEight) {  // (a masked token's scale may be anything)
          p0 = t < c.lim[nt][0] ? p0 * vsc : 0.f;
          p1 = t < c.lim[nt][1] ? p1 * vsc : 0.f;
        }
        split_terms<T, PT>(p0, p1, pt[mt][nt][h]);
#pragma unroll
        for (int k = 0; k < PT; ++k) pt[mt][nt][h][k] = movm_trans(pt[mt][nt][h][k]);
      }
    }
    if (plain) {
#pragma unroll
      for (int i = 0; i < KK / VF::kPer; ++i) {
        VF v;
        v.load(vs, mt, i, lane);
#pragma unroll
        for (int k = 0; k < VF::kPer; ++k)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < PT; ++q)
              MmaOp<T>::run(c.acc[nt][i * VF::kPer + k], v.a[k][0], v.a[k][1], v.a[k][2], v.a[k][3],
                            pt[mt][nt][0][q], pt[mt][nt][1][q]);
      }
    }
  }
  if (plain) return;
  for (int below = 0x7fffffff;;) {
    int top = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (c.lim[nt][e] < below) top = max(top, c.lim[nt][e]);
    top = __reduce_max_sync(0xffffffffu, top);
    if (top <= tok0) break;
    if (top - tok0 < G::kTok) zero_rows<G::kRow, G::kSwz, G::kTok>(vgen, top - tok0, lane);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll 1
      for (int i = 0; i < KK / VF::kPer; ++i) {
        VF v;
        v.load(vs, mt, i, lane);
#pragma unroll
        for (int k = 0; k < VF::kPer; ++k)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = 0; q < PT; ++q)
              MmaOp<T>::run(x, v.a[k][0], v.a[k][1], v.a[k][2], v.a[k][3], pt[mt][nt][0][q], pt[mt][nt][1][q]);
            // (constant indices: the accumulators stay in registers)
#pragma unroll
            for (int j = 0; j < KK; ++j) {
              if (j != i * VF::kPer + k) continue;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (c.lim[nt][e & 1] == top) c.acc[nt][j][e] += x[e];
            }
          }
      }
    below = top;
  }
}

// Fused append: the new tokens of the cursor's sequence that lie in its unit,
// for KV head kvh, written before the unit is copied (slot[u]: first cache slot
// of the unit's u-th 16 tokens).
template <int KV, int D, int SUBS>
__device__ __forceinline__ void append_unit(const AttendArgs& a, const Cursor& cur, int kvh,
                                            const int (&slot)[SUBS], int lane) {
  const int tok0 = cur.jj * SUBS * kUnitTok;
  for (int j = 0; j < cur.s.nq; ++j) {
    const int r = cur.s.row0 + j;
    const int rel = __ldg(a.ctx + r) - 1 - tok0;
    if (rel < 0 || rel >= SUBS * kUnitTok || rel + tok0 >= cur.s.ctx) continue;
    const int base = SUBS == 1 || rel < kUnitTok ? slot[0] : slot[SUBS - 1];
    const int64_t at = base + (rel & (kUnitTok - 1));
    const int64_t row = (at * a.hkv + kvh) * D, src = (int64_t)r * a.new_stride + (int64_t)kvh * D;
    if (KV >= KV_I8) {
      uint8_t* kd = static_cast<uint8_t*>(const_cast<void*>(a.kc)) + row;
      uint8_t* vd = static_cast<uint8_t*>(const_cast<void*>(a.vc)) + row;
      const float ks = encode_row_any<KV == KV_E4M3>(a.new_dtype, a.k_new, src, kd, D, lane);
      const float vs = encode_row_any<KV == KV_E4M3>(a.new_dtype, a.v_new, src, vd, D, lane);
      const int64_t blk = at / a.bs, si = (blk * a.hkv + kvh) * a.bs + (at - blk * a.bs);
      if (lane == 0) {
        const_cast<float*>(a.ks)[si] = ks;
        const_cast<float*>(a.vs)[si] = vs;
      }
    } else {
      uint16_t* kd = static_cast<uint16_t*>(const_cast<void*>(a.kc)) + row;
      uint16_t* vd = static_cast<uint16_t*>(const_cast<void*>(a.vc)) + row;
      for (int d = lane; d < D; d += 32) {
        kd[d] = static_cast<const uint16_t*>(a.k_new)[src + d];
        vd[d] = static_cast<const uint16_t*>(a.v_new)[src + d];
      }
    }
  }
  fence_proxy_async_global();  // the copies read what was just written
  __syncwarp();
}

template <int KV, bool QF32, int D, int NT>
__global__ void __launch_bounds__(kAttendThreads, AttendGeom<KV, QF32, D, NT>::kCtas)
attend_mma_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const AttendArgs a) {
  using G = AttendGeom<KV, QF32, D, NT>;
  constexpr int STAGES = G::kStages;
  constexpr int KK = D / 16;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[kAttendWarps * STAGES];
  __shared__ AttendPlan plan;
  __shared__ int s_stop;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wid = blockIdx.x * kAttendWarps + warp;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kAttendWarps * STAGES; ++i) mbar_init(smem_addr(&bars[i]), 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  pdl_wait();
  // after a bounded wait gave up anywhere, later launches stop at once
  if (threadIdx.x == 0)
    s_stop = a.status != nullptr && (*(volatile int32_t*)a.status & CLOVER_B200_DEV_TIMEOUT);
  __syncthreads();
  if (s_stop) return;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + warp * G::kWarpTiles;
  float* scales = reinterpret_cast<float*>(smem + kAttendWarps * G::kWarpTiles) + warp * STAGES * (G::kScales / 4);
  const uint32_t ring_s = smem_addr(ring), scales_s = smem_addr(scales), bar0 = smem_addr(&bars[warp * STAGES]);
  const int hcmax = a.hkv * a.chunks;

  int per = 1;
  Cursor pc;  // the copies' position
  bool more;
  if (a.whole) {
    // rows of empty sequences have no unit: their zeros are written here
    for (int64_t sg = wid; sg < (int64_t)a.n_seqs * hcmax; sg += a.workers) {
      const int b = (int)sg / hcmax, h = (int)sg - b * hcmax;
      const SeqInfo s = seq_info(a, b);
      if (h == 0 && lane == 0) attend_check_seq(a, s);
      if (h >= s.hc || s.n > 0) continue;
      const int nch = s.hc / a.hkv, kvh = h / nch;
      for (int c = 0; c < 8 * NT; ++c) {
        const AttendCol ci = attend_col(a, s.row0, s.nq, kvh, (h - kvh * nch) * (8 * NT) + c);
        if (!ci.valid || ci.map == 1) continue;
        for (int d = lane; d < D; d += 32)
          attend_store(a, (int64_t)ci.row * a.out_stride + (int64_t)ci.head * D + d, 0.f);
      }
    }
    more = pc.seek(a, wid);
  } else {
    int total;
    per = attend_plan(a, plan, total);
    pdl_trigger();
    const int64_t u0 = (int64_t)wid * per;
    more = u0 < total && plan.start[warp][0] >= 0;
    if (more)
      pc.start(a, plan.start[warp][0], plan.start[warp][1], plan.start[warp][2],
               (int)min((int64_t)per, total - u0));
  }
  if (!more) return;
  Cursor cc = pc;  // the products' position

  // ---- copies.  Block ids of the sequence are held 32 at a time (lane i:
  // block id_base + i); block and sub count 16-token steps of the segment.
  constexpr int SUBS = G::kTok / kUnitTok;
  const int upb = a.bs / kUnitTok;  // 16-token steps per block
  int ids = 0, id_base = -64, p_b = -1, p_h = -1, p_kvh = 0, blk_i = 0, sub = 0, first_new = 0;
  int p_st = 0;
  auto issue = [&]() {
    if (pc.b != p_b || pc.h != p_h) {
      if (pc.b != p_b) id_base = -64;
      p_b = pc.b;
      p_h = pc.h;
      p_kvh = pc.h / (pc.s.hc / a.hkv);
      const int at = pc.jj * SUBS;
      blk_i = at / upb;
      sub = at - blk_i * upb;
      if (a.k_new != nullptr) first_new = __ldg(a.ctx + pc.s.row0) - 1;
    }
    const int n_sub = (pc.s.ctx + kUnitTok - 1) / kUnitTok - pc.jj * SUBS;  // steps left
    if (blk_i < id_base || blk_i + SUBS > id_base + 32) {
      id_base = blk_i;
      const int trow = a.seq_rows ? __ldg(a.seq_rows + pc.b) : pc.b;
      const int nblk = (pc.s.ctx + a.bs - 1) / a.bs;
      ids = 0;
      if (blk_i + lane < nblk) {
        ids = blk_i + lane < a.table_stride
                  ? __ldg(a.tables + (int64_t)trow * a.table_stride + blk_i + lane) : -1;
        if (ids < 0 || ids >= a.num_blocks) {
          raise_status(a.status, CLOVER_B200_DEV_BAD_BLOCK);
          ids = 0;  // keep the pipeline well-formed; the output is flagged
        }
      }
    }
    int slot[SUBS];  // first cache slot of each 16-token step
    int64_t sc_at[SUBS];
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      const int blk = __shfl_sync(0xffffffffu, ids, blk_i - id_base);
      slot[u] = blk * a.bs + sub * kUnitTok;
      sc_at[u] = ((int64_t)blk * a.hkv + p_kvh) * a.bs + sub * kUnitTok;
      if (++sub == upb) {
        sub = 0;
        ++blk_i;
      }
    }
    if (a.k_new != nullptr && (pc.jj + 1) * G::kTok > first_new)
      append_unit<KV, D>(a, pc, p_kvh, slot, lane);
    const int subs = n_sub < SUBS ? n_sub : SUBS;
    const uint32_t bar = bar0 + p_st * 8;
    const uint32_t kd = ring_s + p_st * G::kTiles, vd = kd + G::kTile;
    if (lane == 0) mbar_arrive_expect_tx(bar, subs * (G::kStageB / SUBS));
    __syncwarp();
    // one copy per lane: (step, K or V, chunk), then the scales
    constexpr int kCopies = 2 * G::kChunks;
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      if (u >= subs) break;
      const int i = lane - u * (kCopies + 2);
      if (i >= 0 && i < kCopies) {
        const int ch = i >> 1;
        tma_load_3d((i & 1 ? vd : kd) + (ch * G::kTok + u * kUnitTok) * G::kSwz, i & 1 ? &tmV : &tmK,
                    ch * (G::kSwz / G::kEsz), p_kvh, slot[u], bar);
      }
      if (G::kEight && (i == kCopies || i == kCopies + 1)) {
        const int v = i - kCopies;
        bulk_load(scales_s + p_st * G::kScales + (v * G::kTok + u * kUnitTok) * 4, (v ? a.vs : a.ks) + sc_at[u],
                  kUnitTok * 4, bar);
      }
    }
    p_st = p_st + 1 == STAGES ? 0 : p_st + 1;
  };

  int issued = 0;
  while (issued < STAGES && more) {
    issue();
    ++issued;
    more = pc.next(a);
  }

  AttendCols<KV, QF32, D, NT> c;
  int cur_b = -1, cur_h = -1, first_jj = 0, last_jj = 0, kvh = 0, chunk = 0;
  Cursor seg = cc;  // the segment of the columns in registers

  auto finish = [&]() {
    const bool whole = a.whole || (first_jj == 0 && last_jj == seg.s.n - 1);
    const int64_t slot = 2 * (int64_t)wid + (first_jj == 0 ? 1 : 0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        c.l[nt][0] += __shfl_xor_sync(0xffffffffu, c.l[nt][0], off);
        c.l[nt][1] += __shfl_xor_sync(0xffffffffu, c.l[nt][1], off);
      }
      const int g = lane >> 2, c0 = nt * 8 + (lane & 3) * 2;
      const int d0 = G::kEight ? 2 * g : g, dh = G::kEight ? 1 : 8;  // dims of M rows g, g + 8
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int64_t at = slot * (8 * NT) + c0 + e;
          float* po = a.part + at * D;
#pragma unroll
          for (int i = 0; i < KK; ++i) {
            if (G::kEight) {
              *reinterpret_cast<float2*>(po + i * 16 + d0) = make_float2(c.acc[nt][i][e], c.acc[nt][i][2 + e]);
            } else {
              po[i * 16 + d0] = c.acc[nt][i][e];
              po[i * 16 + d0 + dh] = c.acc[nt][i][2 + e];
            }
          }
          if (lane < 4) a.part_ml[at] = make_float2(c.m[nt][e], c.l[nt][e]);
        }
        continue;
      }
      if (a.maps == 1) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const AttendCol ci = attend_col(a, seg.s.row0, seg.s.nq, kvh, chunk * (8 * NT) + c0 + e);
          if (!ci.valid) continue;
          const bool any = c.lim[nt][e] > 0;
          const float inv = attend_inv(c.l[nt][e], c.lim[nt][e]);
          const int64_t ob = (int64_t)ci.row * a.out_stride + (int64_t)ci.head * D + d0;
#pragma unroll
          for (int i = 0; i < KK; ++i) {
            attend_store(a, ob + i * 16, any ? c.acc[nt][i][e] * inv : 0.f);
            attend_store(a, ob + i * 16 + dh, any ? c.acc[nt][i][2 + e] * inv : 0.f);
          }
        }
      } else {
        // columns 2t and 2t + 1 are the two maps of one head
        const AttendCol ci = attend_col(a, seg.s.row0, seg.s.nq, kvh, chunk * (8 * NT) + c0);
        const bool any = c.lim[nt][0] > 0;
        const float lam = ci.valid ? a.lam[ci.head] : 0.f;
        const float i0 = attend_inv(c.l[nt][0], c.lim[nt][0]), i1 = attend_inv(c.l[nt][1], c.lim[nt][1]);
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < KK; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float o = any ? diff_value(c.acc[nt][i][2 * h] * i0, c.acc[nt][i][2 * h + 1] * i1, lam) : 0.f;
            c.acc[nt][i][2 * h] = o;
            sq = fmaf(o, o, sq);
          }
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
        if (!ci.valid) continue;
        const int64_t ob = (int64_t)ci.row * a.out_stride + (int64_t)ci.head * D;
        const float r = a.norm_w != nullptr ? rsqrtf(sq / D + a.eps) * a.out_scale : 1.f;
#pragma unroll
        for (int i = 0; i < KK; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int d = i * 16 + d0 + h * dh;
            const float w = a.norm_w != nullptr ? a.norm_w[d] : 1.f;
            attend_store(a, ob + d, c.acc[nt][i][2 * h] * (r * w));
          }
        }
      }
    }
    if (!a.whole && first_jj == 0 && lane == 0) {
      const int fw = seg.seg0 / per;
      a.seg[(int64_t)seg.b * hcmax + seg.h] = make_int2(fw, (seg.seg0 + seg.s.n - 1) / per - fw + 1);
    }
  };

  bool timed_out = false;
  int k = 0, st = 0;
  uint32_t parity = 0;
  for (;; ++k) {
    if (cc.b != cur_b || cc.h != cur_h) {
      if (cur_b >= 0) finish();
      cur_b = cc.b;
      cur_h = cc.h;
      seg = cc;
      first_jj = cc.jj;
      const int nch = cc.s.hc / a.hkv;
      kvh = cc.h / nch;
      chunk = cc.h - kvh * nch;
      load_columns<KV, QF32, D, NT>(a, cc, kvh, chunk, c, lane);
    }
    if (!mbar_wait_bounded(bar0 + st * 8, parity, a.wait_ns)) {
      timed_out = true;
      break;
    }
    last_jj = cc.jj;
    const int tok0 = cc.jj * G::kTok;
    const uint32_t ks = ring_s + st * G::kTiles;
    attend_stage<KV, QF32, D, NT>(ks, ks + G::kTile, ring + st * G::kTiles + G::kTile,
                                  scales + st * (G::kScales / 4), tok0, cc.s.ctx - tok0, c, lane);
    __syncwarp();
    if (more) {
      issue();
      ++issued;
      more = pc.next(a);
    }
    if (++st == STAGES) {
      st = 0;
      parity ^= 1;
    }
    if (!cc.next(a)) break;
  }
  if (timed_out) {
    // drain this warp's copies still in flight (bounded) before giving up
    for (int j = k; j < issued; ++j)
      mbar_wait_bounded(bar0 + (j % STAGES) * 8, (j / STAGES) & 1, kWaitLimitNs);
    if (lane == 0) raise_status(a.status, CLOVER_B200_DEV_TIMEOUT);
    return;
  }
  finish();
}

// ------------------------------------------------------------------ host side
static std::mutex g_attend_mu;

// Tiled map of a cache [slots, H, D]: boxes of 16 tokens x one head x one
// swizzled row.  The last 64 maps are kept by everything that defines them.
static int attend_tmap(const void* ptr, int esz, int D, int H, int64_t slots, CUtensorMap* out) {
  struct Entry {
    const void* ptr;
    int esz, D, H;
    int64_t slots;
    CUtensorMap map;
  };
  static Entry cache[64];
  static int used = 0, next = 0;
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  std::lock_guard<std::mutex> lock(g_attend_mu);
  for (int i = 0; i < used; ++i) {
    const Entry& e = cache[i];
    if (e.ptr == ptr && e.esz == esz && e.D == D && e.H == H && e.slots == slots) {
      *out = e.map;
      return CLOVER_B200_OK;
    }
  }
  if (encode == nullptr) {
    cudaDriverEntryPointQueryResult q;
    void* fn = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess || fn == nullptr)
      return set_error(CLOVER_B200_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }
  const int row = D * esz, swz = row < 128 ? row : 128;
  Entry e{ptr, esz, D, H, slots, {}};
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)slots};
  const cuuint64_t strides[2] = {(cuuint64_t)row, (cuuint64_t)H * row};
  const cuuint32_t box[3] = {(cuuint32_t)(swz / esz), 1, (cuuint32_t)kUnitTok};
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult r = encode(&e.map, esz == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3,
                            const_cast<void*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            swz == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                            // a token row at most: its neighbours are other heads' rows
                            row >= 256   ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                            : row == 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B
                                         : CU_TENSOR_MAP_L2_PROMOTION_L2_64B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(CLOVER_B200_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  cache[next] = e;
  next = (next + 1) % 64;
  if (used < 64) ++used;
  *out = e.map;
  return CLOVER_B200_OK;
}

template <int KV, bool QF32, int D, int NT>
static int mma_launch(const AttendArgs* a, cudaStream_t s, int* grid) {
  using G = AttendGeom<KV, QF32, D, NT>;
  auto kern = attend_mma_kernel<KV, QF32, D, NT>;
  static int per_sm[64] = {0}, sms[64] = {0};
  int dev = 0;
  int rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  if (dev >= 64) return set_error(CLOVER_B200_ERR_UNSUPPORTED, "attend: device ordinal %d", dev);
  {
    std::lock_guard<std::mutex> lock(g_attend_mu);
    if (per_sm[dev] == 0) {
      rc = set_smem(kern, G::kSmem);
      if (rc) return rc;
      int n = 0, m = 0;
      rc = check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kAttendThreads, G::kSmem),
                      "attend occupancy");
      if (rc) return rc;
      rc = check_cuda(cudaDeviceGetAttribute(&m, cudaDevAttrMultiProcessorCount, dev), "attend SMs");
      if (rc) return rc;
      if (n < 1) return set_error(CLOVER_B200_ERR_UNSUPPORTED, "attend: kernel does not fit on an SM");
      sms[dev] = m;
      per_sm[dev] = n;
    }
  }
  if (a == nullptr) {
    *grid = per_sm[dev] * sms[dev];
    return CLOVER_B200_OK;
  }
  CUtensorMap tk, tv;
  rc = attend_tmap(a->kc, G::kEsz, D, a->hkv, a->num_blocks * a->bs, &tk);
  if (rc) return rc;
  rc = attend_tmap(a->vc, G::kEsz, D, a->hkv, a->num_blocks * a->bs, &tv);
  if (rc) return rc;
  return check_cuda(launch_pdl(kern, dim3(a->workers / kAttendWarps), dim3(kAttendThreads), G::kSmem, s, tk, tv, *a),
                    "attend_mma launch");
}

template <int KV, bool QF32>
static int mma_shape(int cols, const AttendArgs* a, int D, cudaStream_t s, int* grid) {
  const bool two = cols > kMmaCols;
  switch (D) {
    case 64: return two ? mma_launch<KV, QF32, 64, 2>(a, s, grid) : mma_launch<KV, QF32, 64, 1>(a, s, grid);
    case 128: return two ? mma_launch<KV, QF32, 128, 2>(a, s, grid) : mma_launch<KV, QF32, 128, 1>(a, s, grid);
    default: return mma_launch<KV, QF32, 256, 1>(a, s, grid);
  }
}

bool attend_mma_supported(int kv_dtype, int q_dtype, int D, int bs) {
  return (D == 64 || D == 128 || D == 256) && bs % kUnitTok == 0 && kv_dtype != CLOVER_B200_F32;
}

int attend_mma_unit_log2(int kv_dtype, int D) {
  const bool eight = kv_dtype == CLOVER_B200_INT8 || kv_dtype == CLOVER_B200_FP8_E4M3;
  return D * (eight ? 1 : 2) <= 128 ? 5 : 4;
}

int attend_mma(int kv_dtype, int q_dtype, int cols, const AttendArgs* a, int D, cudaStream_t s, int* grid) {
  const bool f32 = q_dtype == CLOVER_B200_F32;
  switch (kv_dtype) {
    case CLOVER_B200_BF16: return f32 ? mma_shape<KV_BF16, true>(cols, a, D, s, grid) : mma_shape<KV_BF16, false>(cols, a, D, s, grid);
    case CLOVER_B200_F16: return f32 ? mma_shape<KV_F16, true>(cols, a, D, s, grid) : mma_shape<KV_F16, false>(cols, a, D, s, grid);
    case CLOVER_B200_INT8: return f32 ? mma_shape<KV_I8, true>(cols, a, D, s, grid) : mma_shape<KV_I8, false>(cols, a, D, s, grid);
    default: return f32 ? mma_shape<KV_E4M3, true>(cols, a, D, s, grid) : mma_shape<KV_E4M3, false>(cols, a, D, s, grid);
  }
}

}  // namespace clover
