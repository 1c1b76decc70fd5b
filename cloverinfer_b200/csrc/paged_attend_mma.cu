// Tensor-core decode over a 16-bit cache (differential) or an 8-bit cache with
// scales: head_dim 64, 128 or 256, block sizes that are multiples of 16.
//
// One CTA per SM.  A ring of stages belongs to CW warps ("column warps": CW = 1
// for up to 8 columns of a chunk, 2 for 16), which read the same stages, each
// for its own 8 columns; a ring with its warps is a worker of
// attend_common.cuh.  A stage is one unit, 16 tokens of one KV head (32 where a
// token row is at most 128 bytes): the K and V tiles (TMA boxes of 16 tokens,
// 128- or 64-byte swizzle) and, for 8 bits, their scales (16 bytes per lane,
// cp.async), all completing on one mbarrier.  The ring's first warp refills a
// stage when it is done with it.  Two other ways were measured at 8 x 32k
// tokens, e4m3: one warp that issues for all rings (165 us with the scales as
// bulk copies, 179 as here: its own instructions are the limit), and the scales
// as bulk copies (half of all copies for 6 % of the bytes).
// Per 16 tokens (tokens = M, columns = N = 8):
//     S[16 x 8] = K . Q^T,  O^T[D x 8] += V^T . P^T     (mma.sync m16n8k16)
// tcgen05 would need 64 or 128 rows of M per instruction: a decode column tile
// has 8 columns and every product here waits for memory, so the warp
// instruction on fragments in registers is the right size.
//
// 8-bit codes become fp16 in registers, exactly, between ldmatrix and the
// product (no staging pass):
//   * K: ldmatrix moves byte pairs, so thread (g, t) of a 16-byte chunk holds
//     dims 4t .. 4t + 3 of rows g and g + 8.  The order of a dot product's dims
//     is free: the query fragments take the order the conversion gives.
//   * V: the transposing ldmatrix gives tokens (2t, 2t + 1) x dims (2g, 2g + 1)
//     in one word; the conversion picks the bytes of one dim, so M row g is dim
//     2g and row g + 8 dim 2g + 1.
//   * int8: byte ^ 0x80 under 0x64 is the fp16 1024 + 128 + x; subtract 1152.
//     (K's codes left 1152 high, with that times the query's sum taken off each
//     score, save two subtractions per four codes: 121.2 against 123.6 us on 64
//     ragged requests of 1-4 rows.  But the partial sums are then about
//     1152 |sum q| and round accordingly: 128 dims of mean and deviation 8 put
//     scores off by up to 5e-4, against 6e-6 as here.)
//     e4m3: the conversion instruction.
// K's scale multiplies the score; V's scale multiplies the softmax weight.  The
// weights' reference is a bound of score + e, 2^e >= V's scale: a weight times
// its scale is then bounded, so fp16 does not overflow whatever the scales are,
// and only one exponential is needed.  Weights are split into two 16-bit terms:
// 2^-16 of the weight in bf16 (three terms, 2^-24, for fp32 queries); 2^-22 in
// fp16 down to 2^-3, and half of fp16's least step, 2^-25, below.  fp16 weights
// are therefore multiplied by 2^12 before they are rounded (and the result by
// 2^-12): what is lost of a small one is at most 2^-37 of the largest.  (Without
// it 40000 tokens 18 nats below one with a V row of its own lost all that shared
// its piece, 9 to 23 % of their sum.  The sum of the weights is in fp32.  The
// factor is not part of the reference: 12 more in the exponential's argument
// would round by 2^-21 of every weight.)  fp32 queries are split the same way
// (2^-22 of a value over fp16 products, 2^-24 over bf16; a third fp16 term costs
// 8 to 15 % and changes none of the errors measured); columns of fp16 products
// are first scaled by a power of two so that their largest value is in
// [2^14, 2^15).
//
// The reference moves only when a weight exceeds it by 2^3 (fp16: 2^15 with the
// factor) or 2^8 (bf16).  With the running maximum itself about half of the
// stages of a worker rescaled the accumulators, and every stage took the columns'
// maxima over the lanes; 2^8, 2^5 and 2^3 of room measure alike (64 ragged
// requests 124.0, 124.1, 124.1 us; scores five times as wide 124.4, 124.6,
// 125.1).
#include <mutex>

#include <cudaTypedefs.h>

#include "attend_common.cuh"

namespace clover {

enum { KV_BF16 = 0, KV_F16 = 1, KV_I8 = 2, KV_E4M3 = 3 };

template <int KV> struct KvMma { using T = __half; };
template <> struct KvMma<KV_BF16> { using T = __nv_bfloat16; };

constexpr bool attend_fits(int rings, int stage, int budget) { return rings * 2 * stage <= budget; }

template <int KV, bool QF32, int D, int CW_>
struct AttendGeom {
  static constexpr int CW = CW_;
  static constexpr bool kEight = KV >= KV_I8;
  static constexpr int kEsz = kEight ? 1 : 2;
  static constexpr int kRow = D * kEsz;                  // bytes of a token row
  static constexpr int kSwz = kRow < 128 ? kRow : 128;   // bytes of a swizzled row
  static constexpr int kChunks = kRow / kSwz;            // TMA boxes per 16 tokens
  static constexpr int kTok = kRow <= 128 ? 32 : 16;     // tokens of a unit
  static constexpr int kSubs = kTok / kUnitTok;
  static constexpr int kTile = kTok * kRow;
  static constexpr int kTiles = 2 * kTile;               // K, V
  static constexpr int kScales = kEight ? 2 * kTok * 4 : 0;
  static constexpr int kStageB = kTiles + kScales;
  static constexpr int kQTerms = !QF32 ? 1 : KV == KV_BF16 ? 3 : 2;
  static constexpr int kPTerms = KV == KV_BF16 && QF32 ? 3 : 2;
  // What a weight is multiplied by before it is rounded, and the weight (before
  // that) that makes the reference move.
  static constexpr float kUp = KV == KV_BF16 ? 1.f : 4096.f;
  static constexpr float kMaxWeight = KV == KV_BF16 ? 256.f : 8.f;
  // Warps: 16, 12 or 8 (128, 168 or 255 registers each), as many as hold
  // accumulators, query fragments and about 80 more, with rings at least two
  // stages deep; 6 where 8 such rings do not fit (head_dim 256 in 16 bits).
  static constexpr int kRegs = D / 4 + D / 8 * kQTerms + (kEight ? 92 : 80);
  static constexpr int kBudget = 232448 - 1024 - 1024;  // an SM's shared memory, less alignment and barriers
  static constexpr int kWarps = kRegs <= 128 && attend_fits(16 / CW, kStageB, kBudget)   ? 16
                                : kRegs <= 180 && attend_fits(12 / CW, kStageB, kBudget) ? 12
                                : attend_fits(8 / CW, kStageB, kBudget)                  ? 8
                                                                                         : 6;
  static constexpr int kRings = kWarps / CW;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kFit = kBudget / (kRings * kStageB);
  static constexpr int kStages = kFit < 1 ? 1 : kFit > 8 ? 8 : kFit;
  static constexpr int kRingTiles = kStages * kTiles;
  static constexpr int kSmem = kRings * kStages * kStageB + 1024;
};

// Byte offset of 16-byte chunk c of tile row r (SWZ-byte rows, chunk groups of
// SWZ bytes one after the other).
template <int SWZ, int TOK>
__device__ __forceinline__ uint32_t attend_swz(int r, int c) {
  if (SWZ == 128) return (uint32_t)((c >> 3) * TOK * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
  return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// attend_swz(r, c + 2 i) from the address of attend_swz(r, c), c in {0, 1}: the
// swizzle is an exclusive or of the chunk's low bits, so an even step is one
// instruction (tile rows start on a multiple of the swizzled row).
template <int SWZ, int TOK>
__device__ __forceinline__ uint32_t attend_swz_step(uint32_t at, int i) {
  constexpr int kGroup = SWZ / 16;  // chunks of a swizzled row
  return (at ^ (uint32_t)((2 * i % kGroup) << 4)) + (uint32_t)(2 * i / kGroup * TOK * SWZ);
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
// Two fp16 pairs from four codes, in the order bytes (0, 2), (1, 3).
template <int KV>
__device__ __forceinline__ void codes_to_f16(uint32_t x, uint32_t& lo, uint32_t& hi) {
  if (KV == KV_I8) {
    const uint32_t u = x ^ 0x80808080u;
    lo = prmt(u, 0x64646464u, 0x4240u);
    hi = prmt(u, 0x64646464u, 0x4341u);
    lo = hsub2_u(lo, 0x64806480u);
    hi = hsub2_u(hi, 0x64806480u);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(prmt(x, 0u, 0x3120u)));
  }
}
// Two fp16 pairs of e4m3 codes in byte order, (0, 1), (2, 3).
__device__ __forceinline__ void e4m3_to_f16(uint32_t x, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(x));
}
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// One arrival on the barrier when this thread's copy16_async calls so far have landed.
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
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

// A reference below every score (finite, so that differences to -inf stay
// -inf): the weights of a column that has seen nothing are 2^-inf.
constexpr float kNoRef = -1e30f;

// V scales under 2^-80 count as that in the reference (a zero row's is 0, the
// least stored 2^-109), though the weight takes them as they are: a softmax
// weight is then at most 2^(3 + 80), and the sum of 2^31 of them finite.
constexpr float kLeastScale = 8.271806125530277e-25f;

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ------------------------------------------------------------------ consumer
// Columns of a warp: query fragments, accumulators, softmax state.  Lane
// (g, t) = (lane / 4, lane % 4) holds the query of column g and the
// accumulators of columns 2t and 2t + 1.
template <int KV, bool QF32, int D, int CW>
struct AttendCols {
  using G = AttendGeom<KV, QF32, D, CW>;
  uint32_t q[D / 16][2][G::kQTerms];
  float acc[D / 16][4];
  float m[2], l[2], sc[2];  // sc: score scale in base 2
  int lim[2];
  int min_lim;  // least limit of the warp's columns
};

// First of the warp's columns within the (sequence, KV head): chunk * cols + 8 cw.
template <int KV, bool QF32, int D, int CW>
__device__ __forceinline__ void load_columns(const AttendArgs& a, const Cursor& cur, int kvh, int col0,
                                             AttendCols<KV, QF32, D, CW>& c, int lane) {
  using G = AttendGeom<KV, QF32, D, CW>;
  using T = typename KvMma<KV>::T;
  constexpr bool kNorm = G::kEight || (KV == KV_F16 && QF32);
  const int half = D / 2;
  const int cap = cur.s.ctx;
  const AttendCol ci = attend_col(a, cur.s.row0, cur.s.nq, kvh, col0 + (lane >> 2));
  const int64_t qb = (int64_t)ci.row * a.q_stride + (int64_t)ci.head * D;
  float x[D / 16][4];
  uint32_t big = 0;
  // the lane's dims of a 16-dim group, in runs of 4 (8-bit caches) or 2
  constexpr int kRun = G::kEight ? 4 : 2;
  const bool f16 = a.q_dtype == CLOVER_B200_F16;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
    for (int j = 0; j < 4; j += kRun) {
      const int d = kk * 16 + (lane & 3) * kRun + j * (8 / kRun);
      const bool in = ci.valid && (a.maps == 1 || (d >= half) == (ci.map == 1));  // (a run lies in one half)
      float v[kRun];
#pragma unroll
      for (int i = 0; i < kRun; ++i) v[i] = 0.f;
      if (in && QF32) {
        const float* src = static_cast<const float*>(a.q) + qb + d;
        if (a.q_vec && kRun == 4) {
          const float4 f = *reinterpret_cast<const float4*>(src);
          v[0] = f.x, v[1] = f.y, v[kRun - 2] = f.z, v[kRun - 1] = f.w;
        } else if (a.q_vec) {
          const float2 f = *reinterpret_cast<const float2*>(src);
          v[0] = f.x, v[1] = f.y;
        } else {
#pragma unroll
          for (int i = 0; i < kRun; ++i) v[i] = src[i];
        }
      } else if (in) {
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + qb + d;
        uint32_t w[2] = {0, 0};
        if (a.q_vec && kRun == 4) {
          const uint2 u = *reinterpret_cast<const uint2*>(src);
          w[0] = u.x, w[1] = u.y;
        } else if (a.q_vec) {
          w[0] = *reinterpret_cast<const uint32_t*>(src);
        } else {
#pragma unroll
          for (int i = 0; i < kRun; i += 2) w[i / 2] = src[i] | ((uint32_t)src[i + 1] << 16);
        }
#pragma unroll
        for (int i = 0; i < kRun; i += 2) {
          const float2 f = f16 ? Pack<__half>::unpack(w[i / 2]) : Pack<__nv_bfloat16>::unpack(w[i / 2]);
          v[i] = f.x, v[i + 1] = f.y;
        }
      }
      // the order of K's fragments: int8 words give dims 0, 2 then 1, 3
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        x[kk][j + i] = v[KV == KV_I8 ? (i & 1) * 2 + (i >> 1) : i];
        big = max(big, abs_bits(v[i]));
      }
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
    split_terms<T, G::kQTerms>(x[kk][0], x[kk][1], c.q[kk][0]);
    split_terms<T, G::kQTerms>(x[kk][2], x[kk][3], c.q[kk][1]);
  }
  // limits and score scales of columns 2t, 2t + 1 from the lanes that hold them
  int lim = ci.valid ? ci.lim : 0;
  if (lim > cap) {  // a row past its sequence's last row
    raise_status(a.status, CLOVER_B200_DEV_CTX_RANGE);
    lim = cap;
  }
  c.min_lim = __reduce_min_sync(0xffffffffu, ci.valid ? lim : cap);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int src = ((lane & 3) * 2 + e) * 4;
    c.lim[e] = __shfl_sync(0xffffffffu, lim, src);
    c.sc[e] = a.scale_log2 * __shfl_sync(0xffffffffu, inv, src);
    c.m[e] = kNoRef;
    c.l[e] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < D / 16; ++i) c.acc[i][0] = c.acc[i][1] = c.acc[i][2] = c.acc[i][3] = 0.f;
}

// Fragments of V^T of 16 tokens for dims 16 i .. 16 i + 15 (8 bits: 32 i ..
// 32 i + 31, two M tiles).
template <int KV, int SWZ, int TOK>
struct VFrag {
  static constexpr int kPer = KV >= KV_I8 ? 2 : 1;
  uint32_t a[kPer][4];
  // This lane's row and chunk of the first load.
  __device__ __forceinline__ static uint32_t first(int lane) {
    const int grp = lane >> 3;
    return KV >= KV_I8 ? attend_swz<SWZ, TOK>((lane & 7) + (grp & 1) * 8, grp >> 1)
                       : attend_swz<SWZ, TOK>((lane & 7) + (grp >> 1) * 8, grp & 1);
  }
  __device__ __forceinline__ void load(uint32_t va, int i) {
    if (KV >= KV_I8) {
      uint32_t x[4];
      ldsm_x4_trans(attend_swz_step<SWZ, TOK>(va, i), x[0], x[1], x[2], x[3]);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        codes_to_f16<KV>(x[2 * k], a[k][0], a[k][1]);
        codes_to_f16<KV>(x[2 * k + 1], a[k][2], a[k][3]);
      }
    } else {
      ldsm_x4_trans(attend_swz_step<SWZ, TOK>(va, i), a[0][0], a[0][1], a[0][2], a[0][3]);
    }
  }
  // Zero the tokens at and past n: lo masks tokens 2t, 2t + 1, hi the tokens 8
  // later.
  __device__ __forceinline__ void mask(int n, int lane) {
    const int t = (lane & 3) * 2;
    const uint32_t lo = (t < n ? 0xffffu : 0u) | (t + 1 < n ? 0xffff0000u : 0u);
    const uint32_t hi = (t + 8 < n ? 0xffffu : 0u) | (t + 9 < n ? 0xffff0000u : 0u);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      a[k][0] &= lo;
      a[k][1] &= lo;
      a[k][2] &= hi;
      a[k][3] &= hi;
    }
  }
};

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

// Sixteen tokens of one warp: rows 0 .. 15 at ks / vs (tile row 16 j of the
// stage: the swizzle repeats every 8 rows), first token tok0, nvalid of them in
// the context; scales: their K scales, V's kTok floats on.
template <int KV, bool QF32, int D, int CW>
__device__ __forceinline__ void attend_step(uint32_t ks, uint32_t vs, const uint8_t* vgen, const float* scales,
                                            int tok0, int nvalid, AttendCols<KV, QF32, D, CW>& c, int lane) {
  using G = AttendGeom<KV, QF32, D, CW>;
  using T = typename KvMma<KV>::T;
  using VF = VFrag<KV, G::kSwz, G::kTok>;
  constexpr int KK = D / 16, QT = G::kQTerms, PT = G::kPTerms;
  const int g = lane >> 2;

  // ---- S = K . Q^T (two chains), times K's scale
  float ch[2][4], s[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) ch[0][e] = ch[1][e] = 0.f;
  const uint32_t ka = ks + attend_swz<G::kSwz, G::kTok>((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
  const uint32_t va = vs + VF::first(lane);
  if (G::kEight) {
#pragma unroll
    for (int i = 0; i < KK / 2; ++i) {
      uint32_t x[4];
      ldsm_x4(attend_swz_step<G::kSwz, G::kTok>(ka, i), x[0], x[1], x[2], x[3]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t a0, a1, a2, a3;
        if (KV == KV_E4M3) {
          e4m3_to_f16(x[2 * k], a0, a2);
          e4m3_to_f16(x[2 * k + 1], a1, a3);
        } else {
          codes_to_f16<KV>(x[2 * k], a0, a2);
          codes_to_f16<KV>(x[2 * k + 1], a1, a3);
        }
#pragma unroll
        for (int q = 0; q < QT; ++q)
          MmaOp<T>::run(ch[k], a0, a1, a2, a3, c.q[2 * i + k][0][q], c.q[2 * i + k][1][q]);
      }
    }
  } else {
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      uint32_t a0, a1, a2, a3;
      ldsm_x4(attend_swz_step<G::kSwz, G::kTok>(ka, kk), a0, a1, a2, a3);
#pragma unroll
      for (int q = 0; q < QT; ++q)
        MmaOp<T>::run(ch[kk & 1], a0, a1, a2, a3, c.q[kk][0][q], c.q[kk][1][q]);
    }
  }
  // V's scales, and their bounds for the reference
  float vsc[2] = {1.f, 1.f}, vref[2] = {1.f, 1.f};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (G::kEight) {
      vsc[h] = scales[G::kTok + g + 8 * h];
      vref[h] = fmaxf(fabsf(vsc[h]), kLeastScale);
    }
    const float ksc = G::kEight ? scales[g + 8 * h] : 1.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x = ch[0][2 * h + e] + ch[1][2 * h + e];
      s[2 * h + e] = G::kEight ? x * ksc : x;
    }
  }
  // Steps that every column sees whole need no mask.
  const bool edge = tok0 + kUnitTok > c.min_lim;
  auto masked = [&](int h, int e) { return edge && tok0 + g + 8 * h >= c.lim[e]; };

  // ---- weights; the reference moves when one outgrows it.  Each lane looks at
  // its own; only a move takes the columns' maxima over the lanes.
  float p[4], w[4], big = 0.f;
  auto weigh = [&](int h, int e) {
    const int i = 2 * h + e;
    p[i] = masked(h, e) ? 0.f : fast_exp2(fmaf(s[i], c.sc[e], -c.m[e]));
    // (a masked token's scale may be anything: its weight stays 0)
    const float up = p[i] * G::kUp;
    w[i] = G::kEight ? (masked(h, e) ? 0.f : up * vsc[h]) : up;
  };
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      weigh(h, e);
      big = fmaxf(big, p[2 * h + e] * vref[h]);
    }
  if (__any_sync(0xffffffffu, big > G::kMaxWeight)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float mx = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (!masked(h, e)) mx = fmaxf(mx, fmaf(s[2 * h + e], c.sc[e], G::kEight ? fast_log2(vref[h]) : 0.f));
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float nm = fmaxf(c.m[e], mx);
      const float al = fast_exp2(c.m[e] - nm);
      c.m[e] = nm;
      c.l[e] *= al;
#pragma unroll
      for (int i = 0; i < KK; ++i) {
        c.acc[i][e] *= al;
        c.acc[i][2 + e] *= al;
      }
      weigh(0, e);
      weigh(1, e);
    }
  }
  c.l[0] += p[0] + p[2];
  c.l[1] += p[1] + p[3];
  uint32_t pt[2][PT];  // split and transposed
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    split_terms<T, PT>(w[2 * h], w[2 * h + 1], pt[h]);
#pragma unroll
    for (int k = 0; k < PT; ++k) pt[h][k] = movm_trans(pt[h][k]);
  }

  // ---- O^T += V^T . P^T
  if (KV == KV_I8 || !edge) {  // (every int8 code is finite)
#pragma unroll
    for (int i = 0; i < KK / VF::kPer; ++i) {
      VF v;
      v.load(va, i);
#pragma unroll
      for (int q = 0; q < PT; ++q)
#pragma unroll
        for (int k = 0; k < VF::kPer; ++k)
          MmaOp<T>::run(c.acc[i * VF::kPer + k], v.a[k][0], v.a[k][1], v.a[k][2], v.a[k][3], pt[0][q], pt[1][q]);
    }
    return;
  }
  // Tokens that some column does not see.  Past the context they are masked in
  // V; an infinity or NaN of a later token must not meet the zero weight of an
  // earlier row (multi-token rows), so a step that holds one takes its columns
  // limit by limit, each with V masked from its limit on.
  const int lo = max(0, c.min_lim - tok0), hi = min(nvalid, kUnitTok);
  const bool plain = !(lo < hi && rows_nonfinite<KV, G::kRow, G::kSwz, G::kTok>(vgen, lo, hi, lane));
  for (int below = 0x7fffffff;;) {
    int top = plain ? tok0 + hi : 0;
    if (!plain) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (c.lim[e] < below) top = max(top, c.lim[e]);
      top = __reduce_max_sync(0xffffffffu, top);
      if (top <= tok0) break;
    }
#pragma unroll
    for (int i = 0; i < KK / VF::kPer; ++i) {
      VF v;
      v.load(va, i);
      v.mask(top - tok0, lane);
#pragma unroll
      for (int k = 0; k < VF::kPer; ++k) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < PT; ++q)
          MmaOp<T>::run(x, v.a[k][0], v.a[k][1], v.a[k][2], v.a[k][3], pt[0][q], pt[1][q]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (plain || c.lim[e & 1] == top) c.acc[i * VF::kPer + k][e] += x[e];
      }
    }
    if (plain) break;
    below = top;
  }
}

// The end of a segment's piece: the output, or a partial for the join.
template <int KV, bool QF32, int D, int CW>
__device__ __forceinline__ void finish_piece(const AttendArgs& a, const Cursor& cur, int wid, const AttendSplit& sp,
                                             int first_jj, int kvh, int chunk, int cw,
                                             AttendCols<KV, QF32, D, CW>& c, int lane) {
  using G = AttendGeom<KV, QF32, D, CW>;
  constexpr int KK = D / 16, COLS = 8 * CW;
  constexpr float kDown = 1.f / G::kUp;  // (a power of two: exact)
  const bool whole = a.whole || (first_jj == 0 && cur.jj == cur.s.n - 1);
#pragma unroll
  for (int off = 4; off < 32; off <<= 1) {
    c.l[0] += __shfl_xor_sync(0xffffffffu, c.l[0], off);
    c.l[1] += __shfl_xor_sync(0xffffffffu, c.l[1], off);
  }
  const int g = lane >> 2, c0 = cw * 8 + (lane & 3) * 2;
  const int d0 = G::kEight ? 2 * g : g, dh = G::kEight ? 1 : 8;  // dims of M rows g, g + 8
  if (!whole) {
    const int64_t slot = attend_slot(sp, wid, first_jj);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t at = slot * COLS + c0 + e;
      float* po = a.part + at * D;
#pragma unroll
      for (int i = 0; i < KK; ++i) {
        if (G::kEight) {
          *reinterpret_cast<float2*>(po + i * 16 + d0) = make_float2(c.acc[i][e] * kDown, c.acc[i][2 + e] * kDown);
        } else {
          po[i * 16 + d0] = c.acc[i][e] * kDown;
          po[i * 16 + d0 + dh] = c.acc[i][2 + e] * kDown;
        }
      }
      if (lane < 4) a.part_ml[at] = make_float2(c.m[e], c.l[e]);
    }
  } else if (a.maps == 1) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const AttendCol ci = attend_col(a, cur.s.row0, cur.s.nq, kvh, chunk * COLS + c0 + e);
      if (!ci.valid) continue;
      const bool any = c.lim[e] > 0;
      const float inv = attend_inv(c.l[e], c.lim[e]) * kDown;
      const int64_t ob = (int64_t)ci.row * a.out_stride + (int64_t)ci.head * D + d0;
#pragma unroll
      for (int i = 0; i < KK; ++i) {
        attend_store(a, ob + i * 16, any ? c.acc[i][e] * inv : 0.f);
        attend_store(a, ob + i * 16 + dh, any ? c.acc[i][2 + e] * inv : 0.f);
      }
    }
  } else {
    // columns 2t and 2t + 1 are the two maps of one head
    const AttendCol ci = attend_col(a, cur.s.row0, cur.s.nq, kvh, chunk * COLS + c0);
    const bool any = c.lim[0] > 0;
    const float lam = ci.valid ? a.lam[ci.head] : 0.f;
    const float i0 = attend_inv(c.l[0], c.lim[0]) * kDown, i1 = attend_inv(c.l[1], c.lim[1]) * kDown;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < KK; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float o = any ? diff_value(c.acc[i][2 * h] * i0, c.acc[i][2 * h + 1] * i1, lam) : 0.f;
        c.acc[i][2 * h] = o;
        sq = fmaf(o, o, sq);
      }
    }
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
    if (ci.valid) {
      const int64_t ob = (int64_t)ci.row * a.out_stride + (int64_t)ci.head * D;
      // (a row without tokens is 0, and eps may be)
      const float r = a.norm_w == nullptr ? 1.f : any ? rsqrtf(sq / D + a.eps) * a.out_scale : 0.f;
#pragma unroll
      for (int i = 0; i < KK; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int d = i * 16 + d0 + h * dh;
          const float w = a.norm_w != nullptr ? a.norm_w[d] : 1.f;
          attend_store(a, ob + d, c.acc[i][2 * h] * (r * w));
        }
      }
    }
    __syncwarp();
  }
  if (!a.whole && first_jj == 0 && cw == 0 && lane == 0)
    attend_record(a, sp, cur.b, cur.h, cur.seg0, cur.s, wid);
}

// ------------------------------------------------------------------ copies
// Fused append: the new tokens of a sequence (rows row0 .. row0 + nq - 1) that
// lie in the unit [tok0, tok0 + 16 SUBS), for KV head kvh, written by the warp
// before the unit is copied (slot0, slot1: first cache slot of its 16-token
// steps, negative where the step's block id is bad: its tokens are skipped).
template <int KV, int D, int SUBS>
__device__ __forceinline__ void append_unit(const AttendArgs& a, int row0, int nq, int ctx, int tok0, int kvh,
                                            int slot0, int slot1, int lane) {
  for (int j = 0; j < nq; ++j) {
    const int r = row0 + j;
    const int rel = __ldg(a.ctx + r) - 1 - tok0;
    if (rel < 0 || rel >= SUBS * kUnitTok || rel + tok0 >= ctx) continue;
    const int first = rel < kUnitTok ? slot0 : slot1;
    if (first < 0) continue;
    const int64_t at = first + (rel & (kUnitTok - 1));
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

// The copies of a ring: the unit after the last one issued, and where its
// tokens are.  Block ids are held 32 at a time (lane i: block id_base + i), a
// bad one as -1.
template <int KV, bool QF32, int D, int CW>
struct RingCopies {
  using G = AttendGeom<KV, QF32, D, CW>;
  Cursor cur;
  bool more;
  int ids, id_base, blk, sub, kvh, first_new, st;

  // Start (or go on in) a segment: the block and 16-token step of its unit jj.
  __device__ __forceinline__ void enter(const AttendArgs& a, bool new_seq) {
    const int upb = a.bs / kUnitTok;
    if (new_seq) id_base = -64;
    kvh = cur.h / (cur.s.hc / a.hkv);
    const int at = cur.jj * G::kSubs;
    blk = at / upb;
    sub = at - blk * upb;
    if (a.k_new != nullptr) first_new = __ldg(a.ctx + cur.s.row0) - 1;
  }

  __device__ __forceinline__ void issue(const AttendArgs& a, const CUtensorMap* tmK, const CUtensorMap* tmV,
                                        uint32_t ring, uint32_t scales, uint32_t full, int lane) {
    constexpr int SUBS = G::kSubs;
    const int upb = a.bs / kUnitTok;
    if (blk < id_base || blk + SUBS > id_base + 32) {
      id_base = blk;
      const int trow = a.seq_rows ? __ldg(a.seq_rows + cur.b) : cur.b;
      const int n = (cur.s.ctx + a.bs - 1) / a.bs;
      ids = 0;
      if (blk + lane < n) {
        ids = blk + lane < a.table_stride ? __ldg(a.tables + (int64_t)trow * a.table_stride + blk + lane) : -1;
        if (ids < 0 || ids >= a.num_blocks) {
          raise_status(a.status, CLOVER_B200_DEV_BAD_BLOCK);
          ids = -1;
        }
      }
    }
    // First cache slot of each 16-token step: what is copied (a bad block reads
    // block 0, so that the pipeline stays well-formed; the output is flagged),
    // and what an append may write to (a bad block: nothing).
    int slot[SUBS], own[SUBS];
    int id[SUBS], off[SUBS];
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      const int got = __shfl_sync(0xffffffffu, ids, blk - id_base);
      id[u] = max(got, 0);
      off[u] = sub * kUnitTok;
      slot[u] = id[u] * a.bs + off[u];
      own[u] = got < 0 ? -1 : slot[u];
      if (++sub == upb) {
        sub = 0;
        ++blk;
      }
    }
    if (a.k_new != nullptr && (cur.jj + 1) * G::kTok > first_new)
      append_unit<KV, D, SUBS>(a, cur.s.row0, cur.s.nq, cur.s.ctx, cur.jj * G::kTok, kvh, own[0], own[SUBS - 1],
                               lane);
    const int left = (cur.s.ctx + kUnitTok - 1) / kUnitTok - cur.jj * SUBS;  // steps of the segment
    const int subs = left < SUBS ? left : SUBS;
    const uint32_t bar = full + st * 8;
    const uint32_t kd = ring + st * G::kTiles, vd = kd + G::kTile;
    if (lane == 0) mbar_arrive_expect_tx(bar, subs * (G::kTiles / SUBS));
    __syncwarp();
    // one tile copy per lane: (step, chunk, K or V)
    constexpr int kPer = 2 * G::kChunks;
    const int u = lane / kPer, i = lane - u * kPer;
    if (u < subs) {
      const int ch = i >> 1;
      tma_load_3d((i & 1 ? vd : kd) + (ch * G::kTok + u * kUnitTok) * G::kSwz, i & 1 ? tmV : tmK,
                  ch * (G::kSwz / G::kEsz), kvh, u == 0 ? slot[0] : slot[SUBS - 1], bar);
    }
    if (G::kEight) {
      // 16 bytes of the scales per lane: (K or V, step, quarter)
      const int su = SUBS > 1 ? (lane >> 2) & 1 : 0, v = SUBS > 1 ? lane >> 3 : lane >> 2;
      if (v < 2 && su < subs) {
        const int64_t at = ((int64_t)(su ? id[SUBS - 1] : id[0]) * a.hkv + kvh) * a.bs + (su ? off[SUBS - 1] : off[0]);
        copy16_async(scales + st * G::kScales + (v * G::kTok + su * kUnitTok) * 4 + (lane & 3) * 16,
                     (v ? a.vs : a.ks) + at + (lane & 3) * 4);
      }
      copies_arrive(bar);
    }
    st = st + 1 == G::kStages ? 0 : st + 1;
    const int b = cur.b, h = cur.h;
    more = cur.next(a);
    if (more && (cur.b != b || cur.h != h)) enter(a, cur.b != b);
  }
};

template <int KV, bool QF32, int D, int CW>
__global__ void __launch_bounds__(AttendGeom<KV, QF32, D, CW>::kThreads, 1)
attend_mma_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const AttendArgs a) {
  using G = AttendGeom<KV, QF32, D, CW>;
  constexpr int STAGES = G::kStages, RINGS = G::kRings, COLS = 8 * CW;
  constexpr int LAG = CW > 1 ? 1 : 0;  // a shared stage is refilled one unit later
  static_assert(STAGES > LAG, "a refill may not wait for itself");
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[RINGS * STAGES], s_empty[RINGS * STAGES];
  __shared__ AttendPlan<G::kWarps, RINGS> plan;
  __shared__ int s_stop;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // after a bounded wait gave up anywhere, later launches stop at once
  if (threadIdx.x == 0)
    s_stop = a.status != nullptr && (*(volatile int32_t*)a.status & CLOVER_B200_DEV_TIMEOUT);
  for (int i = threadIdx.x; i < RINGS * STAGES; i += G::kThreads) {
    mbar_init(smem_addr(&s_full[i]), G::kEight ? 33 : 1);  // the tiles, and each lane's scales
    mbar_init(smem_addr(&s_empty[i]), 1);                  // the ring's other warp
    fence_mbar_init();
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  pdl_wait();
  __syncthreads();
  if (s_stop) return;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_sc = smem + RINGS * G::kRingTiles;
  AttendSplit sp{1, 0, 0, false};
  if (!a.whole) {
    sp = attend_plan<G::kWarps, RINGS>(a, plan);
    pdl_trigger();
  }

  const int ring = warp / CW, cw = warp % CW;
  const int wid = a.whole ? ring * gridDim.x + blockIdx.x : attend_worker(sp, ring);
  if (a.whole && cw == 0) {
    // rows of empty sequences have no unit: their zeros are written here
    const int hcmax = a.hkv * a.chunks;
    for (int64_t sg = wid; sg < (int64_t)a.n_seqs * hcmax; sg += a.workers) {
      const int b = (int)sg / hcmax, h = (int)sg - b * hcmax;
      const SeqInfo s = seq_info(a, b);
      if (h == 0 && lane == 0) attend_check_seq(a, s);
      if (h >= s.hc || s.n > 0) continue;
      const int nch = s.hc / a.hkv, kvh = h / nch;
      for (int c = 0; c < COLS; ++c) {
        const AttendCol ci = attend_col(a, s.row0, s.nq, kvh, (h - kvh * nch) * COLS + c);
        if (!ci.valid || ci.map == 1) continue;
        for (int d = lane; d < D; d += 32)
          attend_store(a, (int64_t)ci.row * a.out_stride + (int64_t)ci.head * D + d, 0.f);
      }
    }
  }
  Cursor cur;
  if (!(a.whole ? cur.seek(a, wid) : attend_start(a, plan, ring, cur))) return;
  const uint32_t ring_s = smem_addr(smem) + ring * G::kRingTiles;
  const uint32_t scales_s = smem_addr(smem_sc) + ring * STAGES * G::kScales;
  const uint32_t full = smem_addr(&s_full[ring * STAGES]), empty = smem_addr(&s_empty[ring * STAGES]);

  RingCopies<KV, QF32, D, CW> copies;
  copies.cur = cur;
  copies.more = cw == 0;
  copies.st = 0;
  copies.first_new = 0x7fffffff;
  int issued = 0;
  if (cw == 0) {
    copies.enter(a, true);
    while (issued < STAGES && copies.more) {
      copies.issue(a, &tmK, &tmV, ring_s, scales_s, full, lane);
      ++issued;
    }
  }

  AttendCols<KV, QF32, D, CW> c;
  int first_jj = 0, kvh = 0, chunk = 0, st = 0, k = 0;
  uint32_t parity = 0;
  bool fresh = true, cols = false, timed_out = false;
  for (;; ++k) {
    if (fresh) {
      first_jj = cur.jj;
      const int nch = cur.s.hc / a.hkv;
      kvh = cur.h / nch;
      chunk = cur.h - kvh * nch;
      // (a column warp past the sequence's columns only passes the stages on)
      cols = chunk * COLS + cw * 8 < cur.s.nq * a.group * a.maps;
      if (cols) load_columns<KV, QF32, D, CW>(a, cur, kvh, chunk * COLS + cw * 8, c, lane);
    }
    if (!mbar_wait_bounded(full + st * 8, parity, a.wait_ns)) {
      timed_out = true;
      break;
    }
    if (cols) {
      const uint32_t ks = ring_s + st * G::kTiles;
      const uint8_t* vgen = smem + ring * G::kRingTiles + st * G::kTiles + G::kTile;
      const float* sc = reinterpret_cast<const float*>(smem_sc + (ring * STAGES + st) * G::kScales);
      // (a loop, not unrolled: half the code in the instruction cache)
#pragma unroll 1
      for (int u = 0; u < G::kSubs; ++u) {
        const int tok0 = cur.jj * G::kTok + u * kUnitTok;
        if (tok0 >= cur.s.ctx) break;
        attend_step<KV, QF32, D, CW>(ks + u * kUnitTok * G::kSwz, ks + G::kTile + u * kUnitTok * G::kSwz,
                                     vgen + u * kUnitTok * G::kSwz, sc + u * kUnitTok, tok0, cur.s.ctx - tok0, c,
                                     lane);
      }
    }
    __syncwarp();
    if (CW > 1 && cw > 0 && lane == 0) mbar_arrive(empty + st * 8);
    if (copies.more && k >= LAG) {
      // (the stage refilled is copies.st: unit k - LAG was in it)
      if (CW > 1 && !mbar_wait_bounded(empty + copies.st * 8, ((k - LAG) / STAGES) & 1, a.wait_ns)) {
        timed_out = true;
        break;
      }
      copies.issue(a, &tmK, &tmV, ring_s, scales_s, full, lane);
      ++issued;
    }
    if (++st == STAGES) {
      st = 0;
      parity ^= 1;
    }
    Cursor nx = cur;
    const bool on = nx.next(a);
    fresh = !on || nx.b != cur.b || nx.h != cur.h;
    if (fresh && cols) finish_piece<KV, QF32, D, CW>(a, cur, wid, sp, first_jj, kvh, chunk, cw, c, lane);
    if (!on) break;
    cur = nx;
  }
  if (timed_out) {
    // the copies in flight land (bounded) before the CTA's memory goes
    for (int j = max(0, issued - STAGES); j < issued; ++j)
      mbar_wait_bounded(full + (j % STAGES) * 8, (j / STAGES) & 1, kWaitLimitNs);
    if (lane == 0) raise_status(a.status, CLOVER_B200_DEV_TIMEOUT);
  }
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

template <int KV, bool QF32, int D, int CW>
static int mma_launch(const AttendArgs* a, cudaStream_t s, int* rings) {
  using G = AttendGeom<KV, QF32, D, CW>;
  if (a == nullptr) {
    *rings = G::kRings;
    return CLOVER_B200_OK;
  }
  auto kern = attend_mma_kernel<KV, QF32, D, CW>;
  static uint64_t configured = 0;  // one bit per device ordinal
  int dev = 0;
  int rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  {
    std::lock_guard<std::mutex> lock(g_attend_mu);
    if (dev >= 64 || !(configured >> dev & 1)) {
      rc = set_smem(kern, G::kSmem);
      if (rc) return rc;
      if (dev < 64) configured |= 1ull << dev;
    }
  }
  CUtensorMap tk, tv;
  rc = attend_tmap(a->kc, G::kEsz, D, a->hkv, a->num_blocks * a->bs, &tk);
  if (rc) return rc;
  rc = attend_tmap(a->vc, G::kEsz, D, a->hkv, a->num_blocks * a->bs, &tv);
  if (rc) return rc;
  return check_cuda(launch_pdl(kern, dim3(a->workers / G::kRings), dim3(G::kThreads), G::kSmem, s, tk, tv, *a),
                    "attend_mma launch");
}

template <int KV, bool QF32>
static int mma_shape(int cols, const AttendArgs* a, int D, cudaStream_t s, int* rings) {
  const bool two = cols > kMmaCols;
  switch (D) {
    case 64: return two ? mma_launch<KV, QF32, 64, 2>(a, s, rings) : mma_launch<KV, QF32, 64, 1>(a, s, rings);
    case 128: return two ? mma_launch<KV, QF32, 128, 2>(a, s, rings) : mma_launch<KV, QF32, 128, 1>(a, s, rings);
    default: return two ? mma_launch<KV, QF32, 256, 2>(a, s, rings) : mma_launch<KV, QF32, 256, 1>(a, s, rings);
  }
}

bool attend_mma_supported(int kv_dtype, int q_dtype, int D, int bs) {
  return (D == 64 || D == 128 || D == 256) && bs % kUnitTok == 0 && kv_dtype != CLOVER_B200_F32;
}

int attend_mma_unit_log2(int kv_dtype, int D) {
  const bool eight = kv_dtype == CLOVER_B200_INT8 || kv_dtype == CLOVER_B200_FP8_E4M3;
  return D * (eight ? 1 : 2) <= 128 ? 5 : 4;
}

int attend_mma(int kv_dtype, int q_dtype, int cols, const AttendArgs* a, int D, cudaStream_t s, int* rings) {
  const bool f32 = q_dtype == CLOVER_B200_F32;
  switch (kv_dtype) {
    case CLOVER_B200_BF16: return f32 ? mma_shape<KV_BF16, true>(cols, a, D, s, rings) : mma_shape<KV_BF16, false>(cols, a, D, s, rings);
    case CLOVER_B200_F16: return f32 ? mma_shape<KV_F16, true>(cols, a, D, s, rings) : mma_shape<KV_F16, false>(cols, a, D, s, rings);
    case CLOVER_B200_INT8: return f32 ? mma_shape<KV_I8, true>(cols, a, D, s, rings) : mma_shape<KV_I8, false>(cols, a, D, s, rings);
    default: return f32 ? mma_shape<KV_E4M3, true>(cols, a, D, s, rings) : mma_shape<KV_E4M3, false>(cols, a, D, s, rings);
  }
}

}  // namespace clover
