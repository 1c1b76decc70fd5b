// Quantising KV append: new tokens' K/V rows (f32, f16 or bf16) into an 8-bit
// paged cache with one scale per (token, KV head); quantise.cuh has the
// formula.  The slot arithmetic, the skipped and the flagged slots are those
// of clover_b200_kv_append (KVCacheManager.write_new_kv / load_initial_kv,
// src/core/memory_manager.py:74-93, :123-132).
#include "quantise.cuh"

namespace clover {

struct AppendScaledArgs {
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  int64_t cache_layer, scale_layer;  // elements between layers
  const void* kn;
  const void* vn;
  int64_t new_layer, new_token;  // elements between layers / tokens
  const int64_t* slots;
  int64_t n_tokens;
  int32_t heads, dim, bs;
  int64_t n_slots;
  int32_t* status;
};

// Rows of a multiple of 16 bytes, 16-byte aligned (dst: 8): a power of two of
// lanes holds a row, up to NV vectors each; blockIdx.y is the layer, blockIdx.z
// K or V.  Bound: HBM (read the row, write one byte per value), with the
// instructions close behind: one vector per lane repeats the row's scale, slot
// and division in every lane (16381 tokens x 8 heads x 128, f16 -> e4m3: 46 us; a
// warp per row without vectors 92; two rows in flight per thread, with fewer
// warps on an SM, 27.5; this 21.5, 72 % of the copy peak).
template <bool FP8, typename TI, int NV>
__global__ void __launch_bounds__(256)
kv_append_scaled_vec_kernel(const AppendScaledArgs a, int lpr) {
  constexpr int VEC = 16 / (int)sizeof(TI);
  const int lane = threadIdx.x & 31;
  const int64_t layer = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const int vecs = a.dim / VEC;
  const int rpw = 32 / lpr, sub = lane / lpr, l = lane - sub * lpr;  // rows per warp, this lane's row and vector
  const int64_t rows = a.n_tokens * a.heads;
  const TI* src = static_cast<const TI*>(is_v ? a.vn : a.kn) + layer * a.new_layer;
  uint8_t* cache = (is_v ? a.vc : a.kc) + layer * a.cache_layer;
  float* scales = (is_v ? a.vs : a.ks) + layer * a.scale_layer;
  const int64_t step = (int64_t)gridDim.x * 8 * rpw;
  for (int64_t r = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * rpw + sub; r - sub < rows; r += step) {
    uint4 x[NV];
    int64_t slot = -1;
    int head = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) x[k] = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const int64_t t = rows <= INT32_MAX ? (int)r / a.heads : r / a.heads;
      head = (int)(r - t * a.heads);
      slot = __ldg(a.slots + t);
      const uint4* row = reinterpret_cast<const uint4*>(src + t * a.new_token + (int64_t)head * a.dim);
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (l + k * lpr < vecs) x[k] = __ldg(row + l + k * lpr);
      if (slot >= a.n_slots) {
        if (l == 0 && head == 0 && !is_v) raise_status(a.status, CLOVER_B200_DEV_BAD_SLOT);
        slot = -1;
      }
    }
    float v[NV][VEC];
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (VEC == 4) {
          v[k][i] = __uint_as_float(w[i]);
          m = max(m, abs_bits(v[k][i]));
        } else {
          const float2 p = Pack<TI>::unpack(w[i]);
          v[k][2 * i] = p.x;
          v[k][2 * i + 1] = p.y;
          m = max(m, max(abs_bits(p.x), abs_bits(p.y)));
        }
      }
    }
    for (int off = lpr >> 1; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
    float factor;
    const float s = row_scale(m, code_top<FP8>(), factor);
    if (slot < 0) continue;  // padding token
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (l + k * lpr >= vecs) continue;
      uint8_t* dst = cache + (slot * a.heads + head) * a.dim + (l + k * lpr) * VEC;
      if constexpr (VEC == 4) {
        *reinterpret_cast<uint32_t*>(dst) = encode4<FP8>(v[k], factor);
      } else {
        *reinterpret_cast<uint2*>(dst) = make_uint2(encode4<FP8>(v[k], factor), encode4<FP8>(v[k] + 4, factor));
      }
    }
    if (l == 0) {
      const int64_t blk = slot <= INT32_MAX ? (int)slot / a.bs : slot / a.bs;
      scales[(blk * a.heads + head) * a.bs + (slot - blk * a.bs)] = s;
    }
  }
}

// One warp per (token, K or V, head) row; any head_dim and alignment.
template <bool FP8, typename TI>
__global__ void __launch_bounds__(256)
kv_append_scaled_kernel(const AppendScaledArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t layer = blockIdx.y;
  const int64_t rows = a.n_tokens * 2 * a.heads;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    const int64_t t = r / (2 * a.heads);
    const int rest = (int)(r - t * 2 * a.heads);
    const bool is_v = rest >= a.heads;
    const int h = is_v ? rest - a.heads : rest;
    const int64_t slot = __ldg(a.slots + t);
    if (slot < 0) continue;  // padding token
    if (slot >= a.n_slots) {
      if (lane == 0 && rest == 0) raise_status(a.status, CLOVER_B200_DEV_BAD_SLOT);
      continue;
    }
    const TI* src = static_cast<const TI*>(is_v ? a.vn : a.kn) + layer * a.new_layer + t * a.new_token +
                    (int64_t)h * a.dim;
    uint8_t* dst = (is_v ? a.vc : a.kc) + layer * a.cache_layer + (slot * a.heads + h) * a.dim;
    const float s = encode_row_warp<FP8, TI>(src, dst, a.dim, lane);
    const int64_t blk = slot / a.bs;
    if (lane == 0)
      (is_v ? a.vs : a.ks)[layer * a.scale_layer + (blk * a.heads + h) * a.bs + (slot - blk * a.bs)] = s;
  }
}

template <bool FP8>
static cudaError_t launch_append_scaled(int dtype, dim3 grid, cudaStream_t s,
                                        const AppendScaledArgs& a) {
  switch (dtype) {
    case CLOVER_B200_F32: kv_append_scaled_kernel<FP8, float><<<grid, 256, 0, s>>>(a); break;
    case CLOVER_B200_F16: kv_append_scaled_kernel<FP8, __half><<<grid, 256, 0, s>>>(a); break;
    default: kv_append_scaled_kernel<FP8, __nv_bfloat16><<<grid, 256, 0, s>>>(a); break;
  }
  return cudaGetLastError();
}

template <bool FP8>
static cudaError_t launch_append_vec(int dtype, dim3 grid, cudaStream_t s, const AppendScaledArgs& a,
                                     int lpr) {
  switch (dtype) {
    case CLOVER_B200_F32: kv_append_scaled_vec_kernel<FP8, float, 4><<<grid, 256, 0, s>>>(a, lpr); break;
    case CLOVER_B200_F16: kv_append_scaled_vec_kernel<FP8, __half, 4><<<grid, 256, 0, s>>>(a, lpr); break;
    default: kv_append_scaled_vec_kernel<FP8, __nv_bfloat16, 4><<<grid, 256, 0, s>>>(a, lpr); break;
  }
  return cudaGetLastError();
}

}  // namespace clover

using namespace clover;

extern "C" int clover_b200_kv_append_scaled(
    void* k_cache, void* v_cache, float* k_scales, float* v_scales, int32_t kv_dtype,
    int64_t cache_layer_stride, int64_t scale_layer_stride, const void* k_new, const void* v_new,
    int32_t new_dtype, int64_t new_layer_stride, int64_t new_token_stride,
    const int64_t* slot_mapping, int64_t n_tokens, int32_t n_layers, int32_t num_kv_heads,
    int32_t head_dim, int32_t block_size, int64_t num_blocks, int32_t* dev_status, void* stream) {
  if (n_tokens < 0 || n_layers < 0 || n_layers > 65535 || num_kv_heads <= 0 || head_dim <= 0 ||
      block_size <= 0 || num_blocks < 0)
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "kv_append_scaled: bad sizes");
  if (kv_dtype != CLOVER_B200_INT8 && kv_dtype != CLOVER_B200_FP8_E4M3)
    return set_error(CLOVER_B200_ERR_UNSUPPORTED, "kv_append_scaled: cache dtype %d", kv_dtype);
  if (new_dtype != CLOVER_B200_F32 && new_dtype != CLOVER_B200_F16 && new_dtype != CLOVER_B200_BF16)
    return set_error(CLOVER_B200_ERR_UNSUPPORTED, "kv_append_scaled: new K/V dtype %d", new_dtype);
  if (n_tokens == 0 || n_layers == 0) return CLOVER_B200_OK;
  if (!k_cache || !v_cache || !k_scales || !v_scales || !k_new || !v_new || !slot_mapping)
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "kv_append_scaled: null pointer");
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (new_token_stride < row)
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "kv_append_scaled: token stride < heads*head_dim");
  const int64_t n_slots = num_blocks * (int64_t)block_size;
  if (n_layers > 1 && (cache_layer_stride < n_slots * row ||
                       scale_layer_stride < n_slots * (int64_t)num_kv_heads ||
                       new_layer_stride < 0))
    return set_error(CLOVER_B200_ERR_INVALID_ARG, "kv_append_scaled: layer strides overlap");
  AppendScaledArgs a{(uint8_t*)k_cache, (uint8_t*)v_cache, k_scales, v_scales, cache_layer_stride,
                     scale_layer_stride, k_new, v_new, new_layer_stride, new_token_stride,
                     slot_mapping, n_tokens, num_kv_heads, head_dim, block_size, n_slots,
                     dev_status};
  const int64_t want = (n_tokens * 2 * num_kv_heads + 7) / 8;
  const int64_t cap = (148 * 16 + n_layers - 1) / n_layers;
  const dim3 grid((unsigned)(want < cap ? want : cap), (unsigned)n_layers);
  const int esz = new_dtype == CLOVER_B200_F32 ? 4 : 2, vec = 16 / esz, vecs = head_dim / vec;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new);
  const uintptr_t caches = reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache);
  if (head_dim % vec == 0 && vecs <= 128 && !(bases & 15) && !(caches & 7) && head_dim % 8 == 0 &&
      (new_token_stride * esz) % 16 == 0 && (n_layers == 1 || (new_layer_stride * esz) % 16 == 0) &&
      (n_layers == 1 || cache_layer_stride % 8 == 0)) {
    int lpr = 1;
    while (lpr * 4 < vecs) lpr *= 2;
    const int64_t warps = (n_tokens * num_kv_heads + 32 / lpr - 1) / (32 / lpr);
    const int64_t want_v = (warps + 7) / 8;
    const int64_t cap_v = (148 * 16 + 2 * n_layers - 1) / (2 * n_layers);
    const dim3 gv((unsigned)(want_v < cap_v ? want_v : cap_v), (unsigned)n_layers, 2);
    const cudaError_t ev = kv_dtype == CLOVER_B200_INT8
                               ? launch_append_vec<false>(new_dtype, gv, (cudaStream_t)stream, a, lpr)
                               : launch_append_vec<true>(new_dtype, gv, (cudaStream_t)stream, a, lpr);
    return check_cuda(ev, "kv_append_scaled launch");
  }
  const cudaError_t e = kv_dtype == CLOVER_B200_INT8
                            ? launch_append_scaled<false>(new_dtype, grid, (cudaStream_t)stream, a)
                            : launch_append_scaled<true>(new_dtype, grid, (cudaStream_t)stream, a);
  return check_cuda(e, "kv_append_scaled launch");
}
