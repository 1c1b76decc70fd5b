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
  const cudaError_t e = kv_dtype == CLOVER_B200_INT8
                            ? launch_append_scaled<false>(new_dtype, grid, (cudaStream_t)stream, a)
                            : launch_append_scaled<true>(new_dtype, grid, (cudaStream_t)stream, a);
  return check_cuda(e, "kv_append_scaled launch");
}
