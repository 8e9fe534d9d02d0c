// Attention of one new token per sequence over a paged key-value cache.
//
//   o[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[b, h] . k_j - max),  j over the visible keys of row b:
//   j < len, and with a window: j >= len - window or j < sinks.  A row without visible keys gives zeros.
//
// Simple form: one warp per query head, one key at a time, the running maximum and sum in fp32.
#include "kernels.cuh"

namespace cq {

__device__ __forceinline__ float load_cache(const void* p, int64_t i, int dt) {
  if (dt == CQ_DT_FP8_E4M3) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<const __nv_fp8_storage_t*>(p)[i], __NV_E4M3);
    return __half2float(__half(h));
  }
  return dt == CQ_DT_F16 ? __half2float(static_cast<const __half*>(p)[i])
                         : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__global__ void __launch_bounds__(128) paged_attention_kernel(const PagedAttnArgs a) {
  const int lane = threadIdx.x & 31;
  const int h = blockIdx.x * 4 + (threadIdx.x >> 5), b = blockIdx.y;
  if (h >= a.Hq) return;
  const int hk = h / (a.Hq / a.Hkv);
  const int row = a.rows != nullptr ? a.rows[b] : b;
  int64_t len = (row >= 0 && row < a.table_rows) ? a.lens[row] : 0;
  if (len > static_cast<int64_t>(a.table_width) * a.page_size) len = static_cast<int64_t>(a.table_width) * a.page_size;
  const float ks = a.k_scale != nullptr ? a.k_scale[hk] : 1.0f, vs = a.v_scale != nullptr ? a.v_scale[hk] : 1.0f;
  float q[8], o[8] = {};
  const int per = a.D / 32;
  for (int i = 0; i < per; ++i) q[i] = load_cache(a.q, b * a.q_sb + h * a.q_sh + lane + 32 * i, a.dtype) * a.scale * ks;
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = 0; j < len; ++j) {
    if (a.window > 0 && j < len - a.window && j >= a.sinks) continue;
    const int page = a.table[row * a.table_stride + j / a.page_size];
    if (page < 0 || page >= a.num_pages) continue;
    const int64_t at = page * a.page_stride + hk * a.head_stride + (j % a.page_size) * a.tok_stride + lane;
    float s = 0.0f;
    for (int i = 0; i < per; ++i) s = fmaf(q[i], load_cache(a.k, at + 32 * i, a.cache_dtype), s);
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.0f : mn;   // every score so far may be -inf
    const float f = expf(m - base), p = expf(s - base);
    m = mn;
    l = l * f + p;
    for (int i = 0; i < per; ++i) o[i] = o[i] * f + p * load_cache(a.v, at + 32 * i, a.cache_dtype);
  }
  for (int i = 0; i < per; ++i) {
    const float y = l > 0.0f ? o[i] / l * vs : l;
    const int64_t at = (static_cast<int64_t>(b) * a.Hq + h) * a.D + lane + 32 * i;
    if (a.dtype == CQ_DT_F16) static_cast<__half*>(a.out)[at] = __float2half_rn(y);
    else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
  }
  if (a.lse != nullptr && lane == 0) a.lse[static_cast<int64_t>(b) * a.Hq + h] = l > 0.0f ? m + logf(l) : -INFINITY;
}

int64_t paged_attention_workspace(int64_t batch, int Hq, int Hkv, int D) { return 0; }

cudaError_t launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st) {
  const dim3 grid((a.Hq + 3) / 4, a.B);
  paged_attention_kernel<<<grid, 128, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace cq
