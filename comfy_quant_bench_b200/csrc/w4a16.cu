// W4A16 linear: 16-bit activations against packed 4-bit weights with a scale and a zero per group (the awq_w4a16
// layout the converter writes), for the few tokens of a decode step.
//
//   y[m, n] = sum_g ( s[g, n] sum_{k in g} x[m, k] (q[n, k] - 8) + z[g, n] sum_{k in g} x[m, k] ) + bias[n]
//
// Simple form: one warp per output row and eight tokens, one 8-column word per lane and step, sums in fp32.
#include "kernels.cuh"

namespace cq {

namespace w4a16 {
constexpr int kWarps = 8;
constexpr int kTokens = 8;
}  // namespace w4a16

__device__ __forceinline__ float load16(const void* p, int64_t i, bool f16) {
  return f16 ? __half2float(static_cast<const __half*>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__global__ void __launch_bounds__(w4a16::kWarps * 32) w4a16_kernel(const W4A16Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * w4a16::kWarps + (threadIdx.x >> 5);
  const int m0 = blockIdx.y * w4a16::kTokens;
  if (n >= a.N) return;
  float acc[w4a16::kTokens] = {};
  const uint32_t* w = reinterpret_cast<const uint32_t*>(a.b + n * (a.K >> 1));
  for (int c = lane; c < a.K / 8; c += 32) {
    const uint32_t word = __ldg(w + c);
    const int64_t gi = static_cast<int64_t>(8 * c / a.group) * a.N + n;
    const float s = __bfloat162float(a.s[gi]), z = __bfloat162float(a.z[gi]);
    for (int t = 0; t < w4a16::kTokens; ++t) {
      if (m0 + t >= a.M) break;
      for (int j = 0; j < 8; ++j) {
        const float x = load16(a.x, (m0 + t) * a.ldx + 8 * c + j, a.f16);
        const float q = static_cast<float>(static_cast<int>((word >> (4 * j)) & 15u) - 8);
        acc[t] = fmaf(x, fmaf(q, s, z), acc[t]);
      }
    }
  }
  for (int t = 0; t < w4a16::kTokens; ++t) {
    for (int o = 16; o > 0; o >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);
    if (lane == 0 && m0 + t < a.M) {
      const float y = acc[t] + (a.bias != nullptr ? load16(a.bias, n, a.f16) : 0.0f);
      const int64_t at = (m0 + t) * static_cast<int64_t>(a.N) + n;
      if (a.f16) static_cast<__half*>(a.out)[at] = __float2half_rn(y);
      else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
    }
  }
}

cudaError_t launch_w4a16(const W4A16Args& a, cudaStream_t st) {
  const dim3 grid((a.N + w4a16::kWarps - 1) / w4a16::kWarps, (a.M + w4a16::kTokens - 1) / w4a16::kTokens);
  w4a16_kernel<<<grid, w4a16::kWarps * 32, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace cq
