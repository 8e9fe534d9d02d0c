// The tokens of a W4A16 product of more than eight, as its kernels read them.
//
// Codes are widened in pairs (j, j + 4) of a word, so the tokens are written with each eight columns in the order 0, 4, 1,
// 5, 2, 6, 3, 7; and R, their sums over the scale groups, once for all weight rows.  bf16 tokens become f16, each divided
// by the power of two that brings its largest element to [2^13, 2^14), which f16 holds exactly down to 2^-28 of that
// element and to 2^-38 of it below; the products are multiplied by it again at the end.
#include "decode_common.cuh"

namespace cq {

struct W4Tokens {
  const uint16_t* x;           // [M, K] f16, permuted
  const float* r;              // [token tiles][groups, padded to whole chunks][tile], or null
  const __nv_bfloat16* parts;  // [M, 128 blocks], or null
  const float* factor;         // [M] what a bf16 token was divided by
  int64_t blocks;              // of 32 groups
};

// One token per CTA: f16 columns in the order 0, 4, 1, 5, 2, 6, 3, 7 of each eight, their sums over the scale groups,
// and the power of two a bf16 token was divided by.  Sums: fp32, tokens past the last one zero; or (parts) three bf16
// values that add up to each, as columns 32 p + i of block q for part p of group 32 q + i, groups past the last zero.
template <bool F16>
__global__ void __launch_bounds__(256) w4a16_tokens_kernel(const void* x, int64_t ldx, int M, int K, int G, int ntok,
                                                           int groups_padded, uint4* xp, float* r, __nv_bfloat16* parts,
                                                           float* factor) {
  __shared__ float tops[8];
  grid_dep_launch();
  const int m = blockIdx.x, per = G / 8;                      // lanes of a group: 4, 8 or 16
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + m * ldx);
  float down = 1.0f;
  if constexpr (!F16) {
    float top = 0.0f;
    if (m < M)
      for (int c = threadIdx.x; c < K / 8; c += 256) {
        const uint4 v = src[c];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[j] << 16)), fabsf(__uint_as_float(w[j] & 0xffff0000u))));
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, tops[i]);
    // from 2^-126 on both powers are normal numbers, and the smallest bf16 becomes 2^-7; a token with an infinity keeps its
    // values and overflows
    const int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    const int by = top > 0.0f && ex < 128 ? max(ex - 13, -126) : 0;
    down = __uint_as_float(static_cast<uint32_t>(127 - by) << 23);
    if (m < M && threadIdx.x == 0) factor[m] = __uint_as_float(static_cast<uint32_t>(127 + by) << 23);
  }
  const int last = parts == nullptr ? K / 8 : max(K / 8, groups_padded * per);
  for (int c0 = 0; c0 < last; c0 += 256) {
    const int c = c0 + threadIdx.x;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (m < M && c < K / 8) v = src[c];
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (!F16) {
        const __half2 h = __floats2half2_rn(__uint_as_float(w[j] << 16) * down, __uint_as_float(w[j] & 0xffff0000u) * down);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      sum += f.x;
      sum += f.y;
    }
    if (m < M && c < K / 8)
      xp[static_cast<int64_t>(m) * (K / 8) + c] = make_uint4(__byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632),
                                                             __byte_perm(w[1], w[3], 0x5410), __byte_perm(w[1], w[3], 0x7632));
    for (int o = per / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int grp = c / per;
    if (c % per == 0 && parts == nullptr) {
      if (c < K / 8) r[(static_cast<int64_t>(m / ntok) * groups_padded + grp) * ntok + m % ntok] = sum;
    } else if (c % per == 0 && m < M && grp < groups_padded) {
      __nv_bfloat16* to = parts + static_cast<int64_t>(m) * (4 * groups_padded) + (grp >> 5) * 128 + (grp & 31);
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        const __nv_bfloat16 v = __float2bfloat16_rn(sum);
        to[32 * p] = v;
        sum -= __bfloat162float(v);
      }
    }
  }
}

namespace {
// tokens of a tile; from 33 on the tensor-memory form takes 64
int w4a16_tile(int M) { return M <= 16 ? 16 : M <= 24 ? 24 : M <= 32 ? 32 : 64; }
bool w4a16_tensor_memory(int M) { return M > 32; }
int64_t w4a16_tokens_bytes(int M, int K) { return (static_cast<int64_t>(M) * K * 2 + 255) / 256 * 256; }
int64_t w4a16_sums_bytes(int M, int K, int G) {
  if (w4a16_tensor_memory(M)) return static_cast<int64_t>(M) * ((K / G + 31) / 32) * 256;
  const int tile = w4a16_tile(M);
  return static_cast<int64_t>((M + tile - 1) / tile) * tile * ((K + 127) / 128) * (128 / G) * 4;
}
}  // namespace

bool w4a16_shares_tokens(int M) { return M > 8; }

int64_t w4a16_workspace(int M, int K, int G) {
  if (!w4a16_shares_tokens(M)) return 0;
  return w4a16_tokens_bytes(M, K) + w4a16_sums_bytes(M, K, G) + static_cast<int64_t>(M) * 4;
}

cudaError_t launch_w4a16_tokens(const W4A16Args& a, void* ws, W4Tokens& t, cudaStream_t st) {
  const bool split = w4a16_tensor_memory(a.M);
  const int tile = w4a16_tile(a.M);
  uint8_t* at = static_cast<uint8_t*>(ws);
  uint8_t* sums = at + w4a16_tokens_bytes(a.M, a.K);
  float* factor = reinterpret_cast<float*>(sums + w4a16_sums_bytes(a.M, a.K, a.group));
  float* r = split ? nullptr : reinterpret_cast<float*>(sums);
  __nv_bfloat16* parts = split ? reinterpret_cast<__nv_bfloat16*>(sums) : nullptr;
  t = W4Tokens{reinterpret_cast<const uint16_t*>(at), r, parts, factor, (a.K / a.group + 31) / 32};
  const int groups = split ? static_cast<int>(t.blocks) * 32 : (a.K + 127) / 128 * (128 / a.group);
  const int rows = split ? a.M : (a.M + tile - 1) / tile * tile;
  auto kern = a.f16 ? w4a16_tokens_kernel<true> : w4a16_tokens_kernel<false>;
  kern<<<rows, 256, 0, st>>>(a.x, a.ldx, a.M, a.K, a.group, tile, groups, reinterpret_cast<uint4*>(at), r, parts, factor);
  return cudaGetLastError();
}

}  // namespace cq
