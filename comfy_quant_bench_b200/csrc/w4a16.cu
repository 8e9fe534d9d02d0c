// W4A16 linear: 16-bit activations against packed 4-bit weights with a scale and a zero per group (the awq_w4a16
// layout the converter writes), for the few tokens of a decode step.
//
//   y[m, n] = sum_g ( s[g, n] sum_{k in g} x[m, k] (q[n, k] - 8) + z[g, n] sum_{k in g} x[m, k] ) + bias[n]
//
// Bound by reading the packed weights once: a lane has about three instructions per weight at that rate, too few to
// widen a weight to fp32 and multiply it for even one token.  So the products run as mma.sync tiles of 16 weight rows
// x 16 columns x 8 tokens whose weight operand is formed in registers, two instructions per pair of weights: a shift
// and one three-input logic operation put two 4-bit codes into the mantissas of a pair of 16-bit numbers 16 + q
// (exact).  With P = sum x (16 + q) and R = sum x over a group (R from the same tile shape against ones), the group
// adds s P + (z - 24 s) R in fp32.
//
// A CTA owns 32 weight rows and its eight warps split K in chunks of 128 columns; each warp keeps a ring of
// asynchronous copies of its weights and tokens in flight and nothing is exchanged before the end, when the partial
// sums are added in the order of the warps (equal calls give equal bits).
#include "decode_common.cuh"

namespace cq {

namespace w4a16 {
constexpr int kWarps = 8;
constexpr int kRt = 2;                     // 16-row tiles of a CTA
constexpr int kRows = 16 * kRt;
constexpr int kChunk = 128;                // columns of a ring stage
constexpr int kStages = 3;
constexpr int kWBytes = kRows * kChunk / 2;
constexpr int kRedStride = kRows + 4;      // floats between tokens of a partial tile: no bank conflicts
}  // namespace w4a16

// codes of nibbles j and j + 4 of a word as the pair 16 + q of 16-bit floats (j = 0..3)
template <bool F16>
__device__ __forceinline__ uint32_t codes16(uint32_t w, int j) {
  // bf16: the code in mantissa bits 3..6 of 2^4; f16: in bits 6..9
  const int up = (F16 ? 6 : 3) - 4 * j;
  const uint32_t v = up >= 0 ? w << up : w >> -up;
  return F16 ? ((v & 0x03C003C0u) | 0x4C004C00u) : ((v & 0x00780078u) | 0x41804180u);
}

template <bool F16, int G, int NT>
__global__ void __launch_bounds__(w4a16::kWarps * 32, 1) w4a16_kernel(const W4A16Args a, const int tokens) {
  using namespace w4a16;
  constexpr int kGroups = kChunk / G;      // scale groups of a chunk
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * kRows, m0 = blockIdx.y * tokens;
  const int mt = min(tokens, a.M - m0);                       // tokens of this tile
  const int stage_bytes = kWBytes + tokens * 2 * kChunk;
  uint8_t* ring = smem + warp * kStages * stage_bytes;
  const uint32_t ring_u = smem_u32(ring);
  const int chunks = (a.K + kChunk - 1) / kChunk;

  auto issue = [&](int ch, int stage) {
    if (ch < chunks) {
      const uint32_t dst = ring_u + stage * stage_bytes;
#pragma unroll
      for (int i = 0; i < kRt * 2; ++i) {
        const int r = 8 * i + (lane >> 2);
        const bool ok = n0 + r < a.N && ch * kChunk + 32 * c < a.K;
        const uint8_t* src = a.b + (ok ? static_cast<int64_t>(n0 + r) * (a.K >> 1) + ch * (kChunk / 2) + 16 * c : 0);
        cp_async16(dst + r * (kChunk / 2) + ((c ^ (r >> 1 & 3)) << 4), src, ok);
      }
      for (int t = lane >> 4; t < mt; t += 2) {
        const int q = lane & 15;
        const bool ok = ch * kChunk + 8 * q < a.K;
        const uint16_t* src = static_cast<const uint16_t*>(a.x) + (ok ? (m0 + t) * a.ldx + ch * kChunk + 8 * q : 0);
        cp_async16(dst + kWBytes + t * (2 * kChunk) + ((q ^ ((t & 1) << 2)) << 4), src, ok);
      }
    }
    cp_async_commit();
  };
  // scale and zero of row n0 + lane in each group of a chunk, packed
  auto load_sz = [&](int ch, uint32_t (&sz)[kGroups]) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int grp = ch * kGroups + i;
      sz[i] = 0;
      if (ch < chunks && grp * G < a.K && lane < kRows && n0 + lane < a.N) {
        const int64_t at = static_cast<int64_t>(grp) * a.N + n0 + lane;
        sz[i] = __ldg(reinterpret_cast<const unsigned short*>(a.s) + at) |
                static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(a.z) + at)) << 16;
      }
    }
  };

  float acc[kRt][NT][4] = {};
  uint32_t sz_next[kGroups];
  load_sz(warp, sz_next);
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(warp + s * kWarps, s);
  const uint32_t one = F16 ? 0x3C003C00u : 0x3F803F80u;
  const uint32_t ones[4] = {one, one, one, one};
  int stage = 0;
  for (int ch = warp; ch < chunks; ch += kWarps) {
    uint32_t sz[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) sz[i] = sz_next[i];
    load_sz(ch + kWarps, sz_next);
    cp_async_wait<kStages - 2>();
    __syncwarp();
    const uint8_t* st = ring + stage * stage_bytes;
    float p[kRt][NT][4], r[NT][4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {                             // blocks of 32 columns: lane c holds columns 8c .. 8c + 7
      if (b % (G / 32) == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            r[n][j] = 0.0f;
#pragma unroll
            for (int t = 0; t < kRt; ++t) p[t][n][j] = 0.0f;
          }
      }
      uint32_t xb[NT][4];                                     // token g's columns j and j + 4 as pairs
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int t = 8 * n + g;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (t < mt) v = *reinterpret_cast<const uint4*>(st + kWBytes + t * (2 * kChunk) + (((4 * b + c) ^ ((t & 1) << 2)) << 4));
        xb[n][0] = __byte_perm(v.x, v.z, 0x5410);
        xb[n][1] = __byte_perm(v.x, v.z, 0x7632);
        xb[n][2] = __byte_perm(v.y, v.w, 0x5410);
        xb[n][3] = __byte_perm(v.y, v.w, 0x7632);
        mma_16816<F16>(r[n], ones, xb[n][0], xb[n][1]);
        mma_16816<F16>(r[n], ones, xb[n][2], xb[n][3]);
      }
#pragma unroll
      for (int t = 0; t < kRt; ++t) {
        const int r0 = 16 * t + g, r1 = r0 + 8;
        const uint32_t w0 = *reinterpret_cast<const uint32_t*>(st + r0 * (kChunk / 2) + ((b ^ (r0 >> 1 & 3)) << 4) + 4 * c);
        const uint32_t w1 = *reinterpret_cast<const uint32_t*>(st + r1 * (kChunk / 2) + ((b ^ (r1 >> 1 & 3)) << 4) + 4 * c);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t wa[4] = {codes16<F16>(w0, 2 * h), codes16<F16>(w1, 2 * h), codes16<F16>(w0, 2 * h + 1),
                                  codes16<F16>(w1, 2 * h + 1)};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16816<F16>(p[t][n], wa, xb[n][2 * h], xb[n][2 * h + 1]);
        }
      }
      if ((b + 1) % (G / 32) == 0) {                          // the group's end
        const uint32_t mine = sz[b / (G / 32)];
#pragma unroll
        for (int t = 0; t < kRt; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t v = __shfl_sync(0xffffffffu, mine, 16 * t + 8 * h + g);
            const float s = __uint_as_float(v << 16), z = fmaf(-24.0f, s, __uint_as_float(v & 0xffff0000u));
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                acc[t][n][2 * h + j] = fmaf(s, p[t][n][2 * h + j], fmaf(z, r[n][j], acc[t][n][2 * h + j]));
          }
      }
    }
    __syncwarp();
    issue(ch + (kStages - 1) * kWarps, stage == 0 ? kStages - 1 : stage - 1);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  __syncthreads();                                            // the rings are free: partial tiles [warp][token][row]
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int t = 0; t < kRt; ++t)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        red[(warp * 8 * NT + 8 * n + 2 * c + (j & 1)) * kRedStride + 16 * t + g + 8 * (j >> 1)] = acc[t][n][j];
  __syncthreads();
  for (int i = threadIdx.x; i < mt * kRows; i += kWarps * 32) {
    const int m = i / kRows, r = i - m * kRows, n = n0 + r;
    if (n >= a.N) continue;
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) y += red[(w * 8 * NT + m) * kRedStride + r];
    const int64_t at = static_cast<int64_t>(m0 + m) * a.N + n;
    if constexpr (F16) {
      if (a.bias != nullptr) y += __half2float(static_cast<const __half*>(a.bias)[n]);
      static_cast<__half*>(a.out)[at] = __float2half_rn(y);
    } else {
      if (a.bias != nullptr) y += __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[n]);
      static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
    }
  }
}

template <bool F16, int G, int NT>
cudaError_t run_w4a16(const W4A16Args& a, cudaStream_t st) {
  using namespace w4a16;
  const int tokens = a.M < 8 * NT ? a.M : 8 * NT;
  const int ring = kWarps * kStages * (kWBytes + tokens * 2 * kChunk), red = kWarps * 8 * NT * kRedStride * 4;
  const int smem = ring > red ? ring : red;
  constexpr int kMost = kWarps * kStages * (kWBytes + 8 * NT * 2 * kChunk);
  static bool ready = false;                                  // set once; setting it twice is harmless
  if (!ready) {
    const cudaError_t e = cudaFuncSetAttribute(w4a16_kernel<F16, G, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e != cudaSuccess) return e;
    ready = true;
  }
  const dim3 grid((a.N + kRows - 1) / kRows, (a.M + tokens - 1) / tokens);
  w4a16_kernel<F16, G, NT><<<grid, kWarps * 32, smem, st>>>(a, tokens);
  return cudaGetLastError();
}

template <bool F16, int G>
cudaError_t pick_w4a16(const W4A16Args& a, cudaStream_t st) {
  return a.M <= 8 ? run_w4a16<F16, G, 1>(a, st) : run_w4a16<F16, G, 2>(a, st);
}

cudaError_t launch_w4a16(const W4A16Args& a, cudaStream_t st) {
  switch (a.group) {
    case 32: return a.f16 ? pick_w4a16<true, 32>(a, st) : pick_w4a16<false, 32>(a, st);
    case 64: return a.f16 ? pick_w4a16<true, 64>(a, st) : pick_w4a16<false, 64>(a, st);
    default: return a.f16 ? pick_w4a16<true, 128>(a, st) : pick_w4a16<false, 128>(a, st);
  }
}

}  // namespace cq
