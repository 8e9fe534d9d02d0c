// W4A16 linear: 16-bit activations against packed 4-bit weights with a scale and a zero per group (the awq_w4a16
// layout the converter writes), for the few tokens of a decode step.
//
//   y[m, n] = sum_g ( s[g, n] sum_{k in g} x[m, k] (q[n, k] - 8) + z[g, n] sum_{k in g} x[m, k] ) + bias[n]
//
// Bound by reading the packed weights once: a lane has about three instructions per weight at that rate, too few to
// widen a weight to fp32 and multiply it for even one token.  So the products run as mma.sync tiles of 16 weight rows
// x 16 columns x 8 tokens whose weight operand is formed in registers, about two instructions per pair of weights, as
// q - 8 (f16) or 16 + q (bf16), both exact.  With P the group's sum of x times those and R = sum x (from the same tile
// shape against ones), the group adds s P + z R (f16) or s P + (z - 24 s) R (bf16) in fp32.
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
constexpr int kSBytes = 80;                // scales (or zeros) of a group's 32 rows, and room for a shift
constexpr int kRedStride = kRows + 4;      // floats between tokens of a partial tile: no bank conflicts
}  // namespace w4a16

template <bool F16, int G, int NT>
__global__ void __launch_bounds__(w4a16::kWarps * 32, 1) w4a16_kernel(const W4A16Args a, const int tokens) {
  using namespace w4a16;
  constexpr int kGroups = kChunk / G;      // scale groups of a chunk
  constexpr int kXAt = kWBytes + 2 * kGroups * kSBytes;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * kRows, m0 = blockIdx.y * tokens;
  const int mt = min(tokens, a.M - m0);                       // tokens of this tile
  const int stage_bytes = kXAt + tokens * 2 * kChunk;
  const unsigned short* sp = reinterpret_cast<const unsigned short*>(a.s) + n0;
  const unsigned short* zp = reinterpret_cast<const unsigned short*>(a.z) + n0;
  uint8_t* ring = smem + warp * kStages * stage_bytes;
  const uint32_t ring_u = smem_u32(ring);
  const int chunks = (a.K + kChunk - 1) / kChunk;
  const int w_at = g * (kChunk / 2) + 4 * c, w_swz = g >> 1 & 3;   // rows g, g + 8, ... share their chunks' swizzle

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
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        const int64_t at = static_cast<int64_t>(ch * kGroups + i) * a.N;
        if ((ch * kGroups + i) * G < a.K) {
          cp_async_halves(dst + kWBytes + 2 * i * kSBytes, sp + at, min(kRows, a.N - n0), lane);
          cp_async_halves(dst + kWBytes + (2 * i + 1) * kSBytes, zp + at, min(kRows, a.N - n0), lane);
        }
      }
      for (int t = lane >> 4; t < mt; t += 2) {
        const int q = lane & 15;
        const bool ok = ch * kChunk + 8 * q < a.K;
        const uint16_t* src = static_cast<const uint16_t*>(a.x) + (ok ? (m0 + t) * a.ldx + ch * kChunk + 8 * q : 0);
        cp_async16(dst + kXAt + t * (2 * kChunk) + ((q ^ ((t & 1) << 2)) << 4), src, ok);
      }
    }
    cp_async_commit();
  };
  float acc[kRt][NT][4] = {};
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(warp + s * kWarps, s);
  const uint32_t one = F16 ? 0x3C003C00u : 0x3F803F80u;
  const uint32_t ones[4] = {one, one, one, one};
  int stage = 0;
  for (int ch = warp; ch < chunks; ch += kWarps) {
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
        if (t < mt) v = *reinterpret_cast<const uint4*>(st + kXAt + t * (2 * kChunk) + (((4 * b + c) ^ ((t & 1) << 2)) << 4));
        xb[n][0] = __byte_perm(v.x, v.z, 0x5410);
        xb[n][1] = __byte_perm(v.x, v.z, 0x7632);
        xb[n][2] = __byte_perm(v.y, v.w, 0x5410);
        xb[n][3] = __byte_perm(v.y, v.w, 0x7632);
        mma_16816<F16>(r[n], ones, xb[n][0], xb[n][1]);
        mma_16816<F16>(r[n], ones, xb[n][2], xb[n][3]);
      }
      const uint8_t* wrow = st + w_at + ((b ^ w_swz) << 4);
#pragma unroll
      for (int t = 0; t < kRt; ++t) {
        uint32_t p0[4], p1[4];
        widen8<F16>(*reinterpret_cast<const uint32_t*>(wrow + t * (16 * kChunk / 2)), p0);
        widen8<F16>(*reinterpret_cast<const uint32_t*>(wrow + t * (16 * kChunk / 2) + 8 * kChunk / 2), p1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t wa[4] = {p0[2 * h], p1[2 * h], p0[2 * h + 1], p1[2 * h + 1]};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16816<F16>(p[t][n], wa, xb[n][2 * h], xb[n][2 * h + 1]);
        }
      }
      if ((b + 1) % (G / 32) == 0) {                          // the group's end
        // scale and zero of row `lane`; past the last group there are none, and the tokens there are zeros
        const int grp = ch * kGroups + b / (G / 32);
        const int64_t at = static_cast<int64_t>(grp) * a.N;
        uint32_t mine = 0;
        if (grp * G < a.K) {
          const unsigned short* sz = reinterpret_cast<const unsigned short*>(st + kWBytes + 2 * (b / (G / 32)) * kSBytes) + lane;
          mine = sz[half_shift(sp + at)] | static_cast<uint32_t>(sz[kSBytes / 2 + half_shift(zp + at)]) << 16;
        }
#pragma unroll
        for (int t = 0; t < kRt; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t v = __shfl_sync(0xffffffffu, mine, 16 * t + 8 * h + g);
            const float s = __uint_as_float(v << 16), z = fmaf(-widen_offset<F16>(), s, __uint_as_float(v & 0xffff0000u));
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
  const int ring = kWarps * kStages * (kWBytes + 2 * (kChunk / G) * kSBytes + tokens * 2 * kChunk), red = kWarps * 8 * NT * kRedStride * 4;
  const int smem = ring > red ? ring : red;
  constexpr int kMost = kWarps * kStages * (kWBytes + 2 * (kChunk / G) * kSBytes + 8 * NT * 2 * kChunk);
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

// Up to eight tokens one tile of this kernel holds them all; beyond, w4a16_tc.cu.
cudaError_t launch_w4a16(const W4A16Args& a, void* ws, cudaStream_t st) {
  if (w4a16_uses_tc(a.M)) return launch_w4a16_tc(a, ws, st);
  switch (a.group) {
    case 32: return a.f16 ? run_w4a16<true, 32, 1>(a, st) : run_w4a16<false, 32, 1>(a, st);
    case 64: return a.f16 ? run_w4a16<true, 64, 1>(a, st) : run_w4a16<false, 64, 1>(a, st);
    default: return a.f16 ? run_w4a16<true, 128, 1>(a, st) : run_w4a16<false, 128, 1>(a, st);
  }
}

}  // namespace cq
