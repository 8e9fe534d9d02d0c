// W4A16 linear for more than eight tokens: the tiles of w4a16.cu, with the tokens shared by a CTA.
//
// A CTA owns 256 weight rows, 32 for each of its eight warps, and up to 32 tokens.  With more tokens the tokens are most
// of what a tile reads, so they are brought into shared memory once per CTA and chunk of 128 columns; weights, scales,
// tokens and their sums arrive through one ring of asynchronous copies.  A warp forms q - 8 as f16 in registers (nine
// instructions per eight codes), multiplies it with every eight tokens in mma.sync tiles, and after each scale group
// adds s P + z R (P = sum x (q - 8), R = sum x) to its fp32 sums.
//
// Bound by the tiles' rate (a tile of 16 x 8 x 16 takes eight cycles of an SM's quarter): 18 tokens of a 5120 x 13824
// weight need 16 us of them with four tiles of tokens, 12 us with three.  Measured (device time, the tokens' kernel
// included): 27 us with groups of 64, 31 us with groups of 32, whose ends, s P + z R, come twice as often.
//
// The tokens come from w4a16_tokens.cu, as f16 in the order the codes are widened in, with R.  The product is launched as
// its programmatic dependent: its weights are on their way while the tokens are written.
//
// With few row tiles a cluster of CTAs splits K and adds its partial sums over distributed shared memory in rank order.
#include "decode_common.cuh"

namespace cq {

namespace w4mid {
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kRt = 2;                         // 16-row tiles of a warp
constexpr int kRows = 16 * kRt * kWarps;
constexpr int kChunk = 128;                    // columns of a ring stage
constexpr int kStages = 3;
constexpr int kWBytes = kRows * kChunk / 2;
constexpr int kScaleBytes = 544;               // 256 scales (or zeros) of a group, and room for a shift

template <int G, int NT>
struct Plan {
  static constexpr int kTokens = 8 * NT;
  static constexpr int kGroups = kChunk / G;
  static constexpr int kXAt = kWBytes;
  static constexpr int kSAt = kXAt + kTokens * 2 * kChunk;
  static constexpr int kRAt = kSAt + 2 * kGroups * kScaleBytes;
  static constexpr int kStageBytes = (kRAt + kGroups * kTokens * 4 + 255) / 256 * 256;
  static constexpr int kPartStride = kRows + 4;               // floats between tokens of a partial tile
  static constexpr int kRing = kStages * kStageBytes, kPart = kTokens * kPartStride * 4;
  static constexpr int kSmem = kRing > kPart ? kRing : kPart;
};

struct Args {
  const uint8_t* b;            // [N, K/2]
  const uint16_t* x;           // [M, K] f16, permuted
  const __nv_bfloat16* s;
  const __nv_bfloat16* z;
  const float* factor;         // [M] what a bf16 token was divided by
  const float* r;              // [token tiles][groups, padded to whole chunks][8 NT]
  const void* bias;
  void* out;
  int M, N, K, ksplit;
};
}  // namespace w4mid

template <bool F16, int G, int NT>
__global__ void __launch_bounds__(w4mid::kThreads, 2) w4a16_mid_kernel(const w4mid::Args a) {
  using namespace w4mid;
  using P = Plan<G, NT>;
  constexpr int kGroups = P::kGroups;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t ring = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int rank = a.ksplit > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int n0 = blockIdx.x * kRows, m0 = blockIdx.y * P::kTokens, mt = min(P::kTokens, a.M - m0);
  const int chunks = (a.K + kChunk - 1) / kChunk;
  const int c0 = rank * chunks / a.ksplit, c1 = (rank + 1) * chunks / a.ksplit;
  const int rows = min(kRows, a.N - n0);

  // rows past the last are copies of it (nothing of them is stored); columns past the last are zeros
  const int wr = tid >> 2;                                    // rows wr, wr + 64, ...: 16 bytes each, chunk tid & 3
  auto copy_weights = [&](int ch, int stage) {
    const uint32_t dst = ring + stage * P::kStageBytes;
    const bool ok = ch * kChunk + 32 * (tid & 3) < a.K;
#pragma unroll
    for (int i = 0; i < kRows / 64; ++i) {
      const int r = wr + 64 * i;
      const uint8_t* src = a.b + static_cast<int64_t>(n0 + min(r, rows - 1)) * (a.K >> 1) + ch * (kChunk / 2) + 16 * (tid & 3);
      cp_async16(dst + r * (kChunk / 2) + (((tid & 3) ^ (r >> 1 & 3)) << 4), ok ? src : a.b, ok);
    }
    // a warp per group and array: the aligned words that hold its scales (or zeros)
#pragma unroll
    for (int i = 0; i < (2 * kGroups + kWarps - 1) / kWarps; ++i) {
      const int k = warp + i * kWarps, grp = ch * kGroups + (k >> 1);
      if (k < 2 * kGroups && grp * G < a.K)
        cp_async_halves(dst + P::kSAt + k * kScaleBytes,
                        reinterpret_cast<const unsigned short*>(k & 1 ? a.z : a.s) + static_cast<int64_t>(grp) * a.N + n0, rows, lane);
    }
  };
  auto copy_tokens = [&](int ch, int stage) {
    const uint32_t dst = ring + stage * P::kStageBytes;
    const bool ok = ch * kChunk + 8 * (tid & 15) < a.K;
    for (int t = tid >> 4; t < P::kTokens; t += w4mid::kThreads / 16) {
      const bool here = ok && t < mt;                         // tokens past the last one are zeros
      const uint16_t* src = a.x + (here ? static_cast<int64_t>(m0 + t) * a.K + ch * kChunk + 8 * (tid & 15) : 0);
      cp_async16(dst + P::kXAt + t * (2 * kChunk) + (((tid & 15) ^ ((t & 1) << 2)) << 4), src, here);
    }
    const float* r = a.r + (static_cast<int64_t>(blockIdx.y) * chunks + ch) * kGroups * P::kTokens;
    if (tid < kGroups * P::kTokens / 4) cp_async16(dst + P::kRAt + 16 * tid, r + 4 * tid, true);
  };

  const int first = min(kStages - 1, c1 - c0);
  for (int i = 0; i < first; ++i) copy_weights(c0 + i, i);
  grid_dep_wait();                                            // the tokens and their sums are written
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < first) copy_tokens(c0 + i, i);
    cp_async_commit();
  }

  float2 acc[kRt][NT][2];                                     // rows g and g + 8 of a tile, tokens 2c and 2c + 1
#pragma unroll
  for (int t = 0; t < kRt; ++t)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[t][n][0] = acc[t][n][1] = make_float2(0.0f, 0.0f);
  const int s_odd = half_shift(reinterpret_cast<const unsigned short*>(a.s) + n0);
  const int z_odd = half_shift(reinterpret_cast<const unsigned short*>(a.z) + n0);
  const int w_at = (warp * 16 * kRt + g) * (kChunk / 2) + 4 * c, w_swz = g >> 1 & 3;
  const int x_at = P::kXAt + g * (2 * kChunk) + ((c ^ ((g & 1) << 2)) << 4);
  int stage = 0;
  for (int ch = c0; ch < c1; ++ch) {
    cp_async_wait<kStages - 2>();
    __syncthreads();                                          // the chunk is here, and the stage before it is free
    {
      const int next = ch + kStages - 1, to = stage == 0 ? kStages - 1 : stage - 1;
      if (next < c1) {
        copy_weights(next, to);
        copy_tokens(next, to);
      }
      cp_async_commit();
    }
    const uint8_t* st = smem + stage * P::kStageBytes;
    stage = stage + 1 == kStages ? 0 : stage + 1;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      if (i > 0 && (ch * kGroups + i) * G >= a.K) break;
      float p[kRt][NT][4];
#pragma unroll
      for (int b = i * (G / 32); b < (i + 1) * (G / 32); ++b) {   // 32 columns: lane c holds columns 8c .. 8c + 7
        uint32_t wp[kRt][2][4];
#pragma unroll
        for (int t = 0; t < kRt; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            widen8<true>(*reinterpret_cast<const uint32_t*>(st + w_at + ((b ^ w_swz) << 4) + (16 * t + 8 * h) * (kChunk / 2)), wp[t][h]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 v = *reinterpret_cast<const uint4*>(st + (x_at ^ (b << 6)) + n * (16 * kChunk));
#pragma unroll
          for (int t = 0; t < kRt; ++t) {
            if (b == i * (G / 32)) p[t][n][0] = p[t][n][1] = p[t][n][2] = p[t][n][3] = 0.0f;
            const uint32_t lo[4] = {wp[t][0][0], wp[t][1][0], wp[t][0][1], wp[t][1][1]};
            const uint32_t hi[4] = {wp[t][0][2], wp[t][1][2], wp[t][0][3], wp[t][1][3]};
            mma_16816<true>(p[t][n], lo, v.x, v.y);
            mma_16816<true>(p[t][n], hi, v.z, v.w);
          }
        }
      }
      const int odd = (ch * kGroups + i) & a.N & 1;           // an odd N moves every other group's values by a half
      const unsigned short* sp = reinterpret_cast<const unsigned short*>(st + P::kSAt + 2 * i * kScaleBytes) +
                                 (s_odd ^ odd) + warp * 16 * kRt + g;
      const unsigned short* zp = reinterpret_cast<const unsigned short*>(st + P::kSAt + (2 * i + 1) * kScaleBytes) +
                                 (z_odd ^ odd) + warp * 16 * kRt + g;
      float2 r[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n)
        r[n] = *reinterpret_cast<const float2*>(st + P::kRAt + (i * P::kTokens + 8 * n + 2 * c) * 4);
#pragma unroll
      for (int t = 0; t < kRt; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float s = bf16_bits_to_f32(sp[16 * t + 8 * h]), z = bf16_bits_to_f32(zp[16 * t + 8 * h]);
          const float2 s2 = make_float2(s, s), z2 = make_float2(z, z);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            acc[t][n][h] = fma2(s2, make_float2(p[t][n][2 * h], p[t][n][2 * h + 1]), fma2(z2, r[n], acc[t][n][h]));
        }
    }
  }
  cp_async_wait<0>();
  __syncthreads();                                            // the ring is free: sums as [token][row]
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int t = 0; t < kRt; ++t)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float* to = part + (8 * n + 2 * c) * P::kPartStride + (warp * kRt + t) * 16 + 8 * h + g;
        to[0] = acc[t][n][h].x;
        to[P::kPartStride] = acc[t][n][h].y;
      }
  if (a.ksplit > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
  if (tid < rows) {
    for (int m = rank; m < mt; m += a.ksplit) {
      const float factor = F16 ? 1.0f : a.factor[m0 + m];     // written while this grid may be there already: a plain load
      float y = part[m * P::kPartStride + tid];
      if (a.ksplit > 1) {
        y = 0.0f;
        for (int q = 0; q < a.ksplit; ++q) {
          float v;
          asm volatile("ld.shared::cluster.f32 %0, [%1];"
                       : "=f"(v) : "r"(mapa_shared(smem_u32(part + m * P::kPartStride + tid), q)));
          y += v;
        }
      }
      const int64_t at = static_cast<int64_t>(m0 + m) * a.N + n0 + tid;
      if constexpr (F16) {
        if (a.bias != nullptr) y += __half2float(static_cast<const __half*>(a.bias)[n0 + tid]);
        static_cast<__half*>(a.out)[at] = __float2half_rn(y);
      } else {
        y *= factor;
        if (a.bias != nullptr) y += __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[n0 + tid]);
        static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
      }
    }
  }
  if (a.ksplit > 1)                                           // a CTA's sums stay until every rank has read them
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <bool F16, int G, int NT>
cudaError_t run_w4a16_mid(const W4A16Args& a, const W4Tokens& t, cudaStream_t st) {
  using P = w4mid::Plan<G, NT>;
  auto kern = w4a16_mid_kernel<F16, G, NT>;
  static unsigned long long devices = 0;
  const cudaError_t e = allow_shared(kern, P::kSmem, devices);
  if (e != cudaSuccess) return e;
  const int tiles = (a.M + P::kTokens - 1) / P::kTokens, chunks = (a.K + w4mid::kChunk - 1) / w4mid::kChunk;
  const int row_tiles = (a.N + w4mid::kRows - 1) / w4mid::kRows;
  // K split over a cluster while that leaves no resident CTA (two per SM) without work and each has two chunks
  int ksplit = 1;
  while (ksplit < 8 && row_tiles * tiles * ksplit * 2 <= 2 * num_sms() && chunks / (2 * ksplit) >= 2) ksplit *= 2;
  const w4mid::Args args{a.b, t.x, a.s, a.z, t.factor, t.r, a.bias, a.out, a.M, a.N, a.K, ksplit};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = static_cast<unsigned>(ksplit);
  cfg.gridDim = dim3(row_tiles, tiles, ksplit);
  cfg.blockDim = dim3(w4mid::kThreads);
  cfg.dynamicSmemBytes = P::kSmem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, args);
}

}  // namespace cq
