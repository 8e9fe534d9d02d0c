// W4A16 linear: 16-bit activations against packed 4-bit weights with a scale and a zero per group (the awq_w4a16
// layout the converter writes), for the few tokens of a decode step.
//
//   y[m, n] = sum_g ( s[g, n] sum_{k in g} x[m, k] (q[n, k] - 8) + z[g, n] sum_{k in g} x[m, k] ) + bias[n]
//
// Bound by reading the packed weights once: a lane has about three instructions per weight at that rate, too few to
// widen a weight to fp32 and multiply it for even one token.  So the products run as mma.sync tiles of 16 weight rows
// x 16 columns x 8 tokens whose weight operand is formed in registers, about two instructions per pair of weights, as
// q - 8 (f16) or 16 + q (bf16), both exact.  With P the group's sum of x times those and R = sum x (from the same tile
// shape against ones), the group adds s P + z R (f16) or s P + (z - 24 s) R (bf16) in fp32; for bf16 the rounding is thus that
// of sum |x| (16 + q), some five times that of sum |x| |q - 8|.
//
// A CTA owns 32 weight rows and its eight warps split K in chunks of 128 columns; each warp keeps a ring of
// asynchronous copies of its weights and tokens in flight and nothing is exchanged before the end, when the partial
// sums are added in the order of the warps (equal calls give equal bits).
//
// Measured on a B200 (device time): one token at 4096 x 16384, groups of 128: 13.0 us, 2.7 TB/s; one and eight tokens at
// 8192 x 28672: 38 and 44 us, 3.2 and 2.8 TB/s; one token at 1024 x 1001: 2.5 us, launch and latency.  No unit is full: at
// the first size an SM with work issues in 54 % of its cycles, its integer pipe (forming the operands) is at 40 % and HBM at
// 42 %.  What is lost is rounds of CTAs - 512 for 296 places are two rounds for 1.73, 896 at the second size four for 3.03 -
// and a CTA's start and end, with four chunks a warp at K = 4096 through a ring of three.  At eight tokens and the second
// size 65 % and 54 %.
#include "decode_common.cuh"

namespace cq {

namespace w4a16 {
constexpr int kWarps = 8;
constexpr int kChunk = 128;                // columns of a ring stage
constexpr int kStages = 3;                 // of a warp's ring
constexpr int kRt = 2;                     // tiles of 16 weight rows of a CTA
constexpr int kRows = 16 * kRt;
constexpr int kWBytes = kRows * kChunk / 2;
constexpr int kSBytes = 128;               // scales (or zeros) of a group's rows, and room for a shift
constexpr int kRedStride = kRows + 4;      // floats between tokens of a partial tile: no bank conflicts

template <int G>
struct Plan {
  static constexpr int kGroups = kChunk / G;             // scale groups of a chunk
  static constexpr int kXAt = kWBytes + 2 * kGroups * kSBytes;
  static constexpr int stage(int tokens) { return kXAt + tokens * 2 * kChunk; }
  static constexpr int shared(int tokens) {
    const int ring = kWarps * kStages * stage(tokens), red = kWarps * 8 * kRedStride * 4;
    return ring > red ? ring : red;
  }
};
}  // namespace w4a16

template <bool F16, int G>
__global__ void __launch_bounds__(w4a16::kWarps * 32, 1) w4a16_kernel(const W4A16Args a, const int tokens) {
  using namespace w4a16;
  using P = Plan<G>;
  constexpr int kGroups = P::kGroups, kXAt = P::kXAt;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * kRows, m0 = blockIdx.y * tokens;
  const int mt = min(tokens, a.M - m0);                       // tokens of this tile
  const int stage_bytes = P::stage(tokens);
  uint8_t* ring = smem + warp * kStages * stage_bytes;
  const uint32_t ring_u = smem_u32(ring);
  const int chunks = (a.K + kChunk - 1) / kChunk;

  // What a lane copies into every stage, as addresses in the next chunk to copy.  Rows past the last are copies of it
  // (nothing of them is stored); columns past the last are zeros, in the tokens too.
  const int row_bytes = a.K >> 1;
  const uint8_t* w_src[kRt * 2];                              // 16 bytes of rows g, g + 8, ...
#pragma unroll
  for (int i = 0; i < kRt * 2; ++i)
    w_src[i] = a.b + static_cast<int64_t>(min(n0 + 8 * i + g, a.N - 1)) * row_bytes + warp * (kChunk / 2) + 16 * c;
  const uint16_t* x_src = static_cast<const uint16_t*>(a.x) + (m0 + (lane >> 4)) * a.ldx + warp * kChunk + 8 * (lane & 15);
  uintptr_t s_src = reinterpret_cast<uintptr_t>(a.s + static_cast<int64_t>(warp) * kGroups * a.N + n0);
  uintptr_t z_src = reinterpret_cast<uintptr_t>(a.z + static_cast<int64_t>(warp) * kGroups * a.N + n0);
  const int s_ends = 2 * min(kRows, a.N - n0) - 4 * lane;     // bytes of a group's scales from this lane's word on
  const uint32_t w_dst = g * (kChunk / 2) + ((c ^ (g >> 1 & 3)) << 4);
  const uint32_t x_dst = kXAt + (lane >> 4) * (2 * kChunk) + (((lane & 15) ^ ((lane >> 4) << 2)) << 4);
  int left = a.K - warp * kChunk;                             // columns from the next chunk to copy on

  // the aligned words of 16-bit values that this lane copies from `src` on; bytes past the last value are not read
  auto copy_halves = [&](uint32_t dst, uintptr_t src) {
#pragma unroll
    for (int q = 0; q <= kRows / 2; q += 32) {
      const int bytes = min(4, s_ends - 4 * q + static_cast<int>(src & 2));
      if (bytes > 0)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * (lane + q)),
                     "l"((src & ~static_cast<uintptr_t>(3)) + 4 * (lane + q)), "r"(bytes) : "memory");
    }
  };
  auto issue = [&](int stage) {
    if (left > 0) {
      const uint32_t dst = ring_u + stage * stage_bytes;
      const bool w_ok = left > 32 * c;
#pragma unroll
      for (int i = 0; i < kRt * 2; ++i) {
        cp_async16(dst + w_dst + i * (8 * kChunk / 2), w_ok ? w_src[i] : a.b, w_ok);
        w_src[i] += kWarps * (kChunk / 2);
      }
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        if (i == 0 || left > i * G) {
          copy_halves(dst + kWBytes + 2 * i * kSBytes, s_src + i * 2 * static_cast<int64_t>(a.N));
          copy_halves(dst + kWBytes + (2 * i + 1) * kSBytes, z_src + i * 2 * static_cast<int64_t>(a.N));
        }
      }
      const bool x_ok = left > 8 * (lane & 15);
      for (int t = lane >> 4; t < mt; t += 2)
        cp_async16(dst + x_dst + (t >> 1) * (4 * kChunk), x_ok ? x_src + (t >> 1) * 2 * a.ldx : a.x, x_ok);
      x_src += kWarps * kChunk;
      s_src += 2 * kWarps * kGroups * static_cast<int64_t>(a.N);
      z_src += 2 * kWarps * kGroups * static_cast<int64_t>(a.N);
      left -= kWarps * kChunk;
    }
    cp_async_commit();
  };

  float acc[kRt][4] = {};
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s);
  // where the row's scale and zero lie in a group's words: at an odd half where the group's address is one
  const int s_odd = half_shift(reinterpret_cast<const unsigned short*>(a.s) + n0);
  const int z_odd = half_shift(reinterpret_cast<const unsigned short*>(a.z) + n0);
  const int w_at = g * (kChunk / 2) + 4 * c, w_swz = g >> 1 & 3;   // rows g, g + 8, ... share their chunks' swizzle
  const int x_at = kXAt + g * (2 * kChunk) + ((c ^ ((g & 1) << 2)) << 4);
  const uint32_t one = F16 ? 0x3C003C00u : 0x3F803F80u;
  const uint32_t ones[4] = {one, one, one, one};
  int stage = 0;
  for (int ch = warp; ch < chunks; ch += kWarps) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    const uint8_t* st = ring + stage * stage_bytes;
    float p[kRt][4], r[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {                             // blocks of 32 columns: lane c holds columns 8c .. 8c + 7
      if (b % (G / 32) == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          r[j] = 0.0f;
#pragma unroll
          for (int t = 0; t < kRt; ++t) p[t][j] = 0.0f;
        }
      }
      uint4 v = make_uint4(0, 0, 0, 0);
      if (g < mt) v = *reinterpret_cast<const uint4*>(st + (x_at ^ (b << 6)));
      // token g's columns j and j + 4 as pairs
      const uint32_t xb[4] = {__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                              __byte_perm(v.y, v.w, 0x7632)};
      mma_16816<F16>(r, ones, xb[0], xb[1]);
      mma_16816<F16>(r, ones, xb[2], xb[3]);
      const uint8_t* wrow = st + w_at + ((b ^ w_swz) << 4);
#pragma unroll
      for (int t = 0; t < kRt; ++t) {
        uint32_t p0[4], p1[4];
        widen8<F16>(*reinterpret_cast<const uint32_t*>(wrow + t * (16 * kChunk / 2)), p0);
        widen8<F16>(*reinterpret_cast<const uint32_t*>(wrow + t * (16 * kChunk / 2) + 8 * kChunk / 2), p1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t wa[4] = {p0[2 * h], p1[2 * h], p0[2 * h + 1], p1[2 * h + 1]};
          mma_16816<F16>(p[t], wa, xb[2 * h], xb[2 * h + 1]);
        }
      }
      if ((b + 1) % (G / 32) == 0) {                          // the group's end
        // the scale and zero of row `lane`; past the last group there are none, and the tokens are zeros
        const int i = b / (G / 32), odd = (ch * kGroups + i) & a.N & 1;
        uint32_t mine = 0;
        if (i == 0 || (ch * kGroups + i) * G < a.K) {
          const unsigned short* sz = reinterpret_cast<const unsigned short*>(st + kWBytes + 2 * i * kSBytes) + lane;
          mine = sz[s_odd ^ odd] | static_cast<uint32_t>(sz[kSBytes / 2 + (z_odd ^ odd)]) << 16;
        }
#pragma unroll
        for (int t = 0; t < kRt; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t u = __shfl_sync(0xffffffffu, mine, 16 * t + 8 * h + g);
            const float s = __uint_as_float(u << 16), z = fmaf(-widen_offset<F16>(), s, __uint_as_float(u & 0xffff0000u));
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[t][2 * h + j] = fmaf(s, p[t][2 * h + j], fmaf(z, r[j], acc[t][2 * h + j]));
          }
      }
    }
    __syncwarp();
    issue(stage == 0 ? kStages - 1 : stage - 1);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  __syncthreads();                                            // the rings are free: partial tiles [warp][token][row]
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int t = 0; t < kRt; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      red[(warp * 8 + 2 * c + (j & 1)) * kRedStride + 16 * t + g + 8 * (j >> 1)] = acc[t][j];
  __syncthreads();
  for (int i = threadIdx.x; i < mt * kRows; i += kWarps * 32) {
    const int m = i / kRows, r = i - m * kRows, n = n0 + r;
    if (n >= a.N) continue;
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) y += red[(w * 8 + m) * kRedStride + r];
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

template <bool F16, int G>
cudaError_t run_w4a16(const W4A16Args& a, cudaStream_t st) {
  using P = w4a16::Plan<G>;
  static unsigned long long devices = 0;
  const cudaError_t e = allow_shared(w4a16_kernel<F16, G>, P::shared(8), devices);
  if (e != cudaSuccess) return e;
  const int tokens = a.M < 8 ? a.M : 8;
  w4a16_kernel<F16, G><<<dim3((a.N + w4a16::kRows - 1) / w4a16::kRows, (a.M + tokens - 1) / tokens), w4a16::kWarps * 32,
                         P::shared(tokens), st>>>(a, tokens);
  return cudaGetLastError();
}

template <bool F16, int G>
cudaError_t pick_w4a16_shared(const W4A16Args& a, const W4Tokens& t, cudaStream_t st) {
  if (w4a16_tensor_memory(a.M)) return run_w4a16_tc<F16, G>(a, t, st);
  switch (w4a16_tile(a.M)) {
    case 16: return run_w4a16_mid<F16, G, 2>(a, t, st);
    case 24: return run_w4a16_mid<F16, G, 3>(a, t, st);
    default: return run_w4a16_mid<F16, G, 4>(a, t, st);
  }
}

// Up to eight tokens this file's kernel; up to 32 the one that shares the tokens between a CTA's rows (it needs them
// written first, a launch of about 5 us); beyond, the one in tensor memory.  Us, device time, at 4096 x 4096 (groups of 128,
// bf16) and 5120 x 13824 (groups of 64, f16):
//   8 tokens: 4.9 and 15.6, shared 10.7 and 21.9;   9: shared 10.8 and 22.3;   32: shared 16.0 and 32.8
//   33: tensor memory 17.5 and 37.8, shared 18.9 and 58.0;   64: tensor memory 14.9 and 40.7, shared 23.8 and 58.6
cudaError_t launch_w4a16(const W4A16Args& a, void* ws, cudaStream_t st) {
  if (w4a16_shares_tokens(a.M)) {
    W4Tokens t;
    const cudaError_t e = launch_w4a16_tokens(a, ws, t, st);
    if (e != cudaSuccess) return e;
    switch (a.group) {
      case 32: return a.f16 ? pick_w4a16_shared<true, 32>(a, t, st) : pick_w4a16_shared<false, 32>(a, t, st);
      case 64: return a.f16 ? pick_w4a16_shared<true, 64>(a, t, st) : pick_w4a16_shared<false, 64>(a, t, st);
      default: return a.f16 ? pick_w4a16_shared<true, 128>(a, t, st) : pick_w4a16_shared<false, 128>(a, t, st);
    }
  }
  switch (a.group) {
    case 32: return a.f16 ? run_w4a16<true, 32>(a, st) : run_w4a16<false, 32>(a, st);
    case 64: return a.f16 ? run_w4a16<true, 64>(a, st) : run_w4a16<false, 64>(a, st);
    default: return a.f16 ? run_w4a16<true, 128>(a, st) : run_w4a16<false, 128>(a, st);
  }
}

}  // namespace cq
