// W4A16 linear for more than a few tokens: the product of w4a16.cu on tcgen05 tensor cores.
//
// A CTA owns 128 weight rows and up to 64 tokens.  Thread r of four widening warps is weight row r = TMEM lane r: it
// takes its packed codes from shared memory, forms q - 8 as f16 in registers (nine instructions per eight codes) and
// stores them straight into the A operand in tensor memory, so the widened weights never pass through shared
// memory.  The tokens are the B operand, in K-major 128-byte-swizzled tiles.  Each scale group is one accumulation
// P = sum x (q - 8) in TMEM; four adding warps per 32 tokens read it back and add s P + z R to their fp32 sums, with R = sum x per group and token.  A and P are double buffered, and the roles only meet at mbarriers: a
// group's latency (copy, widening, product, read-back) is several times its work, so the roles run ahead of one
// another instead of taking turns.
//
// Codes are widened in pairs (j, j + 4) of a word, so a small kernel first writes the tokens with each eight columns in
// the order 0, 4, 1, 5, 2, 6, 3, 7 and sums the groups (R).  The product is launched as its programmatic dependent: its
// weights are on their way while the tokens are written.
//
// With few row tiles a cluster of CTAs splits K and adds its partial sums over distributed shared memory in rank order.
#include "decode_common.cuh"

namespace cq {

namespace w4tc {
constexpr int kRows = 128;
constexpr int kChunk = 128;                    // columns of a ring stage
constexpr int kAheadWarps = 4;                 // widening warps, one per TMEM lane quadrant
constexpr int kWBytes = kRows * kChunk / 2;
constexpr int kSite = 120;                     // device status sites of the waits

template <int G, int NTOK>
struct Plan {
  static constexpr int kXBytes = NTOK * kChunk * 2;
  static constexpr int kRBytes = kChunk / G * NTOK * 4;
  static constexpr int kScaleBytes = 272;                      // 128 scales (or zeros) of a group, and room for a shift
  static constexpr int kStageBytes = (kWBytes + kXBytes + kRBytes + kChunk / G * 2 * kScaleBytes + 1023) / 1024 * 1024;
  static constexpr int kStages = 100 * 1024 / kStageBytes < 8 ? 100 * 1024 / kStageBytes : 8;
  static constexpr int kSmem = kStages * kStageBytes + 1024 + 256;      // alignment, barriers
  static constexpr int kSums = NTOK < 32 ? NTOK : 32;          // tokens of an adding warp
  static constexpr int kAddWarps = 4 * (NTOK / kSums);
  static constexpr int kThreads = 32 * (kAheadWarps + kAddWarps + 3);   // and two copying warps and the multiplying one
  static_assert(kRows * NTOK * 4 <= kStages * kStageBytes, "partial sums fit the ring");
};

struct Args {
  const __nv_bfloat16* s;
  const __nv_bfloat16* z;
  const float* factor;         // [M] what a bf16 token was divided by
  const float* r;              // [token tiles][groups, padded to whole chunks][NTOK]
  const void* bias;
  void* out;
  int M, N, K, ksplit;
};
}  // namespace w4tc

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 lanes x 16 columns; the registers hold them after the wait, which names them so that no read moves before it
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld_x16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               : : "memory");
}
// D(tmem) (+)= A(tmem, 16-bit pairs per column) * B(smem desc), fp32 accumulation
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// (a.x, a.y) * (b.x, b.y) + (c.x, c.y) in one instruction, each rounded once
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
        "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// mbar_wait with its clock reads out of line: one suspending wait (0.5 ms at most) where the roles' loops run
__device__ __noinline__ bool mbar_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int where) {
  return mbar_wait(bar, parity, abort_flag, where);
}
__device__ __forceinline__ bool mbar_wait_short(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int where) {
  return mbar_try_wait(bar, parity) || mbar_wait_long(bar, parity, abort_flag, where);
}

// One token per CTA: f16 columns in the order 0, 4, 1, 5, 2, 6, 3, 7 of each eight, their sums over the scale groups,
// and the power of two a bf16 token was divided by.  Tokens past the last one get sums of zero.
template <bool F16>
__global__ void __launch_bounds__(256) w4a16_tokens_kernel(const void* x, int64_t ldx, int M, int K, int G, int ntok,
                                                           int groups_padded, uint4* xp, float* r, float* factor) {
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
    // both powers are normal numbers; a token with an infinity keeps its values and overflows
    const int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    const int by = top > 0.0f && ex < 128 ? min(max(ex - 13, -100), 114) : 0;
    down = __uint_as_float(static_cast<uint32_t>(127 - by) << 23);
    if (m < M && threadIdx.x == 0) factor[m] = __uint_as_float(static_cast<uint32_t>(127 + by) << 23);
  }
  for (int c0 = 0; c0 < K / 8; c0 += 256) {
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
    if (c < K / 8 && c % per == 0) r[(static_cast<int64_t>(m / ntok) * groups_padded + c / per) * ntok + m % ntok] = sum;
  }
}

template <bool F16, int G, int NTOK>
__global__ void __launch_bounds__(w4tc::Plan<G, NTOK>::kThreads, 2)
    w4a16_tc_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const w4tc::Args a) {
  using namespace w4tc;
  using P = Plan<G, NTOK>;
  constexpr int kStages = P::kStages, kSteps = kChunk / G, kSums = P::kSums;
  constexpr int kCopyWarp = kAheadWarps + P::kAddWarps, kScaleWarp = kCopyWarp + 1, kMmaWarp = kCopyWarp + 2;
  constexpr uint32_t kCols = 256;                             // TMEM: two P of NTOK columns, two A of G / 2
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * P::kStageBytes);
  uint64_t* empty = full + kStages;
  uint64_t* a_full = empty + kStages;                         // [2] a group's codes are in TMEM
  uint64_t* p_full = a_full + 2;                              // [2] its product is done: P to be read, A free
  uint64_t* p_empty = p_full + 2;                             // [2] P is read
  uint32_t* holder = reinterpret_cast<uint32_t*>(p_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(holder + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = a.ksplit > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int n0 = blockIdx.x * kRows, m0 = blockIdx.y * NTOK;
  const int chunks = (a.K + kChunk - 1) / kChunk;
  const int c0 = rank * chunks / a.ksplit, c1 = (rank + 1) * chunks / a.ksplit;
  const int steps = min(c1 * kSteps, a.K / G) - c0 * kSteps;  // groups of this CTA

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1 + 32);                            // the bulk copies, and each lane of the scale warp
      mbar_init(&empty[s], kAheadWarps + P::kAddWarps + 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&a_full[b], kAheadWarps);
      mbar_init(&p_full[b], 1);
      mbar_init(&p_empty[b], P::kAddWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(holder, kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t d_col = *holder, a_col = d_col + 2 * NTOK;
  const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;    // the warp's quadrant of TMEM lanes
  const int row = (warp & 3) * 32 + lane, n = n0 + row;       // this thread's weight row (widening and adding warps)
  float2 acc[kSums / 2];
#pragma unroll
  for (int j = 0; j < kSums / 2; ++j) acc[j] = make_float2(0.0f, 0.0f);
  const int first_sum = warp >= kAheadWarps && warp < kCopyWarp ? (warp - kAheadWarps) / 4 * kSums : 0;   // of the tile's tokens

  if (warp == kCopyWarp) {
    if (lane == 0) {
      // ---- codes, tokens and group sums of a chunk per stage ----
      auto weights = [&](int ch, int s) {
        mbar_arrive_expect_tx(&full[s], kWBytes + P::kXBytes + P::kRBytes);
        tma_load_2d(smem + s * P::kStageBytes + P::kXBytes, &tm_w, &full[s], ch * (kChunk / 2), n0);
      };
      auto rest = [&](int ch, int s) {
        uint8_t* st = smem + s * P::kStageBytes;
        tma_load_2d(st, &tm_x, &full[s], ch * kChunk * 2, m0);
        tma_load_2d(st + P::kXBytes / 2, &tm_x, &full[s], ch * kChunk * 2 + 128, m0);
        const int64_t at = (static_cast<int64_t>(blockIdx.y) * chunks + ch) * kSteps * NTOK;
        bulk_load(st + P::kXBytes + kWBytes, a.r + at, P::kRBytes, &full[s]);
      };
      const int first = min(kStages, c1 - c0);
      for (int i = 0; i < first; ++i) weights(c0 + i, i);
      grid_dep_wait();                                        // the tokens and their sums are written
      for (int i = 0; i < first; ++i) rest(c0 + i, i);
      uint32_t issued = first, phase = 0;
      int s = 0;
      for (int ch = c0 + first; ch < c1; ++ch) {
        if (!mbar_wait_short(&empty[s], phase, abort_flag, kSite)) break;
        weights(ch, s);
        rest(ch, s);
        ++issued;
        if (++s == kStages) { s = 0; phase ^= 1u; }
      }
      drain_ring(full, kStages, issued, 50000000ull);
    }
    __syncwarp();
  } else if (warp == kScaleWarp) {
    // ---- scales and zeros of a chunk's groups, any alignment (rows of N 16-bit values) ----
    uint32_t phase = 1;
    int s = 0;
    for (int ch = c0; ch < c1; ++ch) {
      if (!mbar_wait_short(&empty[s], phase, abort_flag, kSite + 8)) break;
      const uint32_t dst = smem_u32(smem + s * P::kStageBytes + P::kXBytes + kWBytes + P::kRBytes);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int grp = ch * kSteps + i;
        if (grp * G >= a.K) break;
        const int64_t at = static_cast<int64_t>(grp) * a.N + n0;
        const int count = min(kRows, a.N - n0);
        cp_async_halves(dst + 2 * i * P::kScaleBytes, reinterpret_cast<const unsigned short*>(a.s) + at, count, lane);
        cp_async_halves(dst + (2 * i + 1) * P::kScaleBytes, reinterpret_cast<const unsigned short*>(a.z) + at, count, lane);
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[s])) : "memory");
      if (++s == kStages) { s = 0; phase ^= 1u; }
    }
    cp_async_wait_all();
  } else if (warp == kMmaWarp) {
    // ---- products: a group's P = codes x tokens ----
    constexpr uint32_t idesc =
        (1u << 4) | (static_cast<uint32_t>(NTOK >> 3) << 17) | (8u << 24);   // f32 += f16 x f16, M = 128
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < steps && ok; ++stage, phase ^= stage == kStages, stage = stage == kStages ? 0 : stage) {
      if (!(ok = mbar_wait_short(&full[stage], phase, abort_flag, kSite + 1))) break;
      const uint64_t x = smem_desc_k_sw128(smem_u32(smem + stage * P::kStageBytes));
#pragma unroll
      for (int sub = 0; sub < kSteps; ++sub) {
        if (i >= steps || !ok) break;
        const int buf = i & 1;
        if (!(ok = mbar_wait_short(&p_empty[buf], ((i >> 1) & 1) ^ 1u, abort_flag, kSite + 2))) break;
        if (!(ok = mbar_wait_short(&a_full[buf], (i >> 1) & 1, abort_flag, kSite + 3))) break;
        tc_fence_after();
        if (lane == 0) {
#pragma unroll
          for (int k = 0; k < G / 16; ++k) {
            const int col = sub * G + 16 * k;                 // 64 columns per 128-byte-wide half
            mma_f16_ts(d_col + buf * NTOK, a_col + buf * (G / 2) + 8 * k,
                       x + ((col >> 6) * (P::kXBytes / 2) + (col & 63) * 2) / 16, idesc, k != 0);
          }
          tc_commit(&p_full[buf]);
          if (sub == kSteps - 1) tc_commit(&empty[stage]);
        }
        __syncwarp();
        issued = ++i;
      }
    }
    // after a wait that ran out: the products in flight end before TMEM and the ring go away
    if (!ok && lane == 0)
      for (int i = max(issued - 2, 0); i < issued; ++i) mbar_wait_drain(&p_full[i & 1], (i >> 1) & 1, 50000000ull);
    __syncwarp();
  } else if (warp < kAheadWarps) {
    // ---- codes of a group, widened into the A operand ----
    const uint8_t* w = smem + P::kXBytes + row * 64;
    const int sw = (row >> 1 & 3) << 4;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < steps && ok; ++stage, phase ^= stage == kStages, stage = stage == kStages ? 0 : stage) {
      if (!mbar_wait_short(&full[stage], phase, abort_flag, kSite + 4)) break;
#pragma unroll
      for (int sub = 0; sub < kSteps; ++sub) {
        if (i >= steps) break;
        const int buf = i & 1;
        uint4 codes[G / 32];
#pragma unroll
        for (int b = 0; b < G / 32; ++b)                      // 32 columns: 16 bytes
          codes[b] = *reinterpret_cast<const uint4*>(w + stage * P::kStageBytes + (((sub * (G / 32) + b) << 4) ^ sw));
        // A's buffer is free when the product of the group two before is done
        if (!(ok = mbar_wait_short(&p_full[buf], ((i >> 1) & 1) ^ 1u, abort_flag, kSite + 5))) break;
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int b = 0; b < G / 32; ++b) {
          const uint32_t v[4] = {codes[b].x, codes[b].y, codes[b].z, codes[b].w};
          uint32_t pairs[16];
#pragma unroll
          for (int j = 0; j < 4; ++j) widen8<true>(v[j], reinterpret_cast<uint32_t(&)[4]>(pairs[4 * j]));
          tmem_st_x16(a_col + buf * (G / 2) + 16 * b + lane_base, pairs);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&a_full[buf]);
          if (sub == kSteps - 1) mbar_arrive(&empty[stage]);
        }
        ++i;
      }
    }
  } else {
    // ---- a group's product, scaled and added ----
    // places of the row's scale and zero: a group's values begin at an odd half where its address does
    const int s_odd = half_shift(reinterpret_cast<const unsigned short*>(a.s) + n0);
    const int z_odd = half_shift(reinterpret_cast<const unsigned short*>(a.z) + n0);
    const int flip = a.N & 1;
    const uint8_t* base = smem + P::kXBytes + kWBytes;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < steps && ok; ++stage, phase ^= stage == kStages, stage = stage == kStages ? 0 : stage) {
      if (!mbar_wait_short(&full[stage], phase, abort_flag, kSite + 6)) break;
      const uint8_t* sums = base + stage * P::kStageBytes;
#pragma unroll
      for (int sub = 0; sub < kSteps; ++sub) {
        if (i >= steps) break;
        const int buf = i & 1, odd = (c0 * kSteps + i) & flip;
        const float4* r4 = reinterpret_cast<const float4*>(sums + (sub * NTOK + first_sum) * 4);
        const unsigned short* sz = reinterpret_cast<const unsigned short*>(sums + P::kRBytes + 2 * sub * P::kScaleBytes) + row;
        const float sf = bf16_bits_to_f32(sz[s_odd ^ odd]), zf = bf16_bits_to_f32(sz[P::kScaleBytes / 2 + (z_odd ^ odd)]);
        const float2 s2 = make_float2(sf, sf), z2 = make_float2(zf, zf);
        if (!(ok = mbar_wait_short(&p_full[buf], (i >> 1) & 1, abort_flag, kSite + 7))) break;
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < kSums / 16; ++q) {
          uint32_t v[16];
          tmem_ld_x16(d_col + buf * NTOK + first_sum + 16 * q + lane_base, v);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 r = r4[4 * q + j];
            acc[8 * q + 2 * j] = fma2(z2, make_float2(r.x, r.y), acc[8 * q + 2 * j]);
            acc[8 * q + 2 * j + 1] = fma2(z2, make_float2(r.z, r.w), acc[8 * q + 2 * j + 1]);
          }
          tmem_wait_ld_x16(v);
          if (q == kSums / 16 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&p_empty[buf]);
              if (sub == kSteps - 1) mbar_arrive(&empty[stage]);
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            acc[8 * q + j] = fma2(s2, make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), acc[8 * q + j]);
        }
        ++i;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(d_col, kCols);
  }

  auto store = [&](int m, int col, float y) {
    const int64_t at = static_cast<int64_t>(m) * a.N + col;
    if constexpr (F16) {
      if (a.bias != nullptr) y += __half2float(static_cast<const __half*>(a.bias)[col]);
      static_cast<__half*>(a.out)[at] = __float2half_rn(y);
    } else {
      y *= __ldg(a.factor + m);
      if (a.bias != nullptr) y += __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[col]);
      static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
    }
  };
  const bool adds = warp >= kAheadWarps && warp < kCopyWarp;
  const int mt = min(NTOK, a.M - m0);
  if (a.ksplit == 1) {
    if (adds && n < a.N) {
#pragma unroll
      for (int j = 0; j < kSums; ++j)
        if (first_sum + j < mt) store(m0 + first_sum + j, n, j & 1 ? acc[j / 2].y : acc[j / 2].x);
    }
    return;
  }
  // ---- partial sums of the cluster: [token][row] in each CTA's ring, added in rank order ----
  float* part = reinterpret_cast<float*>(smem);
  if (adds) {
#pragma unroll
    for (int j = 0; j < kSums; ++j) part[(first_sum + j) * kRows + row] = j & 1 ? acc[j / 2].y : acc[j / 2].x;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (adds && n < a.N) {
    for (int m = rank + first_sum / kSums * a.ksplit; m < mt; m += a.ksplit * (P::kAddWarps / 4)) {
      float y = 0.0f;
      for (int q = 0; q < a.ksplit; ++q) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(part + m * kRows + row), q)));
        y += v;
      }
      store(m0 + m, n, y);
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

namespace {
int w4a16_tile(int M) { return M <= 16 ? 16 : M <= 32 ? 32 : 64; }
int64_t w4a16_groups_padded(int K, int G) { return static_cast<int64_t>((K + 127) / 128) * (128 / G); }
bool w4a16_map(CUtensorMap* map, const void* base, int64_t rows, int64_t bytes, int box_bytes, int box_rows, CUtensorMapSwizzle sw) {
  EncodeTiledFn fn = get_encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(bytes), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(bytes)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_bytes), static_cast<cuuint32_t>(box_rows)}, estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}
}  // namespace

bool w4a16_uses_tc(int M) { return M > 8; }

int64_t w4a16_workspace(int M, int K, int G) {
  if (!w4a16_uses_tc(M)) return 0;
  const int tile = w4a16_tile(M);
  const int64_t tokens = (static_cast<int64_t>(M) * K * 2 + 255) / 256 * 256;
  return tokens + static_cast<int64_t>((M + tile - 1) / tile) * tile * (w4a16_groups_padded(K, G) + 1) * 4;
}

template <bool F16, int G, int NTOK>
cudaError_t run_w4a16_tc(const W4A16Args& a, void* ws, cudaStream_t st) {
  using P = w4tc::Plan<G, NTOK>;
  auto kern = w4a16_tc_kernel<F16, G, NTOK>;
  static unsigned long long devices = 0;
  cudaError_t e = allow_shared(kern, P::kSmem, devices);
  if (e != cudaSuccess) return e;
  const int tiles = (a.M + NTOK - 1) / NTOK, chunks = (a.K + w4tc::kChunk - 1) / w4tc::kChunk;
  const int groups = static_cast<int>(w4a16_groups_padded(a.K, G));
  uint4* xp = static_cast<uint4*>(ws);
  float* r = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + (static_cast<int64_t>(a.M) * a.K * 2 + 255) / 256 * 256);
  float* factor = r + static_cast<int64_t>(tiles) * NTOK * groups;
  CUtensorMap tm_w, tm_x;
  if (!w4a16_map(&tm_w, a.b, a.N, a.K / 2, 64, w4tc::kRows, CU_TENSOR_MAP_SWIZZLE_64B) ||
      !w4a16_map(&tm_x, xp, a.M, static_cast<int64_t>(a.K) * 2, 128, NTOK, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  w4a16_tokens_kernel<F16><<<tiles * NTOK, 256, 0, st>>>(a.x, a.ldx, a.M, a.K, G, NTOK, groups, xp, r, factor);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int row_tiles = (a.N + w4tc::kRows - 1) / w4tc::kRows;
  // K split over a cluster while the grid leaves half of the resident CTAs (two per SM) idle and each still has four
  // chunks
  int ksplit = 1;
  while (ksplit < 8 && row_tiles * tiles * ksplit * 2 <= 2 * num_sms() && chunks / (2 * ksplit) >= 4) ksplit *= 2;
  const w4tc::Args args{a.s, a.z, factor, r, a.bias, a.out, a.M, a.N, a.K, ksplit};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = static_cast<unsigned>(ksplit);
  cfg.gridDim = dim3(row_tiles, tiles, ksplit);
  cfg.blockDim = dim3(P::kThreads);
  cfg.dynamicSmemBytes = P::kSmem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, tm_w, tm_x, args);
}

template <bool F16, int G>
cudaError_t pick_w4a16_tc(const W4A16Args& a, void* ws, cudaStream_t st) {
  switch (w4a16_tile(a.M)) {
    case 16: return run_w4a16_tc<F16, G, 16>(a, ws, st);
    case 32: return run_w4a16_tc<F16, G, 32>(a, ws, st);
    default: return run_w4a16_tc<F16, G, 64>(a, ws, st);
  }
}

cudaError_t launch_w4a16_tc(const W4A16Args& a, void* ws, cudaStream_t st) {
  switch (a.group) {
    case 32: return a.f16 ? pick_w4a16_tc<true, 32>(a, ws, st) : pick_w4a16_tc<false, 32>(a, ws, st);
    case 64: return a.f16 ? pick_w4a16_tc<true, 64>(a, ws, st) : pick_w4a16_tc<false, 64>(a, ws, st);
    default: return a.f16 ? pick_w4a16_tc<true, 128>(a, ws, st) : pick_w4a16_tc<false, 128>(a, ws, st);
  }
}

}  // namespace cq
