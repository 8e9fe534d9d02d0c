// W4A16 linear for more than a few tokens: the product of w4a16.cu on tcgen05 tensor cores.
//
// A CTA owns 128 weight rows and up to 64 tokens.  Thread r of four widening warps is weight row r = TMEM lane r: it
// takes its packed codes from shared memory, forms q - 8 as f16 in registers (nine instructions per eight codes) and
// stores them straight into the A operand in tensor memory, so the widened weights never pass through shared
// memory.  The tokens are the B operand, in K-major 128-byte-swizzled tiles.  Each scale group is one accumulation
// P = sum x (q - 8) in TMEM; four adding warps per 32 tokens read it back and add s P to their fp32 sums.  The zeros'
// term, sum over the groups of z R with R = sum x, is one more product of bf16 zeros and R in three bf16 parts, before the
// groups'.  A and P are double buffered, and the roles only meet at mbarriers: a group's latency (copy, widening,
// product, read-back) is several times its work, so the roles run ahead of one another instead of taking turns.  Codes
// and tokens have rings of their own, since codes are free again as soon as they are widened, and scales are loaded
// straight into registers, four groups ahead (together 82 -> 75 us at the first size below).
//
// The tokens come from w4a16_tokens.cu, as f16 in the order the codes are widened in, with R's parts.  The product is
// launched as its programmatic dependent: its weights are on their way while the tokens are written.
//
// Measured on a B200 (device time, the tokens' kernel included): 64 tokens at 8192 x 28672, groups of 128: 66 us, 450
// TFLOP/s; at 5120 x 13824, groups of 64: 41 us (f16) and 42 us (bf16).  Bound by the hand-overs from one role to the next
// at each group: an SM with two CTAs issues in two thirds of its slots, the polling of waiting warps among them, has its
// integer pipe half and its tensor pipe a third full, and its warps stall at the mbarriers more than anywhere else.
//
// With few row tiles a cluster of CTAs splits K and adds its partial sums over distributed shared memory in rank order.
#include "decode_common.cuh"

namespace cq {

namespace w4tc {
constexpr int kRows = 128;
constexpr int kChunk = 128;                    // columns of a ring stage
constexpr int kTokens = 64;                    // of a CTA
constexpr int kAheadWarps = 4;                 // widening warps, one per TMEM lane quadrant
constexpr int kWBytes = kRows * kChunk / 2;
constexpr int kAheadScales = 4;
constexpr int kSite = 120;                     // device status sites of the waits
constexpr int kTokenBytes = kTokens * kChunk * 2;
constexpr int kXStages = 3, kWStages = 7;
constexpr int kRing = kXStages * kTokenBytes + kWStages * kWBytes;
constexpr int kSmem = kRing + 1024 + 256;      // alignment, barriers
constexpr int kSums = 32;                      // tokens of an adding warp
constexpr int kAddWarps = 4 * (kTokens / kSums);
constexpr int kThreads = 32 * (kAheadWarps + kAddWarps + 2);   // and the copying and the multiplying warp
static_assert(kRows * kTokens * 4 <= kRing, "partial sums fit the rings");
static_assert(kWStages >= kXStages, "the copying warp's order");

struct Args {
  const __nv_bfloat16* s;
  const __nv_bfloat16* z;
  const float* factor;         // [M] what a bf16 token was divided by
  const void* bias;
  void* out;
  int M, N, K, ksplit;
};
}  // namespace w4tc

template <bool F16, int G>
__global__ void __launch_bounds__(w4tc::kThreads, 2)
    w4a16_tc_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                    const __grid_constant__ CUtensorMap tm_r, const w4tc::Args a) {
  using namespace w4tc;
  constexpr int kSteps = kChunk / G;                          // scale groups of a chunk
  constexpr int kCopyWarp = kAheadWarps + kAddWarps, kMmaWarp = kCopyWarp + 1;
  constexpr uint32_t kCols = 256;                             // TMEM: two P of kTokens columns, A's buffers in the rest
  static_assert(2 * kTokens + 128 <= kCols, "two 128-column A operands");
  extern __shared__ __align__(128) uint8_t smem_any[];
  uint8_t* smem = smem_any + ((1024 - (smem_u32(smem_any) & 1023)) & 1023);
  uint8_t* codes_at = smem + kXStages * kTokenBytes;              // the ring of codes comes after the tokens'
  uint64_t* x_full = reinterpret_cast<uint64_t*>(smem + kRing);
  uint64_t* x_empty = x_full + kXStages;
  uint64_t* w_full = x_empty + kXStages;
  uint64_t* w_empty = w_full + kWStages;
  uint64_t* a_full = w_empty + kWStages;                      // [2] an operand's codes (or zeros) are in TMEM
  uint64_t* p_full = a_full + 2;                              // [2] a product is done: P to be read, A free
  uint64_t* p_empty = p_full + 2;                             // [2] P is read
  uint64_t* z_done = p_empty + 2;                             // [2] A's buffer of the zeros' product is free
  uint32_t* holder = reinterpret_cast<uint32_t*>(z_done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(holder + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = a.ksplit > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int n0 = blockIdx.x * kRows, m0 = blockIdx.y * kTokens;
  const int chunks = (a.K + kChunk - 1) / kChunk;
  const int c0 = rank * chunks / a.ksplit, c1 = (rank + 1) * chunks / a.ksplit;
  const int steps = min(c1 * kSteps, a.K / G) - c0 * kSteps;  // groups of this CTA
  // the zeros' term sum_g z R: products of 32 groups each, this rank's share of them; they come before the groups'
  const int blocks = (a.K / G + 31) / 32, z0 = rank * blocks / a.ksplit, z1 = (rank + 1) * blocks / a.ksplit;
  const int nz = z1 - z0;

  if (tid == 0) {
    for (int s = 0; s < kXStages; ++s) {
      mbar_init(&x_full[s], 1);
      mbar_init(&x_empty[s], 1);
    }
    for (int s = 0; s < kWStages; ++s) {
      mbar_init(&w_full[s], 1);
      mbar_init(&w_empty[s], kAheadWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&a_full[b], kAheadWarps);
      mbar_init(&p_full[b], 1);
      mbar_init(&p_empty[b], kAddWarps);
      mbar_init(&z_done[b], 1);
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
  const uint32_t d_col = *holder, a_col = d_col + 2 * kTokens;
  const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;    // the warp's quadrant of TMEM lanes
  const int row = (warp & 3) * 32 + lane, n = n0 + row;       // this thread's weight row (widening and adding warps)
  float2 acc[kSums / 2];
#pragma unroll
  for (int j = 0; j < kSums / 2; ++j) acc[j] = make_float2(0.0f, 0.0f);
  const int first_sum = warp >= kAheadWarps && warp < kCopyWarp ? (warp - kAheadWarps) / 4 * kSums : 0;   // of the tile's tokens

  if (warp == kCopyWarp) {
    // ---- a ring of codes, freed when they are widened, and one of tokens (the zeros' nz blocks of sums first), freed by
    // the products ----
    const int wloads = c1 - c0, xloads = nz + wloads;
    int wi = 0, ws = 0, xi = 0, xs = 0;
    auto codes = [&]() {
      mbar_arrive_expect_tx(&w_full[ws], kWBytes);
      tma_load_2d(codes_at + ws * kWBytes, &tm_w, &w_full[ws], (c0 + wi) * (kChunk / 2), n0);
      ++wi;
      if (++ws == kWStages) ws = 0;
    };
    auto tokens = [&]() {
      uint8_t* st = smem + xs * kTokenBytes;
      const CUtensorMap* map = xi < nz ? &tm_r : &tm_x;
      const int at = (xi < nz ? z0 + xi : c0 + xi - nz) * kChunk * 2;
      mbar_arrive_expect_tx(&x_full[xs], kTokenBytes);
      tma_load_2d(st, map, &x_full[xs], at, m0);
      tma_load_2d(st + kTokenBytes / 2, map, &x_full[xs], at + 128, m0);
      ++xi;
      if (++xs == kXStages) xs = 0;
    };
    if (lane == 0) {
      while (wi < min(kWStages, wloads)) codes();             // no earlier kernel writes them
      grid_dep_wait();                                        // the tokens and their sums are written
      while (xi < min(kXStages, xloads)) tokens();
      // one after the other: a block's codes are widened before its product is done
      while (wi < wloads || xi < xloads) {
        if (wi < wloads && xi - kXStages - nz >= wi - kWStages) {
          if (!mbar_wait_short(&w_empty[ws], ((wi / kWStages) & 1) ^ 1u, abort_flag, kSite)) break;
          codes();
        }
        if (xi < xloads) {
          if (!mbar_wait_short(&x_empty[xs], ((xi / kXStages) & 1) ^ 1u, abort_flag, kSite + 1)) break;
          tokens();
        }
      }
      drain_ring(w_full, kWStages, wi, 50000000ull);
      drain_ring(x_full, kXStages, xi, 50000000ull);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---- products: the zeros' first, then each group's P = codes x tokens.  One thread, which neither waits for the
    // warp's other lanes nor makes them poll: it paces the CTA ----
    if (elect_one()) {
      constexpr uint32_t shape = (1u << 4) | (static_cast<uint32_t>(kTokens >> 3) << 17) | (8u << 24);   // f32, M = 128
      constexpr uint32_t idesc_z = shape | (1u << 7) | (1u << 10);                                    // bf16 x bf16
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      auto next_stage = [&]() {
        if (++stage == kXStages) { stage = 0; phase ^= 1u; }
      };
      for (int j = 0; j < nz; ++j) {
        const int buf = j & 1;
        ok = ok && mbar_wait_short(&x_full[stage], phase, abort_flag, kSite + 2) &&
             mbar_wait_short(&a_full[buf], (j >> 1) & 1, abort_flag, kSite + 3);
        if (!ok) break;
        tc_fence_after();
        const uint64_t x = smem_desc_k_sw128(smem_u32(smem + stage * kTokenBytes));
#pragma unroll
        for (int k = 0; k < 6; ++k) {                         // three parts of 32 sums; the last 32 columns are empty
          const int col = 16 * k;
          mma_f16_ts(d_col, a_col + buf * 64 + 8 * k, x + ((col >> 6) * (kTokenBytes / 2) + (col & 63) * 2) / 16, idesc_z,
                     j + k != 0);
        }
        tc_commit(&z_done[buf]);
        tc_commit(&x_empty[stage]);
        if (j + 1 == nz) tc_commit(&p_full[0]);
        issued = 1;
        next_stage();
      }
      if (nz == 0) mbar_arrive(&p_full[0]);
      // product i (0: the zeros', 1 ..: the groups') takes P buffer i & 1; a_full goes on counting from the zeros' blocks
      for (int i = 1; i <= steps && ok; next_stage()) {
        if (!(ok = mbar_wait_short(&x_full[stage], phase, abort_flag, kSite + 4))) break;
        const uint64_t x = smem_desc_k_sw128(smem_u32(smem + stage * kTokenBytes));
#pragma unroll
        for (int sub = 0; sub < kSteps; ++sub) {
          if (i > steps) break;
          const int buf = i & 1, use = nz + i - 1;
          ok = mbar_wait_short(&p_empty[buf], ((i >> 1) & 1) ^ 1u, abort_flag, kSite + 5) &&
               mbar_wait_short(&a_full[use & 1], (use >> 1) & 1, abort_flag, kSite + 6);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < G / 16; ++k) {
            const int col = sub * G + 16 * k;                 // 64 columns per 128-byte-wide half
            mma_f16_ts(d_col + buf * kTokens, a_col + (use & 1) * 64 + 8 * k,
                       x + ((col >> 6) * (kTokenBytes / 2) + (col & 63) * 2) / 16, shape, k != 0);
          }
          tc_commit(&p_full[buf]);
          if (sub == kSteps - 1) tc_commit(&x_empty[stage]);
          issued = ++i;
        }
      }
      // after a wait that ran out: the products in flight end before TMEM and the ring go away
      if (!ok) {
        for (int j = max(nz - 2, 0); j < nz && issued <= 1; ++j) mbar_wait_drain(&z_done[j & 1], (j >> 1) & 1, 50000000ull);
        for (int i = max(issued - 2, 0); i < issued; ++i) mbar_wait_drain(&p_full[i & 1], (i >> 1) & 1, 50000000ull);
      }
    }
    __syncwarp();
  } else if (warp < kAheadWarps) {
    // ---- operands: 32 groups' zeros, three times, then each group's codes widened ----
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto hand_over = [&](int buf) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_full[buf]);
    };
    for (int j = 0; j < nz && ok; ++j) {
      const int buf = j & 1;
      uint32_t pairs[16];
      const unsigned short* zp = reinterpret_cast<const unsigned short*>(a.z) + static_cast<int64_t>(z0 + j) * 32 * a.N + n;
      const int left = n < a.N ? a.K / G - (z0 + j) * 32 : 0;
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const uint32_t lo = 2 * q < left ? __ldg(zp + static_cast<int64_t>(2 * q) * a.N) : 0;
        const uint32_t hi = 2 * q + 1 < left ? __ldg(zp + static_cast<int64_t>(2 * q + 1) * a.N) : 0;
        pairs[q] = lo | hi << 16;
      }
      if (j >= 2 && !(ok = mbar_wait_short(&z_done[buf], ((j - 2) >> 1) & 1, abort_flag, kSite + 7))) break;
      __syncwarp();
      tc_fence_after();
#pragma unroll
      for (int part = 0; part < 3; ++part) tmem_st_x16(a_col + buf * 64 + 16 * part + lane_base, pairs);
      hand_over(buf);
    }
    const uint8_t* w = codes_at + row * 64;
    const int sw = (row >> 1 & 3) << 4;
    for (int i = 1; i <= steps && ok;) {
      if (!(ok = mbar_wait_short(&w_full[stage], phase, abort_flag, kSite + 8))) break;
#pragma unroll
      for (int sub = 0; sub < kSteps; ++sub) {
        if (i > steps) break;
        const int buf = (nz + i - 1) & 1;
        uint4 codes[G / 32];
#pragma unroll
        for (int b = 0; b < G / 32; ++b)                      // 32 columns: 16 bytes
          codes[b] = *reinterpret_cast<const uint4*>(w + stage * kWBytes + (((sub * (G / 32) + b) << 4) ^ sw));
        auto widen = [&](int b, uint32_t (&pairs)[16]) {
          const uint32_t v[4] = {codes[b].x, codes[b].y, codes[b].z, codes[b].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) widen8<true>(v[j], reinterpret_cast<uint32_t(&)[4]>(pairs[4 * j]));
        };
        uint32_t first[16];
        widen(0, first);
        if (sub == kSteps - 1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&w_empty[stage]);
        }
        // A's buffer is free when the product two before is done; the zeros' products took both
        const int free_at = i <= 2 ? 0 : i - 2;
        if ((i > 2 || nz > 0) && !(ok = mbar_wait_short(&p_full[free_at & 1], (free_at >> 1) & 1, abort_flag, kSite + 9))) break;
        __syncwarp();
        tc_fence_after();
        tmem_st_x16(a_col + buf * 64 + lane_base, first);
#pragma unroll
        for (int b = 1; b < G / 32; ++b) {
          uint32_t pairs[16];
          widen(b, pairs);
          tmem_st_x16(a_col + buf * 64 + 16 * b + lane_base, pairs);
        }
        hand_over(buf);
        ++i;
      }
      if (++stage == kWStages) { stage = 0; phase ^= 1u; }
    }
  } else {
    // ---- the zeros' product, and each group's scaled, added up; scales are loaded kAheadScales groups ahead ----
    const unsigned short* sp = reinterpret_cast<const unsigned short*>(a.s) + static_cast<int64_t>(c0) * kSteps * a.N + min(n, a.N - 1);
    uint32_t scales[kAheadScales];
#pragma unroll
    for (int u = 0; u < kAheadScales; ++u) scales[u] = u < steps ? __ldg(sp + static_cast<int64_t>(u) * a.N) : 0;
    bool ok = true;
    auto add = [&](int i, float scale) {
      const int buf = i & 1;
      if (!(ok = mbar_wait_short(&p_full[buf], (i >> 1) & 1, abort_flag, kSite + 10))) return;
      __syncwarp();
      tc_fence_after();
      const float2 s2 = make_float2(scale, scale);
#pragma unroll
      for (int q = 0; q < kSums / 16; ++q) {
        uint32_t v[16];
        tmem_ld_x16(d_col + buf * kTokens + first_sum + 16 * q + lane_base, v);
        tmem_wait_ld_x16(v);
        if (q == kSums / 16 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_empty[buf]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          acc[8 * q + j] = fma2(s2, make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), acc[8 * q + j]);
      }
    };
    if (nz > 0) add(0, 1.0f);
    else if (lane == 0) mbar_arrive(&p_empty[0]);             // product 0 has nothing in it
    for (int i = 0; i < steps && ok; i += kAheadScales) {
#pragma unroll
      for (int u = 0; u < kAheadScales; ++u) {
        if (i + u >= steps || !ok) break;
        add(i + u + 1, bf16_bits_to_f32(static_cast<unsigned short>(scales[u])));
        if (i + u + kAheadScales < steps) scales[u] = __ldg(sp + static_cast<int64_t>(i + u + kAheadScales) * a.N);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(d_col, kCols);
  }

  // What a bf16 token was divided by is written while this grid may be there already: a plain load, not a read-only one.
  // At 64 tokens, 8192 x 28672: beside each store 66 us, as with a read-only load; from L2 70 us; once per warp, ahead of the
  // stores, 68 us.
  auto factor_of = [&](int m) { return F16 ? 1.0f : a.factor[m]; };
  auto store = [&](int m, int col, float y, float factor) {
    const int64_t at = static_cast<int64_t>(m) * a.N + col;
    if constexpr (F16) {
      if (a.bias != nullptr) y += __half2float(static_cast<const __half*>(a.bias)[col]);
      static_cast<__half*>(a.out)[at] = __float2half_rn(y);
    } else {
      y *= factor;
      if (a.bias != nullptr) y += __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[col]);
      static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
    }
  };
  const bool adds = warp >= kAheadWarps && warp < kCopyWarp;
  const int mt = min(kTokens, a.M - m0);
  if (a.ksplit == 1) {
    if (adds && n < a.N) {
#pragma unroll
      for (int j = 0; j < kSums; ++j)
        if (first_sum + j < mt) store(m0 + first_sum + j, n, j & 1 ? acc[j / 2].y : acc[j / 2].x, factor_of(m0 + first_sum + j));
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
    for (int m = rank + first_sum / kSums * a.ksplit; m < mt; m += a.ksplit * (kAddWarps / 4)) {
      const float factor = factor_of(m0 + m);
      float y = 0.0f;
      for (int q = 0; q < a.ksplit; ++q) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(part + m * kRows + row), q)));
        y += v;
      }
      store(m0 + m, n, y, factor);
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

namespace {
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

template <bool F16, int G>
cudaError_t run_w4a16_tc(const W4A16Args& a, const W4Tokens& t, cudaStream_t st) {
  auto kern = w4a16_tc_kernel<F16, G>;
  static unsigned long long devices = 0;
  const cudaError_t e = allow_shared(kern, w4tc::kSmem, devices);
  if (e != cudaSuccess) return e;
  const int tiles = (a.M + w4tc::kTokens - 1) / w4tc::kTokens, chunks = (a.K + w4tc::kChunk - 1) / w4tc::kChunk;
  CUtensorMap tm_w, tm_x, tm_r;
  if (!w4a16_map(&tm_w, a.b, a.N, a.K / 2, 64, w4tc::kRows, CU_TENSOR_MAP_SWIZZLE_64B) ||
      !w4a16_map(&tm_x, t.x, a.M, static_cast<int64_t>(a.K) * 2, 128, w4tc::kTokens, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !w4a16_map(&tm_r, t.parts, a.M, t.blocks * 256, 128, w4tc::kTokens, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  const int row_tiles = (a.N + w4tc::kRows - 1) / w4tc::kRows;
  // K split over a cluster while that leaves no resident CTA (two per SM) without work and each has four chunks
  int ksplit = 1;
  while (ksplit < 8 && row_tiles * tiles * ksplit * 2 <= 2 * num_sms() && chunks / (2 * ksplit) >= 4) ksplit *= 2;
  const w4tc::Args args{a.s, a.z, t.factor, a.bias, a.out, a.M, a.N, a.K, ksplit};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = static_cast<unsigned>(ksplit);
  cfg.gridDim = dim3(row_tiles, tiles, ksplit);
  cfg.blockDim = dim3(w4tc::kThreads);
  cfg.dynamicSmemBytes = w4tc::kSmem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, tm_w, tm_x, tm_r, args);
}

}  // namespace cq
