// Attention of one new token per sequence where all sequences begin with the same tokens: the shared prefix is read once
// for the whole batch.
//
//   o[b, h] = (sum over the prefix + sum over the row's own tokens) of p_j v_j / the same sums of p_j
//
// The prefix: the batch's B (q_heads / kv_heads) query rows of a key-value head are the rows of a matrix product with its
// keys, so unlike decode's eight heads per key they fill tcgen05 tiles: S = Q K^T and O += P V on tiles of 128 rows and 128
// keys (64 at D 256), S, P and O in tensor memory.  A CTA holds two row tiles (one at D 256) against the same keys; where
// there is one row tile only, its two tile slots take every other key tile.  Four warps a slot turn S into P in place, a row
// a thread; one thread issues the products; four warps gather keys and values from their pages (8-bit caches are widened on
// the way, which is exact).  A row's maximum is only raised when a score exceeds it by 2^8 (f16: 2), since raising it rewrites O.
//
// Work: teams of CTAs, a CTA for each pair of row tiles, take equal runs of key tiles, through as many key-value heads as
// that covers; the team's CTAs read the same keys at the same time, from L2.  Every run leaves its sums (fp32) in the
// workspace, the row's own tokens go through the kernel of paged_attention.cu, and a last kernel joins them in a fixed order.
// The second kernel is launched early, but a CTA of the first leaves no room for one of it on an SM (225 KB of shared memory): it
// begins on the SMs that are done.
//
// Weights enter P V in 16 bits: in two parts of the type, as in paged_attention.cu, or in one, which errs about as much as
// rounding the output does.  256 rows of 64 heads behind 30011 tokens: 358 us a call with one part and a relative L2 error of
// 2.3e-3, 433 us with two and 1.7e-3, what rounding the exact result costs; two parts add half to the products.  The caller
// chooses; without a choice two where the batch has no more rows than one CTA takes (64 rows behind 16003 tokens: 52 us with
// the join, 46 with one part), else one.
//
// Measured on a B200 (device time of the prefix's kernel): 256 rows of 64 heads on 8 of 128 behind 30011 tokens: 284 to 290
// us, 870 to 890 TFLOP/s.  Bound by the chain from scores to weights to product to scores: with 128 x 128 tiles a slot's maximum, exponentials
// and conversions take about 2400 cycles, the two products 1300, and two slots hide each other's only in part (a pair of
// tiles takes 4200; the exponential unit and the tensor pipe are both busy for 2000 to 2600 of them).  Measured and left: a
// quarter of the exponentials as polynomials (no change), two threads a row (no change), tiles of 64 keys with the scores double
// buffered (342 us against 274 in the same run: products of 64 columns wait for shared memory).  64 rows behind 16003 tokens: 45
// us, half of it the start and end of a run; 40 rows of 16 heads on 4 of 256 behind 20000 tokens in 8 bits: 67 us, bound by the
// gathers, which hold one operand in flight at a time.
#include <type_traits>

#include "decode_common.cuh"

namespace cq {

namespace pfx {
constexpr int kSite = 130;                     // device status sites of the waits
constexpr int kRows = 128;
template <int D>
struct Cfg {
  static constexpr int kSlots = D == 256 ? 1 : 2;            // row tiles of a CTA
  static constexpr int kBufs = D == 256 ? 2 : 1;             // score buffers of a slot
  static constexpr int kKeys = D == 256 ? 64 : 128;
  static constexpr int kStages = D == 64 ? 8 : 5;
  static constexpr int kLag = D == 64 ? 3 : 1;               // loads in flight before one is waited for
  static constexpr int kStageBytes = kKeys * D * 2;
  static constexpr int kQBytes = kRows * D * 2;
  // warpgroups: softmax of each slot, gathers, products (one warp works)
  static constexpr int kSoftWarps = 4 * kSlots;
  static constexpr int kLoadWarp = kSoftWarps, kMmaWarp = kSoftWarps + 4;
  static constexpr int kThreads = 32 * (kSoftWarps + 8);
  static constexpr int kSmem = kSlots * kQBytes + kStages * kStageBytes + 256;
  static constexpr uint32_t kCols = 512;
  static constexpr int kSCols = kKeys;                       // columns of a score buffer
  static_assert(kSlots * (kBufs * kSCols + D) <= 512, "tensor memory");
};
// weights are raised by 2^lift, and the running maximum once a score exceeds it by 2^slack.  bf16 parts have fp32's range; f16
// parts reach 2^15 and hold 2^-25, so 2^-39 of the running maximum: a long tail behind one strong key keeps its values
template <bool F16>
__host__ __device__ constexpr float lift() { return F16 ? 14.0f : 0.0f; }
template <bool F16>
__host__ __device__ constexpr float slack() { return F16 ? 1.0f : 8.0f; }
// floats of a row tile's part: O as [D / 4][128 rows][4], then the rows' (maximum, sum)
__host__ __device__ constexpr int64_t part_floats(int d) { return 128ll * d + 256; }
}  // namespace pfx

// shared memory descriptor of an operand whose contiguous dimension is not the product's: 64 columns (128 bytes, swizzled)
// by 8 rows are a block; blocks along the columns lie `lbo` bytes apart, along the rows 1024
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t saddr, uint32_t lbo) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(lbo >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
// D(tmem) (+)= A(smem) * B(smem), 16-bit operands of one type
__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  mma_bf16(d_tmem, adesc, bdesc, idesc, accumulate);         // kind::f16: the descriptor names the type
}
// mbar_wait_short all inline: a kernel that moves registers between its warps has room for no call
__device__ __forceinline__ bool thread_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int where) {
  unsigned long long since = 0;
  for (uint32_t i = 1;; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    if (ok) return true;
    if ((i & 255u) == 0) {
      const unsigned long long now = globaltimer_ns();
      if (since == 0) since = now;
      if (*abort_flag) return false;
      if (now - since > kWaitLimitNs) {
        record_status(CQ_ERR_TIMEOUT, where);
        *abort_flag = 1;
        return false;
      }
    }
  }
}
// a wait of a whole warp: all lanes go on, or none does
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int where) {
  return __all_sync(0xffffffffu, thread_wait(bar, parity, abort_flag, where));
}
// four e4m3 values as two pairs of the type, exactly
template <bool F16>
__device__ __forceinline__ void widen_e4m3x4(uint32_t x, uint32_t& lo, uint32_t& hi) {
  e4m3x4_to_f16(x, lo, hi);
  if constexpr (!F16) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    lo = bf16x2_bits(a.x, a.y);
    hi = bf16x2_bits(b.x, b.y);
  }
}

// The prefix that this call joins, and the first query row that holds it (-1: none, and then nothing is shared).
__device__ __forceinline__ int prefix_leader(const PrefixArgs& a, int prefix, int* shared) {
  if (threadIdx.x == 0) *shared = 0x7fffffff;
  __syncthreads();
  for (int b = threadIdx.x; b < a.own.B; b += blockDim.x) {
    const int row = a.own.rows != nullptr ? __ldg(a.own.rows + b) : b;
    if (row < 0 || row >= a.own.table_rows) continue;
    const int n = min(__ldg(a.own.lens + row), a.own.table_width * a.own.page_size);
    if (n >= prefix) {
      atomicMin(shared, b);
      break;
    }
  }
  __syncthreads();
  return *shared == 0x7fffffff ? -1 : *shared;
}

template <bool F16, bool FP8, int D, int PARTS>
__global__ void __launch_bounds__(pfx::Cfg<D>::kThreads, 1) prefix_attention_kernel(const PrefixArgs a) {
  using C = pfx::Cfg<D>;
  constexpr int kKeys = C::kKeys, kStages = C::kStages, kSlots = C::kSlots, kBufs = C::kBufs;
  // with two slots the gathers and products give registers to the softmax, whose threads hold a row of scores
  constexpr int kSoftRegs = FP8 ? 168 : 184, kLoadRegs = FP8 ? 104 : 72, kMmaRegs = 72;
  static_assert(2 * kSoftRegs + kLoadRegs + kMmaRegs <= 4 * 128, "the registers that 512 threads are launched with");
  extern __shared__ __align__(1024) uint8_t smem[];           // the kernel has no other shared memory: it begins aligned
  uint8_t* q_at = smem;
  uint8_t* ring = smem + kSlots * C::kQBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * C::kStageBytes);
  uint64_t* empty = full + kStages;
  uint64_t* q_full = empty + kStages;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;                             // [kSlots * kBufs] scores are in tensor memory
  uint64_t* p_full = s_full + 2;                              // [..][2] half of the weights are
  uint64_t* o_done = p_full + 4;                              // [kSlots] a product with the values is done
  uint64_t* run_done = o_done + 2;                            // [kSlots] a run's last product is done
  uint64_t* all_done = run_done + 2;
  uint32_t* holder = reinterpret_cast<uint32_t*>(all_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(holder + 1);
  int* leader_at = reinterpret_cast<int*>(holder + 2);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const PagedAttnArgs& g = a.own;
  grid_dep_launch();                                          // the rows' own tokens are started where this is done

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 4);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 4);
    mbar_init(q_empty, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[2 * s], 4);
      mbar_init(&p_full[2 * s + 1], 4);
      mbar_init(&o_done[s], 1);
      mbar_init(&run_done[s], 1);
    }
    mbar_init(all_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == C::kMmaWarp) {
    tmem_alloc(holder, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  const int prefix = prefix_of(g);
  const int leader = prefix_leader(a, prefix, leader_at);     // and the barriers and the holder are written
  tc_fence_after();
  const uint32_t tmem = *holder;
  const uint32_t o_col = tmem, s_col = tmem + kSlots * D;     // O of each slot, then the score buffers

  // ---- this CTA: its row tiles, its team's run of key tiles ----
  const int group = g.Hq / g.Hkv, rows = g.B * group, tiles = (rows + pfx::kRows - 1) / pfx::kRows;
  const int team = blockIdx.x / a.members, tile0 = (blockIdx.x - team * a.members) * kSlots;
  const bool pair = kSlots == 2 && tile0 + 1 < tiles;         // two row tiles, or one that both slots share
  const int key_tiles = leader < 0 ? 0 : (prefix + kKeys - 1) / kKeys;
  const int64_t units = static_cast<int64_t>(g.Hkv) * key_tiles;
  const int64_t teams = min(static_cast<int64_t>(a.teams), units);     // each with a key tile or more
  const int64_t u0 = team < teams ? team * units / teams : 0, u1 = team < teams ? (team + 1) * units / teams : 0;
  const int64_t padded = static_cast<int64_t>(a.members) * kSlots;

  struct Segment {
    int head, j0, n;
  };
  auto segment = [&](int64_t u) {
    Segment s;
    s.head = static_cast<int>(u / key_tiles);
    s.j0 = static_cast<int>(u - static_cast<int64_t>(s.head) * key_tiles);
    s.n = static_cast<int>(min(u1 - u, static_cast<int64_t>(key_tiles - s.j0)));
    return s;
  };
  const int row_of_leader = leader < 0 ? 0 : g.rows != nullptr ? __ldg(g.rows + leader) : leader;
  const int* table = g.table + row_of_leader * g.table_stride;
  const int page_shift = 31 - __clz(g.page_size), page_mask = g.page_size - 1;

  if (warp >= C::kMmaWarp) {
    if constexpr (kSlots == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
    // ---- products, by one thread ----
    if (warp == C::kMmaWarp && elect_one()) {
      constexpr uint32_t type = F16 ? 0u : (1u << 7) | (1u << 10);
      constexpr uint32_t idesc_s = (1u << 4) | type | (static_cast<uint32_t>(kKeys >> 3) << 17) | (8u << 24);
      constexpr uint32_t idesc_o = (1u << 4) | type | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (8u << 24);
      int base = 0;                                           // ring loads before this segment
      uint32_t q_phase = 0, p_phase[2] = {0, 0}, o_phase[2] = {0, 0};
      bool ok = true;
      for (int64_t u = u0; u < u1 && ok;) {
        const Segment seg = segment(u);
        const int jobs = pair ? 2 * seg.n : seg.n;            // job i: slot i & 1 (where there are two)
        auto tile_of = [&](int i) { return pair ? i >> 1 : i; };
        auto last_of_tile = [&](int i) { return !pair || (i & 1); };
        auto scores = [&](int i) {
          const int slot = kSlots == 2 ? i & 1 : 0, buf = kBufs == 2 ? i & 1 : slot;
          const int l = base + 2 * tile_of(i), stage = l % kStages;
          if (!thread_wait(&full[stage], (l / kStages) & 1, abort_flag, pfx::kSite + 2)) return false;
          tc_fence_after();
          const uint64_t q = smem_desc_k_sw128(smem_u32(q_at + (pair ? slot : 0) * C::kQBytes));
          const uint64_t k = smem_desc_k_sw128(smem_u32(ring + stage * C::kStageBytes));
#pragma unroll
          for (int x = 0; x < D / 16; ++x)
            mma_f16_ss(s_col + buf * C::kSCols, q + ((x >> 2) * (pfx::kRows * 128) + (x & 3) * 32) / 16,
                       k + ((x >> 2) * (kKeys * 128) + (x & 3) * 32) / 16, idesc_s, x != 0);
          tc_commit(&s_full[buf]);
          if (last_of_tile(i)) tc_commit(&empty[stage]);
          if (i + 1 == jobs) tc_commit(q_empty);
          return true;
        };
        ok = thread_wait(q_full, q_phase, abort_flag, pfx::kSite + 3);
        q_phase ^= 1u;
        if (!ok) break;
        const int ahead = kSlots == 2 ? 2 : 1;                // jobs whose scores come before a job's weights
        for (int i = 0; i < min(ahead, jobs) && ok; ++i) ok = scores(i);
        for (int i = 0; i < jobs && ok; ++i) {
          const int slot = kSlots == 2 ? i & 1 : 0, buf = kBufs == 2 ? i & 1 : slot;
          if (kBufs == 2 && i + 1 < jobs) {
            // the other buffer's weights are consumed when the product before is done
            if (i > 0) {
              ok = thread_wait(&o_done[0], o_phase[0], abort_flag, pfx::kSite + 4);
              o_phase[0] ^= 1u;
            }
            ok = ok && scores(i + 1);
            if (!ok) break;
          } else if (kBufs == 2 && i > 0) {
            ok = thread_wait(&o_done[0], o_phase[0], abort_flag, pfx::kSite + 4);
            o_phase[0] ^= 1u;
            if (!ok) break;
          }
          const int l = base + 2 * tile_of(i) + 1, stage = l % kStages;
          if (!(ok = thread_wait(&full[stage], (l / kStages) & 1, abort_flag, pfx::kSite + 5))) break;
          const uint32_t v = smem_u32(ring + stage * C::kStageBytes);
          const bool first = kSlots == 2 ? i < 2 : i == 0;
#pragma unroll
          for (int x = 0; x < kKeys / 16; ++x) {
            if (x % (kKeys / 32) == 0) {
              if (!(ok = thread_wait(&p_full[2 * buf + x / (kKeys / 32)], p_phase[buf], abort_flag, pfx::kSite + 6))) break;
              tc_fence_after();
            }
            const uint64_t vd = smem_desc_mn_sw128(v + x * 2048, kKeys * 128);
            const uint32_t p = s_col + buf * C::kSCols + 32 * (x >> 1) + 8 * (x & 1);
            mma_f16_ts(o_col + slot * D, p, vd, idesc_o, !first || x != 0);
            if constexpr (PARTS == 2) mma_f16_ts(o_col + slot * D, p + 16, vd, idesc_o, 1);
          }
          p_phase[buf] ^= 1u;
          if (!ok) break;
          tc_commit(&o_done[slot]);
          if (i + kSlots >= jobs) tc_commit(&run_done[slot]);
          if (last_of_tile(i)) tc_commit(&empty[stage]);
          if (kSlots == 2 && i + 2 < jobs) {
            // this slot's scores take the place of the weights just used
            ok = thread_wait(&o_done[slot], o_phase[slot], abort_flag, pfx::kSite + 7) && scores(i + 2);
            o_phase[slot] ^= 1u;
          }
        }
        // the segment's last products: the next one's scores take the place of their weights
        for (int i = max(0, jobs - kSlots); i < jobs && ok; ++i) {
          const int slot = kSlots == 2 ? i & 1 : 0;
          ok = thread_wait(&o_done[slot], o_phase[slot], abort_flag, pfx::kSite + 4);
          o_phase[slot] ^= 1u;
        }
        base += 2 * seg.n;
        u += seg.n;
      }
      tc_commit(all_done);
      mbar_wait_drain(all_done, 0, 50000000ull);
    }
    __syncwarp();
  } else if (warp >= C::kLoadWarp) {
    if constexpr (kSlots == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
    // ---- gathers: Q of a segment, then its keys and values, tile by tile ----
    const int w = warp - C::kLoadWarp;
    constexpr int kChunks = D / 8;                            // 16-byte chunks of a 16-bit row
    int load = 0, landed = 0;                                 // ring loads issued, and handed over
    uint32_t q_phase = 0;
    bool ok = true;
    auto place = [&](int rows_of, int r, int c) {             // in a tile of `rows_of` rows: 64 columns wide blocks, swizzled
      return (c >> 3) * (rows_of * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    };
    auto hand_over = [&](uint64_t* bar) {                     // this warp's share has landed
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    for (int64_t u = u0; u < u1 && ok;) {
      const Segment seg = segment(u);
      if (u > u0) {
        ok = warp_wait(q_empty, q_phase, abort_flag, pfx::kSite);
        q_phase ^= 1u;
        if (!ok) break;
      }
      // Q: 32 rows of each tile a warp
      for (int s = 0; s < (pair ? 2 : 1); ++s) {
        constexpr int kRowsAtOnce = 32 / kChunks > 0 ? 32 / kChunks : 1;
        const uint32_t dst = smem_u32(q_at + s * C::kQBytes);
        for (int r0 = 0; r0 < 32; r0 += kRowsAtOnce) {
          const int r = 32 * w + r0 + lane / kChunks, c = lane % kChunks;
          const int at = (tile0 + s) * pfx::kRows + r;
          const bool valid = at < rows;
          const int b = valid ? at / group : 0, h = valid ? at - b * group : 0;
          const uint16_t* src = static_cast<const uint16_t*>(g.q) + b * g.q_sb + (seg.head * group + h) * g.q_sh;
          cp_async16(dst + place(pfx::kRows, r, c), src + 8 * c, valid);
        }
      }
      cp_async_commit();
      bool q_landed = false;
      if constexpr (FP8) {
        cp_async_wait<0>();
        hand_over(q_full);
      }
      const int64_t head_at = seg.head * g.head_stride;
      constexpr int kPerWarp = kKeys / 4;                     // keys of a warp: 32 or 16
      // lane r looks its key of a tile up
      struct Keys {
        int64_t off;
        uint32_t mask;
      };
      auto look_up = [&](int j) {
        const int key = j * kKeys + w * kPerWarp + (lane & (kPerWarp - 1));
        int page = -1;
        if (j < seg.j0 + seg.n && key < prefix) page = __ldg(table + (key >> page_shift));
        const bool there = page >= 0 && page < g.num_pages;
        return Keys{there ? page * g.page_stride + head_at + (key & page_mask) * g.tok_stride : 0, __ballot_sync(0xffffffffu, there)};
      };
      if constexpr (FP8) {
        // 16 codes a lane, through registers: an operand's next rows are on their way while the other's are widened
        constexpr int kLanes = D / 16, kAtOnce = 32 / kLanes, kLoads = kPerWarp / kAtOnce;
        uint4 raw[2][kLoads];
        const int c = lane % kLanes;
        auto fetch = [&](int kv, const Keys& keys) {
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const int r = i * kAtOnce + lane / kLanes;
            const int64_t o = __shfl_sync(0xffffffffu, keys.off, r) + 16 * c;
            uint4& x = raw[kv][i];
            x = make_uint4(0, 0, 0, 0);
            if (keys.mask >> r & 1u)
              asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                           : "l"(static_cast<const uint8_t*>(kv ? g.v : g.k) + o));
          }
        };
        auto store = [&](int kv) {
          const int stage = load % kStages;
          if (load >= kStages && !(ok = warp_wait(&empty[stage], (load / kStages - 1) & 1, abort_flag, pfx::kSite + 1))) return;
          uint8_t* dst = ring + stage * C::kStageBytes;
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const int r = kPerWarp * w + i * kAtOnce + lane / kLanes;
            uint4 lo, hi;
            widen_e4m3x4<F16>(raw[kv][i].x, lo.x, lo.y);
            widen_e4m3x4<F16>(raw[kv][i].y, lo.z, lo.w);
            widen_e4m3x4<F16>(raw[kv][i].z, hi.x, hi.y);
            widen_e4m3x4<F16>(raw[kv][i].w, hi.z, hi.w);
            *reinterpret_cast<uint4*>(dst + place(kKeys, r, 2 * c)) = lo;
            *reinterpret_cast<uint4*>(dst + place(kKeys, r, 2 * c + 1)) = hi;
          }
          hand_over(&full[stage]);
          ++load;
        };
        Keys next = look_up(seg.j0);
        fetch(0, next);
        fetch(1, next);
        next = look_up(seg.j0 + 1);
        for (int j = seg.j0; j < seg.j0 + seg.n; ++j) {
          store(0);
          if (!ok) break;
          fetch(0, next);
          store(1);
          if (!ok) break;
          fetch(1, next);
          next = look_up(j + 2);
        }
      }
      for (int j = seg.j0; !FP8 && j < seg.j0 + seg.n && ok; ++j) {
        const Keys keys = look_up(j);
        if constexpr (!FP8) {
          for (int kv = 0; kv < 2 && ok; ++kv) {
            const int stage = load % kStages;
            if (load >= kStages && !(ok = warp_wait(&empty[stage], (load / kStages - 1) & 1, abort_flag, pfx::kSite + 1))) break;
            const uint32_t dst = smem_u32(ring + stage * C::kStageBytes);
            const uint16_t* base = static_cast<const uint16_t*>(kv ? g.v : g.k);
            constexpr int kRowsAtOnce = 32 / kChunks > 0 ? 32 / kChunks : 1;
            const int c = lane % kChunks;
#pragma unroll 8
            for (int r0 = 0; r0 < kPerWarp; r0 += kRowsAtOnce) {
              const int r = r0 + lane / kChunks;
              const int64_t o = __shfl_sync(0xffffffffu, keys.off, r) + 8 * c;
              cp_async16(dst + place(kKeys, kPerWarp * w + r, c), base + o, keys.mask >> r & 1u);
            }
            cp_async_commit();
            ++load;
            if (!q_landed) {                                  // the first keys are on their way behind it
              cp_async_wait<1>();
              hand_over(q_full);
              q_landed = true;
            }
            if (load - landed > C::kLag) {
              cp_async_wait<C::kLag>();
              hand_over(&full[landed % kStages]);
              ++landed;
            }
          }
        }
      }
      if constexpr (!FP8) {
        cp_async_wait<0>();
        for (; landed < load; ++landed) hand_over(&full[landed % kStages]);
      }
      u += seg.n;
    }
    cp_async_wait<0>();
  } else {
    // ---- softmax: thread = row of the slot's tile ----
    if constexpr (kSlots == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    const int slot = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    constexpr float kLift = pfx::lift<F16>(), kSlackUp = pfx::slack<F16>();
    uint32_t s_phase[2] = {0, 0}, o_phase = 0, run_phase = 0;   // o_phase: products of earlier runs
    bool ok = true;
    for (int64_t u = u0; u < u1 && ok;) {
      const Segment seg = segment(u);
      const float mul = g.scale * 1.4426950408889634f * (FP8 && g.k_scale != nullptr ? __ldg(g.k_scale + seg.head) : 1.0f);
      float m = -INFINITY, l = 0.0f;
      const int step = kSlots == 2 && !pair ? 2 : 1;          // key tiles of this slot: first, first + step, ...
      int done = 0;
      // which keys of a tile are there: looked up a tile ahead
      int page[kKeys / 32];
      auto look_up = [&](int j) {
#pragma unroll
        for (int x = 0; x < kKeys / 32; ++x) {
          const int key = (seg.j0 + j) * kKeys + 32 * x + lane;
          page[x] = j < seg.n && key < prefix ? __ldg(table + (key >> page_shift)) : -1;
        }
      };
      look_up(kSlots == 2 && !pair ? slot : 0);
      for (int j = kSlots == 2 && !pair ? slot : 0; j < seg.n && ok; j += step, ++done) {
        const int buf = kBufs == 2 ? done & 1 : slot;
        if (!(ok = warp_wait(&s_full[buf], s_phase[buf], abort_flag, pfx::kSite + 8))) break;
        s_phase[buf] ^= 1u;
        tc_fence_after();
        uint32_t masks[kKeys / 32];
        bool whole = true;
#pragma unroll
        for (int x = 0; x < kKeys / 32; ++x) {
          masks[x] = __ballot_sync(0xffffffffu, page[x] >= 0 && page[x] < g.num_pages);
          whole = whole && masks[x] == 0xffffffffu;
        }
        look_up(j + step);
        const uint32_t s_at = s_col + buf * C::kSCols + lanes;
        // a row of scores; NaN is passed over here and shows in the weights
        uint32_t v[kKeys / 32][32];
#pragma unroll
        for (int x = 0; x < kKeys / 32; ++x) tmem_ld_32x32b_x32(s_at + 32 * x, v[x]);
#pragma unroll
        for (int x = 0; x < kKeys / 32; ++x) tmem_wait_ld_dep(v[x]);
        float top = -INFINITY, top2 = -INFINITY;
        auto largest = [&](auto whole_tile, float sign) {     // a negative scale turns the order around
#pragma unroll
          for (int x = 0; x < kKeys / 32; ++x)
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float s0 = __uint_as_float(v[x][i]) * sign, s1 = __uint_as_float(v[x][i + 1]) * sign;
              if (whole_tile || masks[x] >> i & 1u) top = fmaxf(top, s0);
              if (whole_tile || masks[x] >> (i + 1) & 1u) top2 = fmaxf(top2, s1);
            }
        };
        if (whole && mul >= 0.0f) largest(std::true_type{}, 1.0f);
        else largest(std::false_type{}, mul < 0.0f ? -1.0f : 1.0f);
        top = fmaxf(top, top2);
        top = top == -INFINITY ? top : top * fabsf(mul);
        const bool raise = top > m + kSlackUp || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, raise)) {
          const float to = raise ? top : m, f = raise ? exp2_fast(m - to) : 1.0f;
          m = to;
          l *= f;
          if (done > 0) {
            // with two buffers the product before may still add to O; those before it are done, since one of them was the
            // last use of this buffer.  With one, these scores came after the product
            if (kBufs == 2) {
              ok = warp_wait(&o_done[slot], (o_phase + static_cast<uint32_t>(done) - 1u) & 1u, abort_flag, pfx::kSite + 9);
              if (!ok) break;
              tc_fence_after();
            }
#pragma unroll 2
            for (int x = 0; x < D / 16; ++x) {
              uint32_t o[16];
              const uint32_t at = o_col + slot * D + lanes + 16 * x;
              tmem_ld_x16(at, o);
              tmem_wait_ld_x16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st_x16(at, o);
            }
          }
        }
        const float base = (m == -INFINITY ? 0.0f : m) - kLift;
        float2 sums[2] = {};
        auto weights = [&](auto whole_tile) {
#pragma unroll
          for (int x = 0; x < kKeys / 32; ++x) {
            uint32_t p[PARTS == 2 ? 32 : 16];                 // the first part's pairs, then the second's
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 y = fma2(make_float2(__uint_as_float(v[x][i]), __uint_as_float(v[x][i + 1])), make_float2(mul, mul), make_float2(-base, -base));
              float2 w = make_float2(exp2_fast(y.x), exp2_fast(y.y));
              if (!whole_tile) {
                w.x = masks[x] >> i & 1u ? w.x : 0.0f;
                w.y = masks[x] >> (i + 1) & 1u ? w.y : 0.0f;
              }
              sums[i / 2 & 1] = fma2(w, make_float2(1.0f, 1.0f), sums[i / 2 & 1]);
              p[i / 2] = narrow16<F16>(w.x, w.y);
              if constexpr (PARTS == 2) {
                const float2 rest = fma2(widen16<F16>(p[i / 2]), make_float2(-1.0f, -1.0f), w);
                p[16 + i / 2] = narrow16<F16>(rest.x, rest.y);
              }
            }
            if constexpr (PARTS == 2) tmem_st_x32(s_at + 32 * x, p);
            else tmem_st_x16(s_at + 32 * x, p);
            if ((x + 1) % (kKeys / 64) == 0) {                // a half: the product may begin with it
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_full[2 * buf + x / (kKeys / 64)]);
            }
          }
        };
        if (whole) weights(std::true_type{});
        else weights(std::false_type{});
        l += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
      }
      // ---- this run's sums ----
      if (!ok) break;
      if (done > 0) {
        ok = warp_wait(&run_done[slot], run_phase, abort_flag, pfx::kSite + 10);
        run_phase ^= 1u;
        o_phase += static_cast<uint32_t>(done);
        if (!ok) break;
        tc_fence_after();
      }
      float* part = a.parts + ((team + seg.head) * padded + tile0 + slot) * pfx::part_floats(D);
      if (done > 0) {
#pragma unroll 1
        for (int x = 0; x < D / 16; ++x) {
          uint32_t o[16];
          tmem_ld_x16(o_col + slot * D + lanes + 16 * x, o);
          tmem_wait_ld_x16(o);
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            reinterpret_cast<uint4*>(part)[(4 * x + i / 4) * pfx::kRows + row] = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
      reinterpret_cast<float2*>(part + 128 * D)[row] = make_float2(m, l);
      tc_fence_before();
      u += seg.n;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) tmem_dealloc(tmem, C::kCols);
}

// Joins a row's runs over the prefix, in their order, with its own tokens.  A block: 128 rows of a row tile, one head, eight
// columns; thread = row.  What the runs left is in L2: eight runs' loads are in flight at a time.
template <bool F16, int D>
__global__ void __launch_bounds__(128) prefix_join_kernel(const PrefixArgs a) {
  using C = pfx::Cfg<D>;
  constexpr int kKeys = C::kKeys, kAtOnce = 8;
  const PagedAttnArgs& g = a.own;
  const int tile = blockIdx.x, head = blockIdx.y, d4 = blockIdx.z * 2, tid = threadIdx.x;
  const int group = g.Hq / g.Hkv, rows = g.B * group, tiles = (rows + pfx::kRows - 1) / pfx::kRows;
  const int prefix = prefix_of(g);
  const int key_tiles = (prefix + kKeys - 1) / kKeys;
  const int64_t units = static_cast<int64_t>(g.Hkv) * key_tiles, padded = static_cast<int64_t>(a.members) * C::kSlots;
  const int subs = C::kSlots == 2 && tile + 1 == tiles && !(tile & 1) ? 2 : 1;
  const int at = tile * pfx::kRows + tid;
  const bool live = at < rows;
  const int b = live ? at / group : 0, h = head * group + (live ? at - b * group : 0);
  const int row = g.rows != nullptr ? g.rows[b] : b;
  const int n = row >= 0 && row < g.table_rows ? min(g.lens[row], g.table_width * g.page_size) : 0;
  int parts = 0;
  const float* first = a.parts;
  if (live && prefix > 0 && n >= prefix) {                    // the row has the prefix: the teams with a run over this head
    const int64_t teams = min(static_cast<int64_t>(a.teams), units);
    const int64_t t0 = ((static_cast<int64_t>(head) * key_tiles + 1) * teams - 1) / units;
    const int64_t t1 = (static_cast<int64_t>(head + 1) * key_tiles * teams - 1) / units;
    parts = static_cast<int>(t1 - t0 + 1) * subs;
    first += ((t0 + head) * padded + tile) * pfx::part_floats(D);
  }
  const int64_t stride = padded * pfx::part_floats(D);
  grid_dep_wait();
  const int64_t own = static_cast<int64_t>(b) * g.Hq + h;
  const float vs = g.cache_dtype == CQ_DT_FP8_E4M3 && g.v_scale != nullptr ? g.v_scale[head] : 1.0f;
  constexpr float kLift = pfx::lift<F16>();
  // the running maximum is of what the weights were raised by, a power of 2; own tokens first (-inf: none)
  float top = live ? g.lse[own] * 1.4426950408889634f + kLift : -INFINITY;
  const bool has_own = top != -INFINITY;
  float sum = has_own ? 1.0f : 0.0f, o[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 v = has_own ? *reinterpret_cast<const float4*>(g.out32 + own * D + 4 * (d4 + i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    o[4 * i] = v.x, o[4 * i + 1] = v.y, o[4 * i + 2] = v.z, o[4 * i + 3] = v.w;
  }
  for (int i0 = 0; i0 < parts; i0 += kAtOnce) {
    float2 ml[kAtOnce];
    float4 v[kAtOnce][2];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = min(i0 + j, parts - 1);
      const float* p = first + (subs == 2 ? i >> 1 : i) * stride + (subs == 2 && (i & 1) ? pfx::part_floats(D) : 0);
      ml[j] = reinterpret_cast<const float2*>(p + 128 * D)[tid];
      v[j][0] = reinterpret_cast<const float4*>(p)[d4 * pfx::kRows + tid];
      v[j][1] = reinterpret_cast<const float4*>(p)[(d4 + 1) * pfx::kRows + tid];
    }
    float most = top;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (i0 + j < parts) most = fmaxf(most, ml[j].x);
    const float down = top == -INFINITY ? 1.0f : exp2f(top - most);   // -inf so far: what is there weighs nothing, or is NaN
    sum *= down;
#pragma unroll
    for (int x = 0; x < 8; ++x) o[x] *= down;
    top = most;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (i0 + j >= parts || ml[j].y == 0.0f) continue;       // a slot without a key tile, or keys that weigh nothing
      const float f = ml[j].x == -INFINITY ? 1.0f : exp2f(ml[j].x - top);
      sum = fmaf(ml[j].y, f, sum);
      const float fv = f * vs;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        o[4 * i] = fmaf(v[j][i].x, fv, o[4 * i]);
        o[4 * i + 1] = fmaf(v[j][i].y, fv, o[4 * i + 1]);
        o[4 * i + 2] = fmaf(v[j][i].z, fv, o[4 * i + 2]);
        o[4 * i + 3] = fmaf(v[j][i].w, fv, o[4 * i + 3]);
      }
    }
  }
  if (!live) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = narrow16<F16>(o[2 * i] * inv, o[2 * i + 1] * inv);
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(g.out) + own * D + 4 * d4) = make_uint4(out[0], out[1], out[2], out[3]);
  if (a.lse_out != nullptr && d4 == 0)
    a.lse_out[own] = sum == 0.0f ? -INFINITY : (top - kLift + log2f(sum)) / 1.4426950408889634f;
}

namespace {
int prefix_members(int64_t rows, int D) {
  const int per = D == 256 ? pfx::kRows : 2 * pfx::kRows;
  return static_cast<int>((rows + per - 1) / per);
}
int prefix_teams(int members) { return members < num_sms() ? num_sms() / members : 1; }
}  // namespace

// Sharing pays from about 128 MB of shared keys and values that the rows would read one by one: four launches and the split
// of the rows' sums cost 14 to 20 us, and reading runs at 5 to 6 TB/s.  Us one by one and shared: 16 rows of 8 heads of 128
// behind 1000 tokens (70 MB) 15 and 22, 32 rows (139 MB) 22 and 22, 16 rows behind 4000 (266 MB) 38 and 36, 64 rows behind
// 1000 (279 MB) 40 and 27; 8-bit codes of 256: 139 MB 28 and 26; heads of 64: 133 MB 31 and 31.  So many tokens they are; a
// prefix on the device that has fewer is left to the rows' own kernel, whose results are those of a call that shares nothing.
int64_t prefix_share_from(int64_t batch, int Hkv, int D, int size) {
  return 134217728 / (batch * Hkv * D * 2 * size) + 1;
}

// the runs' sums, the rows' own outputs and their logs, and the workspace of their kernel
int64_t prefix_attention_workspace(int64_t batch, int Hq, int Hkv, int D, int64_t span) {
  if (batch == 0) return 0;
  if (span < prefix_share_from(batch, Hkv, D, 2)) return paged_attention_workspace(batch, Hq, Hkv, D, span, 0, 0);
  const int members = prefix_members(batch * (Hq / Hkv), D);
  const int64_t parts = static_cast<int64_t>(prefix_teams(members) + Hkv) * members * (D == 256 ? 1 : 2) * pfx::part_floats(D) * 4;
  return parts + batch * Hq * (D + 4) * 4 + (paged_attention_workspace(batch, Hq, Hkv, D, span, 0, 0) + 255) / 256 * 256;
}

template <bool F16, bool FP8, int D, int PARTS>
cudaError_t run_prefix(const PrefixArgs& a, cudaStream_t st) {
  using C = pfx::Cfg<D>;
  auto kern = prefix_attention_kernel<F16, FP8, D, PARTS>;
  static unsigned long long devices = 0;
  cudaError_t e = allow_shared(kern, C::kSmem, devices);
  if (e != cudaSuccess) return e;
  kern<<<static_cast<unsigned>(a.teams * a.members), C::kThreads, C::kSmem, st>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if ((e = launch_paged_attention(a.own, st)) != cudaSuccess) return e;
  const int group = a.own.Hq / a.own.Hkv, tiles = (a.own.B * group + pfx::kRows - 1) / pfx::kRows;
  return launch_early(prefix_join_kernel<F16, D>, dim3(tiles, a.own.Hkv, D / 8), 128, 0, st, a);
}
template <bool F16, bool FP8, int D>
cudaError_t pick_prefix(const PrefixArgs& a, int weight_parts, cudaStream_t st) {
  const bool two = weight_parts == 0 ? a.members == 1 : weight_parts == 2;
  return two ? run_prefix<F16, FP8, D, 2>(a, st) : run_prefix<F16, FP8, D, 1>(a, st);
}
template <bool F16, bool FP8>
cudaError_t pick_prefix_dim(const PrefixArgs& a, int weight_parts, cudaStream_t st) {
  switch (a.own.D) {
    case 64: return pick_prefix<F16, FP8, 64>(a, weight_parts, st);
    case 128: return pick_prefix<F16, FP8, 128>(a, weight_parts, st);
    default: return pick_prefix<F16, FP8, 256>(a, weight_parts, st);
  }
}

// a.own: the whole call's arguments, its ws the whole workspace
cudaError_t launch_prefix_attention(const PagedAttnArgs& call, int weight_parts, cudaStream_t st) {
  const int64_t span = static_cast<int64_t>(call.table_width) * call.page_size;
  const int64_t from = prefix_share_from(call.B, call.Hkv, call.D, call.cache_dtype == CQ_DT_FP8_E4M3 ? 1 : 2);
  if ((call.prefix != nullptr || call.prefix_len > span ? span : call.prefix_len) < from)
    return launch_paged_attention(call, st);                  // every row through its own table
  PrefixArgs a{};
  a.own = call;
  a.own.share_from = static_cast<int>(from);                  // at most the span
  a.members = prefix_members(static_cast<int64_t>(call.B) * (call.Hq / call.Hkv), call.D);
  a.teams = prefix_teams(a.members);
  a.lse_out = call.lse;
  a.parts = static_cast<float*>(call.ws);
  float* next = a.parts + static_cast<int64_t>(a.teams + call.Hkv) * a.members * (call.D == 256 ? 1 : 2) * pfx::part_floats(call.D);
  const int64_t heads = static_cast<int64_t>(call.B) * call.Hq;
  a.own.out32 = next;
  a.own.lse = next + heads * call.D;
  a.own.ws = next + heads * (call.D + 4);
  const bool fp8 = call.cache_dtype == CQ_DT_FP8_E4M3;
  if (call.dtype == CQ_DT_F16)
    return fp8 ? pick_prefix_dim<true, true>(a, weight_parts, st) : pick_prefix_dim<true, false>(a, weight_parts, st);
  return fp8 ? pick_prefix_dim<false, true>(a, weight_parts, st) : pick_prefix_dim<false, false>(a, weight_parts, st);
}

}  // namespace cq
