// Attention of one new token per sequence over a paged key-value cache.
//
//   o[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[b, h] . k_j - max),  j over the visible keys of row b:
//   j < len, and with a window: j >= len - window or j < sinks.  A row without visible keys gives zeros.
//
// Bound by reading the visible keys and values once.  The query heads of a key-value head share its tiles, so the
// products run on tensor cores with the keys as rows and the heads as columns:
//   S^T [16 keys x 8 heads] = K Q^T,  O^T [D x 8 heads] += V^T P^T.
// At decode there are at most 16 heads per key-value head: mma.sync with its operands in registers does a tile in
// tens of instructions, while a tcgen05 tile would be filled to an eighth; HBM, not the tensor pipe, is the limit.
//
// Work: a unit is 64 visible keys of one segment (a row and a tile of heads), 16 for each of the CTA's four warps.
// Every CTA of a resident grid takes an equal run of units, through as many segments as that covers, so ragged lengths
// balance and one long row uses every SM; a row that several CTAs share is joined by a second small kernel in the order
// of its parts.  Short rows go whole to a CTA instead, and few segments of moderate length to a cluster of CTAs each,
// which join over distributed shared memory.  Each warp keeps its own ring of asynchronous 16-byte copies in flight and
// never waits for the others inside a run; the ring runs on across segments.  Where a segment ends (or the run does)
// the warps' running maxima, sums and outputs are joined in the stages they have just consumed.  All orders are fixed,
// so equal calls give equal bits.
//
// Behind a shared prefix (prefix_attention.cu) a row that holds it sees only its own tokens, and its output stays fp32 with
// the log of its sum, for that file's join.
//
// Softmax statistics, scores and outputs are fp32.  The weights p enter the second product as two parts of the cache's
// 16-bit type, p = hi + lo, since one part alone would add up to as much error as rounding the output does.  f16 parts
// hold 2^15 p, and the sum is taken over the same: without it a weight of 2^-25 of the largest, which a long tail behind
// one strong key has many of, would count in the sum alone.  So they are held to 2^-40 of the largest.
// 8-bit caches are widened exactly to f16; a bf16 query is scaled by a power of two per head so that f16 holds it to
// 2^-24 of its largest element.
//
// Measured on a B200 (device time): 64 ragged rows of up to 8000 keys, 32 heads on 8, D 128, bf16: 174 us, 6.1 TB/s, and
// 16 rows of up to 8000 keys at D 256: 129 us, 6.2 TB/s, HBM's rate; 2 rows of up to 200,000 keys, 28 heads on 4, f16: 141
// us, 5.7 TB/s; 48 rows that see 1028 keys of an 8-bit cache, 16 heads on 8, D 256: 56 us, 3.5 TB/s, bound by the chain of
// loads, products and exponentials from one tile to the next; one row of 333 keys: 6.5 us, launch and latency.
#include "decode_common.cuh"

namespace cq {

namespace pattn {
constexpr int kWarps = 4;
constexpr int kTile = 16;                    // keys per warp and step
constexpr int kUnit = kWarps * kTile;
// A row is split no finer than this: a part costs its CTA a start and an end (about two units' time), and the join; 2 and
// 8 measured the same.
constexpr int kMinUnits = 4;
// Segments of at most kWholeUnits go whole to CTAs, one launch and no join, where that keeps the SMs busy: all of them at
// once, or in waves whose last one idles for less than kJoinUnits a CTA, about what runs pay for their parts and join.  Us
// whole and as runs, 8 heads of D 128: 30 rows of 500 keys 14 and 19, of 1500 32 and 36; 64 rows of 500 27 and 31; but 40
// rows (320 segments) of 500 26 and 24, of 1000 47 and 37.
constexpr int kWholeUnits = 24;
constexpr int kJoinUnits = 5;
// CTAs of a resident grid (two per SM; at D 256 with 16-bit caches one fits, and the rules above and below, measured at D
// 64 and 128, count two all the same), and the most units of a cluster's CTA: with few segments of up to so many units a
// cluster each is quicker than runs over all SMs and their join (8 segments of 4000 keys: 12 and 14 us).
constexpr int kMaxRuns = 2 * 148;
constexpr int kClusterUnits = 16;

// shared memory: ring (a consumed stage holds its warp's outputs while the warps are joined), query fragments, statistics
template <int D, int ES, int NT>
struct Cfg {
  static constexpr int kRow = D * ES;                          // bytes of one key
  static constexpr int kTileBytes = kTile * kRow;              // one operand's tile
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kQ = D / 16 * NT * 256;
  static constexpr int kMisc = 8 * NT * 4 * (2 * kWarps + 1) + 16;
  static constexpr int kFixed = kQ + kMisc;
  static constexpr int kCtas = 3 * kWarps * kStageBytes + kFixed <= 112 * 1024 ? 2 : 1;
  static constexpr int kFit = ((kCtas == 2 ? 112 : 224) * 1024 - kFixed) / (kWarps * kStageBytes);
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kMaskBytes = kWarps * kStages * 4;
  static constexpr int kSmem = kWarps * kStages * kStageBytes + kFixed + kMaskBytes;
  static_assert(kStages >= 3, "ring of three stages");
  static_assert(8 * D * 4 <= kStageBytes, "eight heads' outputs fit a stage");
};

// How the units are dealt out: equal runs of units, joined by a second kernel where a row is split; runs of whole
// segments; or a cluster of CTAs per segment, which join over distributed shared memory.
enum Mode { kRuns, kSegments, kClusters };

struct Meta {          // one CTA's run, for the join: its first part's segment, first unit there, the segment's units
  int seg, unit0, units, count;
};
}  // namespace pattn

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {   // transpose of the warp's 8 x 8 matrix of 16-bit values
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
// four e4m3 values as two f16 pairs: exact; NaN stays NaN
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t x, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(x));
}
// two fp32 values as 16-bit pairs: hi = the nearest, lo = the nearest of what is left
template <bool F16>
__device__ __forceinline__ void split16(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  }
}
// 16-byte chunk c of row r of a tile whose rows are kRow bytes: the chunks a matrix load reads from eight rows at one
// c fall on different banks
template <int kRow>
__device__ __forceinline__ int swz(int r, int c) {
  if constexpr (kRow >= 128) return r * kRow + ((c ^ (r & 7)) << 4);
  return r * kRow + ((c ^ ((r >> 1) & 3)) << 4);
}

// the visible keys of a row: vis of them, the i-th at position i below nsink and at n - vis + i from there on
struct RowView {
  int row, n, vis, nsink, units;
};
// the tokens that this call reads once for all rows: none where that would not pay
__device__ __forceinline__ int prefix_of(const PagedAttnArgs& a) {
  const int n = min(a.prefix != nullptr ? __ldg(a.prefix) : a.prefix_len, a.table_width * a.page_size);
  return n >= a.share_from ? n : 0;
}
__device__ __forceinline__ RowView row_view(const PagedAttnArgs& a, int b) {
  RowView v;
  v.row = a.rows != nullptr ? __ldg(a.rows + b) : b;
  int n = v.row >= 0 && v.row < a.table_rows ? __ldg(a.lens + v.row) : 0;
  n = min(max(n, 0), a.table_width * a.page_size);
  v.n = n;
  v.vis = n;
  v.nsink = 0;
  if (a.window > 0 && n > a.window) {
    v.nsink = min(a.sinks, n - a.window);
    v.vis = a.window + v.nsink;
  }
  if (a.out32 != nullptr) {                             // behind a shared prefix, where the row holds it
    const int prefix = prefix_of(a);
    if (n >= prefix) v.vis = n - prefix;
  }
  v.units = (v.vis + pattn::kUnit - 1) / pattn::kUnit;
  return v;
}

// a place in the sequence of units: row b, key-value head, tile of its query heads, unit of that segment
struct UnitIter {
  int b, hk, ht, unit;
  RowView v;
  __device__ __forceinline__ void next(const PagedAttnArgs& a, int head_tiles) {
    if (++unit < v.units) return;
    unit = 0;
    if (++ht < head_tiles) return;
    ht = 0;
    if (++hk < a.Hkv) return;
    hk = 0;
    while (++b < a.B) {
      v = row_view(a, b);
      if (v.units > 0) break;
    }
  }
};

// two neighbouring outputs: element `to` and the next
template <bool F16>
__device__ __forceinline__ void store_out(const PagedAttnArgs& a, int64_t to, float x, float y) {
  if (a.out32 != nullptr) *reinterpret_cast<float2*>(a.out32 + to) = make_float2(x, y);
  else if constexpr (F16) *reinterpret_cast<__half2*>(static_cast<__half*>(a.out) + to) = __floats2half2_rn(x, y);
  else *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(a.out) + to) = __floats2bfloat162_rn(x, y);
}

// what the weights' exponents are raised by: f16 parts reach up to 2^15, bf16 parts have fp32's range
template <bool F16Math>
__device__ __forceinline__ constexpr float weight_lift() { return F16Math ? 15.0f : 0.0f; }
// log of the softmax's sum, from the largest score (a power of 2) and the sum of the raised weights
__device__ __forceinline__ float log_sum(float top, float sum, float lift) {
  return sum == 0.0f ? -INFINITY : (top + (log2f(sum) - lift)) / 1.4426950408889634f;
}

// 2^x to 2^-22 of it; below 2^-126 zero
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// kCluster: the form for Mode kClusters, apart so that the others do not hold its registers
template <bool F16, bool FP8, int D, int NT, bool kCluster>
__global__ void __launch_bounds__(pattn::kWarps * 32, pattn::Cfg<D, FP8 ? 1 : 2, NT>::kCtas)
    paged_attention_kernel(const PagedAttnArgs a, const int head_tiles, const pattn::Mode mode, const int cluster) {
  using C = pattn::Cfg<D, FP8 ? 1 : 2, NT>;
  constexpr int ES = FP8 ? 1 : 2, kRow = C::kRow, kStages = C::kStages;
  constexpr bool kF16Math = F16 || FP8;
  constexpr float kLift = weight_lift<kF16Math>();
  constexpr int kHeads = 8 * NT;                        // heads of a tile
  constexpr int kMt = D / 16;                           // 16-wide slices of the head dim
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  uint2* qfrag = reinterpret_cast<uint2*>(smem + pattn::kWarps * kStages * C::kStageBytes);
  float* sm_m = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(qfrag) + C::kQ);   // [kWarps][kHeads]
  float* sm_l = sm_m + pattn::kWarps * kHeads;
  float* qmul = sm_l + pattn::kWarps * kHeads;          // [kHeads] score multiplier
  int* start = reinterpret_cast<int*>(qmul + kHeads);   // the run's first (b, head, unit)
  uint32_t* masks = reinterpret_cast<uint32_t*>(start + 4);   // [kWarps][kStages] valid keys of a tile
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int group = a.Hq / a.Hkv, heads = a.Hkv * head_tiles;
  if (mode == pattn::kRuns) grid_dep_launch();                        // the join may be set up while this grid runs

  // ---- this CTA's run of units --------------------------------------------------------------
  int64_t count = 0;
  UnitIter it;
  if constexpr (kCluster) {                             // this CTA's share of the cluster's segment
    const int seg = blockIdx.x / cluster, rank = static_cast<int>(cluster_ctarank());
    it.b = seg / heads;
    const int head = seg - it.b * heads, units = row_view(a, it.b).units;
    it.hk = head / head_tiles;
    it.ht = head - it.hk * head_tiles;
    it.unit = static_cast<int>(static_cast<int64_t>(rank) * units / cluster);
    count = static_cast<int64_t>(rank + 1) * units / cluster - it.unit;
  } else if (mode == pattn::kSegments) {                // runs of whole segments
    const int64_t segs = static_cast<int64_t>(a.B) * heads;
    const int64_t s0 = blockIdx.x * segs / gridDim.x, s1 = (blockIdx.x + 1) * segs / gridDim.x;
    int b0 = static_cast<int>(s0 / heads), h0 = static_cast<int>(s0 % heads);
    for (int64_t s = s0; s < s1;) {
      const int b = static_cast<int>(s / heads);
      const int64_t upto = min(s1, static_cast<int64_t>(b + 1) * heads);
      const int u = row_view(a, b).units;
      if (count == 0 && u > 0) { b0 = b; h0 = static_cast<int>(s % heads); }
      count += u * (upto - s);
      s = upto;
    }
    it.b = b0;
    it.hk = h0 / head_tiles;
    it.ht = h0 - it.hk * head_tiles;
    it.unit = 0;
  } else {                                              // equal runs of units
    __shared__ int64_t wsum[pattn::kWarps];
    const int each = (a.B + blockDim.x - 1) / blockDim.x, first = tid * each, last = min(a.B, first + each);
    int64_t mine = 0;
    for (int b = first; b < last; ++b) mine += row_view(a, b).units;
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < pattn::kWarps; ++w) {
      if (w == warp) incl += total;
      total += wsum[w];
    }
    total *= heads;
    const int64_t runs = max(static_cast<int64_t>(1), min(static_cast<int64_t>(gridDim.x), total / pattn::kMinUnits));
    const int64_t u0 = min(static_cast<int64_t>(blockIdx.x), runs) * total / runs;
    const int64_t u1 = min(static_cast<int64_t>(blockIdx.x) + 1, runs) * total / runs;
    count = u1 - u0;
    const int64_t from = (incl - mine) * heads, to = incl * heads;
    if (count > 0 && u0 >= from && u0 < to) {
      int64_t left = u0 - from;
      for (int b = first; b < last; ++b) {
        const int u = row_view(a, b).units;
        if (left < static_cast<int64_t>(u) * heads) {
          start[0] = b;
          start[1] = static_cast<int>(left / u);
          start[2] = static_cast<int>(left % u);
          break;
        }
        left -= static_cast<int64_t>(u) * heads;
      }
    }
    __syncthreads();
    it.b = count > 0 ? start[0] : 0;
    const int head = count > 0 ? start[1] : 0;
    it.hk = head / head_tiles;
    it.ht = head - it.hk * head_tiles;
    it.unit = count > 0 ? start[2] : 0;
  }
  // rows that see nothing belong to no unit: their zeros
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if (row_view(a, b).units > 0) continue;
    if (a.lse != nullptr)
      for (int i = tid; i < a.Hq; i += blockDim.x) a.lse[static_cast<int64_t>(b) * a.Hq + i] = -INFINITY;
    if (a.out32 != nullptr) continue;                   // its log says that it has none
    uint32_t* o = static_cast<uint32_t*>(a.out) + static_cast<int64_t>(b) * a.Hq * (D / 2);
    for (int i = tid; i < a.Hq * (D / 2); i += blockDim.x) o[i] = 0;
  }
  float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + gridDim.x * sizeof(pattn::Meta));
  if (mode == pattn::kRuns && tid == 0) {
    pattn::Meta m{0, 0, 0, static_cast<int>(count)};
    if (count > 0) m = {it.b * heads + it.hk * head_tiles + it.ht, it.unit, row_view(a, it.b).units, static_cast<int>(count)};
    static_cast<pattn::Meta*>(a.ws)[blockIdx.x] = m;
  }
  it.v = row_view(a, it.b);
  if (count == 0 && (!kCluster || it.v.units == 0)) {
    if (a.out32 != nullptr) grid_dep_wait();
    return;
  }

  // ---- the warp's ring ----------------------------------------------------------------------
  uint8_t* my_ring = ring + warp * kStages * C::kStageBytes;
  const uint32_t my_ring_u = smem_u32(my_ring);
  uint32_t* my_masks = masks + warp * kStages;
  const int page_shift = 31 - __clz(a.page_size), page_mask = a.page_size - 1;
  // lane r < 16 looks after key r of the tile; its page index is loaded a step before the copies need it
  struct Place {
    int page;
    int64_t inner;
  };
  UnitIter ahead = it;
  auto look_up = [&]() {
    const int i = ahead.unit * pattn::kUnit + warp * pattn::kTile + (lane & 15);
    Place p{-1, 0};
    if (i < ahead.v.vis) {
      const int j = i < ahead.v.nsink ? i : ahead.v.n - ahead.v.vis + i;
      p.page = __ldg(a.table + ahead.v.row * a.table_stride + (j >> page_shift));
      p.inner = ahead.hk * a.head_stride + (j & page_mask) * a.tok_stride;
    }
    ahead.next(a, head_tiles);
    return p;
  };
  auto copy = [&](int stage, const Place& p) {
    const bool ok = p.page >= 0 && p.page < a.num_pages;
    const uint32_t mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
    if (lane == 0) my_masks[stage] = mask;
    if (mask == 0) return;
    const int64_t off = ok ? (p.page * a.page_stride + p.inner) * ES : 0;
    constexpr int kChunks = kRow / 16;                  // 16-byte chunks of a row: 4 to 32
    constexpr int kRows = 32 / kChunks;                 // rows of one copy instruction
    const uint32_t dst = my_ring_u + stage * C::kStageBytes;
    const int ch = lane % kChunks;
#pragma unroll
    for (int r0 = 0; r0 < pattn::kTile; r0 += kRows) {
      const int r = r0 + lane / kChunks;
      const int64_t o = __shfl_sync(0xffffffffu, off, r) + 16 * ch;
      const bool valid = mask >> r & 1u;
      const uint32_t to = dst + swz<kRow>(r, ch);
      cp_async16(to, static_cast<const uint8_t*>(a.k) + o, valid);
      cp_async16(to + C::kTileBytes, static_cast<const uint8_t*>(a.v) + o, valid);
    }
  };
  Place place[kStages], next_place{-1, 0};
#pragma unroll
  for (int s = 0; s < kStages; ++s)                     // the first pages' indexes are loaded together
    if (s < count) place[s] = look_up();
#pragma unroll
  for (int s = 0; s < kStages; ++s) {
    if (s < count) copy(s, place[s]);
    cp_async_commit();
  }
  if (kStages < count) next_place = look_up();

  // ---- units --------------------------------------------------------------------------------
  const float log2e = 1.4426950408889634f;
  float o[kMt][NT][4], m[NT][2], l[NT][2], mul[NT][2];
  int part = 0, part_begin = 0, h0 = it.hk * group + it.ht * kHeads, nh = min(kHeads, (it.hk + 1) * group - h0);
  // a cluster's CTA: its part of the segment, as the join's parts are
  float2 mine_o[NT][D / 32];
  float mine_top[NT], mine_sum[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    mine_top[n] = -INFINITY;
    mine_sum[n] = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) mine_o[n][i] = make_float2(0.0f, 0.0f);
  }
  bool fresh = true;
  int stage = 0;
  for (int64_t t = 0; t < count; ++t) {
    if (fresh) {
      fresh = false;
      part_begin = it.unit;
      h0 = it.hk * group + it.ht * kHeads;
      nh = min(kHeads, (it.hk + 1) * group - h0);
      // the tile's query heads as the second operand's fragments, one warp per head
      for (int h = warp; h < kHeads; h += pattn::kWarps) {
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + it.b * a.q_sb + (h0 + h) * a.q_sh;
        uint2 w[(D / 4 + 31) / 32];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < (D / 4 + 31) / 32; ++i) {
          const int e = lane + 32 * i;                  // slice e / 4, column pair e % 4
          w[i] = make_uint2(0, 0);
          if (h < nh && e < D / 4) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(src + 16 * (e >> 2));
            w[i] = FP8 ? make_uint2(__ldg(p + 2 * (e & 3)), __ldg(p + 2 * (e & 3) + 1))
                       : make_uint2(__ldg(p + (e & 3)), __ldg(p + (e & 3) + 4));
          }
          if constexpr (FP8 && !F16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t word = j < 2 ? w[i].x : w[i].y;
              top = fmaxf(top, fabsf(__uint_as_float((j & 1 ? word >> 16 : word & 0xffffu) << 16)));
            }
          }
        }
        float factor = 1.0f;
        if constexpr (FP8 && !F16) {
#pragma unroll
          for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          // top in [2^e, 2^(e + 1)) is taken to [2^13, 2^14); from 2^-126 on both powers are normal numbers
          const int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
          const int by = top > 0.0f && ex < 128 ? max(ex - 13, -126) : 0;
          factor = __uint_as_float(static_cast<uint32_t>(127 + by) << 23);
          const float down = __uint_as_float(static_cast<uint32_t>(127 - by) << 23);
#pragma unroll
          for (int i = 0; i < (D / 4 + 31) / 32; ++i) {
            uint32_t* u = &w[i].x;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const __half2 x = __floats2half2_rn(__uint_as_float(u[j] << 16) * down,
                                                  __uint_as_float(u[j] & 0xffff0000u) * down);
              u[j] = *reinterpret_cast<const uint32_t*>(&x);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < (D / 4 + 31) / 32; ++i) {
          const int e = lane + 32 * i;
          if (e < D / 4) qfrag[((e >> 2) * NT + (h >> 3)) * 32 + (h & 7) * 4 + (e & 3)] = w[i];
        }
        if (lane == 0)
          qmul[h] = a.scale * log2e * factor * (FP8 && a.k_scale != nullptr ? __ldg(a.k_scale + it.hk) : 1.0f);
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
        mul[n][0] = qmul[8 * n + 2 * c];
        mul[n][1] = qmul[8 * n + 2 * c + 1];
#pragma unroll
        for (int i = 0; i < kMt; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][n][j] = 0.0f;
      }
    }
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const uint32_t mask = my_masks[stage];
    if (mask != 0) {
      const uint32_t kt = my_ring_u + stage * C::kStageBytes, vt = kt + C::kTileBytes;
      float s[NT][4], s2[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = s2[n][j] = 0.0f;
      const int kr = (lane & 7) + (lane >> 3 & 1) * 8, kc = lane >> 4;
      if constexpr (!FP8) {
#pragma unroll
        for (int ks = 0; ks < kMt; ++ks) {
          uint32_t ka[4];
          ldsm_x4(ka, kt + swz<kRow>(kr, 2 * ks + kc));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint2 q = qfrag[(ks * NT + n) * 32 + lane];
            mma_16816<kF16Math>(ks & 1 ? s2[n] : s[n], ka, q.x, q.y);
          }
        }
      } else {
#pragma unroll
        for (int kp = 0; kp < kMt / 2; ++kp) {
          uint32_t raw[4];
          ldsm_x4(raw, kt + swz<kRow>(kr, 2 * kp + kc));
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t ka[4];
            e4m3x4_to_f16(raw[2 * half], ka[0], ka[2]);
            e4m3x4_to_f16(raw[2 * half + 1], ka[1], ka[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint2 q = qfrag[((2 * kp + half) * NT + n) * 32 + lane];
              mma_16816<true>(half ? s2[n] : s[n], ka, q.x, q.y);
            }
          }
        }
      }
      // s[n][0..1]: key g, heads 2c, 2c + 1 of the tile's n-th eight; s[n][2..3]: key g + 8
      const bool ok0 = mask >> g & 1u, ok1 = mask >> (g + 8) & 1u;
      uint32_t ph[NT][2], pl[NT][2];
      bool grew = false;
      float f[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float x0 = ok0 ? (s[n][j] + s2[n][j]) * mul[n][j] : -INFINITY;
          const float x1 = ok1 ? (s[n][2 + j] + s2[n][2 + j]) * mul[n][j] : -INFINITY;
          float top = fmaxf(x0, x1);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float mn = fmaxf(m[n][j], top), base = mn == -INFINITY ? 0.0f : mn;   // all may be -inf so far
          f[n][j] = exp2_fast(m[n][j] - base);
          grew |= mn != m[n][j];
          m[n][j] = mn;
          const float y0 = x0 - base, y1 = x1 - base;      // never above 0: a lift of the base could round past it
          s[n][j] = exp2_fast(kF16Math ? y0 + kLift : y0);
          s[n][2 + j] = exp2_fast(kF16Math ? y1 + kLift : y1);
          l[n][j] = l[n][j] * f[n][j] + (s[n][j] + s[n][2 + j]);
        }
        split16<kF16Math>(s[n][0], s[n][1], ph[n][0], pl[n][0]);
        split16<kF16Math>(s[n][2], s[n][3], ph[n][1], pl[n][1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ph[n][j] = movmatrix_t(ph[n][j]);
          pl[n][j] = movmatrix_t(pl[n][j]);
        }
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int i = 0; i < kMt; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][n][j] *= f[n][j & 1];
      }
      if constexpr (!FP8) {
        const int vr = (lane & 7) + (lane >> 4) * 8, vc = lane >> 3 & 1;
#pragma unroll
        for (int i = 0; i < kMt; ++i) {
          uint32_t va[4];
          ldsm_x4_t(va, vt + swz<kRow>(vr, 2 * i + vc));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_16816<kF16Math>(o[i][n], va, ph[n][0], ph[n][1]);
            mma_16816<kF16Math>(o[i][n], va, pl[n][0], pl[n][1]);
          }
        }
      } else {
        // a transposed load gives the columns in pairs: row g of slice i is column 2g, row g + 8 column 2g + 1
#pragma unroll
        for (int ip = 0; ip < kMt / 2; ++ip) {
          uint32_t raw[4];
          ldsm_x4_t(raw, vt + swz<kRow>(kr, 2 * ip + kc));
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t va[4];
            e4m3x4_to_f16(__byte_perm(raw[2 * half], 0, 0x3120), va[0], va[1]);
            e4m3x4_to_f16(__byte_perm(raw[2 * half + 1], 0, 0x3120), va[2], va[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_16816<true>(o[2 * ip + half][n], va, ph[n][0], ph[n][1]);
              mma_16816<true>(o[2 * ip + half][n], va, pl[n][0], pl[n][1]);
            }
          }
        }
      }
    }
    __syncwarp();
    const bool seg_end = it.unit + 1 == it.v.units;
    if (seg_end || t + 1 == count) {
      // ---- the end of this CTA's part of the segment: join the warps, eight heads at a time ------
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
          if (g == 0) {
            sm_m[warp * kHeads + 8 * n + 2 * c + j] = m[n][j];
            sm_l[warp * kHeads + 8 * n + 2 * c + j] = l[n][j];
          }
        }
      __syncthreads();                                    // and every warp is done with its tile
      const bool complete = seg_end && part_begin == 0 && !kCluster;
      const float vs = FP8 && a.v_scale != nullptr ? __ldg(a.v_scale + it.hk) : 1.0f;
      const uint8_t* slot = ring + stage * C::kStageBytes;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* mine = reinterpret_cast<float*>(my_ring + stage * C::kStageBytes);   // [D][8]
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int h = 8 * n + 2 * c + j;
          float top = sm_m[h];
#pragma unroll
          for (int w = 1; w < pattn::kWarps; ++w) top = fmaxf(top, sm_m[w * kHeads + h]);
          const float f = m[n][j] == -INFINITY ? 0.0f : exp2_fast(m[n][j] - top);
#pragma unroll
          for (int i = 0; i < kMt; ++i) {
            o[i][n][j] *= f;
            o[i][n][2 + j] *= f;
          }
        }
#pragma unroll
        for (int i = 0; i < kMt; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int d = FP8 ? 16 * i + 2 * g + r : 16 * i + g + 8 * r;
            *reinterpret_cast<float2*>(mine + d * 8 + 2 * c) = make_float2(o[i][n][2 * r], o[i][n][2 * r + 1]);
          }
        __syncthreads();
        const int h8 = tid & 7, h = 8 * n + h8;           // this thread's head
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < pattn::kWarps; ++w) top = fmaxf(top, sm_m[w * kHeads + h]);
#pragma unroll
        for (int w = 0; w < pattn::kWarps; ++w) {
          const float mw = sm_m[w * kHeads + h], lw = sm_l[w * kHeads + h];
          sum += mw == -INFINITY ? lw : lw * exp2_fast(mw - top);   // without a maximum: zero, or NaN where a score was NaN
        }
        if (h < nh) {
          const float inv = sum == 0.0f ? 0.0f : vs / sum;
          float* p = parts + (static_cast<int64_t>(blockIdx.x) * 2 + min(part, 1)) * kHeads * (D + 2);
          const int64_t to = (static_cast<int64_t>(it.b) * a.Hq + h0 + h) * D;
          mine_top[n] = top;
          mine_sum[n] = sum;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const int d = 2 * (tid >> 3) + 32 * i;
            float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < pattn::kWarps; ++w) {     // in the order of the warps
              const float* from = reinterpret_cast<const float*>(slot + w * kStages * C::kStageBytes) + d * 8 + h8;
              v.x += from[0];
              v.y += from[8];
            }
            if constexpr (kCluster) {
              mine_o[n][i] = v;
            } else if (!complete) {
              *reinterpret_cast<float2*>(p + h * D + d) = v;
            } else {
              store_out<F16>(a, to + d, v.x * inv, v.y * inv);
            }
          }
          if (tid < 8 && !complete && !kCluster) {
            p[kHeads * D + h] = top;
            p[kHeads * D + kHeads + h] = sum;
          }
          if (tid < 8 && complete && a.lse != nullptr)
            a.lse[static_cast<int64_t>(it.b) * a.Hq + h0 + h] = log_sum(top, sum, kLift);
        }
        __syncthreads();                                  // the slots and the statistics are read
      }
      ++part;
      fresh = true;
    }
    // the consumed stage takes the tile kStages ahead
    if (t + kStages < count) {
      copy(stage, next_place);
      if (t + kStages + 1 < count) next_place = look_up();
    }
    cp_async_commit();
    stage = stage + 1 == kStages ? 0 : stage + 1;
    if (t + 1 < count) it.next(a, head_tiles);
  }
  cp_async_wait<0>();
  if constexpr (kCluster) {
    // ---- the cluster's join: every rank's part in its shared memory, the outputs dealt out over the ranks -------
    __syncthreads();                                        // the ring is free
    float* box = reinterpret_cast<float*>(ring);            // [kHeads][D] outputs, maxima, sums
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = 8 * n + (tid & 7);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) *reinterpret_cast<float2*>(box + h * D + 2 * (tid >> 3) + 32 * i) = mine_o[n][i];
      if (tid < 8) {
        box[kHeads * D + h] = mine_top[n];
        box[kHeads * D + kHeads + h] = mine_sum[n];
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int rank = static_cast<int>(cluster_ctarank());
    const float vs = FP8 && a.v_scale != nullptr ? __ldg(a.v_scale + it.hk) : 1.0f;
    const uint32_t box_u = smem_u32(box);
    auto remote = [&](int q, int i) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(box_u + 4 * i, q)));
      return v;
    };
    for (int i = rank * blockDim.x + tid; i < nh * (D / 2); i += cluster * blockDim.x) {
      const int h = i / (D / 2), d = 2 * (i - h * (D / 2));
      float top = -INFINITY, sum = 0.0f;
      for (int q = 0; q < cluster; ++q) top = fmaxf(top, remote(q, kHeads * D + h));
      float2 v = make_float2(0.0f, 0.0f);
      for (int q = 0; q < cluster; ++q) {                   // in the order of the ranks
        const float m = remote(q, kHeads * D + h), s = remote(q, kHeads * D + kHeads + h);
        const float f = m == -INFINITY ? 0.0f : exp2_fast(m - top);
        sum += m == -INFINITY ? s : s * f;
        v.x = fmaf(remote(q, h * D + d), f, v.x);
        v.y = fmaf(remote(q, h * D + d + 1), f, v.y);
      }
      const float inv = sum == 0.0f ? 0.0f : vs / sum;
      const int64_t to = (static_cast<int64_t>(it.b) * a.Hq + h0 + h) * D + d;
      store_out<F16>(a, to, v.x * inv, v.y * inv);
      if (d == 0 && a.lse != nullptr)
        a.lse[static_cast<int64_t>(it.b) * a.Hq + h0 + h] = log_sum(top, sum, kLift);
    }
    // a CTA's part stays until every rank has read it
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  // behind a shared prefix this grid may run beside the one before it: it ends after that, so that what waits for this one
  // finds the results of both
  if (a.out32 != nullptr) grid_dep_wait();
}

// Joins the parts of a row that several CTAs shared, in their order.  CTA (r, h): the segment whose first boundary
// between two runs lies before run r, head h of its tile; most have nothing to do.  Warps take every fourth part.
template <bool F16, int D, int NT>
__global__ void __launch_bounds__(128) paged_attention_join_kernel(const PagedAttnArgs a, const int runs, const int head_tiles) {
  constexpr int kHeads = 8 * NT, kPer = D / 32;           // columns per lane
  __shared__ float sum_o[4][D];
  grid_dep_wait();
  const int r = blockIdx.x + 1, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const pattn::Meta* metas = static_cast<const pattn::Meta*>(a.ws);
  const pattn::Meta me = metas[r];
  if (me.count == 0 || me.unit0 == 0) return;             // no run, or it begins with a segment of its own
  const int before = metas[r - 1].count;
  if (before < me.unit0) return;                          // the segment's first boundary is an earlier one
  const int heads = a.Hkv * head_tiles, group = a.Hq / a.Hkv;
  const int b = me.seg / heads, head = me.seg - b * heads, hk = head / head_tiles;
  const int h0 = hk * group + (head - hk * head_tiles) * kHeads;
  if (h >= min(kHeads, (hk + 1) * group - h0)) return;
  const float* parts = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.ws) + runs * sizeof(pattn::Meta));
  // part 0 is run r - 1's last one (its only one where that run begins with this segment), part i run r - 1 + i's first
  auto at = [&](int i) {
    const int slot = i == 0 && before > me.unit0 ? 1 : 0;
    return parts + (static_cast<int64_t>(r - 1 + i) * 2 + slot) * kHeads * (D + 2);
  };
  int n = 1;
  for (int left = me.units - me.unit0; left > 0; ++n) left -= metas[r - 1 + n].count;
  float top = -INFINITY;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, at(i)[kHeads * D + h]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  float o[kPer] = {}, l = 0.0f;
#pragma unroll 4
  for (int i = warp; i < n; i += 4) {
    const float* p = at(i);
    const float m = p[kHeads * D + h], f = m == -INFINITY ? 0.0f : exp2f(m - top);
#pragma unroll
    for (int j = 0; j < kPer; ++j) o[j] = fmaf(p[h * D + lane + 32 * j], f, o[j]);
  }
  for (int i = lane; i < n; i += 32) {
    const float m = at(i)[kHeads * D + h], s = at(i)[kHeads * D + kHeads + h];
    l += m == -INFINITY ? s : s * exp2f(m - top);
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
  for (int j = 0; j < kPer; ++j) sum_o[warp][lane + 32 * j] = o[j];
  __syncthreads();
  const bool fp8 = a.cache_dtype == CQ_DT_FP8_E4M3;
  const float vs = fp8 && a.v_scale != nullptr ? __ldg(a.v_scale + hk) : 1.0f;
  const float inv = l == 0.0f ? 0.0f : vs / l;
  const int64_t to = (static_cast<int64_t>(b) * a.Hq + h0 + h) * D;
  for (int d = threadIdx.x; d < D; d += 128) {
    const float y = ((sum_o[0][d] + sum_o[1][d]) + (sum_o[2][d] + sum_o[3][d])) * inv;
    if (a.out32 != nullptr) a.out32[to + d] = y;
    else if constexpr (F16) static_cast<__half*>(a.out)[to + d] = __float2half_rn(y);
    else static_cast<__nv_bfloat16*>(a.out)[to + d] = __float2bfloat16_rn(y);
  }
  if (threadIdx.x == 0 && a.lse != nullptr)
    a.lse[static_cast<int64_t>(b) * a.Hq + h0 + h] = log_sum(top, l, fp8 ? weight_lift<true>() : weight_lift<F16>());
}

namespace {
// By what the table's width allows, not by the lengths on the device, so that a captured launch stays right as rows grow: a
// short row in a wide table is dealt out as runs (333 keys: 8.8 us, and 6.1 as a cluster).
struct Deal {
  pattn::Mode mode;
  int64_t units, segs;         // of the row with the most visible keys; segments
  int cluster;
};
Deal deal_units(int64_t batch, int Hq, int Hkv, int64_t span, int64_t window, int64_t sinks) {
  if (window > 0 && window < span) span = sinks < span - window ? window + sinks : span;
  const int group = Hq / Hkv, tile = group <= 8 ? 8 : 16;
  Deal d{pattn::kRuns, (span + pattn::kUnit - 1) / pattn::kUnit, batch * Hkv * ((group + tile - 1) / tile), 1};
  while (d.cluster < 8 && d.cluster < d.units && d.segs * d.cluster * 2 <= pattn::kMaxRuns) d.cluster *= 2;
  if (d.cluster > 1 && d.units <= static_cast<int64_t>(pattn::kClusterUnits) * d.cluster) d.mode = pattn::kClusters;
  else if (d.units <= pattn::kWholeUnits) {
    const int64_t idle = (d.segs + pattn::kMaxRuns - 1) / pattn::kMaxRuns * pattn::kMaxRuns - d.segs;   // in the last wave
    if (d.segs <= pattn::kMaxRuns || idle * d.units <= pattn::kJoinUnits * pattn::kMaxRuns) d.mode = pattn::kSegments;
  }
  return d;
}
}  // namespace

int64_t paged_attention_workspace(int64_t batch, int Hq, int Hkv, int D, int64_t span, int64_t window, int64_t sinks) {
  const int heads = Hq / Hkv <= 8 ? 8 : 16;
  return batch == 0 || deal_units(batch, Hq, Hkv, span, window, sinks).mode != pattn::kRuns
             ? 0
             : pattn::kMaxRuns * static_cast<int64_t>(sizeof(pattn::Meta) + 2 * heads * (D + 2) * sizeof(float));
}

template <bool F16, bool FP8, int D, int NT>
cudaError_t run_paged_attention(const PagedAttnArgs& a, cudaStream_t st) {
  using C = pattn::Cfg<D, FP8 ? 1 : 2, NT>;
  const int group = a.Hq / a.Hkv, tiles = (group + 8 * NT - 1) / (8 * NT);
  const Deal deal = deal_units(a.B, a.Hq, a.Hkv, static_cast<int64_t>(a.table_width) * a.page_size, a.window, a.sinks);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (deal.mode == pattn::kClusters) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(deal.cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(deal.segs * deal.cluster));
    cfg.blockDim = dim3(pattn::kWarps * 32);
    cfg.dynamicSmemBytes = C::kSmem;
    auto kern = paged_attention_kernel<F16, FP8, D, NT, true>;
    static unsigned long long devices = 0;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = a.out32 != nullptr ? 2 : 1;          // beside the kernel of the shared prefix
    const cudaError_t e = allow_shared(kern, C::kSmem, devices);
    return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, kern, a, tiles, deal.mode, deal.cluster);
  }
  auto kern = paged_attention_kernel<F16, FP8, D, NT, false>;
  static unsigned long long devices = 0;
  cudaError_t e = allow_shared(kern, C::kSmem, devices);
  if (e != cudaSuccess) return e;
  int64_t grid = static_cast<int64_t>(num_sms()) * C::kCtas;
  if (grid > pattn::kMaxRuns) grid = pattn::kMaxRuns;
  const int64_t most = deal.mode == pattn::kSegments ? deal.segs
                                                     : deal.segs * ((deal.units + pattn::kMinUnits - 1) / pattn::kMinUnits);
  if (most < grid) grid = most;
  if (a.out32 != nullptr) {                             // beside the kernel of the shared prefix
    e = launch_early(kern, dim3(static_cast<unsigned>(grid)), pattn::kWarps * 32, C::kSmem, st, a, tiles, deal.mode, 1);
  } else {
    kern<<<static_cast<unsigned>(grid), pattn::kWarps * 32, C::kSmem, st>>>(a, tiles, deal.mode, 1);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess || deal.mode != pattn::kRuns || grid == 1) return e;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(grid - 1), group < 8 * NT ? group : 8 * NT);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<F16, D, NT>, a, static_cast<int>(grid), tiles);
}

template <bool F16, bool FP8>
cudaError_t pick_paged_attention(const PagedAttnArgs& a, cudaStream_t st) {
  const bool wide = a.Hq / a.Hkv > 8;                     // heads of a tile: 16, or 8
  switch (a.D) {
    case 64: return wide ? run_paged_attention<F16, FP8, 64, 2>(a, st) : run_paged_attention<F16, FP8, 64, 1>(a, st);
    case 128: return wide ? run_paged_attention<F16, FP8, 128, 2>(a, st) : run_paged_attention<F16, FP8, 128, 1>(a, st);
    default: return wide ? run_paged_attention<F16, FP8, 256, 2>(a, st) : run_paged_attention<F16, FP8, 256, 1>(a, st);
  }
}

cudaError_t launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st) {
  const bool fp8 = a.cache_dtype == CQ_DT_FP8_E4M3;
  if (a.dtype == CQ_DT_F16) return fp8 ? pick_paged_attention<true, true>(a, st) : pick_paged_attention<true, false>(a, st);
  return fp8 ? pick_paged_attention<false, true>(a, st) : pick_paged_attention<false, false>(a, st);
}

}  // namespace cq
