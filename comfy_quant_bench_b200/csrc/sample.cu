// The next token of each row from its logits and one given uniform number: temperature, top-k, top-p, min-p.
//
//   weight_i = exp((l_i - max) / T); the first k tokens in the order (logit descending, index ascending); of those the
//   shortest head whose sum reaches p times theirs; of those the ones with weight >= min_p; then the first token, in the
//   order of the indexes, whose running sum exceeds u times the sum.
//
// The choice has to be the one of exact arithmetic, so weights are integers, round(2^44 weight): sums are exact, in any
// order, and equal calls give equal bits.  2^x comes in 64 bits from a table of 2^(j/64) and a polynomial of degree five in
// the rest, |rest| <= 1/128 (Taylor: the next term is 4e-17, a thousandth of 2^-44; of degree four it would be 4e-14, more
// than half of it).  A token whose weight rounds to 0 can neither be chosen nor count.
//
// A cluster of CTAs takes a row and keeps it in shared memory: one read of the logits.  A cut (of top-k, of top-p) is an
// element's composite, its logit's order in the high half and its index, reversed, in the low: what lies at or above it
// stays.  To find one, tokens are counted into bins by max - logit, the sums of all bins above the border's are exact, and
// the border's few tokens are ranked one against another; a bin with more of them (equal logits) is halved instead.  Where no
// more than 512 tokens can stay, one CTA takes them over, sorts them in registers and finishes, and the others leave.
//
// Measured on a B200, calls in a row: 128 rows of 128257 f32 logits, top-k 200, top-p and min-p: 86 us, 0.8 TB/s; one row of
// 32000 bf16 logits with top-p 0.9: 15 to 20 us by the box (27 alone and cold); 128 rows of 32000 bf16: 49 us with all
// filters, 93 with top-p alone, 35 with none, 18 for the likeliest token.  Bound by the chain of a row's steps (load, maximum,
// counts, candidates, sort: four waits for the cluster of about 0.5 us each among them), of which an SM holds two CTAs at a
// time.
#include "decode_common.cuh"

namespace cq {

namespace samp {
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 1024;                    // tokens of a border bin that are ranked; more are halved
constexpr int kFew = kThreads;                 // candidates that one CTA can finish alone, one a thread
constexpr int kMaxCluster = 8;
constexpr int kFixed = 44;                     // fractional bits of a weight
constexpr float kReach = 31.2f;                // weights below e^-31.2 < 2^-45 round to 0
using u64 = unsigned long long;

struct Shared {
  union {
    u64 wsum[kBins];                           // weights of a bin near top-p's border
    struct {
      u64 list[kList], weight[kList];          // a border bin's tokens
    };
  };
  u64 other[kFew];
  u64 warp_sums[2][kWarps];
  u64 slots[2][kMaxCluster][2];                // what the cluster's CTAs tell one another
  u64 best[kWarps];
  double power[64];                            // 2^(j / 64)
  uint32_t hist[kBins];                        // this CTA's
  uint32_t total[kBins];                       // the row's
  uint32_t warp_counts[kWarps];
  int list_n;                                  // of rank 0: candidates that the ranks have reserved places for
  int list_at, pushed;                         // this CTA's first place, and places used
  int found[4];
  u64 found_sum;
};
}  // namespace samp

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync_all() {
  cluster_arrive();
  cluster_wait();
}
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long ld_cluster_u64(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// A logit's place among all: larger for larger logits; -0 and 0 alike
__device__ __forceinline__ uint32_t logit_order(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float logit_of_order(uint32_t order) {
  return __uint_as_float(order ^ (order >> 31 ? 0x80000000u : 0xffffffffu));
}

template <int TYPE>                            // CQ_DT_BF16, CQ_DT_F16, CQ_DT_F32
struct Sampler {
  using u64 = samp::u64;
  static constexpr int kSize = TYPE == CQ_DT_F32 ? 4 : 2;
  samp::Shared& s;
  const uint8_t* data;                         // this CTA's elements
  int rank, ranks, tid, lane, warp;
  int first, span;                             // this warp's elements: [first, first + span)
  int index0;                                  // row index of element 0; may be negative (before the row's first)
  int count;                                   // elements held
  float top, range, inv_width;
  double by;                                   // log2(e) / T
  int parity;

  __device__ __forceinline__ float logit(int e) const {
    float l;
    if constexpr (TYPE == CQ_DT_F32) l = reinterpret_cast<const float*>(data)[e];
    else l = widen16<TYPE == CQ_DT_F16>(reinterpret_cast<const uint16_t*>(data)[e]).x;
    return l;
  }
  // f(logit, element) for this thread's share of the CTA's elements, 16 bytes at a time; all elements exist (those outside
  // the row are -inf)
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    constexpr int kPer = 16 / kSize;
#pragma unroll 2
    for (int w = tid; w < count / kPer; w += samp::kThreads) {
      const uint4 v = reinterpret_cast<const uint4*>(data)[w];
      const uint32_t* u = &v.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (TYPE == CQ_DT_F32) {
          f(__uint_as_float(u[j]), w * kPer + j);
        } else {
          const float2 l = widen16<TYPE == CQ_DT_F16>(u[j]);
          f(l.x, w * kPer + 2 * j);
          f(l.y, w * kPer + 2 * j + 1);
        }
      }
    }
  }
  // the bin of a logit, -1 where its weight is 0 (or it is NaN)
  __device__ __forceinline__ int bin(float l) const {
    const float d = l == top ? 0.0f : top - l;
    if (!(d <= range)) return -1;
    return min(max(static_cast<int>(d * inv_width), 0), samp::kBins - 1);
  }
  __device__ __forceinline__ double exponent(float l) const {
    return l == top ? 0.0 : (static_cast<double>(l) - static_cast<double>(top)) * by;
  }
  __device__ __forceinline__ u64 weight_of(double y) const {          // round(2^44 2^y), y <= 0
    if (!(y > -46.0)) return 0;
    const double magic = 6755399441055744.0;                          // 1.5 * 2^52: the sum's low bits are the integer
    const double t = fma(y, 64.0, magic);
    const int k = static_cast<int>(__double2loint(t));
    const double f = fma(t - magic, -1.0 / 64.0, y);
    constexpr double l2 = 0.693147180559945309417;
    double p = fma(f, l2 * l2 * l2 * l2 * l2 / 120.0, l2 * l2 * l2 * l2 / 24.0);
    p = fma(f, p, l2 * l2 * l2 / 6.0);
    p = fma(f, p, l2 * l2 / 2.0);
    p = fma(f, p, l2);
    p = fma(f, p, 1.0) * s.power[k & 63];
    const double w = __hiloint2double(__double2hiint(p) + ((samp::kFixed + (k >> 6)) << 20), __double2loint(p));
    return static_cast<u64>(__double_as_longlong(w + 4503599627370496.0)) & ((1ull << 52) - 1);   // 2^52: the sum rounds
  }
  __device__ __forceinline__ u64 composite(float l, int e) const {
    return static_cast<u64>(logit_order(l)) << 32 | (0xffffffffu - static_cast<uint32_t>(index0 + e));
  }
  __device__ __forceinline__ uint32_t there(const void* mine, int r) const { return mapa_shared(smem_u32(mine), r); }

  // rank 0's count of listed tokens, increased; the count before
  __device__ __forceinline__ int add_at_first(int n) const {
    int before;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(before) : "r"(there(&s.list_n, 0)), "r"(n) : "memory");
    return before;
  }
  // the sum over the CTA's threads, in every thread
  __device__ __forceinline__ u64 block_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) s.warp_sums[0][warp] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < samp::kWarps; ++w) v += s.warp_sums[0][w];
    return v;
  }
  // the sum over the threads up to this one; `total`: over all
  __device__ __forceinline__ u64 block_scan(u64 v, u64& total) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) s.warp_sums[0][warp] = v;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < samp::kWarps; ++w) {
      if (w == warp) v += total;
      total += s.warp_sums[0][w];
    }
    return v;
  }
  // two values of each CTA, in every CTA, by rank, in s.slots[parity] after the call (until the call after the next)
  __device__ __forceinline__ const u64 (*exchange(u64 a, u64 b))[2] {
    parity ^= 1;
    if (tid < ranks) {
      const uint32_t to = there(&s.slots[parity][rank][0], tid);
      st_cluster_u64(to, a);
      st_cluster_u64(to + 8, b);
    }
    cluster_sync_all();
    return s.slots[parity];
  }
  __device__ __forceinline__ u64 cluster_sum(u64 v) {
    const u64(*all)[2] = exchange(block_sum(v), 0);
    u64 sum = 0;
    for (int r = 0; r < ranks; ++r) sum += all[r][0];
    return sum;
  }

  // The elements of bin `b` that lie at or above `from`: the composite of the last one that has to stay, so that what is
  // above the bin (`above`) and what stays of it reach `target`.  WEIGHTS: measured by weights, else counted.
  template <bool WEIGHTS>
  __device__ u64 cut_in_bin(int b, u64 from, u64 above, u64 target, u64 n) {
    if (n <= samp::kList) {
      if (tid == 0) s.list_n = 0;
      cluster_sync_all();                                              // lists are empty, and what they held is read
      each([&](float l, int e) {
        if (bin(l) != b) return;
        const u64 c = composite(l, e);
        if (c < from) return;
        const int place = add_at_first(1);
        const u64 w = WEIGHTS ? weight_of(exponent(l)) : 1;
        for (int r = 0; r < ranks; ++r) {
          st_cluster_u64(there(&s.list[place], r), c);
          st_cluster_u64(there(&s.weight[place], r), w);
        }
      });
      cluster_sync_all();
      const int held = static_cast<int>(ld_cluster_u32(there(&s.list_n, 0)));
      u64 best = 0;
      for (int i = tid; i < held; i += samp::kThreads) {
        const u64 c = s.list[i];
        u64 sum = above;
        for (int j = 0; j < held; ++j) sum += s.list[j] >= c ? s.weight[j] : 0;
        if (sum >= target && c > best) best = c;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
      }
      if (lane == 0) s.best[warp] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < samp::kWarps; ++w) best = s.best[w] > best ? s.best[w] : best;
      __syncthreads();
      return best;
    }
    // halving: the largest c whose elements at or above it reach the target
    u64 lo = from, hi = ~0ull;
    while (lo < hi) {
      const u64 mid = lo + (hi - lo) / 2 + 1;
      u64 sum = 0;
      each([&](float l, int e) {
        if (bin(l) == b && composite(l, e) >= mid) sum += WEIGHTS ? weight_of(exponent(l)) : 1;
      });
      if (above + cluster_sum(sum) >= target) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
};

// One key a thread (0: none), in the first SIZE threads, sorted, largest first: bitonic, within a warp by shuffles.
template <int SIZE>
__device__ __forceinline__ unsigned long long sort_keys_of(unsigned long long key, unsigned long long* box) {
  const int i = threadIdx.x;
#pragma unroll
  for (int k = 2; k <= SIZE; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      unsigned long long other;
      if (j >= 32) {
        __syncthreads();
        box[i] = key;
        __syncthreads();
        other = box[i ^ j];
      } else {
        other = __shfl_xor_sync(0xffffffffu, key, j);
      }
      const bool larger = ((i & j) == 0) == ((i & k) == 0);
      key = (other > key) == larger ? other : key;
    }
  }
  return key;
}
__device__ __noinline__ unsigned long long sort_keys(unsigned long long key, int n, unsigned long long* box) {
  if (n <= 64) return sort_keys_of<64>(key, box);
  return n <= 256 ? sort_keys_of<256>(key, box) : sort_keys_of<samp::kFew>(key, box);
}

// The token from a list of n <= kFew candidates: every token that can stay is among them.  `total`: what top-p refers to
// where top-k does not cut (else the sum of those that top-k keeps).  One CTA, one candidate a thread.
template <int TYPE>
__device__ void finish_from_list(const SampleArgs& a, Sampler<TYPE>& s, int64_t row, int n, int top_k, bool cut_p, float top_p,
                                 double floor_y, unsigned long long total, double uniform) {
  using u64 = samp::u64;
  const int i = s.tid;
  // in order: the rank is the thread's number
  const u64 c = sort_keys(i < n ? s.s.list[i] : 0, n, s.s.weight);
  const bool mine = i < n && (top_k == 0 || i < top_k);
  const double y = mine ? s.exponent(logit_of_order(static_cast<uint32_t>(c >> 32))) : -100.0;
  const u64 w = s.weight_of(y);
  u64 sum;
  const u64 through = s.block_scan(w, sum);
  if (top_k != 0) total = sum;
  bool stays = mine && y >= floor_y;
  if (cut_p) {
    const double wanted = ceil(static_cast<double>(fmaxf(top_p, 0.0f)) * static_cast<double>(total));
    const u64 target = wanted >= 9.2e18 ? total : static_cast<u64>(wanted);
    stays = stays && (through - w < target || i == 0);
  }
  // what stays, by index: the composite's low half is the index reversed
  __syncthreads();
  s.s.weight[i] = stays ? w : 0;
  s.s.list[i] = c;
  const u64 by_index = sort_keys(stays ? c << 32 | static_cast<uint32_t>(i) : 0, n, s.s.other);
  const int from = static_cast<int>(by_index & 0xffffffffu);
  __syncthreads();
  const u64 kept = by_index != 0 ? s.s.weight[from] : 0;
  const u64 upto = s.block_scan(kept, sum);
  const double at = uniform * static_cast<double>(sum);
  u64 goal = !(at > 0.0) ? 0 : at >= 9.2e18 ? sum - 1 : static_cast<u64>(at);
  goal = goal > sum - 1 ? sum - 1 : goal;
  if (upto > goal && upto - kept <= goal) {
    a.tokens[row] = static_cast<long long>(0xffffffffu - static_cast<uint32_t>(by_index >> 32));
    if (a.logprobs != nullptr)
      a.logprobs[row] = static_cast<float>(s.exponent(logit_of_order(static_cast<uint32_t>(s.s.list[from] >> 32))) * 0.693147180559945309417 -
                                           log(static_cast<double>(sum) * 5.6843418860808015e-14));   // 2^-44
  }
}

template <int TYPE>
__global__ void __launch_bounds__(samp::kThreads, 2) sample_kernel(const SampleArgs a, const int ranks) {
  using S = Sampler<TYPE>;
  using u64 = samp::u64;
  constexpr int kSize = S::kSize, kPer = 16 / kSize;                   // elements of a 16-byte word
  extern __shared__ __align__(16) uint8_t smem[];
  samp::Shared& sh = *reinterpret_cast<samp::Shared*>(smem);
  uint8_t* data = smem + (sizeof(samp::Shared) + 15) / 16 * 16;
  const int tid = threadIdx.x, rank = ranks > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int64_t row = blockIdx.x / ranks;
  grid_dep_launch();
  if (tid < 64) sh.power[tid] = exp2(tid / 64.0);
  if (tid == 0) sh.list_n = 0;
  for (int i = tid; i < samp::kBins; i += samp::kThreads) sh.hist[i] = 0;
  __syncwarp();
  cluster_arrive();                                                    // this CTA runs: waited for below
  grid_dep_wait();

  const float temperature = a.temperatures != nullptr ? a.temperatures[row] : a.temperature;
  const int top_k = a.top_ks != nullptr ? a.top_ks[row] : a.top_k;
  const float top_p = a.top_ps != nullptr ? a.top_ps[row] : a.top_p;
  const float min_p = a.min_ps != nullptr ? a.min_ps[row] : a.min_p;
  const double uniform = static_cast<double>(a.uniform[row]);

  // ---- this CTA's share of the row's 16-byte words; elements outside the row become -inf ----
  const uintptr_t begin = reinterpret_cast<uintptr_t>(a.logits) + row * a.ld * kSize, end = begin + static_cast<int64_t>(a.vocab) * kSize;
  const uintptr_t word0 = begin >> 4;
  const int words = static_cast<int>((end + 15 >> 4) - word0), each = (words + ranks - 1) / ranks;
  const int w0 = min(words, rank * each), w1 = min(words, w0 + each);
  float most = -INFINITY, least = INFINITY;
  for (int w = w0 + tid; w < w1; w += samp::kThreads) {
    const uintptr_t at = word0 + w << 4;
    uint4 v;
    uint32_t* u = &v.x;
    if (at >= begin && at + 16 <= end) {
      v = *reinterpret_cast<const uint4*>(at);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uintptr_t p = at + 4 * j;
        if constexpr (kSize == 4) {
          u[j] = p >= begin && p + 4 <= end ? *reinterpret_cast<const uint32_t*>(p) : 0xff800000u;
        } else {
          const uint32_t none = TYPE == CQ_DT_F16 ? 0xfc00u : 0xff80u;
          const uint32_t lo = p >= begin && p + 2 <= end ? *reinterpret_cast<const uint16_t*>(p) : none;
          const uint32_t hi = p + 2 >= begin && p + 4 <= end ? *reinterpret_cast<const uint16_t*>(p + 2) : none;
          u[j] = lo | hi << 16;
        }
      }
    }
    *reinterpret_cast<uint4*>(data + (w - w0) * 16) = v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kSize == 4) {
        const float l = __uint_as_float(u[j]);
        most = fmaxf(most, l);                                         // NaN is passed over
        if (l > -INFINITY) least = fminf(least, l);
      } else {
        const float2 l = widen16<TYPE == CQ_DT_F16>(u[j]);
        most = fmaxf(most, fmaxf(l.x, l.y));
        if (l.x > -INFINITY) least = fminf(least, l.x);
        if (l.y > -INFINITY) least = fminf(least, l.y);
      }
    }
  }
  S s{sh, data, rank, ranks, tid, tid & 31, tid >> 5};
  s.count = (w1 - w0) * kPer;
  s.index0 = static_cast<int>((static_cast<int64_t>(word0 + w0 << 4) - static_cast<int64_t>(begin)) / kSize);
  s.parity = 0;
  const int per_warp = ((s.count + samp::kWarps - 1) / samp::kWarps + 31) & ~31;
  s.first = min(s.count, s.warp * per_warp);
  s.span = min(s.count - s.first, per_warp);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  }
  float* box = reinterpret_cast<float*>(sh.warp_sums);                 // [2][kWarps]
  if (s.lane == 0) {
    box[s.warp] = most;
    box[samp::kWarps + s.warp] = least;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < samp::kWarps; ++w) {
    most = fmaxf(most, box[w]);
    least = fminf(least, box[samp::kWarps + w]);
  }
  __syncthreads();
  cluster_wait();                                                      // all of them run: their memory may be written
  {
    const u64(*all)[2] = s.exchange(__float_as_uint(most), __float_as_uint(least));
    for (int r = 0; r < ranks; ++r) {
      most = fmaxf(most, __uint_as_float(static_cast<uint32_t>(all[r][0])));
      least = fminf(least, __uint_as_float(static_cast<uint32_t>(all[r][1])));
    }
  }
  s.top = most;
  if (most == -INFINITY) {                                             // nothing to choose from
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs != nullptr) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  if (!(temperature > 0.0f)) {                                         // the likeliest, lowest index first
    int at = 0x7fffffff;
    for (int e = s.first + s.lane; e < s.first + s.span; e += 32)
      if (s.logit(e) == most) at = min(at, s.index0 + e);
    at = __reduce_min_sync(0xffffffffu, at);
    if (s.lane == 0) sh.warp_counts[s.warp] = at;
    __syncthreads();
    for (int w = 0; w < samp::kWarps; ++w) at = min(at, static_cast<int>(sh.warp_counts[w]));
    const u64(*all)[2] = s.exchange(at, 0);
    for (int r = 0; r < ranks; ++r) at = min(at, static_cast<int>(all[r][0]));
    if (rank == 0 && tid == 0) {
      a.tokens[row] = at;
      if (a.logprobs != nullptr) a.logprobs[row] = 0.0f;
    }
    return;
  }
  s.by = 1.4426950408889634074 / static_cast<double>(temperature);
  s.range = fminf(fminf(samp::kReach * temperature, most - least), 3e38f);
  // finite where the reach is next to nothing (temperatures below 7e-37): bins are then wider than they have to be
  s.inv_width = s.range > 0.0f ? fminf(samp::kBins / s.range, 1e38f) : 0.0f;
  const bool cut_k = top_k > 0 && top_k < a.vocab, cut_p = top_p < 1.0f;

  u64 cut = 0;                                                         // what lies at or above it stays
  if (cut_k || cut_p) {
    // ---- tokens by bins, over the whole row in every CTA ----
    s.each([&](float l, int) {
      const int b = s.bin(l);
      if (b >= 0) atomicAdd(&sh.hist[b], 1u);
    });
    cluster_sync_all();
    const int per = samp::kBins / ranks;
    for (int i = rank * per + tid; i < (rank + 1) * per; i += samp::kThreads) {
      uint32_t sum = 0;
#pragma unroll
      for (int r = 0; r < samp::kMaxCluster; ++r) sum += r < ranks ? ld_cluster_u32(s.there(&sh.hist[i], r)) : 0;
#pragma unroll
      for (int r = 0; r < samp::kMaxCluster; ++r)
        if (r < ranks) st_cluster_u32(s.there(&sh.total[i], r), sum);
    }
    cluster_sync_all();
  }
  constexpr int kEach = samp::kBins / samp::kThreads;                  // bins of a thread in a scan
  const double floor_y = min_p > 0.0f ? log2(static_cast<double>(fminf(min_p, 1.0f))) : -100.0;
  // the tokens of the bins up to `last` into rank 0's list; with `sum` the weights of all tokens are added up, too.
  // A CTA's places are reserved by what its own bins count.
  auto list_up_to = [&](int last, u64* sum) {
    uint32_t mine = 0;
    for (int b = tid; b <= last; b += samp::kThreads) mine += sh.hist[b];
    const int n = static_cast<int>(s.block_sum(mine));
    if (tid == 0) {
      sh.pushed = 0;
      sh.list_at = s.add_at_first(n);
    }
    __syncthreads();
    s.each([&](float l, int e) {
      const int b = s.bin(l);
      if (b < 0 || (sum == nullptr && b > last)) return;
      if (sum != nullptr) *sum += s.weight_of(s.exponent(l));
      if (b > last) return;
      st_cluster_u64(s.there(&sh.list[sh.list_at + atomicAdd(&sh.pushed, 1)], 0), s.composite(l, e));
    });
    if (sum == nullptr) cluster_sync_all();
  };
  if (cut_k) {
    // ---- the bin in which the k-th token lies ----
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) mine += sh.total[tid * kEach + j];
    uint32_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, before, o);
      if (s.lane >= o) before += u;
    }
    if (s.lane == 31) sh.warp_counts[s.warp] = before;
    if (tid == 0) sh.found[0] = -1;
    __syncthreads();
    before -= mine;
    for (int w = 0; w < s.warp; ++w) before += sh.warp_counts[w];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const uint32_t n = sh.total[tid * kEach + j];
      if (before < static_cast<uint32_t>(top_k) && before + n >= static_cast<uint32_t>(top_k)) {
        sh.found[0] = tid * kEach + j;
        sh.found[1] = static_cast<int>(before);
      }
      before += n;
    }
    __syncthreads();
    const int b = sh.found[0];
    if (b >= 0) {
      const int above = sh.found[1], n = above + static_cast<int>(sh.total[b]);
      if (n <= samp::kFew) {
        list_up_to(b, nullptr);
        if (rank == 0) finish_from_list<TYPE>(a, s, row, n, top_k, cut_p, top_p, floor_y, 0, uniform);
        return;
      }
      cut = s.template cut_in_bin<false>(b, 0, above, top_k, sh.total[b]);
    }
  }
  if (cut_p) {
    // ---- bounds of the sums from the counts: a token of bin b weighs 2^-(b + 1) width .. 2^-b width; the border lies in a
    // bin that the bounds allow; sums of the bins before are exact, and those of the allowed bins each ----
    // top-k's cut ends the bins; its own one is counted whole in the upper bounds and not at all in the lower
    const float step = s.inv_width > 0.0f ? static_cast<float>(s.by / s.inv_width) : 0.0f;   // a bin's width, as a power of 2
    // of a bin's bounds (1.001: fp32 bins); what is in a bin weighs 2^-46 at least, however wide the bin
    const float ratio = exp2f(fminf(step * 1.001f, 46.0f));
    const int last = cut != 0 ? sh.found[0] : samp::kBins - 1;         // no token below this bin
    float up[kEach], mine = 0.0f;                                      // upper bounds
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int b = tid * kEach + j;
      up[j] = b <= last ? sh.total[b] * exp2f(-step * b) : 0.0f;
      mine += up[j];
    }
    float before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float u = __shfl_up_sync(0xffffffffu, before, o);
      if (s.lane >= o) before += u;
    }
    float* fbox = reinterpret_cast<float*>(sh.warp_counts);
    __syncthreads();
    if (s.lane == 31) fbox[s.warp] = before;
    if (tid == 0) {
      sh.found[2] = samp::kBins;
      sh.found[3] = -1;
    }
    __syncthreads();
    before -= mine;
    float whole = 0.0f;
    for (int w = 0; w < samp::kWarps; ++w) {
      if (w < s.warp) before += fbox[w];
      whole += fbox[w];
    }
    // exact sum before a bin in [before / ratio, before], the row's in [whole / ratio - its border bin's, whole]
    const float border = cut != 0 ? sh.total[last] * exp2f(-step * last) : 0.0f;
    const float p = fmaxf(top_p, 0.0f), slack = 1.0f + 1e-3f;
    const float least_target = p * fmaxf(whole - border, 0.0f) / (ratio * slack), most_target = p * whole * slack;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int b = tid * kEach + j;
      // bin b can hold the border unless all of it is surely kept, or all of it surely dropped
      if (up[j] > 0.0f && (before + up[j]) * slack >= least_target && before <= most_target * (ratio * slack)) {
        atomicMin(&sh.found[2], b);
        atomicMax(&sh.found[3], b);
      }
      before += up[j];
    }
    __syncthreads();
    const int lo = sh.found[2], hi = sh.found[3];
    u64 above = 0, sum = 0;
    if (cut == 0) {
      // few tokens up to the last bin that the border can lie in: one CTA finishes from a list of them
      uint32_t upto = 0;
      for (int b = tid; b <= hi; b += samp::kThreads) upto += sh.total[b];
      const int n = static_cast<int>(s.block_sum(upto));
      if (n <= samp::kFew) {
        list_up_to(hi, &sum);
        const u64(*all)[2] = s.exchange(s.block_sum(sum), 0);
        if (rank != 0) return;
        u64 whole_sum = 0;
        for (int r = 0; r < ranks; ++r) whole_sum += all[r][0];
        finish_from_list<TYPE>(a, s, row, n, 0, true, top_p, floor_y, whole_sum, uniform);
        return;
      }
    }
    for (int i = tid; i < samp::kBins; i += samp::kThreads) sh.wsum[i] = 0;
    __syncthreads();
    s.each([&](float l, int e) {
      const int b = s.bin(l);
      if (b < 0 || s.composite(l, e) < cut) return;
      const u64 w = s.weight_of(s.exponent(l));
      sum += w;
      if (b < lo) above += w;
      else if (b <= hi) atomicAdd(&sh.wsum[b], w);
    });
    const u64 my_sum = s.block_sum(sum), my_above = s.block_sum(above);
    const u64(*all)[2] = s.exchange(my_sum, my_above);
    u64 total = 0;
    above = 0;
    for (int r = 0; r < ranks; ++r) {
      total += all[r][0];
      above += all[r][1];
    }
    // the allowed bins' sums over the cluster: every CTA adds them all up (they are few)
    if (tid == 0) sh.found_sum = ~0ull;
    const double wanted = ceil(static_cast<double>(p) * static_cast<double>(total));
    u64 target = wanted >= 9.2e18 ? total : static_cast<u64>(wanted);
    target = target < 1 ? 1 : target > total ? total : target;
    __syncthreads();
    // thread i takes the allowed bins in runs, so that a scan gives the sums before each
    const int bins = hi - lo + 1, run = (bins + samp::kThreads - 1) / samp::kThreads;
    u64 part = 0;
    for (int j = 0; j < run; ++j) {
      const int b = lo + tid * run + j;
      if (b <= hi) {
        u64 w = 0;
        for (int r = 0; r < ranks; ++r) w += ld_cluster_u64(s.there(&sh.wsum[b], r));
        part += w;
      }
    }
    u64 incl = part;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 u = __shfl_up_sync(0xffffffffu, incl, o);
      if (s.lane >= o) incl += u;
    }
    if (s.lane == 31) sh.warp_sums[1][s.warp] = incl;
    __syncthreads();
    u64 run_sum = above + incl - part;
    for (int w = 0; w < s.warp; ++w) run_sum += sh.warp_sums[1][w];
    for (int j = 0; j < run; ++j) {
      const int b = lo + tid * run + j;
      if (b <= hi) {
        u64 w = 0;
        for (int r = 0; r < ranks; ++r) w += ld_cluster_u64(s.there(&sh.wsum[b], r));
        if (run_sum < target && run_sum + w >= target) {
          sh.found[2] = b;
          sh.found_sum = run_sum;
        }
        run_sum += w;
      }
    }
    __syncthreads();
    const int b = sh.found[2];
    const u64 sum_above = sh.found_sum;
    cluster_sync_all();                                                // everyone has read the sums
    if (sum_above != ~0ull) cut = s.template cut_in_bin<true>(b, cut, sum_above, target, sh.total[b]);
  }

  // ---- what stays: sums by warps, then the token ----
  auto kept = [&](int e, double& y) {
    const float l = s.logit(e);
    if (s.bin(l) < 0 || s.composite(l, e) < cut) return static_cast<u64>(0);
    y = s.exponent(l);
    return y >= floor_y ? s.weight_of(y) : 0;
  };
  u64 sum = 0;
  double y = 0.0;
  for (int e = s.first + s.lane; e < s.first + s.span; e += 32) sum += kept(e, y);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (s.lane == 0) sh.warp_sums[0][s.warp] = sum;
  __syncthreads();
  u64 mine = 0, before = 0;
  for (int w = 0; w < samp::kWarps; ++w) {
    if (w < s.warp) before += sh.warp_sums[0][w];
    mine += sh.warp_sums[0][w];
  }
  const u64(*all)[2] = s.exchange(mine, 0);
  u64 total = 0;
  for (int r = 0; r < ranks; ++r) {
    if (r < rank) before += all[r][0];
    total += all[r][0];
  }
  const double at = uniform > 0.0 ? uniform * static_cast<double>(total) : 0.0;   // NaN: the first
  u64 goal = at >= 9.2e18 ? total - 1 : static_cast<u64>(at);
  goal = goal > total - 1 ? total - 1 : goal;
  if (goal < before || goal >= before + sum) return;                   // another warp's
  for (int e0 = s.first; e0 < s.first + s.span; e0 += 32) {
    const int e = e0 + s.lane;
    const u64 w = e < s.first + s.span ? kept(e, y) : 0;
    u64 incl = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 v = __shfl_up_sync(0xffffffffu, incl, o);
      if (s.lane >= o) incl += v;
    }
    const uint32_t over = __ballot_sync(0xffffffffu, before + incl > goal);
    if (over != 0) {
      if (s.lane == __ffs(over) - 1) {
        a.tokens[row] = s.index0 + e;
        if (a.logprobs != nullptr)
          a.logprobs[row] = static_cast<float>(y * 0.693147180559945309417 - log(static_cast<double>(total) * 5.6843418860808015e-14));   // 2^-44
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
}

namespace {
template <int TYPE>
cudaError_t run_sample(const SampleArgs& a, cudaStream_t st) {
  constexpr int kSize = TYPE == CQ_DT_F32 ? 4 : 2;
  // a CTA for each 2048 tokens, up to a cluster of eight: one row of 32000 with top-p takes 20 us on eight, 28 on four, 39 on
  // two and 68 on one, 128 rows of 128257 204 us on eight and 253 on four (sixteen were slower at both).  Not the best for many
  // rows of fewer tokens: 32 rows of 32000 take 27 us on eight and 36 on four, but 128 rows 95 on eight, 70 on four and 58 on two
  int ranks = 1;
  while (ranks < samp::kMaxCluster && ranks * 2048 < a.vocab) ranks *= 2;
  const int words = (a.vocab * kSize + 15) / 16 + 1;
  const int bytes = static_cast<int>((sizeof(samp::Shared) + 15) / 16 * 16) + (words + ranks - 1) / ranks * 16;
  static unsigned long long devices = 0;
  auto kern = sample_kernel<TYPE>;
  const cudaError_t e = allow_shared(kern, 227 * 1024, devices);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ranks);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows * ranks));
  cfg.blockDim = dim3(samp::kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, a, ranks);
}
}  // namespace

cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.dtype) {
    case CQ_DT_BF16: return run_sample<CQ_DT_BF16>(a, st);
    case CQ_DT_F16: return run_sample<CQ_DT_F16>(a, st);
    default: return run_sample<CQ_DT_F32>(a, st);
  }
}

}  // namespace cq
