// New queries, keys and values of a decoder's tokens: rotary positions, with an RMS norm of each head before them if asked
// for; queries go to an output, keys and values straight into their rows' pages.
//
//   pairs (a, b) = (x[i], x[i + R/2]) or (x[2i], x[2i + 1]) of a head's first R columns:
//   a' = a cos - b sin, b' = a sin + b cos, angles of the token's position; columns from R on stay.
//
// One rounding, at the end.  A thread holds two eights of a head, in the first layout those whose columns make pairs, so that
// nothing is exchanged but the norm's sums (with the partner's eight from another lane by shuffles: 106 us instead of 90 in
// the first case below, by the host's clock).  A block takes one token: its table entries are looked up once, while its
// first heads are on their way; blocks that stay for several tokens keep fewer loads in flight (139 us).
//
// Bound by reading and writing each head once.  Measured on a B200 (device time): 16001 tokens, 32 query and 8 key-value heads
// of 128, f16, half of each turned: 82 to 85 us, 4.7 TB/s; all of each, with norms, bf16: 101 us, 4.0 TB/s, and into an 8-bit cache
// 113 us, 3.3 TB/s; 64 tokens with norms into an 8-bit cache: 5.8 us, one token 3.7 us, launch and the chain of position, page and angle.
#include "decode_common.cuh"

namespace cq {

namespace rota {
constexpr int kSite = 104;                     // device status: a position beyond the table of angles
constexpr int kThreads = 256;
}  // namespace rota

template <bool F16>
__device__ __forceinline__ void widen_eight(const uint4& v, float2 (&f)[4]) {
  const uint32_t* w = &v.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = widen16<F16>(w[j]);
}
template <bool F16>
__device__ __forceinline__ uint4 narrow_eight(const float2 (&f)[4]) {
  return make_uint4(narrow16<F16>(f[0].x, f[0].y), narrow16<F16>(f[1].x, f[1].y), narrow16<F16>(f[2].x, f[2].y),
                    narrow16<F16>(f[3].x, f[3].y));
}
__device__ __forceinline__ uint2 e4m3_eight(const float2 (&f)[4], float scale) {
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    c[j] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f[j].x, scale), __fdiv_rn(f[j].y, scale)), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}

// AHEAD: heads of a thread that are loaded together
template <bool F16, bool FP8, bool NORM, int AHEAD>
__global__ void __launch_bounds__(AHEAD == 1 ? 1024 : rota::kThreads) rotate_append_kernel(const RotateArgs a) {
  grid_dep_launch();
  const int64_t t = blockIdx.x;
  const int lanes = 1 << a.lane_bits, half = a.R >> 4;  // threads of a head; its units of pairs
  const int unit = threadIdx.x & (lanes - 1), first = threadIdx.x >> a.lane_bits;
  const int heads = a.Hq + 2 * a.Hkv, step = blockDim.x >> a.lane_bits;
  // columns of this thread's two eights; the second may not be there
  const bool pairs = unit < half, spread = pairs && !a.interleaved;
  const int c0 = spread ? 8 * unit : 16 * unit, c1 = spread ? c0 + 8 * half : c0 + 8;
  const bool one = c0 < a.D, two = c1 < a.D;
  grid_dep_wait();
  const int pos = a.positions[t], row = a.rows[t];
  const uint16_t* q_at = static_cast<const uint16_t*>(a.q) + t * a.q_st;
  const uint16_t* k_at = static_cast<const uint16_t*>(a.k_new) + t * a.k_st;
  const uint16_t* v_at = static_cast<const uint16_t*>(a.v_new) + t * a.v_st;
  uint4 raw[AHEAD][2];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int head = h0 + i * step + first;
      const uint16_t* src = head < a.Hq ? q_at + head * a.q_sh
                            : head < a.Hq + a.Hkv ? k_at + (head - a.Hq) * a.k_sh : v_at + (head - a.Hq - a.Hkv) * a.v_sh;
      raw[i][0] = head < heads && one ? __ldcs(reinterpret_cast<const uint4*>(src + c0)) : make_uint4(0, 0, 0, 0);
      raw[i][1] = head < heads && two ? __ldcs(reinterpret_cast<const uint4*>(src + c1)) : make_uint4(0, 0, 0, 0);
    }
  };
  fetch(0);
  const bool far = pos >= a.rope_rows;
  int page = -1;
  if (row >= 0 && row < a.table_rows && pos >= 0 && !far && pos / a.page_size < a.table_width)
    page = a.table[row * a.table_stride + pos / a.page_size];
  if (far && threadIdx.x == 0) record_status(CQ_ERR_SHAPE, rota::kSite);

  float2 cs[4], sn[4];                                  // of the thread's eight pairs
  if (pairs) {
    const float4* angle = reinterpret_cast<const float4*>(a.rope) + (static_cast<int64_t>(min(max(pos, 0), a.rope_rows - 1)) * (a.R / 2) + 8 * unit) / 2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 f = __ldg(angle + j);
      cs[j] = make_float2(f.x, f.z);
      sn[j] = make_float2(f.y, f.w);
    }
    if (far) {
#pragma unroll
      for (int j = 0; j < 4; ++j) cs[j] = sn[j] = make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
    }
  }
  const bool placed = page >= 0 && page < a.num_pages;
  const int64_t base = placed ? page * a.page_stride + (pos % a.page_size) * a.tok_stride : 0;
  uint16_t* q_to = static_cast<uint16_t*>(a.q_out) + t * a.Hq * a.D;
  // the loops are the same for every lane of a warp: shuffles meet
  for (int h0 = 0; h0 < heads; h0 += AHEAD * step) {
    if (h0 > 0) fetch(h0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (h0 + i * step >= heads) break;
      const int head = h0 + i * step + first;
      const bool key = head >= a.Hq, value = head >= a.Hq + a.Hkv;
      float2 x[4], y[4];
      widen_eight<F16>(raw[i][0], x);
      widen_eight<F16>(raw[i][1], y);
      if constexpr (NORM) {
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum = fma2(y[j], y[j], fma2(x[j], x[j], sum));
        float all = sum.x + sum.y;
        for (int o = lanes >> 1; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        const uint16_t* weight = static_cast<const uint16_t*>(value ? nullptr : key ? a.k_norm : a.q_norm);
        if (weight != nullptr) {
          const float inv = rsqrtf(all / static_cast<float>(a.D) + a.eps);
          float2 w[4];
          widen_eight<F16>(one ? __ldg(reinterpret_cast<const uint4*>(weight + c0)) : make_uint4(0, 0, 0, 0), w);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = make_float2(x[j].x * inv * w[j].x, x[j].y * inv * w[j].y);
          widen_eight<F16>(two ? __ldg(reinterpret_cast<const uint4*>(weight + c1)) : make_uint4(0, 0, 0, 0), w);
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = make_float2(y[j].x * inv * w[j].x, y[j].y * inv * w[j].y);
        }
      }
      if (pairs && !value) {
        const float2 none = make_float2(0.0f, 0.0f), minus = make_float2(-1.0f, -1.0f);
        if (spread) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 p = x[j], q = y[j];
            x[j] = fma2(p, cs[j], fma2(fma2(q, sn[j], none), minus, none));
            y[j] = fma2(q, cs[j], fma2(p, sn[j], none));
          }
        } else {                                          // pairs side by side: pair 2j in x[..] of the first eight, and so on
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float2& z = j < 2 ? x[2 * j] : y[2 * j - 4];
            float2& u = j < 2 ? x[2 * j + 1] : y[2 * j - 3];
            z = make_float2(z.x * cs[j].x - z.y * sn[j].x, z.x * sn[j].x + z.y * cs[j].x);
            u = make_float2(u.x * cs[j].y - u.y * sn[j].y, u.x * sn[j].y + u.y * cs[j].y);
          }
        }
      }
      if (head >= heads || !one) continue;
      if (!value) {
        const uint4 out0 = narrow_eight<F16>(x), out1 = narrow_eight<F16>(y);
        if (!key) {
          uint16_t* to = q_to + head * a.D;
          *reinterpret_cast<uint4*>(to + c0) = out0;
          if (two) *reinterpret_cast<uint4*>(to + c1) = out1;
          continue;
        }
        raw[i][0] = out0;
        raw[i][1] = out1;
        if (a.k_out != nullptr) {
          uint16_t* to = static_cast<uint16_t*>(a.k_out) + (t * a.Hkv + head - a.Hq) * a.D;
          *reinterpret_cast<uint4*>(to + c0) = out0;
          if (two) *reinterpret_cast<uint4*>(to + c1) = out1;
        }
      }
      if (!placed) continue;
      const int h = value ? head - a.Hq - a.Hkv : head - a.Hq;
      const int64_t at = base + h * a.head_stride;
      if constexpr (!FP8) {
        uint16_t* to = static_cast<uint16_t*>(value ? a.v : a.k) + at;
        *reinterpret_cast<uint4*>(to + c0) = raw[i][0];
        if (two) *reinterpret_cast<uint4*>(to + c1) = raw[i][1];
      } else {
        const float* scales = value ? a.v_scale : a.k_scale;
        const float scale = scales != nullptr ? scales[h] : 1.0f;
        uint8_t* to = static_cast<uint8_t*>(value ? a.v : a.k) + at;
        *reinterpret_cast<uint2*>(to + c0) = e4m3_eight(x, scale);
        if (two) *reinterpret_cast<uint2*>(to + c1) = e4m3_eight(y, scale);
      }
    }
  }
}

namespace {
template <bool F16, bool FP8, bool NORM>
cudaError_t run_rotate(const RotateArgs& a, int items, cudaStream_t st) {
  // two tokens an SM or fewer: all heads of a token at once; more: two heads a thread on their way together
  if (a.T <= 2 * num_sms()) return launch_early(rotate_append_kernel<F16, FP8, NORM, 1>, dim3(a.T), items < 1024 ? items : 1024, 0, st, a);
  const int threads = (items + 1) / 2 + 31 & ~31;
  return launch_early(rotate_append_kernel<F16, FP8, NORM, 2>, dim3(a.T), threads < rota::kThreads ? threads : rota::kThreads, 0, st, a);
}
template <bool F16, bool FP8>
cudaError_t pick_rotate(const RotateArgs& a, int items, cudaStream_t st) {
  return a.q_norm != nullptr || a.k_norm != nullptr ? run_rotate<F16, FP8, true>(a, items, st) : run_rotate<F16, FP8, false>(a, items, st);
}
}  // namespace

cudaError_t launch_rotate_append(const RotateArgs& args, cudaStream_t st) {
  if (args.T == 0) return cudaSuccess;
  RotateArgs a = args;
  a.lane_bits = 0;
  while (16 << a.lane_bits < a.D) ++a.lane_bits;
  const int items = ((a.Hq + 2 * a.Hkv) << a.lane_bits) + 31 & ~31;
  const bool fp8 = a.cache_dtype == CQ_DT_FP8_E4M3;
  if (a.dtype == CQ_DT_F16) return fp8 ? pick_rotate<true, true>(a, items, st) : pick_rotate<true, false>(a, items, st);
  return fp8 ? pick_rotate<false, true>(a, items, st) : pick_rotate<false, false>(a, items, st);
}

}  // namespace cq
