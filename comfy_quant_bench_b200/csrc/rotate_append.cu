// New queries, keys and values of a decoder's tokens: rotary positions, with an RMS norm of each head before them if asked
// for; queries go to an output, keys and values straight into their rows' pages.
//
//   pairs (a, b) = (x[i], x[i + R/2]) or (x[2i], x[2i + 1]) of a head's first R columns:
//   a' = a cos - b sin, b' = a sin + b cos, angles of the token's position; columns from R on stay.
//
// One rounding, at the end.  A thread holds eight columns of a head; in the first layout the partner's eight come by
// shuffles, from the lane R/16 away.  A block takes one token: its table entries are looked up once.  Bound by reading
// and writing each head once.
#include "decode_common.cuh"

namespace cq {

namespace rota {
constexpr int kSite = 104;                     // device status: a position beyond the table of angles
constexpr int kThreads = 256;
}  // namespace rota

template <bool F16>
__device__ __forceinline__ void widen_eight(const uint4& v, float (&f)[8]) {
  const uint32_t* w = &v.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 g = widen16<F16>(w[j]);
    f[2 * j] = g.x;
    f[2 * j + 1] = g.y;
  }
}

template <bool F16, bool FP8>
__global__ void __launch_bounds__(1024) rotate_append_kernel(const RotateArgs a) {
  grid_dep_launch();
  const int64_t t = blockIdx.x;
  const int lanes = 1 << a.lane_bits, eights = a.D >> 3, half = a.R >> 4;
  const int lane = threadIdx.x & (lanes - 1);           // eight columns of a head: 8 lane ..
  const int heads = a.Hq + 2 * a.Hkv, step = blockDim.x >> a.lane_bits;
  grid_dep_wait();
  const int pos = a.positions[t], row = a.rows[t];
  const bool far = pos >= a.rope_rows;
  int page = -1;
  if (row >= 0 && row < a.table_rows && pos >= 0 && !far && pos / a.page_size < a.table_width)
    page = a.table[row * a.table_stride + pos / a.page_size];
  const bool placed = page >= 0 && page < a.num_pages;
  const int64_t base = placed ? page * a.page_stride + (pos % a.page_size) * a.tok_stride : 0;
  if (far && threadIdx.x == 0) record_status(CQ_ERR_SHAPE, rota::kSite);

  const bool turns = lane < 2 * half;
  const int turn = a.interleaved ? 4 * lane : 8 * (lane < half ? lane : lane - half);   // first pair of this thread
  const int pairs = a.interleaved ? 4 : 8;
  float cs[8], sn[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) cs[j] = 1.0f, sn[j] = 0.0f;
  if (turns) {
    const float2* angle = reinterpret_cast<const float2*>(a.rope) + static_cast<int64_t>(min(max(pos, 0), a.rope_rows - 1)) * (a.R / 2) + turn;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      if (j < pairs) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(angle + j));
        cs[j] = f.x, sn[j] = f.y, cs[j + 1] = f.z, sn[j + 1] = f.w;
      }
    }
    if (far) {
#pragma unroll
      for (int j = 0; j < 8; ++j) cs[j] = sn[j] = __int_as_float(0x7fc00000);
    }
  }
  // the loop is the same for every lane of a warp: shuffles meet
  for (int h0 = 0; h0 < heads; h0 += step) {
    const int head = h0 + (threadIdx.x >> a.lane_bits);
    const bool live = head < heads && lane < eights;
    const int kind = head < a.Hq ? 0 : head < a.Hq + a.Hkv ? 1 : 2;      // query, key, value
    const int h = kind == 0 ? head : kind == 1 ? head - a.Hq : head - a.Hq - a.Hkv;
    const uint16_t* src = static_cast<const uint16_t*>(kind == 0 ? a.q : kind == 1 ? a.k_new : a.v_new) +
                          t * (kind == 0 ? a.q_st : kind == 1 ? a.k_st : a.v_st) + h * (kind == 0 ? a.q_sh : kind == 1 ? a.k_sh : a.v_sh);
    const uint4 raw = live ? *reinterpret_cast<const uint4*>(src + 8 * lane) : make_uint4(0, 0, 0, 0);
    float x[8];
    widen_eight<F16>(raw, x);
    float inv = 1.0f;
    const void* weight = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    if (a.q_norm != nullptr || a.k_norm != nullptr) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
      for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (weight != nullptr) {
        inv = rsqrtf(sum / static_cast<float>(a.D) + a.eps);
        float w[8];
        widen_eight<F16>(live ? __ldg(static_cast<const uint4*>(weight) + lane) : make_uint4(0, 0, 0, 0), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = x[j] * inv * w[j];
      }
    }
    if (a.interleaved) {
      if (kind < 2 && turns) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = x[2 * j], q = x[2 * j + 1];
          x[2 * j] = p * cs[j] - q * sn[j];
          x[2 * j + 1] = p * sn[j] + q * cs[j];
        }
      }
    } else {
      const int partner = lane < half ? lane + half : lane < 2 * half ? lane - half : lane;
      const float sign = lane < half ? -1.0f : 1.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = __shfl_sync(0xffffffffu, x[j], partner, lanes);
        if (kind < 2 && turns) x[j] = x[j] * cs[j] + sign * y * sn[j];
      }
    }
    if (!live) continue;
    uint4 out;
    uint32_t* o = &out.x;
    if (kind == 2) {
      out = raw;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = narrow16<F16>(x[2 * j], x[2 * j + 1]);
      if (kind == 0) {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.q_out) + (t * a.Hq + h) * a.D + 8 * lane) = out;
        continue;
      }
      if (a.k_out != nullptr)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.k_out) + (t * a.Hkv + h) * a.D + 8 * lane) = out;
    }
    if (!placed) continue;
    const int64_t at = base + h * a.head_stride + 8 * lane;
    void* cache = kind == 1 ? a.k : a.v;
    if constexpr (!FP8) {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(cache) + at) = out;
    } else {
      const float* scales = kind == 1 ? a.k_scale : a.v_scale;
      const float scale = scales != nullptr ? scales[h] : 1.0f;
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        c[j] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[2 * j], scale), __fdiv_rn(x[2 * j + 1], scale)), __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<uint2*>(static_cast<__nv_fp8_storage_t*>(cache) + at) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
    }
  }
}

cudaError_t launch_rotate_append(const RotateArgs& args, cudaStream_t st) {
  if (args.T == 0) return cudaSuccess;
  RotateArgs a = args;
  a.lane_bits = 1;
  while (8 << a.lane_bits < a.D) ++a.lane_bits;
  const int items = ((a.Hq + 2 * a.Hkv) << a.lane_bits) + 31 & ~31;
  // few tokens: all heads of a token at once
  const int most = a.T <= 2 * 148 ? 1024 : rota::kThreads, threads = items < most ? items : most;
  const dim3 grid(static_cast<unsigned>(a.T));
  const bool fp8 = a.cache_dtype == CQ_DT_FP8_E4M3;
  if (a.dtype == CQ_DT_F16)
    return fp8 ? launch_early(rotate_append_kernel<true, true>, grid, threads, 0, st, a) : launch_early(rotate_append_kernel<true, false>, grid, threads, 0, st, a);
  return fp8 ? launch_early(rotate_append_kernel<false, true>, grid, threads, 0, st, a) : launch_early(rotate_append_kernel<false, false>, grid, threads, 0, st, a);
}

}  // namespace cq
