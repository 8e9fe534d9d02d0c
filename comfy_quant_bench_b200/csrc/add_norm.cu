// Root-mean-square norm with the residual's addition, and an output in 8 bits with scales.
//
//   h = x + r, rounded to the 16-bit type (the residual stream, written back);  y = h w / sqrt(mean(h^2) + eps)
//
// and y rounded once to the type, or in 8 bits: with p = h w and P the largest |p| of the row (or of a group of 32, 64 or
// 128 columns), code = round(top p / P), scale = P / (top sqrt(mean(h^2) + eps)), top = 127 (int8) or 448 (e4m3).  The
// root cancels in the code, and p is exact in fp32 (16-bit factors), so a code is a function of exact values: the nearest
// one of the exact quotient.
//
// Bound by reading x, r and writing h, y once: a row stays in registers between its sums and its outputs.  One reduction
// serves both the sum of squares and the maximum.
//
// Measured on a B200 (device time): 16384 rows of 4096, bf16 in and out: 82 us, 6.6 TB/s, HBM's rate; 100000 rows of 512 to
// e4m3: 56 us, 6.4 TB/s; 8192 rows of 8192 to e4m3 in groups of 128: 85 us, 5.5 TB/s, and to int8: 107 us, 4.4 TB/s, bound by
// the conversions (an SM's integer and conversion pipes); one row of 4096: 2.3 us, launch and latency.
#include "decode_common.cuh"

namespace cq {

// int8 codes of p against the largest P: `by` is 127 / P, or 0 where P is 0.
struct Coder {
  float most, by;
  bool tiny;                                   // 127 / P would overflow: the quotient first
};
__device__ __forceinline__ Coder coder(float most) {
  Coder c{most, 0.0f, most < 1e-30f};
  if (most > 0.0f) c.by = c.tiny ? 127.0f : __fdiv_rn(127.0f, most);
  return c;
}
// the nearest code in 64 bits: rare, and out of the way of the others
__device__ __noinline__ int int8_code_exactly(float p, float most) {
  return static_cast<int>(rint(static_cast<double>(p) * 127.0 / static_cast<double>(most)));
}
__device__ __forceinline__ uint32_t int8_code(float p, const Coder& c) {
  const float t = c.tiny ? (c.most > 0.0f ? __fdiv_rn(p, c.most) * c.by : 0.0f) : p * c.by, k = rintf(t);
  int code = static_cast<int>(k);
  // t is off by 2^-23 of itself, 1.52e-5 at most: only that near to a border can the nearest code be another one
  if (fabsf(t - k) > 0.5f - 1.6e-5f) code = int8_code_exactly(p, c.most);
  return static_cast<uint32_t>(code) & 0xffu;
}

// e4m3 codes of the quotients 448 p / P.  A border b between two codes has five bits, so 448 p - b P is 0 or, where p has bf16
// factors, 2^-21 of either at least: 448 p is exact then, and a step of Newton's method, t + (448 p - t P) / P, rounds the
// quotient to fp32 but for 2^-45 of itself, to the quotient's side of b or to b with it.  f16 factors have more digits: t is off
// by 2^-23, and near a border the sign of 448 p - b P, exact in two parts, decides.  (Bits that tell where a border is
// near, for bf16 too: 101 us in the first 8-bit case above, since many quotients of 8-bit numbers lie on one.)
struct Quotients {
  float wide, most, inv;                       // 448 and P, times a power of 2 that keeps the products in range, and 1 / P
};
template <bool F16>
__device__ __forceinline__ Quotients quotients(float most) {
  const float scale = F16 ? 1.0f : most > 1e30f ? 0x1p-40f : most < 1e-20f ? 0x1p60f : 1.0f;
  const bool some = most > 0.0f && most < INFINITY;                    // else every finite p has code 0
  return {448.0f * scale, some ? most * scale : 0.0f, some ? __frcp_rn(most * scale) : 0.0f};
}
__device__ __forceinline__ uint32_t e4m3_pair(float2 t) { return __nv_cvt_float2_to_fp8x2(t, __NV_SATFINITE, __NV_E4M3); }
// four bits are kept from 2^-6 on, and a border has 1000... behind them: the bits that follow are moved to the top, and those of
// a value that may lie on the other side of a border are at most kNear
constexpr uint32_t kNear = 6u << 12;
__device__ __forceinline__ uint32_t from_border(float t) { return (__float_as_uint(t) << 12) + (3u << 12) - (0x80000u << 12); }
// t on its quotient's side of the border between two codes, or on it.  Below 2^-6 a code is a multiple of 2^-9, as from there
// to 2^-5: the bits are those of t moved up (short of 2^-6, so that the sum does not round to 2^-5)
__device__ __forceinline__ float settled(float t, float p, float most) {
  const float up = fabsf(t) < 0x1.fffffp-7f ? 0x1p-6f : 0.0f;
  const float border = __uint_as_float((__float_as_uint(fabsf(t) + up) & 0xfff00000u) | 0x80000u) - up;
  const float size = fabsf(p), wide = 448.0f * size, d = fmaf(-border, most, wide) + fmaf(448.0f, size, -wide);
  return copysignf(d == 0.0f ? border : fmaf(border, copysignf(0x1p-20f, d), border), p);
}
// N = 2 or 8 values; two codes to a uint32
template <bool F16, int N>
__device__ __forceinline__ void e4m3_codes(const float (&p)[N], const Quotients& c, uint32_t (&code)[N / 2]) {
  const float2 none = make_float2(0.0f, 0.0f), inv = make_float2(c.inv, c.inv);
  float2 t[N / 2];
  uint32_t from = 0xffffffffu;
  float least = 1.0f;
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    const float2 wide = fma2(make_float2(p[2 * j], p[2 * j + 1]), make_float2(c.wide, c.wide), none);
    t[j] = fma2(wide, inv, none);
    if constexpr (F16) {
      from = min(from, min(from_border(t[j].x), from_border(t[j].y)));
      least = fminf(least, fminf(fabsf(t[j].x), fabsf(t[j].y)));
    } else {
      t[j] = fma2(fma2(t[j], make_float2(-c.most, -c.most), wide), inv, t[j]);
    }
  }
  if (F16 && (from <= kNear || least < 0x1p-6f) && c.most > 0.0f) {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) t[j] = make_float2(settled(t[j].x, p[2 * j], c.most), settled(t[j].y, p[2 * j + 1], c.most));
  }
#pragma unroll
  for (int j = 0; j < N / 2; ++j) code[j] = e4m3_pair(t[j]);
}

// the larger one, or NaN where either is
__device__ __forceinline__ float larger(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
// The sum and the maximum over a row's threads: a warp, or a block of whole warps.
template <bool WARP>
__device__ __forceinline__ void row_reduce(float& sum, float& most, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    most = larger(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) {
      red[warp] = sum;
      red[32 + warp] = most;
    }
    __syncthreads();
    sum = lane < warps ? red[lane] : 0.0f;
    most = lane < warps ? red[32 + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      most = larger(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
  }
}

// Widths that are a multiple of eight: a thread holds CHUNKS eights of its row, which a warp (WARP) or the block shares.
// Blocks of at most 512 threads: 8192 columns take 93 us on 512 threads with two eights each, 102 on 256 with four and 104 on
// 1024 with one (host's clock).
template <bool F16, int OUT, bool GROUPS, int CHUNKS, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : CHUNKS < 4 ? 512 : 1024) add_norm_kernel(const AddNormArgs a) {
  __shared__ float red[64];
  const int team = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = WARP ? blockIdx.x * static_cast<int64_t>(blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  grid_dep_launch();
  grid_dep_wait();
  if (WARP && row >= a.rows) return;
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + row * a.ldx;
  const uint16_t* r = static_cast<const uint16_t*>(a.residual) + row * a.ldr;
  const uint4* w = static_cast<const uint4*>(a.weight);
  const int eights = a.width >> 3;
  uint4 h[CHUNKS];
  float sum = 0.0f, most = 0.0f;
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int c = tid + i * team;
    h[i] = c < eights ? __ldcs(reinterpret_cast<const uint4*>(x + 8 * c)) : make_uint4(0, 0, 0, 0);
  }
  if (a.residual != nullptr) {
    uint4 add[CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = tid + i * team;
      add[i] = c < eights ? __ldcs(reinterpret_cast<const uint4*>(r + 8 * c)) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      uint32_t* u = &h[i].x;
      const uint32_t* v = &add[i].x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = widen16<F16>(u[j]), g = widen16<F16>(v[j]);
        u[j] = narrow16<F16>(f.x + g.x, f.y + g.y);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int c = tid + i * team;
    constexpr bool kMost = OUT != kNormSame && !GROUPS;
    const uint4 wc = kMost && c < eights ? __ldg(w + c) : make_uint4(0, 0, 0, 0);
    const uint32_t *u = &h[i].x, *v = &wc.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = widen16<F16>(u[j]), g = widen16<F16>(v[j]);
      sum = fmaf(f.x, f.x, sum);
      sum = fmaf(f.y, f.y, sum);
      if (kMost) most = larger(most, larger(fabsf(f.x * g.x), fabsf(f.y * g.y)));
    }
    if (c < eights && a.h_out != nullptr) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h_out) + row * a.ldh + 8 * c) = h[i];
  }
  row_reduce<WARP>(sum, most, red);
  const float inv = rsqrtf(sum / static_cast<float>(a.width) + a.eps);
  constexpr float kTop = OUT == kNormInt8 ? 127.0f : 448.0f;
  if (OUT != kNormSame && !GROUPS && tid == 0) a.scale[row] = most * inv / kTop;
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int c = tid + i * team;
    const uint4 wc = c < eights ? __ldg(w + c) : make_uint4(0, 0, 0, 0);
    const uint32_t *u = &h[i].x, *v = &wc.x;
    float p[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = widen16<F16>(u[j]), g = widen16<F16>(v[j]);
      p[2 * j] = f.x * g.x;
      p[2 * j + 1] = f.y * g.y;
    }
    if constexpr (OUT == kNormSame) {
      if (c >= eights) continue;
      uint4 y;
      uint32_t* o = &y.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = narrow16<F16>(p[2 * j] * inv, p[2 * j + 1] * inv);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + row * a.width + 8 * c) = y;
    } else {
      float top = most;
      if constexpr (GROUPS) {
        top = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = larger(top, fabsf(p[j]));
        for (int o = 1; o < a.group >> 3; o <<= 1) top = larger(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (c < eights && (8 * c & (a.group - 1)) == 0) a.scale[8 * c / a.group * a.rows + row] = top * inv / kTop;
      }
      if (c >= eights) continue;
      uint2 q;
      if constexpr (OUT == kNormInt8) {
        const Coder by = coder(top);
        uint32_t b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = int8_code(p[j], by);
        q.x = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
        q.y = b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24;
      } else {
        uint32_t codes[4];
        e4m3_codes<F16>(p, quotients<F16>(top), codes);
        q = make_uint2(codes[0] | codes[1] << 16, codes[2] | codes[3] << 16);
      }
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.out) + row * a.width + 8 * c) = q;
    }
  }
}

// Other widths: element by element, a row a warp or a block; a thread leaves its elements of h in shared memory meanwhile.
template <bool F16, int OUT, bool WARP>
__global__ void __launch_bounds__(256) add_norm_odd_kernel(const AddNormArgs a) {
  extern __shared__ uint16_t rows_h[];
  __shared__ float red[64];
  const int team = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = WARP ? blockIdx.x * static_cast<int64_t>(blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  uint16_t* row_h = rows_h + (WARP ? (threadIdx.x >> 5) * a.width : 0);
  grid_dep_launch();
  grid_dep_wait();
  if (WARP && row >= a.rows) return;
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + row * a.ldx;
  const uint16_t* r = static_cast<const uint16_t*>(a.residual) + row * a.ldr;
  const uint16_t* w = static_cast<const uint16_t*>(a.weight);
  float sum = 0.0f, most = 0.0f;
#pragma unroll 4
  for (int c = tid; c < a.width; c += team) {
    uint32_t h = x[c];
    if (a.residual != nullptr) h = narrow16<F16>(widen16<F16>(h).x + widen16<F16>(r[c]).x, 0.0f) & 0xffffu;
    row_h[c] = static_cast<uint16_t>(h);
    if (a.h_out != nullptr) static_cast<uint16_t*>(a.h_out)[row * a.ldh + c] = static_cast<uint16_t>(h);
    const float f = widen16<F16>(h).x;
    sum = fmaf(f, f, sum);
    most = larger(most, fabsf(f * widen16<F16>(w[c]).x));
  }
  row_reduce<WARP>(sum, most, red);
  const float inv = rsqrtf(sum / static_cast<float>(a.width) + a.eps);
  const Coder by = coder(most);
  const Quotients per = quotients<F16>(most);
  if (OUT != kNormSame && tid == 0) a.scale[row] = most * inv / (OUT == kNormInt8 ? 127.0f : 448.0f);
#pragma unroll 4
  for (int c = tid; c < a.width; c += team) {
    const float p = widen16<F16>(row_h[c]).x * widen16<F16>(w[c]).x;
    const int64_t to = row * a.width + c;
    if constexpr (OUT == kNormSame) static_cast<uint16_t*>(a.out)[to] = static_cast<uint16_t>(narrow16<F16>(p * inv, 0.0f));
    else if constexpr (OUT == kNormInt8) static_cast<uint8_t*>(a.out)[to] = static_cast<uint8_t>(int8_code(p, by));
    else {
      const float twice[2] = {p, p};
      uint32_t code[1];
      e4m3_codes<F16>(twice, per, code);
      static_cast<uint8_t*>(a.out)[to] = static_cast<uint8_t>(code[0]);
    }
  }
}

namespace {
template <bool F16, int OUT, bool GROUPS>
cudaError_t run_add_norm(const AddNormArgs& a, cudaStream_t st) {
  const int eights = a.width / 8;
  if (eights <= 32 * 4) {
    const int warps = 8;
    const dim3 grid(static_cast<unsigned>((a.rows + warps - 1) / warps));
    if (eights <= 32) return launch_early(add_norm_kernel<F16, OUT, GROUPS, 1, true>, grid, 32 * warps, 0, st, a);
    if (eights <= 64) return launch_early(add_norm_kernel<F16, OUT, GROUPS, 2, true>, grid, 32 * warps, 0, st, a);
    return launch_early(add_norm_kernel<F16, OUT, GROUPS, 4, true>, grid, 32 * warps, 0, st, a);
  }
  const dim3 grid(static_cast<unsigned>(a.rows));
  auto threads = [&](int chunks) { return ((eights + chunks - 1) / chunks + 31) / 32 * 32; };
  if (threads(1) <= 512) return launch_early(add_norm_kernel<F16, OUT, GROUPS, 1, false>, grid, threads(1), 0, st, a);
  if (threads(2) <= 512) return launch_early(add_norm_kernel<F16, OUT, GROUPS, 2, false>, grid, threads(2), 0, st, a);
  return launch_early(add_norm_kernel<F16, OUT, GROUPS, 4, false>, grid, threads(4), 0, st, a);
}
template <bool F16>
cudaError_t pick_add_norm(const AddNormArgs& a, cudaStream_t st) {
  if (a.width % 8 != 0) {
    // a warp a row where the rows give every SM 32 short ones or more: 518289 rows of 123 take 235 us, and 763 with a block
    // each; 65536 of 999 158 and 259; but 777 of 1001 13 us, and 6.5 with a block each
    const bool warp = a.width <= 1024 && a.rows >= 32 * num_sms();
    const dim3 grid(static_cast<unsigned>(warp ? (a.rows + 7) / 8 : a.rows));
    const int bytes = 2 * a.width * (warp ? 8 : 1);
    static unsigned long long devices[6] = {};
    auto launch = [&](auto kernel, unsigned long long& d) {
      const cudaError_t e = allow_shared(kernel, 2 * kNormMaxWidth, d);
      return e != cudaSuccess ? e : launch_early(kernel, grid, 256, bytes, st, a);
    };
    switch (a.out_kind) {
      case kNormSame: return warp ? launch(add_norm_odd_kernel<F16, kNormSame, true>, devices[0]) : launch(add_norm_odd_kernel<F16, kNormSame, false>, devices[1]);
      case kNormInt8: return warp ? launch(add_norm_odd_kernel<F16, kNormInt8, true>, devices[2]) : launch(add_norm_odd_kernel<F16, kNormInt8, false>, devices[3]);
      default: return warp ? launch(add_norm_odd_kernel<F16, kNormFp8, true>, devices[4]) : launch(add_norm_odd_kernel<F16, kNormFp8, false>, devices[5]);
    }
  }
  switch (a.out_kind) {
    case kNormSame: return run_add_norm<F16, kNormSame, false>(a, st);
    case kNormInt8: return a.group ? run_add_norm<F16, kNormInt8, true>(a, st) : run_add_norm<F16, kNormInt8, false>(a, st);
    default: return a.group ? run_add_norm<F16, kNormFp8, true>(a, st) : run_add_norm<F16, kNormFp8, false>(a, st);
  }
}
}  // namespace

cudaError_t launch_add_norm(const AddNormArgs& a, cudaStream_t st) {
  if (a.rows == 0 || a.width == 0) return cudaSuccess;
  return a.dtype == CQ_DT_F16 ? pick_add_norm<true>(a, st) : pick_add_norm<false>(a, st);
}

}  // namespace cq
