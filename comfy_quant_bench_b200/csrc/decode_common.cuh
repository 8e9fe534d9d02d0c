// Helpers of the decode-side kernels: asynchronous 16-byte copies, matrix loads and mma.sync tiles.
#pragma once
#include "kernels.cuh"

namespace cq {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  // src-size 0: nothing is read and 16 zero bytes are written
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Asynchronous copies, by one warp, of `count` 16-bit values to shared memory: the aligned 32-bit words that hold them,
// so that any 2-byte aligned source will do.  Value i lands at 16-bit place (source's odd half) + i; the word past the
// last value is not read.
__device__ __forceinline__ int half_shift(const unsigned short* src) {
  return static_cast<int>(reinterpret_cast<uintptr_t>(src) >> 1 & 1);
}
__device__ __forceinline__ void cp_async_halves(uint32_t dst, const unsigned short* src, int count, int lane) {
  const int shift = half_shift(src);
  for (int w = lane; 2 * w < count + shift; w += 32) {
    const int bytes = min(4, 2 * (count + shift - 2 * w));
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * w), "l"(src - shift + 2 * w), "r"(bytes)
                 : "memory");
  }
}

// Lets a kernel use `bytes` of dynamic shared memory, once per device (`devices`: a static of the caller's, one bit each;
// two threads that both set the attribute do no harm).
template <typename Kernel>
inline cudaError_t allow_shared(Kernel kernel, int bytes, unsigned long long& devices) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (devices >> dev & 1))) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) devices |= 1ull << dev;
  return e;
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

// (v & mask) | bits in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(v), "r"(mask), "r"(bits));
  return d;
}
// The eight 4-bit codes of a word as 16-bit floats; pair j holds nibbles j and j + 4.  The published way to widen integer
// codes: masked into the mantissa of a power of two, whose value is then taken off.  Logic operations run at half the
// rate of the floating-point pipe, so f16 takes five of them and four additions or fused multiply-adds:
//   f16:  q - 8, exact, from 1024 + q (the code in mantissa bits 0..3) and 1024 + 16 q (bits 4..7)
//   bf16: 16 + q, exact, the code in mantissa bits 3..6 of 2^4; its seven bits have no room for the other form
template <bool F16>
__device__ __forceinline__ void widen8(uint32_t w, uint32_t (&pairs)[4]) {
  if constexpr (F16) {
    const uint32_t h = w >> 8;
    const uint32_t even = 0xE408E408u, sixteenth = 0x2C002C00u, odd = 0xD480D480u;   // -1032, 1/16, -72
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const uint32_t v = j == 0 ? w : h;
      const uint32_t lo = and_or(v, 0x000F000Fu, 0x64006400u), hi = and_or(v, 0x00F000F0u, 0x64006400u);
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(pairs[j]) : "r"(lo), "r"(even));
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(pairs[j + 1]) : "r"(hi), "r"(sixteenth), "r"(odd));
    }
  } else {
    pairs[0] = and_or(w * 8u, 0x00780078u, 0x41804180u);
    pairs[1] = and_or(w >> 1, 0x00780078u, 0x41804180u);
    pairs[2] = and_or(w >> 5, 0x00780078u, 0x41804180u);
    pairs[3] = and_or(w >> 9, 0x00780078u, 0x41804180u);
  }
}
// what a widened weight has over q - 8: the zero's term makes up for it
template <bool F16>
__device__ __forceinline__ float widen_offset() { return F16 ? 0.0f : 24.0f; }

}  // namespace cq
