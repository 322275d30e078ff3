// e4m3.cuh -- values in 8 bits with scales that are powers of two, and the wait
// of kernels that may start while the kernel before them ends.
#pragma once

#include <cstdint>

namespace ca {

// Exponents that a scale may have.
constexpr int kKv8MinExp = -64, kKv8MaxExp = 120;

// Kernels that call dependency_wait are launched so that they may start while the kernel before
// them in the stream ends (programmatic dependent launch): until
// dependency_wait returns, which is when that kernel is complete and its
// writes are visible, they touch nothing in memory but their arguments. Each
// lets its own successor come up right away in the same manner. What the
// kernel before may have written is read with plain loads: read-only ones
// (__ldg, ld.global.nc) are defined only for data that does not change from
// the start of the kernel that reads it, and that start is before the wait.
__device__ __forceinline__ void dependency_wait() {
  asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
}

// Two fp32 to two e4m3 (round to nearest even, saturating, NaN kept): lo in
// the low byte.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// The four e4m3 values of a word as f16 pairs (exact).
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

__device__ __forceinline__ float2 f16x2_to_f32(uint32_t h) {
  float2 r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(h));
  return r;
}

__device__ __forceinline__ void e4m3x4_to_f32(uint32_t w, float (&x)[4]) {
  uint32_t a, b;
  e4m3x4_to_f16(w, a, b);
  const float2 p = f16x2_to_f32(a), q = f16x2_to_f32(b);
  x[0] = p.x;
  x[1] = p.y;
  x[2] = q.x;
  x[3] = q.y;
}

// The smallest k in [lo, hi] with amax <= 448 * 2^k. 448 = 1.75 * 2^8, so
// amax = m * 2^e (1 <= m < 2) needs e - 8, or e - 7 where m > 1.75; read off
// the fp32 bits, so it is exact.
__device__ __forceinline__ int e4m3_exp(float amax, int lo, int hi) {
  if (!(amax > 0.f)) return lo;
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 127;
  const int k = e - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(k, lo), hi);
}

__device__ __forceinline__ float exp2_int(int k) {  // 2^k, -126 <= k <= 127
  return __int_as_float((k + 127) << 23);
}

}  // namespace ca
