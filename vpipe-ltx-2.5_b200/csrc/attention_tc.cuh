// attention_tc.cuh -- the arithmetic that the tcgen05 attention kernels share:
// exponentials, three-input maxima, packed f32 pairs and bf16 packing.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>

namespace ltx {

__device__ __forceinline__ float fast_exp2(float x)
{
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// max(a, b, c) in one instruction (sm_100 three-input max).
__device__ __forceinline__ float max3f(float a, float b, float c)
{
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Packed f32 pairs (sm_100 f32x2): d = a * b + c and d = a + b, lane-wise.
__device__ __forceinline__ unsigned long long ffma2(unsigned long long a, unsigned long long b,
                                                    unsigned long long c)
{
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

__device__ __forceinline__ unsigned long long fadd2(unsigned long long a, unsigned long long b)
{
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ unsigned long long pair2(uint32_t lo, uint32_t hi)
{
  return ((unsigned long long)hi << 32) | lo;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The 64 exponentials of one half row: p = 2^(s c - m), packed to bf16 pairs
// (low half = even column) and summed in two f32x2 chains.
__device__ __forceinline__ void fa3_exp(const uint32_t (&a)[32], const uint32_t (&b)[32],
                                        unsigned long long c2, unsigned long long nm2,
                                        uint32_t (&pk)[32], unsigned long long& sa,
                                        unsigned long long& sb)
{
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const unsigned long long xa = ffma2(pair2(a[2 * e], a[2 * e + 1]), c2, nm2);
    const unsigned long long xb = ffma2(pair2(b[2 * e], b[2 * e + 1]), c2, nm2);
    const float p0 = fast_exp2(__uint_as_float((uint32_t)xa));
    const float p1 = fast_exp2(__uint_as_float((uint32_t)(xa >> 32)));
    const float p2 = fast_exp2(__uint_as_float((uint32_t)xb));
    const float p3 = fast_exp2(__uint_as_float((uint32_t)(xb >> 32)));
    sa = fadd2(sa, pair2(__float_as_uint(p0), __float_as_uint(p1)));
    sb = fadd2(sb, pair2(__float_as_uint(p2), __float_as_uint(p3)));
    pk[e] = pack_bf16(p0, p1);
    pk[16 + e] = pack_bf16(p2, p3);
  }
}

}  // namespace ltx
