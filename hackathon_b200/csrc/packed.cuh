// Two float32 values in one instruction (f32x2), each half rounded as the scalar
// instruction rounds it, and the hardware's exponential and reciprocal.
#pragma once
#include "common.cuh"

namespace b2e {

struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2(uint32_t a, uint32_t b) { return f2(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ void split(F2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(F2 a) {
  float x, y;
  split(a, x, y);
  return pack_bf16(x, y);
}
__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// z / (1 + exp(-z)) of two values. The hardware's exponential and reciprocal are
// within a few 2^-22; the library's take some forty instructions a value, which
// would bound the kernels that use it ahead of their memory.
__device__ __forceinline__ F2 silu2(F2 z) {
  float a, b;
  split(mul2(z, f2(-1.4426950408889634f, -1.4426950408889634f)), a, b);
  split(add2(f2(ex2(a), ex2(b)), f2(1.f, 1.f)), a, b);
  return mul2(z, f2(rcp(a), rcp(b)));
}

}  // namespace b2e
