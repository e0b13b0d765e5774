// Two fp32 operations of one instruction, each rounded as usual.
#pragma once
#include <cuda_runtime.h>

namespace alpha {

__device__ __forceinline__ unsigned long long both(float2 a) { unsigned long long r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y)); return r; }
__device__ __forceinline__ float2 both(unsigned long long a) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a)); return r; }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { unsigned long long r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b))); return both(r); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { unsigned long long r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b))); return both(r); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { unsigned long long r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(both(a)), "l"(both(b)), "l"(both(c))); return both(r); }
__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }
__device__ __forceinline__ float2 twice(float a) { return make_float2(a, a); }

}  // namespace alpha
