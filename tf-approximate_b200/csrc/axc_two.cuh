// fp32 arithmetic on two values at a time.
#pragma once
#include <cuda_runtime.h>

namespace axc {

// Two fp32 values that one instruction computes with
struct Two {
    unsigned long long v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
    __device__ __forceinline__ float2 both() const
    {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
};
__device__ __forceinline__ Two fma2(Two a, Two b, Two c)
{
    Two d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
__device__ __forceinline__ Two add2(Two a, Two b)
{
    Two d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b)
{
    Two d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}

}  // namespace axc
