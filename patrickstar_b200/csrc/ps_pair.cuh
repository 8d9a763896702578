// Two 32-bit operations in one instruction (sm_100a).
#ifndef PS_B200_PAIR_CUH
#define PS_B200_PAIR_CUH

#include <cuda_runtime.h>

#include <cstdint>

struct Pair {
    uint64_t v;
    __device__ __forceinline__ Pair() {}
    __device__ __forceinline__ Pair(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
    __device__ __forceinline__ float2 get() const
    {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c)
{
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b)
{
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b)
{
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}

#endif
