// Device-side pieces shared by the operators on caller-owned device tensors:
// elements of the three types as floats, and pairs of floats.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace leo_operator {

__device__ __forceinline__ float load(const float* p) { return *p; }
__device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }

// Two floats as the packed instructions take them.
using Pair32 = unsigned long long;
__device__ __forceinline__ Pair32 pair_of(float x, float y) {
    Pair32 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 parts(Pair32 p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ Pair32 fma2(Pair32 a, Pair32 b, Pair32 c) {
    Pair32 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Pair32 mul2(Pair32 a, Pair32 b) {
    Pair32 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair32 add2(Pair32 a, Pair32 b) {
    Pair32 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Two neighbours of a row as they lie in memory, from and to words of 32 bits.
template <typename T> struct PairOf;
template <> struct PairOf<float> {
    static __device__ __forceinline__ Pair32 unpack(const uint32_t* r) {
        return pair_of(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    static __device__ __forceinline__ void pack(Pair32 v, uint32_t* r) {
        const float2 f = parts(v);
        r[0] = __float_as_uint(f.x), r[1] = __float_as_uint(f.y);
    }
};
template <> struct PairOf<__nv_bfloat16> {
    static __device__ __forceinline__ Pair32 unpack(const uint32_t* r) {
        return pair_of(__uint_as_float(r[0] << 16), __uint_as_float(r[0] & 0xffff0000u));
    }
    static __device__ __forceinline__ void pack(Pair32 v, uint32_t* r) {
        const float2 f = parts(v);
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
        r[0] = *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <> struct PairOf<__half> {
    static __device__ __forceinline__ Pair32 unpack(const uint32_t* r) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(r));
        return pair_of(f.x, f.y);
    }
    static __device__ __forceinline__ void pack(Pair32 v, uint32_t* r) {
        const float2 f = parts(v);
        const __half2 h = __floats2half2_rn(f.x, f.y);
        r[0] = *reinterpret_cast<const uint32_t*>(&h);
    }
};

}  // namespace leo_operator
