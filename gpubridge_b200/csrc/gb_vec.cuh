// Vectors of eight values of the three floating types, and reductions over a block.
//
// A vector is one access: 16 bytes of bf16 / fp16, or 32 bytes of fp32 (sm_100a's 256-bit loads
// and stores; the address must be a multiple of the vector's size).  Arithmetic is in fp32;
// a store rounds once, to nearest even.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

// type codes of the entry points, those of gpubridge_b200/ops/_lib.py
enum { GB_F32 = 0, GB_BF16 = 1, GB_F16 = 2 };

__device__ __forceinline__ float gb_up(float v) { return v; }
__device__ __forceinline__ float gb_up(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float gb_up(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T gb_down(float v);
template <> __device__ __forceinline__ float gb_down<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 gb_down<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half gb_down<__half>(float v) { return __float2half_rn(v); }

// Eight values as they lie in memory; `get` converts them.
template <typename T> struct Raw8 {
    uint4 q;
    __device__ __forceinline__ void load(const T* p) { q = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float (&v)[8]) const;
};
template <> __device__ __forceinline__ void Raw8<__nv_bfloat16>::get(float (&v)[8]) const {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <> __device__ __forceinline__ void Raw8<__half>::get(float (&v)[8]) const {
    const __half2* h = reinterpret_cast<const __half2*>(&q);
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}
template <> struct Raw8<float> {
    float f[8];
    __device__ __forceinline__ void load(const float* p) {
        asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]),
                       "=f"(f[6]), "=f"(f[7]) : "l"(p) : "memory");
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = f[i];
    }
};

__device__ __forceinline__ void gb_store8(float* p, const float (&v)[8]) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
                    "f"(v[6]), "f"(v[7]) : "memory");
}
__device__ __forceinline__ void gb_store8(__nv_bfloat16* p, const float (&v)[8]) {
    uint4 q;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
    #pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = q;
}
__device__ __forceinline__ void gb_store8(__half* p, const float (&v)[8]) {
    uint4 q;
    __half2* h = reinterpret_cast<__half2*>(&q);
    #pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = q;
}

// One value of a tensor whose type is known at run time (parameters, read once a block).
__device__ __forceinline__ float gb_read(const void* p, int code, size_t i) {
    if (code == GB_F32) return static_cast<const float*>(p)[i];
    if (code == GB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void gb_write(void* p, int code, size_t i, float v) {
    if (code == GB_F32) static_cast<float*>(p)[i] = v;
    else if (code == GB_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

template <typename V>
__device__ __forceinline__ V gb_warp_sum(V v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
