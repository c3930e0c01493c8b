// 16-byte vectors and single elements of the floating types as fp32 values and back.  Narrowing rounds once, to nearest
// even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32); denormals are kept.
#pragma once

#include "reduce_kernels.hpp"

namespace mi {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct F32Vec {
    typedef uint32_t elem_t;
    static constexpr int VEC = 4;
    static __device__ __forceinline__ float widen1(elem_t x) { return as_f32(x); }
    static __device__ __forceinline__ elem_t narrow1(float x) { return as_u32(x); }
    static __device__ __forceinline__ void widen(u32x4 x, float* f) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = as_f32(x[i]);
    }
    static __device__ __forceinline__ u32x4 narrow(const float* f) {
        return u32x4{ as_u32(f[0]), as_u32(f[1]), as_u32(f[2]), as_u32(f[3]) };
    }
    static __device__ __forceinline__ void widen_half(u32x2, float*) {}         // four elements are a whole vector
    static __device__ __forceinline__ u32x2 narrow_half(const float*) { return u32x2{ 0, 0 }; }
};

struct Bf16Vec {
    typedef uint16_t elem_t;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float widen1(elem_t x) { return as_f32((uint32_t)x << 16); }
    static __device__ __forceinline__ elem_t narrow1(float x) { return __builtin_bit_cast(elem_t, (__bf16)x); }
    static __device__ __forceinline__ void widen(u32x4 x, float* f) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = as_f32(x[i] << 16);
            f[2 * i + 1] = as_f32(x[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void widen_half(u32x2 x, float* f) {      // four elements
#pragma unroll
        for (int i = 0; i < 2; i++) {
            f[2 * i] = as_f32(x[i] << 16);
            f[2 * i + 1] = as_f32(x[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x2 narrow_half(const float* f) {
        const f32x2 a = { f[0], f[1] }, b = { f[2], f[3] };
        return u32x2{ __builtin_bit_cast(uint32_t, __builtin_convertvector(a, bf16x2)),
                      __builtin_bit_cast(uint32_t, __builtin_convertvector(b, bf16x2)) };
    }
    static __device__ __forceinline__ u32x4 narrow(const float* f) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f32x2 p = { f[2 * i], f[2 * i + 1] };
            r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
        }
        return r;
    }
};

struct Fp16Vec {
    typedef uint16_t elem_t;
    static constexpr int VEC = 8;
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float widen1(elem_t x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ __forceinline__ elem_t narrow1(float x) { return __builtin_bit_cast(elem_t, (_Float16)x); }
    static __device__ __forceinline__ void widen(u32x4 x, float* f) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t d = x[i];        // a copy: __builtin_bit_cast of a vector's element reads element 0
            const half2 h = __builtin_bit_cast(half2, d);
            f[2 * i] = (float)h[0];
            f[2 * i + 1] = (float)h[1];
        }
    }
    static __device__ __forceinline__ void widen_half(u32x2 x, float* f) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t d = x[i];
            const half2 h = __builtin_bit_cast(half2, d);
            f[2 * i] = (float)h[0];
            f[2 * i + 1] = (float)h[1];
        }
    }
    static __device__ __forceinline__ u32x2 narrow_half(const float* f) {
        const half2 a = { (_Float16)f[0], (_Float16)f[1] }, b = { (_Float16)f[2], (_Float16)f[3] };
        return u32x2{ __builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b) };
    }
    static __device__ __forceinline__ u32x4 narrow(const float* f) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const half2 h = { (_Float16)f[2 * i], (_Float16)f[2 * i + 1] };
            r[i] = __builtin_bit_cast(uint32_t, h);
        }
        return r;
    }
};

// The sum of a value over the wave, in every lane and in a fixed order.
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
    return x;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
    return x;
}

}  // namespace mi
