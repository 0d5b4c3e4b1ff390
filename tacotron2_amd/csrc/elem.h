// Element types of the operators that take fp32, bf16 and fp16 tensors: four neighbouring elements as one vector access, or
// single elements; all arithmetic is fp32, a store rounds once to nearest even.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef float f32v4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32v2 __attribute__((ext_vector_type(2)));

struct ElemF32 {
    typedef float T;
    typedef f32v4 Raw;                                     // four elements as they are in memory
    static constexpr int size = 4;
    static __device__ __forceinline__ float at(const Raw& r, int j) { return r[j]; }
    static __device__ __forceinline__ float get(const void* p, long long i) { return ((const float*)p)[i]; }
    static __device__ __forceinline__ void put(void* p, long long i, float v) { ((float*)p)[i] = v; }
    static __device__ __forceinline__ void set(Raw& r, int j, float v) { r[j] = v; }
    static __device__ __forceinline__ Raw pack(float a, float b, float c, float d) { Raw r = {a, b, c, d}; return r; }
};

struct ElemBF16 {
    typedef __bf16 T;
    typedef u32v2 Raw;
    static constexpr int size = 2;
    typedef __bf16 V2 __attribute__((ext_vector_type(2)));
    typedef float F2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float at(const Raw& r, int j) {
        const uint32_t w = r[j >> 1];
        return __builtin_bit_cast(float, (j & 1) ? (w & 0xFFFF0000u) : (w << 16));
    }
    static __device__ __forceinline__ float get(const void* p, long long i) { return (float)((const T*)p)[i]; }
    static __device__ __forceinline__ void put(void* p, long long i, float v) { ((T*)p)[i] = (T)v; }
    static __device__ __forceinline__ Raw pack(float a, float b, float c, float d) {
        const F2 lo = {a, b}, hi = {c, d};
        Raw r = {__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, V2)), __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, V2))};
        return r;
    }
};

struct ElemF16 {
    typedef _Float16 T;
    typedef u32v2 Raw;
    static constexpr int size = 2;
    typedef _Float16 V2 __attribute__((ext_vector_type(2)));
    typedef float F2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float at(const Raw& r, int j) { return (float)__builtin_bit_cast(V2, (uint32_t)r[j >> 1])[j & 1]; }
    static __device__ __forceinline__ float get(const void* p, long long i) { return (float)((const T*)p)[i]; }
    static __device__ __forceinline__ void put(void* p, long long i, float v) { ((T*)p)[i] = (T)v; }
    static __device__ __forceinline__ Raw pack(float a, float b, float c, float d) {
        const F2 lo = {a, b}, hi = {c, d};
        Raw r = {__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, V2)), __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, V2))};
        return r;
    }
};

// Four neighbouring elements from element i on: one access, or four where the address is not aligned to the vector or the
// row ends inside it (n: elements that are there, >= 1; the missing ones repeat the last).
template <typename E, bool VEC>
__device__ __forceinline__ typename E::Raw load4(const void* p, long long i, int n) {
    typedef typename E::T T;
    if constexpr (VEC) {
        return *reinterpret_cast<const typename E::Raw*>((const T*)p + i);
    } else {
        const T* q = (const T*)p + i;
        T v[4] __attribute__((aligned(16)));
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = q[j < n ? j : n - 1];
        return *reinterpret_cast<const typename E::Raw*>(v);
    }
}
template <typename E, bool VEC>
__device__ __forceinline__ void store4(void* p, long long i, int n, float a, float b, float c, float d) {
    const typename E::Raw r = E::pack(a, b, c, d);
    if constexpr (VEC) {
        *reinterpret_cast<typename E::Raw*>((typename E::T*)p + i) = r;
    } else {
        typename E::T v[4] __attribute__((aligned(16)));
        *reinterpret_cast<typename E::Raw*>(v) = r;
        typename E::T* q = (typename E::T*)p + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (j < n) q[j] = v[j];
    }
}
