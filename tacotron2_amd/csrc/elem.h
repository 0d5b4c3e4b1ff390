// Element types of the operators that take fp32, bf16 and fp16 tensors: four neighbouring elements as one vector access, or
// single elements; all arithmetic is fp32, a store rounds once to nearest even.
#pragma once
#include "../../include/t2mi.h"
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

// Four neighbouring elements of one row of a sequence [B][T][H], for a workgroup that works on `rows` successive steps of row b from
// step `first` on (the steps of a reversed row run from its position len - 1 down).  Steps are counted from `first`.
//  BUFFER: a buffer descriptor at the tile's lowest address and 32-bit offsets: one vector register an access, and an access that
//  is not wanted gets an offset beyond the descriptor's range, where loads give 0 and stores do nothing (no branches).  Elements need
//  only their own alignment.  The caller sees to it that rows * |stride_t| fits SEQ_RANGE and that H >= 4.
//  NT: stores that do not stay in L2.
//  otherwise: plain pointers, element by element (n of the four are there).
#define SEQ_RANGE 0x40000000

template <typename E, bool BUFFER> struct SeqRows;

template <typename E> struct SeqRows<E, true> {
    __amdgpu_buffer_rsrc_t r;
    int base, pitch;                 // bytes; offset of a step: base + step * pitch
    __device__ __forceinline__ SeqRows(const t2_seq& q, int b, int first, int rows, int len, bool reverse) {
        const long long dt = reverse ? -q.stride_t : q.stride_t, t0 = reverse ? len - 1 - first : first;
        const long long low = dt < 0 ? t0 * q.stride_t + dt * (rows - 1) : t0 * q.stride_t;
        const uint64_t at = (uint64_t)q.ptr + (uint64_t)((b * q.stride_b + low) * E::size);
        // uniform, but the compiler cannot see it behind the tile that was drawn
        const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)at), hi = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
        r = __builtin_amdgcn_make_buffer_rsrc((void*)(((uint64_t)hi << 32) | lo), 0, SEQ_RANGE, 0x00020000);
        pitch = __builtin_amdgcn_readfirstlane((int)(dt * E::size));
        base = dt < 0 ? -pitch * (rows - 1) : 0;
    }
    __device__ __forceinline__ int offset(int step, int c, bool on) const { return on ? base + step * pitch + c * E::size : 0x7FFFFFFF; }
    __device__ __forceinline__ typename E::Raw load(int step, int c, int, bool on) const {
        if constexpr (E::size == 4) return __builtin_bit_cast(typename E::Raw, __builtin_amdgcn_raw_buffer_load_b128(r, offset(step, c, on), 0, 0));
        else return __builtin_bit_cast(typename E::Raw, __builtin_amdgcn_raw_buffer_load_b64(r, offset(step, c, on), 0, 0));
    }
    template <bool NT> __device__ __forceinline__ void store(int step, int c, int, bool on, float v0, float v1, float v2, float v3) const {
        typedef uint32_t u32v4 __attribute__((ext_vector_type(4)));
        const typename E::Raw v = E::pack(v0, v1, v2, v3);
        if constexpr (E::size == 4) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32v4, v), r, offset(step, c, on), 0, NT ? 2 : 0);
        else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32v2, v), r, offset(step, c, on), 0, NT ? 2 : 0);
    }
};

template <typename E> struct SeqRows<E, false> {
    typedef typename E::T T;
    T* p;
    long long pitch;
    __device__ __forceinline__ SeqRows(const t2_seq& q, int b, int first, int rows, int len, bool reverse) {
        pitch = reverse ? -q.stride_t : q.stride_t;
        p = (T*)q.ptr + b * q.stride_b + (reverse ? len - 1 - first : first) * q.stride_t;
    }
    __device__ __forceinline__ typename E::Raw load(int step, int c, int n, bool on) const {
        T v[4] __attribute__((aligned(16))) = {};
        const T* q = p + step * pitch + c;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (on && j < n) v[j] = q[j];
        return *reinterpret_cast<const typename E::Raw*>(v);
    }
    template <bool> __device__ __forceinline__ void store(int step, int c, int n, bool on, float v0, float v1, float v2, float v3) const {
        T v[4] __attribute__((aligned(16)));
        *reinterpret_cast<typename E::Raw*>(v) = E::pack(v0, v1, v2, v3);
        T* q = p + step * pitch + c;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (on && j < n) q[j] = v[j];
    }
};
