// AdamW over many tensors in one pass: decoupled weight decay, clipping by the norm of all gradients, states in fp32 or in 8 bits.
//     g' = gs g      m' = b1 m + (1 - b1) g'      v' = b2 v + (1 - b2) g'^2
//     p' = p (1 - lr decay) - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps)
// 8 bits: m and r = sqrt(v) as e4m3 values times one power of two for 128 neighbouring elements (e8m0), the largest of them in
// [128, 256) so that no rounding overflows.  v' changes by a thousandth a step, far less than half a code: rounding to nearest would
// freeze it, so codes are rounded up with the probability of the cut-off part, by a word that is a function of (seed, step,
// element).  r > 0 never becomes 0: its update would be divided by eps alone.
#include "ctx.h"
#include "elem.h"
#include "rng.h"

#include <float.h>
#include <math.h>
#include <new>
#include <vector>

#define AW_THREADS 256
#define AW_BLOCK 128                 /* elements that share a scale; every tensor's states start at a multiple of it */
#define AW_VEC 8                     /* elements of a thread: 16 lanes (one DPP row) hold one block */
#define AW_CHUNK 8192                /* elements of a workgroup (2048: 1.8 M parameters 18.6 us, 17.4 so) */
// From here on the norm reads gradients past the last-level cache: what it leaves there is gone before the step comes to it, and
// what it would push out are the step before's results (272 M bf16 gradients: 968 us in all, 948 so; 27 M fp32: 177, 180 so).
#define AW_STREAM_FROM (128LL << 20)
#define AW_NORM_BLOCKS 2048
#define AW_GROUPS 32                 /* of the workgroups of the norm, each with a counter on a line of its own */
#define AW_STREAM 20                 /* of the counter-based generator */
#define AW_BIND 96                   /* tensors a binding launch takes by value */

struct AwTensor { long long n, off; float decay; int chunk0; };
struct AwBound { const void* g; void* p; void* c; uint32_t g_type, p_type, c_type, aligned; };
struct AwCtl { float gs, lr, lr_t, ic2; uint32_t t; int skip; uint32_t pad[10]; uint32_t ticket[(AW_GROUPS + 1) * 16]; };

struct t2_adamw {
    int device = 0, n_tensors = 0, n_chunks = 0, bits = 32;
    bool stream = false;
    double b1 = 0, b2 = 0, eps = 0;
    uint32_t seed = 0;
    void *m = nullptr, *v = nullptr;
    uint8_t *ms = nullptr, *vs = nullptr;
    long long* step = nullptr;
    // one allocation: ctl | partial | tensors | chunk_tensor
    AwCtl* ctl = nullptr;
    double* partial = nullptr;
    AwTensor* tensors = nullptr;
    int* chunk_tensor = nullptr;
};

// ------------------------------------------------------------------------------------------------
// eight neighbouring elements of a tensor of any of the three types (type and alignment are the same for a whole workgroup)
// ------------------------------------------------------------------------------------------------
#define AW_GLOBAL __attribute__((address_space(1)))     // addresses out of a table are global memory: the compiler cannot know
template <typename E, bool STREAM = false>
__device__ __forceinline__ typename E::Raw load4(const void* p, long long i) {
    const AW_GLOBAL typename E::Raw* q = (const AW_GLOBAL typename E::Raw*)((const AW_GLOBAL typename E::T*)(uintptr_t)p + i);
    if constexpr (STREAM) return __builtin_nontemporal_load(q);
    else return *q;
}
template <typename E>
__device__ __forceinline__ void load8(const void* p, long long i, int n, bool aligned, float* x) {
    if (aligned && n >= AW_VEC) {
        const typename E::Raw lo = load4<E>(p, i), hi = load4<E>(p, i + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[j] = E::at(lo, j); x[j + 4] = E::at(hi, j); }
    } else {
        const AW_GLOBAL typename E::T* q = (const AW_GLOBAL typename E::T*)(uintptr_t)p + i;
#pragma unroll
        for (int j = 0; j < AW_VEC; ++j) x[j] = j < n ? (float)q[j] : 0.f;
    }
}
template <typename E>
__device__ __forceinline__ void store8(void* p, long long i, int n, bool aligned, const float* x) {
    AW_GLOBAL typename E::T* q = (AW_GLOBAL typename E::T*)(uintptr_t)p + i;
    if (aligned && n >= AW_VEC) {
        *(AW_GLOBAL typename E::Raw*)q = E::pack(x[0], x[1], x[2], x[3]);
        *(AW_GLOBAL typename E::Raw*)(q + 4) = E::pack(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int j = 0; j < AW_VEC; ++j) if (j < n) q[j] = (typename E::T)x[j];
    }
}
__device__ __forceinline__ void load8(const void* p, uint32_t type, long long i, int n, bool aligned, float* x) {
    if (type == T2_F32) load8<ElemF32>(p, i, n, aligned, x);
    else if (type == T2_BF16) load8<ElemBF16>(p, i, n, aligned, x);
    else load8<ElemF16>(p, i, n, aligned, x);
}
__device__ __forceinline__ void store8(void* p, uint32_t type, long long i, int n, bool aligned, const float* x) {
    if (type == T2_F32) store8<ElemF32>(p, i, n, aligned, x);
    else if (type == T2_BF16) store8<ElemBF16>(p, i, n, aligned, x);
    else store8<ElemF16>(p, i, n, aligned, x);
}

// ------------------------------------------------------------------------------------------------
// norm of all gradients and the step's factors
// ------------------------------------------------------------------------------------------------
struct AwNormArgs {
    const AwTensor* tensors; const int* chunk_tensor; const AwBound* bound;
    double* partial; AwCtl* ctl; long long* step;
    float* norm_out;                   // the norm alone is wanted: no step is begun
    const float* lr_dev;
    double lr, b1, b2, clip, grad_scale;
    int n_chunks, skip_nonfinite;
};

__device__ __forceinline__ double power(double b, long long n) {
    double r = 1.0;
    for (; n > 0; n >>= 1, b *= b) if (n & 1) r *= b;
    return r;
}

__device__ void begin_step(const AwNormArgs& a, double norm) {
    AwCtl& c = *a.ctl;
    const int skip = a.skip_nonfinite && !(norm <= 1.7976931348623157e308);
    c.skip = skip;
    if (skip) return;
    const long long t = *a.step + 1;
    *a.step = t;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    c.t = (uint32_t)t;
    c.gs = (float)(a.clip > 0.0 && norm > a.clip ? a.grad_scale * (a.clip / norm) : a.grad_scale);     // a limit of inf: no limit
    c.lr = (float)lr;
    c.lr_t = (float)(lr / (1.0 - power(a.b1, t)));
    c.ic2 = (float)(1.0 / sqrt(1.0 - power(a.b2, t)));
}

// Sums of squares in double, so that the clipping factor does not depend on how the work is split; the last workgroup to
// arrive adds the partial sums in a fixed order.  The sums go through agent-scope accesses that are waited for, not through a
// fence: a release at agent scope writes back a whole L2 for every workgroup (27 M gradients: 153 us with it).
template <typename E, bool STREAM>
__device__ __forceinline__ double chunk_squares(const void* p, long long base, long long n, bool aligned) {
    constexpr int R = AW_CHUNK / (AW_THREADS * 4);
    double s = 0.0;
    if (aligned && base + AW_CHUNK <= n) {                    // all loads of the chunk in flight
        typename E::Raw r[R];
#pragma unroll
        for (int k = 0; k < R; ++k) r[k] = load4<E, STREAM>(p, base + (k * AW_THREADS + (int)threadIdx.x) * 4);
#pragma unroll
        for (int k = 0; k < R; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) { const double x = (double)E::at(r[k], j); s = fma(x, x, s); }
    } else {
        const AW_GLOBAL typename E::T* q = (const AW_GLOBAL typename E::T*)(uintptr_t)p;
        const long long end = base + AW_CHUNK < n ? base + AW_CHUNK : n;
        for (long long i = base + threadIdx.x; i < end; i += AW_THREADS) { const double x = (double)(float)q[i]; s = fma(x, x, s); }
    }
    return s;
}

template <bool STREAM>
__global__ __launch_bounds__(AW_THREADS) void adamw_norm_kernel(AwNormArgs a) {
    __shared__ double sh[AW_THREADS / 64];
    __shared__ bool last;
    double s = 0.0;
    int next = a.chunk_tensor[blockIdx.x];
    for (int chunk = blockIdx.x; chunk < a.n_chunks; chunk += gridDim.x) {
        const int k = next;
        const AwTensor t = a.tensors[k];
        const AwBound b = a.bound[k];
        if (chunk + (int)gridDim.x < a.n_chunks) next = a.chunk_tensor[chunk + gridDim.x];
        const long long base = (long long)(chunk - t.chunk0) * AW_CHUNK;
        s += b.g_type == T2_F32 ? chunk_squares<ElemF32, STREAM>(b.g, base, t.n, b.aligned & 1)
           : b.g_type == T2_BF16 ? chunk_squares<ElemBF16, STREAM>(b.g, base, t.n, b.aligned & 1) : chunk_squares<ElemF16, STREAM>(b.g, base, t.n, b.aligned & 1);
    }
    auto block_sum = [&](double v) {
        for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
        double r = 0.0;
        for (int w = 0; w < AW_THREADS / 64; ++w) r += sh[w];
        return r;
    };
    s = block_sum(s);
    if (threadIdx.x == 0) {
        __hip_atomic_store(a.partial + blockIdx.x, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // the store is at the agent's point of coherence
        // the last of its group, and among those the last of all (2048 additions to one address take 20 us)
        const unsigned group = blockIdx.x % AW_GROUPS, groups = gridDim.x < AW_GROUPS ? gridDim.x : AW_GROUPS;
        uint32_t *mine = a.ctl->ticket + group * 16, *all = a.ctl->ticket + AW_GROUPS * 16;
        last = false;
        if (__hip_atomic_fetch_add(mine, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (gridDim.x - group + AW_GROUPS - 1) / AW_GROUPS - 1) {
            *mine = 0;                 // for the next launch
            last = __hip_atomic_fetch_add(all, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == groups - 1;
            if (last) *all = 0;
        }
    }
    __syncthreads();
    if (!last) return;
    s = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += AW_THREADS) s += __hip_atomic_load(a.partial + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s = block_sum(s);
    if (threadIdx.x == 0) {
        const double norm = fabs(a.grad_scale) * sqrt(s);
        if (a.norm_out) *a.norm_out = (float)norm;
        else begin_step(a, norm);
    }
}

__global__ void adamw_begin_kernel(AwNormArgs a) { begin_step(a, 0.0); }

// ------------------------------------------------------------------------------------------------
// the step
// ------------------------------------------------------------------------------------------------
struct AwStepArgs {
    const AwTensor* tensors; const int* chunk_tensor; const AwBound* bound; const AwCtl* ctl;
    void *m, *v; uint8_t *ms, *vs;
    float b1, omb1, b2, omb2, eps;
    uint32_t seed;
};

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
    return x > y ? x : y;
}
__device__ __forceinline__ uint32_t row_max(uint32_t x) {      // over the 16 lanes of a DPP row
    x = dpp_max<0xB1>(x);      // lanes 1, 0, 3, 2
    x = dpp_max<0x4E>(x);      // lanes 2, 3, 0, 1
    x = dpp_max<0x141>(x);     // mirrored halves
    return dpp_max<0x140>(x);  // mirrored row
}

// Eight values: two at a time by the converter, times the block's power of two (255: NaN, which the product keeps).  Both are exact.
__device__ __forceinline__ void decode8(u32v2 codes, int scale, float* x) {
    typedef float F2 __attribute__((ext_vector_type(2)));
    const float power = scale == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, scale ? (uint32_t)scale << 23 : 0x400000u);      // 0: 2^-127, subnormal
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const F2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[h], true);
        x[4 * h] = lo[0] * power; x[4 * h + 1] = lo[1] * power; x[4 * h + 2] = hi[0] * power; x[4 * h + 3] = hi[1] * power;
    }
}

// Roots within an ulp.  The instruction takes subnormal numbers for zeros (gradients under 1e-17 with an epsilon that small too would be
// divided by epsilon alone): they go through it larger by 2^32.
__device__ __forceinline__ void roots_within_an_ulp(const float* x, float* r) {
    float least = x[0];
#pragma unroll
    for (int j = 1; j < AW_VEC; ++j) least = fminf(least, x[j]);
    if (__all(least >= 0x1p-96f)) {
#pragma unroll
        for (int j = 0; j < AW_VEC; ++j) r[j] = __builtin_amdgcn_sqrtf(x[j]);
    } else {
#pragma unroll
        for (int j = 0; j < AW_VEC; ++j) r[j] = x[j] < 0x1p-96f ? __builtin_amdgcn_sqrtf(x[j] * 0x1p32f) * 0x1p-16f : __builtin_amdgcn_sqrtf(x[j]);
    }
}

// The correctly rounded root of every element.  With x normal: from the reciprocal root (one ulp) one correction by the exact residual,
// a third of what the general function takes (compared with that one for every number from 1e-30 to 1e38: equal); zeros and numbers
// too small or large for it go through that.
__device__ __forceinline__ void roots(const float* x, float* r) {
    float least = x[0], most = x[0];
#pragma unroll
    for (int j = 1; j < AW_VEC; ++j) { least = fminf(least, x[j]); most = fmaxf(most, x[j]); }
    if (__all(least > 1e-30f && most < 1e38f)) {
#pragma unroll
        for (int j = 0; j < AW_VEC; ++j) {
            const float y = __builtin_amdgcn_rsqf(x[j]), s = x[j] * y;
            r[j] = fmaf(fmaf(-s, s, x[j]), 0.5f * y, s);
        }
    } else {
#pragma unroll
        for (int j = 0; j < AW_VEC; ++j) r[j] = sqrtf(x[j]);
    }
}

// codes of eight elements and the block's scale byte
template <bool POSITIVE>
__device__ __forceinline__ u32v2 encode8(const float* x, const uint32_t* word, uint32_t& scale) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < AW_VEC; ++j) {
        const uint32_t b = __builtin_bit_cast(uint32_t, x[j]) & 0x7FFFFFFFu;
        top = b > top ? b : top;
    }
    const int e = (int)(row_max(top) >> 23);
    if (e == 255) { scale = 255; u32v2 zero = {0u, 0u}; return zero; }       // inf or NaN: the block stays NaN
    const int sb = e - 7 < 16 ? 16 : e - 7;
    scale = (uint32_t)sb;
    u32v2 out;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float v = x[4 * h + j];
            // an fp32 number whose exponent field is the code's: the code is its upper bits, gradual underflow included
            const uint32_t y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_ldexpf(__builtin_fabsf(v), 7 - sb));
            const uint32_t r16 = POSITIVE ? word[4 * h + j] >> 16 : word[4 * h + j] & 0xFFFFu;
            uint32_t code = (y + (r16 << 4) + 8u) >> 20;
            if (POSITIVE) { if (v > 0.f && code == 0) code = 1; }
            else code |= (__builtin_bit_cast(uint32_t, v) >> 24) & 0x80u;
            w |= code << (8 * j);
        }
        out[h] = w;
    }
    return out;
}

// One pass over parameters, gradients and states; a workgroup takes 8192 neighbouring elements of one tensor, a thread eight at a
// time, so that one DPP row of 16 lanes finds a block's largest value without shared memory.  Memory bounds it: 27 M elements in
// fp32 take 138 us (5.6 TB/s), 272 M with 8-bit states, fp32 parameters, bf16 gradients and copies 840 us (5.2 TB/s).  With 16-bit
// parameters and 8-bit states (10 bytes an element) arithmetic does: 27 M in 60 us, 4.6 TB/s; 65 vector instructions an element take
// three quarters of it.
template <int BITS>
__global__ __launch_bounds__(AW_THREADS) void adamw_step_kernel(AwStepArgs a) {
#pragma clang fp contract(off)       // every product and sum rounded by itself: codes are the definition's, bit for bit
    if (a.ctl->skip) return;
    const int chunk = (int)(gridDim.x - 1 - blockIdx.x);      // from the end: what the norm read last is still near
    const int k = a.chunk_tensor[chunk];
    const AwTensor t = a.tensors[k];
    const AwBound b = a.bound[k];
    if (b.p == nullptr) return;          // a table that was bound for the norm alone
    const float gs = a.ctl->gs, lr_t = a.ctl->lr_t, ic2 = a.ctl->ic2, keep = (float)(1.0 - (double)a.ctl->lr * (double)t.decay);
    const long long base = (long long)(chunk - t.chunk0) * AW_CHUNK;
    uint32_t key = t2_mix32(a.seed ^ (AW_STREAM * 0x9E3779B9u));
    key = t2_mix32(key ^ (a.ctl->t * 0x85EBCA6Bu + 0x165667B1u));
    for (int it = 0; it < AW_CHUNK / (AW_THREADS * AW_VEC); ++it) {
        const long long i = base + (it * AW_THREADS + threadIdx.x) * AW_VEC;
        if (i >= (t.n + AW_BLOCK - 1) / AW_BLOCK * AW_BLOCK) break;         // the same for all lanes of a block of 128
        const int n = (int)(t.n - i < 0 ? 0 : t.n - i < AW_VEC ? t.n - i : AW_VEC);
        const long long at = t.off + i;
        float g[AW_VEC], p[AW_VEC], m[AW_VEC], v[AW_VEC], r[AW_VEC];
        load8(b.g, b.g_type, i, n, b.aligned & 1, g);
        load8(b.p, b.p_type, i, n, b.aligned & 2, p);
        if constexpr (BITS == 32) {
            load8<ElemF32>(a.m, at, AW_VEC, true, m);
            load8<ElemF32>(a.v, at, AW_VEC, true, v);
        } else {
            const u32v2 mc = *(const u32v2*)((const uint8_t*)a.m + at), vc = *(const u32v2*)((const uint8_t*)a.v + at);
            const int sm = a.ms[at / AW_BLOCK], sv = a.vs[at / AW_BLOCK];
            decode8(mc, sm, m);
            decode8(vc, sv, v);
#pragma unroll
            for (int j = 0; j < AW_VEC; ++j) v[j] = v[j] * v[j];
        }
#pragma unroll
        for (int j = 0; j < AW_VEC; ++j) {
            const float x = g[j] * gs;
            m[j] = m[j] * a.b1 + x * a.omb1;
            v[j] = v[j] * a.b2 + (x * x) * a.omb2;
        }
        if constexpr (BITS == 8) {
            roots(v, r);
        } else {
            roots_within_an_ulp(v, r);
        }
#pragma unroll
        for (int j = 0; j < AW_VEC; ++j) p[j] = p[j] * keep - lr_t * m[j] * __builtin_amdgcn_rcpf(r[j] * ic2 + a.eps);
        store8(b.p, b.p_type, i, n, b.aligned & 2, p);
        if (b.c) store8(b.c, b.c_type, i, n, b.aligned & 4, p);
        if constexpr (BITS == 32) {
            store8<ElemF32>(a.m, at, AW_VEC, true, m);
            store8<ElemF32>(a.v, at, AW_VEC, true, v);
        } else {
            uint32_t word[AW_VEC], sm, sv;
            const uint32_t row = t2_mix32(key ^ ((uint32_t)(at >> 32) * 0xC2B2AE35u + 0x27D4EB2Fu));
#pragma unroll
            for (int j = 0; j < AW_VEC; ++j) word[j] = t2_word(row, (uint32_t)at + j);
            *(u32v2*)((uint8_t*)a.m + at) = encode8<false>(m, word, sm);
            *(u32v2*)((uint8_t*)a.v + at) = encode8<true>(r, word, sv);
            if ((threadIdx.x & 15) == 0) { a.ms[at / AW_BLOCK] = (uint8_t)sm; a.vs[at / AW_BLOCK] = (uint8_t)sv; }
        }
    }
}

struct AwBindArgs { AwBound e[AW_BIND]; };
__global__ void adamw_bind_kernel(AwBindArgs a, AwBound* table, int first, int n) {
    if ((int)threadIdx.x < n) table[first + threadIdx.x] = a.e[threadIdx.x];
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
extern "C" int64_t t2_adamw_elements(int n_tensors, const int64_t* sizes) {
    if (n_tensors < 1 || !sizes) return fail(T2_EINVAL, "at least one tensor is needed");
    int64_t total = 0, chunks = 0;
    for (int i = 0; i < n_tensors; ++i) {
        if (sizes[i] < 1 || sizes[i] > (1LL << 40)) return fail(T2_EINVAL, "tensor %d has %lld elements", i, (long long)sizes[i]);
        total += (sizes[i] + AW_BLOCK - 1) / AW_BLOCK * AW_BLOCK;
        chunks += (sizes[i] + AW_CHUNK - 1) / AW_CHUNK;
        if (chunks > 0xFFFFFF) return fail(T2_EINVAL, "too many elements");      // threads of a launch: 32 bits
    }
    return total;
}

extern "C" int t2_adamw_destroy(t2_adamw* o) {
    if (!o) return T2_OK;
    DeviceScope dev(o->device);
    if (o->ctl) (void)hipFree(o->ctl);
    delete o;
    return T2_OK;
}

static int build(t2_adamw* o, const int64_t* sizes, const double* decay) {
    int64_t chunks = 0;
    for (int i = 0; i < o->n_tensors; ++i) chunks += (sizes[i] + AW_CHUNK - 1) / AW_CHUNK;
    const size_t at_partial = sizeof(AwCtl), at_tensors = at_partial + AW_NORM_BLOCKS * sizeof(double),
                 at_chunks = at_tensors + o->n_tensors * sizeof(AwTensor), bytes = at_chunks + (size_t)chunks * sizeof(int);
    std::vector<char> image(bytes);                          // the control block and the counters start at zero
    AwTensor* ts = (AwTensor*)(image.data() + at_tensors);
    int* map = (int*)(image.data() + at_chunks);
    long long off = 0;
    int chunk = 0;
    for (int i = 0; i < o->n_tensors; ++i) {
        ts[i] = {sizes[i], off, (float)decay[i], chunk};
        off += (sizes[i] + AW_BLOCK - 1) / AW_BLOCK * AW_BLOCK;
        for (int64_t k = 0; k < (sizes[i] + AW_CHUNK - 1) / AW_CHUNK; ++k) map[chunk++] = i;
    }
    o->n_chunks = chunk;
    char* dev = nullptr;
    HIP_TRY(hipMalloc(&dev, bytes));
    o->ctl = (AwCtl*)dev;
    o->partial = (double*)(dev + at_partial);
    o->tensors = (AwTensor*)(dev + at_tensors);
    o->chunk_tensor = (int*)(dev + at_chunks);
    HIP_TRY(hipMemcpy(dev, image.data(), bytes, hipMemcpyHostToDevice));
    return T2_OK;
}
static_assert(sizeof(AwCtl) % 8 == 0 && sizeof(AwTensor) % 8 == 0, "parts of the allocation are aligned");

extern "C" int t2_adamw_create(t2_ctx* ctx, int n_tensors, const int64_t* sizes, const double* decay, double beta1, double beta2, double epsilon,
                               int state_bits, uint32_t seed, void* m, void* v, void* m_scale, void* v_scale, int64_t* step, t2_adamw** out) {
    if (!ctx || !sizes || !decay || !m || !v || !step || !out) return fail(T2_EINVAL, "null argument");
    if (t2_adamw_elements(n_tensors, sizes) < 0) return T2_EINVAL;
    // the reciprocal of epsilon is a number: an element whose moments are zero stays where it is
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !((float)epsilon >= FLT_MIN && (float)epsilon <= FLT_MAX))
        return fail(T2_EINVAL, "AdamW needs 0 <= beta < 1 and an epsilon from 1.2e-38 on");
    if (state_bits != 32 && state_bits != 8) return fail(T2_EINVAL, "states have 32 or 8 bits, not %d", state_bits);
    if (state_bits == 8 && (!m_scale || !v_scale)) return fail(T2_EINVAL, "states in 8 bits need scales");
    if ((((uintptr_t)m) | ((uintptr_t)v)) & 15) return fail(T2_EINVAL, "the states must be 16-byte aligned");
    for (int i = 0; i < n_tensors; ++i) if (!(decay[i] >= 0.0 && decay[i] <= 1e6)) return fail(T2_EINVAL, "weight decay %d is %g", i, decay[i]);
    DeviceScope dev(ctx->device);
    HIP_TRY(dev.err);
    t2_adamw* o = new (std::nothrow) t2_adamw();
    if (!o) return fail(T2_ENOMEM, "out of host memory");
    o->device = ctx->device; o->n_tensors = n_tensors; o->bits = state_bits;
    o->stream = t2_adamw_elements(n_tensors, sizes) >= AW_STREAM_FROM;
    o->b1 = beta1; o->b2 = beta2; o->eps = epsilon; o->seed = seed;
    o->m = m; o->v = v; o->ms = (uint8_t*)m_scale; o->vs = (uint8_t*)v_scale; o->step = (long long*)step;
    int rc;
    try {
        rc = build(o, sizes, decay);
    } catch (const std::bad_alloc&) {
        rc = fail(T2_ENOMEM, "out of host memory");
    }
    if (rc != T2_OK) { t2_adamw_destroy(o); return rc; }
    *out = o;
    return T2_OK;
}

static int check_call(const t2_ctx* ctx, const t2_adamw* o) {
    if (!ctx || !o) return fail(T2_EINVAL, "null argument");
    if (ctx->device != o->device) return fail(T2_EINVAL, "optimizer on device %d, context on %d", o->device, ctx->device);
    return T2_OK;
}

extern "C" int64_t t2_adamw_table_bytes(const t2_adamw* o) { return o ? (int64_t)o->n_tensors * (int64_t)sizeof(AwBound) : (int64_t)fail(T2_EINVAL, "null argument"); }

extern "C" int t2_adamw_bind(t2_ctx* ctx, t2_adamw* o, const void* const* grads, const int32_t* grad_types, void* const* params, const int32_t* param_types,
                             void* const* copies, const int32_t* copy_types, void* table) {
    T2_TRY(check_call(ctx, o));
    if (!grads || !grad_types || !table || (params && !param_types) || (copies && (!copy_types || !params))) return fail(T2_EINVAL, "null argument");
    if ((uintptr_t)table & 15) return fail(T2_EINVAL, "the table must be 16-byte aligned");
    for (int i = 0; i < o->n_tensors; ++i) {
        if (!grads[i] || (params && !params[i])) return fail(T2_EINVAL, "tensor %d is null", i);
        if ((unsigned)grad_types[i] > T2_F16 || (params && (unsigned)param_types[i] > T2_F16) || (copies && copies[i] && (unsigned)copy_types[i] > T2_F16))
            return fail(T2_EINVAL, "tensor %d has an unknown type", i);
    }
    DeviceScope dev(ctx->device);
    HIP_TRY(dev.err);
    for (int first = 0; first < o->n_tensors; first += AW_BIND) {
        AwBindArgs a = {};
        const int n = o->n_tensors - first < AW_BIND ? o->n_tensors - first : AW_BIND;
        for (int i = 0; i < n; ++i) {
            AwBound& e = a.e[i];
            const int k = first + i;
            e.g = grads[k]; e.g_type = (uint32_t)grad_types[k];
            e.p = params ? params[k] : nullptr; e.p_type = params ? (uint32_t)param_types[k] : 0;
            e.c = copies ? copies[k] : nullptr; e.c_type = e.c ? (uint32_t)copy_types[k] : 0;
            // accesses of four elements: 16 bytes of fp32, 8 of the 16-bit types
            auto fits = [](const void* p, uint32_t type) { return ((uintptr_t)p & (type == T2_F32 ? 15 : 7)) == 0; };
            e.aligned = (fits(e.g, e.g_type) ? 1u : 0u) | (fits(e.p, e.p_type) ? 2u : 0u) | (fits(e.c, e.c_type) ? 4u : 0u);
        }
        hipLaunchKernelGGL(adamw_bind_kernel, dim3(1), dim3(AW_BIND <= 64 ? 64 : 128), 0, ctx->stream, a, (AwBound*)table, first, n);
    }
    HIP_TRY(hipGetLastError());
    return T2_OK;
}

static AwNormArgs norm_args(const t2_adamw* o, const void* table, double grad_scale) {
    AwNormArgs a = {};
    a.tensors = o->tensors; a.chunk_tensor = o->chunk_tensor; a.bound = (const AwBound*)table;
    a.partial = o->partial; a.ctl = o->ctl; a.step = o->step;
    a.b1 = o->b1; a.b2 = o->b2; a.grad_scale = grad_scale; a.n_chunks = o->n_chunks;
    return a;
}
static void launch_norm(const t2_ctx* ctx, const t2_adamw* o, const AwNormArgs& a) {
    const dim3 grid(o->n_chunks < AW_NORM_BLOCKS ? o->n_chunks : AW_NORM_BLOCKS), threads(AW_THREADS);
    if (o->stream) hipLaunchKernelGGL(adamw_norm_kernel<true>, grid, threads, 0, ctx->stream, a);
    else hipLaunchKernelGGL(adamw_norm_kernel<false>, grid, threads, 0, ctx->stream, a);
}

// the factors of a step are fp32 on the device
static bool fits_f32(double x) { return fabs(x) <= FLT_MAX; }

extern "C" int t2_adamw_global_norm(t2_ctx* ctx, t2_adamw* o, const void* table, double grad_scale, float* norm_out) {
    if (!fits_f32(grad_scale)) return fail(T2_EINVAL, "grad_scale is %g", grad_scale);
    T2_TRY(check_call(ctx, o));
    if (!table || !norm_out) return fail(T2_EINVAL, "null argument");
    DeviceScope dev(ctx->device);
    HIP_TRY(dev.err);
    AwNormArgs a = norm_args(o, table, grad_scale);
    a.norm_out = norm_out;
    launch_norm(ctx, o, a);
    HIP_TRY(hipGetLastError());
    return T2_OK;
}

extern "C" int t2_adamw_step(t2_ctx* ctx, t2_adamw* o, const void* table, double learning_rate, const float* learning_rate_dev, double clip_norm,
                             double grad_scale, int skip_nonfinite) {
    if (!fits_f32(grad_scale)) return fail(T2_EINVAL, "grad_scale is %g", grad_scale);
    if (!learning_rate_dev && !fits_f32(learning_rate)) return fail(T2_EINVAL, "learning_rate is %g", learning_rate);
    if (clip_norm != clip_norm) return fail(T2_EINVAL, "clip_norm is NaN");
    T2_TRY(check_call(ctx, o));
    if (!table) return fail(T2_EINVAL, "null argument");
    DeviceScope dev(ctx->device);
    HIP_TRY(dev.err);
    AwNormArgs a = norm_args(o, table, grad_scale);
    a.lr = learning_rate; a.lr_dev = learning_rate_dev; a.clip = clip_norm; a.skip_nonfinite = skip_nonfinite != 0;
    if (clip_norm > 0.0 || skip_nonfinite) launch_norm(ctx, o, a);
    else hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(1), 0, ctx->stream, a);
    AwStepArgs s = {};
    s.tensors = o->tensors; s.chunk_tensor = o->chunk_tensor; s.bound = (const AwBound*)table; s.ctl = o->ctl;
    s.m = o->m; s.v = o->v; s.ms = o->ms; s.vs = o->vs;
    s.b1 = (float)o->b1; s.omb1 = (float)(1.0 - o->b1); s.b2 = (float)o->b2; s.omb2 = (float)(1.0 - o->b2); s.eps = (float)o->eps; s.seed = o->seed;
    if (o->bits == 32) hipLaunchKernelGGL(adamw_step_kernel<32>, dim3(o->n_chunks), dim3(AW_THREADS), 0, ctx->stream, s);
    else hipLaunchKernelGGL(adamw_step_kernel<8>, dim3(o->n_chunks), dim3(AW_THREADS), 0, ctx->stream, s);
    HIP_TRY(hipGetLastError());
    return T2_OK;
}
