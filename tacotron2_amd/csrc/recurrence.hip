// Gated linear recurrence: a = sigmoid(f), h' = a h + (1 - a) z, y = sigmoid(o) h', forward, backward and for one position.
#include "ctx.h"
#include "elem.h"

#define SCAN_LOG2E 1.4426950408889634f

// a = sigmoid(f) and b = 1 - a.  b comes from the same exponential, not from 1 - a: near a = 1 (long memories) that
// difference would have lost its digits.  The reciprocal gets one correction: the instruction's own error leans to one side, and a
// memory of n steps collects n of them (800 steps, memories up to 1000: the final state was off by 1.5e-6, now by what the
// rounding of a itself leaves).  exp2 of more than 126 would overflow and make b inf * 0; NaN passes through.
__device__ __forceinline__ void gate(float f, float& a, float& b) {
    float x = -SCAN_LOG2E * f;
    x = x > 126.f ? 126.f : x;
    const float e = __builtin_amdgcn_exp2f(x), d = 1.f + e, r = __builtin_amdgcn_rcpf(d);
    a = fmaf(fmaf(-d, r, 1.f), r, r);
    b = e * a;
}
// the output gate: used once, nothing collects
__device__ __forceinline__ float sigmoid1(float f) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-SCAN_LOG2E * f)); }

__device__ __forceinline__ int row_length(const int64_t* lens, int b, int T) {
    if (lens == nullptr) return T;
    const int64_t n = lens[b];
    return n < 0 ? 0 : n > T ? T : (int)n;
}

template <typename E>
__global__ __launch_bounds__(64) void scan_rows_kernel(t2_scan_args a) {
    const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (c >= a.H) return;
    const int len = row_length(a.lens, b, a.T), ntape = (a.T + T2_SCAN_SPAN - 1) / T2_SCAN_SPAN;
    float h = a.state ? a.state[(long long)b * a.H + c] : 0.f;
    for (int s = 0; s < a.T; ++s) {
        if (s >= len) { E::put((void*)a.y.ptr, b * a.y.stride_b + s * a.y.stride_t + c, 0.f); continue; }
        const long long t = a.reverse ? len - 1 - s : s;
        if (a.tape && s % T2_SCAN_SPAN == 0) a.tape[((long long)b * ntape + s / T2_SCAN_SPAN) * a.H + c] = h;
        float g, k;
        gate(E::get(a.f.ptr, b * a.f.stride_b + t * a.f.stride_t + c), g, k);
        h = fmaf(g, h, k * E::get(a.z.ptr, b * a.z.stride_b + t * a.z.stride_t + c));
        const float y = a.o.ptr ? h * sigmoid1(E::get(a.o.ptr, b * a.o.stride_b + t * a.o.stride_t + c)) : h;
        E::put((void*)a.y.ptr, b * a.y.stride_b + t * a.y.stride_t + c, y);
    }
    if (a.final_state) a.final_state[(long long)b * a.H + c] = h;
}

template <typename E>
__global__ __launch_bounds__(64) void scan_rows_backward_kernel(t2_scan_args a) {
    const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (c >= a.H) return;
    const int len = row_length(a.lens, b, a.T), ntape = (a.T + T2_SCAN_SPAN - 1) / T2_SCAN_SPAN;
    auto put = [&](const t2_seq& q, long long t, float v) { E::put((void*)q.ptr, b * q.stride_b + t * q.stride_t + c, v); };
    auto get = [&](const t2_seq& q, long long t) { return E::get(q.ptr, b * q.stride_b + t * q.stride_t + c); };
    for (int t = len; t < a.T; ++t) {
        put(a.dz, t, 0.f); put(a.df, t, 0.f);
        if (a.o.ptr) put(a.do_, t, 0.f);
    }
    float d = a.dfinal ? a.dfinal[(long long)b * a.H + c] : 0.f;         // gradient of the state behind the step
    for (int j = (len + T2_SCAN_SPAN - 1) / T2_SCAN_SPAN - 1; j >= 0; --j) {
        const int s0 = j * T2_SCAN_SPAN, n = len - s0 < T2_SCAN_SPAN ? len - s0 : T2_SCAN_SPAN;
        float before[T2_SCAN_SPAN];
        float h = a.tape[((long long)b * ntape + j) * a.H + c];
        for (int i = 0; i < n; ++i) {
            const long long t = a.reverse ? len - 1 - (s0 + i) : s0 + i;
            before[i] = h;
            float g, k;
            gate(get(a.f, t), g, k);
            h = fmaf(g, h, k * get(a.z, t));
        }
        for (int i = n - 1; i >= 0; --i) {
            const long long t = a.reverse ? len - 1 - (s0 + i) : s0 + i;
            float g, k;
            gate(get(a.f, t), g, k);
            const float z = get(a.z, t), dy = get(a.dy, t);
            if (a.o.ptr) {
                float so, sn;
                gate(get(a.o, t), so, sn);
                d = fmaf(dy, so, d);
                put(a.do_, t, dy * so * sn * fmaf(g, before[i], k * z));
            } else {
                d += dy;
            }
            put(a.dz, t, k * d);
            put(a.df, t, d * (before[i] - z) * g * k);
            d *= g;
        }
    }
    if (a.dstate) a.dstate[(long long)b * a.H + c] = d;
}

struct StepArgs {
    const void *z, *f, *o;
    void* y;
    float* state;
    const uint8_t* active;
    long long zs, fs, os, ys, ss;
    int H;
};

template <typename E>
__global__ __launch_bounds__(64) void scan_step_kernel(StepArgs a) {
    const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (c >= a.H) return;
    if (a.active && !a.active[b]) { E::put(a.y, b * a.ys + c, 0.f); return; }
    float g, k;
    gate(E::get(a.f, b * a.fs + c), g, k);
    const float h = fmaf(g, a.state[b * a.ss + c], k * E::get(a.z, b * a.zs + c));
    a.state[b * a.ss + c] = h;
    E::put(a.y, b * a.ys + c, a.o ? h * sigmoid1(E::get(a.o, b * a.os + c)) : h);
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
static bool sizes_ok(int B, int T, int H) { return B >= 1 && B <= 65535 && T >= 1 && T <= (1 << 30) && H >= 1 && H <= (1 << 24); }

extern "C" int64_t t2_gated_scan_tape(int B, int T, int H) {
    if (!sizes_ok(B, T, H)) return fail(T2_EINVAL, "bad shape [%d,%d,%d]", B, T, H);
    return (int64_t)B * ((T + T2_SCAN_SPAN - 1) / T2_SCAN_SPAN) * H;
}

extern "C" int64_t t2_gated_scan_ws(int B, int T, int H) {
    if (!sizes_ok(B, T, H)) return fail(T2_EINVAL, "bad shape [%d,%d,%d]", B, T, H);
    return 0;
}

static int check_args(const t2_ctx* ctx, const t2_scan_args* a, bool backward) {
    if (!ctx || !a) return fail(T2_EINVAL, "null argument");
    if (a->dtype < T2_F32 || a->dtype > T2_F16) return fail(T2_EINVAL, "unknown type %d", a->dtype);
    if (!sizes_ok(a->B, a->T, a->H)) return fail(T2_EINVAL, "bad shape [%d,%d,%d]", a->B, a->T, a->H);
    if (!a->z.ptr || !a->f.ptr) return fail(T2_EINVAL, "z and f are needed");
    if (!backward && !a->y.ptr) return fail(T2_EINVAL, "y is null");
    if (backward && (!a->dy.ptr || !a->dz.ptr || !a->df.ptr || (a->o.ptr && !a->do_.ptr))) return fail(T2_EINVAL, "dy, dz, df (and do with o) are needed");
    if (backward && !a->tape) return fail(T2_EINVAL, "the tape of the forward call is needed");
    const int64_t ws = t2_gated_scan_ws(a->B, a->T, a->H);
    if (a->ws_bytes < ws || (ws > 0 && (!a->ws || ((uintptr_t)a->ws & 15)))) return fail(T2_EINVAL, "workspace of %lld bytes, 16-byte aligned, needed", (long long)ws);
    return T2_OK;
}

extern "C" int t2_gated_scan(t2_ctx* ctx, const t2_scan_args* a) {
    T2_TRY(check_args(ctx, a, false));
    DeviceScope dev(ctx->device);
    HIP_TRY(dev.err);
    const dim3 grid((a->H + 63) / 64, a->B);
    if (a->dtype == T2_F32) hipLaunchKernelGGL(scan_rows_kernel<ElemF32>, grid, dim3(64), 0, ctx->stream, *a);
    else if (a->dtype == T2_BF16) hipLaunchKernelGGL(scan_rows_kernel<ElemBF16>, grid, dim3(64), 0, ctx->stream, *a);
    else hipLaunchKernelGGL(scan_rows_kernel<ElemF16>, grid, dim3(64), 0, ctx->stream, *a);
    HIP_TRY(hipGetLastError());
    return T2_OK;
}

extern "C" int t2_gated_scan_backward(t2_ctx* ctx, const t2_scan_args* a) {
    T2_TRY(check_args(ctx, a, true));
    DeviceScope dev(ctx->device);
    HIP_TRY(dev.err);
    const dim3 grid((a->H + 63) / 64, a->B);
    if (a->dtype == T2_F32) hipLaunchKernelGGL(scan_rows_backward_kernel<ElemF32>, grid, dim3(64), 0, ctx->stream, *a);
    else if (a->dtype == T2_BF16) hipLaunchKernelGGL(scan_rows_backward_kernel<ElemBF16>, grid, dim3(64), 0, ctx->stream, *a);
    else hipLaunchKernelGGL(scan_rows_backward_kernel<ElemF16>, grid, dim3(64), 0, ctx->stream, *a);
    HIP_TRY(hipGetLastError());
    return T2_OK;
}

extern "C" int t2_gated_scan_step(t2_ctx* ctx, int dtype, int B, int H, const void* z, int64_t z_stride, const void* f, int64_t f_stride, const void* o,
                                  int64_t o_stride, float* state, int64_t state_stride, const uint8_t* active, void* y, int64_t y_stride) {
    if (!ctx || !z || !f || !state || !y) return fail(T2_EINVAL, "null argument");
    if (dtype < T2_F32 || dtype > T2_F16) return fail(T2_EINVAL, "unknown type %d", dtype);
    if (!sizes_ok(B, 1, H)) return fail(T2_EINVAL, "bad shape [%d,%d]", B, H);
    if (B > 1 && (state_stride < H || y_stride < H)) return fail(T2_EINVAL, "rows of the state or of y overlap");
    DeviceScope dev(ctx->device);
    HIP_TRY(dev.err);
    const StepArgs a = {z, f, o, y, state, active, z_stride, f_stride, o_stride, y_stride, state_stride, H};
    const dim3 grid((H + 63) / 64, B);
    if (dtype == T2_F32) hipLaunchKernelGGL(scan_step_kernel<ElemF32>, grid, dim3(64), 0, ctx->stream, a);
    else if (dtype == T2_BF16) hipLaunchKernelGGL(scan_step_kernel<ElemBF16>, grid, dim3(64), 0, ctx->stream, a);
    else hipLaunchKernelGGL(scan_step_kernel<ElemF16>, grid, dim3(64), 0, ctx->stream, a);
    HIP_TRY(hipGetLastError());
    return T2_OK;
}
