// Gated linear recurrence: a = sigmoid(f), h' = a h + (1 - a) z, y = sigmoid(o) h', forward, backward and for one position.
#include "ctx.h"
#include "elem.h"

#define SCAN_LOG2E 1.4426950408889634f

// a = sigmoid(f) and b = 1 - a.  b comes from the same exponential, not from 1 - a: near a = 1 (long memories) that
// difference would have lost its digits.  The reciprocal gets one correction: the instruction's own error leans to one side, and a
// memory of n steps collects n of them (800 steps, memories up to 1000: the final state was off by 1.5e-6, now by what the
// rounding of a itself leaves).  exp2 of more than 126 would overflow and make b inf * 0; NaN passes through.
__device__ __forceinline__ void gate(float f, float& a, float& b) {
    const float x = __builtin_elementwise_minimum(-SCAN_LOG2E * f, 126.f);
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

// ------------------------------------------------------------------------------------------------
// A sequence is cut into tiles of C = TG * L steps by 64 channels, one workgroup each.  A thread holds L consecutive steps of 4
// channels in registers (16 lanes read 64 neighbouring channels of a row: 128 bytes or more), so every input is read once and
// every output written once.  Inside a tile: each thread composes its steps into h' = A h + B; one wave composes the TG pieces of
// every channel, finds the state in front of the tile, and hands every thread the state in front of its steps.
//
// Across tiles: a tile publishes its composition; the state in front of it is that in front of its group of SCAN_GROUP tiles, taken
// through the compositions in between in their order; the first tile of a group finds it through the whole group before and
// publishes it.  The order of every sum is fixed, so results do not depend on timing, and only one hand-over in SCAN_GROUP
// has to wait for another.  Every word is a value that carries its own validity (all ones: not there yet; a computed NaN is never
// that pattern), so one relaxed agent-scope access hands it over, without flags or fences.  Tiles are numbered by a counter that
// workgroups draw from as they start, all tiles of a step range before those that follow it: a workgroup waits only for workgroups
// that have started before it and that wait for none behind them, so every wait ends.
// ------------------------------------------------------------------------------------------------
#define SCAN_CH 64
#define SCAN_GROUP 16
#define SCAN_WAIT_TICKS 200000000ull   /* 2 s of the 100 MHz clock; a wait never comes near it.  Beyond: NaN, not a hang */

struct ScanWs {                        // counter | compositions [ntile][chains][64] | states in front of the groups [ngroup][chains][64]
    unsigned* next;
    unsigned long long* piece;
    unsigned* state;
};
static __host__ __device__ inline ScanWs scan_ws(void* p, long long slots) {
    ScanWs w;
    w.next = (unsigned*)p;
    w.piece = (unsigned long long*)((char*)p + 16);
    w.state = (unsigned*)(w.piece + slots);
    return w;
}

__global__ __launch_bounds__(256) void scan_ws_kernel(uint4* ws, long long n16) {
    const uint4 ones = {~0u, ~0u, ~0u, ~0u}, zero = {0u, 0u, 0u, 0u};
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n16; i += (long long)gridDim.x * 256) ws[i] = i == 0 ? zero : ones;
}

__device__ __forceinline__ unsigned valid_bits(float v) { return v != v ? 0x7FC00000u : __builtin_bit_cast(unsigned, v); }
__device__ __forceinline__ void publish(unsigned long long* p, float A, float B) {
    __hip_atomic_store(p, ((unsigned long long)valid_bits(B) << 32) | valid_bits(A), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish(unsigned* p, float v) { __hip_atomic_store(p, valid_bits(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The value that enters the i-th tile of a chain (i = 0: `first`), for one channel a lane.  slot: the tile's place among the
// compositions; hop: from one tile of the chain to the next; row: the group's place among the states, row_hop: to the group before.
__device__ __forceinline__ float look_back(const ScanWs& w, int i, float first, long long slot, long long hop, long long row, long long row_hop) {
    if (i == 0) return first;
    const bool head = i % SCAN_GROUP == 0;             // the first tile of a group folds the whole group before it
    const int m = head ? SCAN_GROUP : i % SCAN_GROUP, group = i / SCAN_GROUP - (head ? 1 : 0);
    const unsigned* start = w.state + (head ? row - row_hop : row);
    const unsigned long long* from = w.piece + (slot - hop * m);
    unsigned long long pc[SCAN_GROUP];
    unsigned st = 0;
    const unsigned long long t0 = __builtin_amdgcn_s_memrealtime();
    for (;;) {
        bool there = true;
        if (group > 0) { st = __hip_atomic_load(start, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); there = st != ~0u; }
#pragma unroll
        for (int k = 0; k < SCAN_GROUP; ++k) pc[k] = __hip_atomic_load(from + hop * (k < m ? k : m - 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int k = 0; k < SCAN_GROUP; ++k) there = there && pc[k] != ~0ull;
        if (!__any(!there)) break;
        if (__builtin_amdgcn_s_memrealtime() - t0 > SCAN_WAIT_TICKS) { first = __builtin_nanf(""); st = 0x7FC00000u; break; }
    }
    float h = group > 0 ? __builtin_bit_cast(float, st) : first;
#pragma unroll
    for (int k = 0; k < SCAN_GROUP; ++k)
        if (k < m) h = fmaf(__builtin_bit_cast(float, (unsigned)pc[k]), h, __builtin_bit_cast(float, (unsigned)(pc[k] >> 32)));
    if (head) publish(w.state + row, h);
    return h;
}

struct TileIds { int tile, b, c0, len; long long chain, chains; };

template <int C>
__device__ __forceinline__ TileIds tile_ids(const t2_scan_args& a, const ScanWs& w, int ntile, bool from_end) {
    __shared__ unsigned s_id;
    unsigned id = blockIdx.x;
    if (ntile > 1) {
        if (threadIdx.x == 0) s_id = atomicAdd(w.next, 1u);
        __syncthreads();
        id = s_id;
    }
    TileIds t;
    const int ncb = (a.H + SCAN_CH - 1) / SCAN_CH;
    t.chains = (long long)a.B * ncb;
    t.tile = (int)(id / (unsigned)t.chains);
    t.chain = id - (unsigned)t.tile * (unsigned)t.chains;
    t.b = (int)(t.chain / ncb);
    t.c0 = (int)(t.chain - (long long)t.b * ncb) * SCAN_CH;
    if (from_end) t.tile = ntile - 1 - t.tile;
    t.len = row_length(a.lens, t.b, a.T);
    return t;
}

// L rows of four channels; rows at or behind the row's length repeat its last position (discarded by the caller)
template <typename E, bool VEC, int L>
__device__ __forceinline__ void load_rows(typename E::Raw* r, const t2_seq& q, int b, int c, int nc, int s0, int len, bool reverse) {
    const int last = len > 0 ? len - 1 : 0;
    const long long base = (long long)b * q.stride_b + c, dt = reverse ? -q.stride_t : q.stride_t;
    const long long first = base + (long long)(reverse ? last : 0) * q.stride_t;
    if (s0 + L <= len) {
        long long at = first + (long long)s0 * dt;
#pragma unroll
        for (int l = 0; l < L; ++l, at += dt) r[l] = load4<E, VEC>(q.ptr, at, nc);
    } else {
#pragma unroll
        for (int l = 0; l < L; ++l) r[l] = load4<E, VEC>(q.ptr, first + (long long)(s0 + l < last ? s0 + l : last) * dt, nc);
    }
}

template <typename E, bool VEC, int L>
__device__ __forceinline__ void zero_rows(const t2_seq& q, int b, int c, int nc, int s0, int from, int T) {
#pragma unroll
    for (int l = 0; l < L; ++l)
        if (s0 + l >= from && s0 + l < T) store4<E, VEC>((void*)q.ptr, (long long)b * q.stride_b + (long long)(s0 + l) * q.stride_t + c, nc, 0.f, 0.f, 0.f, 0.f);
}

template <typename E, bool GATE, bool VEC, int TG, int L>
__global__ __launch_bounds__(16 * TG) void scan_tile_kernel(t2_scan_args a, ScanWs w, int ntile) {
    constexpr int C = TG * L;
    __shared__ float2 s_piece[TG][SCAN_CH];
    __shared__ f32v4 s_in[TG][SCAN_CH / 4];
    const TileIds t = tile_ids<C>(a, w, ntile, false);
    const int len = t.len, tg = threadIdx.x >> 4, ch = (threadIdx.x & 15) * 4, s0 = t.tile * C + tg * L;
    // lanes beyond the last channel repeat it and store nothing
    const int here = a.H - (t.c0 + ch), c = here > 0 ? t.c0 + ch : (VEC ? a.H - 4 : a.H - 1), nc = here > 4 ? 4 : here > 0 ? here : 1;
    if (t.tile * C >= len && t.tile > 0) {
        if (here > 0) zero_rows<E, VEC, L>(a.y, t.b, c, nc, s0, len, a.T);
        return;
    }
    typename E::Raw zr[L], fr[L], orr[L];
    load_rows<E, VEC, L>(fr, a.f, t.b, c, nc, s0, len, a.reverse);
    load_rows<E, VEC, L>(zr, a.z, t.b, c, nc, s0, len, a.reverse);
    if (GATE) load_rows<E, VEC, L>(orr, a.o, t.b, c, nc, s0, len, a.reverse);
    float ga[L][4], x[L][4], A[4] = {1.f, 1.f, 1.f, 1.f}, B[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float b;
            gate(E::at(fr[l], j), ga[l][j], b);
            x[l][j] = b * E::at(zr[l], j);
        }
    if (s0 + L > len) {                                      // padding: h stays
#pragma unroll
        for (int l = 0; l < L; ++l)
#pragma unroll
            for (int j = 0; j < 4; ++j) if (s0 + l >= len) { ga[l][j] = 1.f; x[l][j] = 0.f; }
    }
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            B[j] = fmaf(ga[l][j], B[j], x[l][j]);
            A[j] *= ga[l][j];
        }
#pragma unroll
    for (int j = 0; j < 4; ++j) s_piece[tg][ch + j] = make_float2(A[j], B[j]);
    __syncthreads();
    if (threadIdx.x < SCAN_CH) {
        const int lane = threadIdx.x, cc = t.c0 + lane;
        float2 p[TG];
        float At = 1.f, Bt = 0.f;
#pragma unroll
        for (int i = 0; i < TG; ++i) {
            p[i] = s_piece[i][lane];
            Bt = fmaf(p[i].x, Bt, p[i].y);
            At *= p[i].x;
        }
        const long long slot = (t.tile * t.chains + t.chain) * SCAN_CH + lane;
        const bool more = (t.tile + 1) * C < len;               // a tile behind this one will look back
        if (more) publish(w.piece + slot, At, Bt);
        const long long line = t.chains * SCAN_CH, row = (t.tile / SCAN_GROUP) * line + t.chain * SCAN_CH + lane;
        float h = look_back(w, t.tile, a.state && cc < a.H ? a.state[(long long)t.b * a.H + cc] : 0.f, slot, line, row, line);
        if (!more && a.final_state && cc < a.H) a.final_state[(long long)t.b * a.H + cc] = fmaf(At, h, Bt);
#pragma unroll
        for (int i = 0; i < TG; ++i) {
            ((float*)s_in[i])[lane] = h;
            h = fmaf(p[i].x, h, p[i].y);
        }
    }
    __syncthreads();
    if (here <= 0) return;
    const f32v4 hin = s_in[tg][threadIdx.x & 15];
    float h[4] = {hin[0], hin[1], hin[2], hin[3]};
    if (a.tape && s0 < len && s0 % T2_SCAN_SPAN == 0) {
        float* q = a.tape + ((long long)t.b * ((a.T + T2_SCAN_SPAN - 1) / T2_SCAN_SPAN) + s0 / T2_SCAN_SPAN) * a.H + c;
        for (int j = 0; j < nc; ++j) q[j] = h[j];
    }
    const long long dt = a.reverse ? -a.y.stride_t : a.y.stride_t;
    long long at = (long long)t.b * a.y.stride_b + c + (long long)(a.reverse ? len - 1 - s0 : s0) * a.y.stride_t;
#pragma unroll
    for (int l = 0; l < L; ++l, at += dt) {
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = fmaf(ga[l][j], h[j], x[l][j]);
            y[j] = GATE ? h[j] * sigmoid1(E::at(orr[l], j)) : h[j];
        }
        if (s0 + l < len) store4<E, VEC>((void*)a.y.ptr, at, nc, y[0], y[1], y[2], y[3]);
    }
    if (s0 + L > len) zero_rows<E, VEC, L>(a.y, t.b, c, nc, s0, len, a.T);
}

// Backward: l_t = the gradient that leaves step t for the state in front of it obeys l_t = a_t (l_{t+1} + g_t), g = dy sigmoid(o), the same
// recurrence from the other end; tiles are drawn from the last to the first and look back at the tiles behind them.  The states inside
// the tile come from the tape's, which needs no other tile.
template <typename E, bool GATE, bool VEC, int TG, int L>
__global__ __launch_bounds__(16 * TG) void scan_tile_backward_kernel(t2_scan_args a, ScanWs w, int ntile) {
    constexpr int C = TG * L;
    static_assert(C % T2_SCAN_SPAN == 0 && T2_SCAN_SPAN % L == 0, "tiles start where the tape has a state");
    __shared__ float2 s_fwd[TG][SCAN_CH], s_bwd[TG][SCAN_CH];
    __shared__ f32v4 s_h[TG][SCAN_CH / 4], s_l[TG][SCAN_CH / 4];
    const TileIds t = tile_ids<C>(a, w, ntile, true);
    const int len = t.len, tg = threadIdx.x >> 4, ch = (threadIdx.x & 15) * 4, s0 = t.tile * C + tg * L;
    const int here = a.H - (t.c0 + ch), c = here > 0 ? t.c0 + ch : (VEC ? a.H - 4 : a.H - 1), nc = here > 4 ? 4 : here > 0 ? here : 1;
    if (t.tile * C >= len && t.tile > 0) {
        if (here > 0) {
            zero_rows<E, VEC, L>(a.dz, t.b, c, nc, s0, len, a.T);
            zero_rows<E, VEC, L>(a.df, t.b, c, nc, s0, len, a.T);
            if (GATE) zero_rows<E, VEC, L>(a.do_, t.b, c, nc, s0, len, a.T);
        }
        return;
    }
    typename E::Raw zr[L], fr[L], orr[L], dr[L];
    load_rows<E, VEC, L>(fr, a.f, t.b, c, nc, s0, len, a.reverse);
    load_rows<E, VEC, L>(zr, a.z, t.b, c, nc, s0, len, a.reverse);
    load_rows<E, VEC, L>(dr, a.dy, t.b, c, nc, s0, len, a.reverse);
    if (GATE) load_rows<E, VEC, L>(orr, a.o, t.b, c, nc, s0, len, a.reverse);
    float ga[L][4], gb[L][4], g[L][4], gn[GATE ? L : 1][4];        // gn: g (1 - sigmoid(o)), do but for h
    float A[4] = {1.f, 1.f, 1.f, 1.f}, B[4] = {0.f, 0.f, 0.f, 0.f}, Q[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            gate(E::at(fr[l], j), ga[l][j], gb[l][j]);
            g[l][j] = E::at(dr[l], j);
            float z = E::at(zr[l], j);
            if (GATE) {
                float so, sn;
                gate(E::at(orr[l], j), so, sn);
                g[l][j] *= so;
                gn[l][j] = g[l][j] * sn;
            }
            if (s0 + l >= len) { ga[l][j] = 1.f; gb[l][j] = 0.f; g[l][j] = 0.f; z = 0.f; }
            B[j] = fmaf(ga[l][j], B[j], gb[l][j] * z);
            A[j] *= ga[l][j];
        }
#pragma unroll
    for (int l = L - 1; l >= 0; --l)
#pragma unroll
        for (int j = 0; j < 4; ++j) Q[j] = ga[l][j] * (Q[j] + g[l][j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        s_fwd[tg][ch + j] = make_float2(A[j], B[j]);
        s_bwd[tg][ch + j] = make_float2(A[j], Q[j]);
    }
    __syncthreads();
    if (threadIdx.x < SCAN_CH) {                                   // one wave: the states, from the tape's
        const int lane = threadIdx.x, cc = t.c0 + lane, ntape = (a.T + T2_SCAN_SPAN - 1) / T2_SCAN_SPAN;
        const float* tape = a.tape + ((long long)t.b * ntape + t.tile * (C / T2_SCAN_SPAN)) * a.H + cc;
        float h = 0.f;
#pragma unroll
        for (int i = 0; i < TG; ++i) {
            const int j = i * L / T2_SCAN_SPAN;
            if (i * L % T2_SCAN_SPAN == 0) h = cc < a.H && t.tile * C + j * T2_SCAN_SPAN < len ? tape[(long long)j * a.H] : 0.f;
            ((float*)s_h[i])[lane] = h;
            h = fmaf(s_fwd[i][lane].x, h, s_fwd[i][lane].y);
        }
    } else if (threadIdx.x < 2 * SCAN_CH) {                        // another: the gradients that enter
        const int lane = threadIdx.x - SCAN_CH, cc = t.c0 + lane;
        float2 p[TG];
        float At = 1.f, Qt = 0.f;
#pragma unroll
        for (int i = TG - 1; i >= 0; --i) {
            p[i] = s_bwd[i][lane];
            Qt = fmaf(p[i].x, Qt, p[i].y);
            At *= p[i].x;
        }
        const long long slot = (t.tile * t.chains + t.chain) * SCAN_CH + lane;
        const int last = len > 0 ? (len - 1) / C : 0;              // the last tile that is not all padding
        if (t.tile > 0) publish(w.piece + slot, At, Qt);
        const long long line = t.chains * SCAN_CH, row = ((last - t.tile) / SCAN_GROUP) * line + t.chain * SCAN_CH + lane;
        float l = look_back(w, last - t.tile, a.dfinal && cc < a.H ? a.dfinal[(long long)t.b * a.H + cc] : 0.f, slot, -line, row, line);
        if (t.tile == 0 && a.dstate && cc < a.H) a.dstate[(long long)t.b * a.H + cc] = fmaf(At, l, Qt);
#pragma unroll
        for (int i = TG - 1; i >= 0; --i) {
            ((float*)s_l[i])[lane] = l;
            l = fmaf(p[i].x, l, p[i].y);
        }
    }
    __syncthreads();
    if (here <= 0) return;
    const f32v4 hin = s_h[tg][threadIdx.x & 15], lin = s_l[tg][threadIdx.x & 15];
    float h[4] = {hin[0], hin[1], hin[2], hin[3]}, d[4] = {lin[0], lin[1], lin[2], lin[3]};
    const long long t0 = a.reverse ? len - 1 - s0 : s0, sign = a.reverse ? -1 : 1;
    float wf[L][4];                                                // df but for the gradient of h
#pragma unroll
    for (int l = 0; l < L; ++l) {
        float o4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float z = E::at(zr[l], j);
            wf[l][j] = (h[j] - z) * (ga[l][j] * gb[l][j]);
            h[j] = fmaf(ga[l][j], h[j], gb[l][j] * z);
            if (GATE) o4[j] = gn[l][j] * h[j];
        }
        if (GATE && s0 + l < len)
            store4<E, VEC>((void*)a.do_.ptr, (long long)t.b * a.do_.stride_b + c + (t0 + sign * l) * a.do_.stride_t, nc, o4[0], o4[1], o4[2], o4[3]);
    }
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
        float z4[4], f4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            d[j] += g[l][j];
            z4[j] = gb[l][j] * d[j];
            f4[j] = wf[l][j] * d[j];
            d[j] *= ga[l][j];
        }
        if (s0 + l < len) {
            store4<E, VEC>((void*)a.dz.ptr, (long long)t.b * a.dz.stride_b + c + (t0 + sign * l) * a.dz.stride_t, nc, z4[0], z4[1], z4[2], z4[3]);
            store4<E, VEC>((void*)a.df.ptr, (long long)t.b * a.df.stride_b + c + (t0 + sign * l) * a.df.stride_t, nc, f4[0], f4[1], f4[2], f4[3]);
        }
    }
    if (s0 + L > len) {
        zero_rows<E, VEC, L>(a.dz, t.b, c, nc, s0, len, a.T);
        zero_rows<E, VEC, L>(a.df, t.b, c, nc, s0, len, a.T);
        if (GATE) zero_rows<E, VEC, L>(a.do_, t.b, c, nc, s0, len, a.T);
    }
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

// Steps of a tile (16 lanes x TG threads of L steps)
template <bool BACKWARD> static int tile_steps(int T) { return BACKWARD ? (T <= 64 ? 64 : T <= 256 ? 256 : 64) : (T <= 64 ? 64 : 256); }

static int64_t ws_bytes(int B, int T, int H, int steps) {
    const int64_t ntile = (T + steps - 1) / steps, chains = (int64_t)B * ((H + SCAN_CH - 1) / SCAN_CH);
    if (ntile * chains > 0x7FFFFFFF) return fail(T2_EINVAL, "[%d,%d,%d] is too large for one call", B, T, H);
    return ntile < 2 ? 0 : 16 + (ntile * 8 + (ntile + SCAN_GROUP - 1) / SCAN_GROUP * 4) * chains * SCAN_CH;
}

extern "C" int64_t t2_gated_scan_ws(int B, int T, int H) {
    if (!sizes_ok(B, T, H)) return fail(T2_EINVAL, "bad shape [%d,%d,%d]", B, T, H);
    const int64_t f = ws_bytes(B, T, H, tile_steps<false>(T)), g = ws_bytes(B, T, H, tile_steps<true>(T));
    return f < 0 || g < 0 ? T2_EINVAL : f > g ? f : g;
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
    if (ws < 0) return T2_EINVAL;
    if (a->ws_bytes < ws || (ws > 0 && (!a->ws || ((uintptr_t)a->ws & 15)))) return fail(T2_EINVAL, "workspace of %lld bytes, 16-byte aligned, needed", (long long)ws);
    return T2_OK;
}

// Vector accesses need whole groups of four channels and rows that start at a multiple of four elements' size.
static bool vectors(const t2_scan_args* a, const t2_seq* const* q, int n) {
    const int size = a->dtype == T2_F32 ? 4 : 2;
    if (a->H % 4 != 0) return false;
    for (int i = 0; i < n; ++i)
        if (q[i]->ptr && ((uintptr_t)q[i]->ptr % (4 * size) != 0 || q[i]->stride_b % 4 != 0 || q[i]->stride_t % 4 != 0)) return false;
    return true;
}

template <typename E, bool GATE, bool VEC, bool BACKWARD, int TG, int L>
static int launch_tiles(t2_ctx* ctx, const t2_scan_args* a) {
    const int ntile = (a->T + TG * L - 1) / (TG * L);
    const int64_t blocks = (int64_t)ntile * a->B * ((a->H + SCAN_CH - 1) / SCAN_CH);
    ScanWs w = {};
    if (ntile > 1) {
        w = scan_ws(a->ws, blocks * SCAN_CH);
        const long long n16 = ws_bytes(a->B, a->T, a->H, TG * L) / 16, nb = (n16 + 1023) / 1024;
        hipLaunchKernelGGL(scan_ws_kernel, dim3((unsigned)(nb < 2048 ? nb : 2048)), dim3(256), 0, ctx->stream, (uint4*)a->ws, n16);
    }
    if constexpr (BACKWARD) hipLaunchKernelGGL((scan_tile_backward_kernel<E, GATE, VEC, TG, L>), dim3((unsigned)blocks), dim3(16 * TG), 0, ctx->stream, *a, w, ntile);
    else hipLaunchKernelGGL((scan_tile_kernel<E, GATE, VEC, TG, L>), dim3((unsigned)blocks), dim3(16 * TG), 0, ctx->stream, *a, w, ntile);
    HIP_TRY(hipGetLastError());
    return T2_OK;
}

template <typename E, bool GATE, bool VEC, bool BACKWARD>
static int launch(t2_ctx* ctx, const t2_scan_args* a) {
    const int steps = tile_steps<BACKWARD>(a->T);
    if constexpr (BACKWARD) return steps == 64 ? launch_tiles<E, GATE, VEC, true, 16, 4>(ctx, a) : launch_tiles<E, GATE, VEC, true, 64, 4>(ctx, a);
    else return steps == 64 ? launch_tiles<E, GATE, VEC, false, 8, 8>(ctx, a) : launch_tiles<E, GATE, VEC, false, 32, 8>(ctx, a);
}

template <bool BACKWARD>
static int launch_any(t2_ctx* ctx, const t2_scan_args* a, bool vec) {
    DeviceScope dev(ctx->device);
    HIP_TRY(dev.err);
    const bool gated = a->o.ptr != nullptr;
#define SCAN_CASE(E) (gated ? vec ? launch<E, true, true, BACKWARD>(ctx, a) : launch<E, true, false, BACKWARD>(ctx, a)                     \
                            : vec ? launch<E, false, true, BACKWARD>(ctx, a) : launch<E, false, false, BACKWARD>(ctx, a))
    return a->dtype == T2_F32 ? SCAN_CASE(ElemF32) : a->dtype == T2_BF16 ? SCAN_CASE(ElemBF16) : SCAN_CASE(ElemF16);
#undef SCAN_CASE
}

extern "C" int t2_gated_scan(t2_ctx* ctx, const t2_scan_args* a) {
    T2_TRY(check_args(ctx, a, false));
    const t2_seq* q[] = {&a->z, &a->f, &a->o, &a->y};
    return launch_any<false>(ctx, a, vectors(a, q, 4));
}

extern "C" int t2_gated_scan_backward(t2_ctx* ctx, const t2_scan_args* a) {
    T2_TRY(check_args(ctx, a, true));
    const t2_seq* q[] = {&a->z, &a->f, &a->o, &a->dy, &a->dz, &a->df, &a->do_};
    return launch_any<true>(ctx, a, vectors(a, q, 7));
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
