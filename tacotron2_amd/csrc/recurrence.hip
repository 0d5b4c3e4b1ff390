// Gated linear recurrence: a = sigmoid(f), h' = a h + (1 - a) z, y = sigmoid(o) h', forward, backward and for one position.
#include "ctx.h"
#include "elem.h"

// Sums are fused where fmaf says so and nowhere else: every instance of a kernel rounds alike, whatever the layout it is for.
#pragma clang fp contract(off)

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
// A sequence is cut into tiles of C = TG * L steps by 4 LANES channels, one workgroup each.  A thread holds L consecutive steps of 4
// channels in registers (LANES threads read neighbouring channels of a row: 128 bytes and more), so every input is read once and
// every output written once: the memory rate bounds it, at T = 65536 the forward pass takes 4.9 TB/s (220 us, a copy's 211), and
// arithmetic takes 40 % of that time.  Inside a tile: each thread composes its steps into h' = A h + B; the first waves compose the
// TG pieces of every channel, find the state in front of the tile, and hand every thread the state in front of its steps.
//
// Across tiles: a tile publishes its composition; the state in front of it is that in front of its group of SCAN_GROUP tiles, taken
// through the compositions in between in their order; the first tile of a group finds it through the whole group before and
// publishes it.  The order of every sum is fixed, so results do not depend on timing, and only one hand-over in SCAN_GROUP
// has to wait for another (16 tiles a group: more registers, 5 to 20 us more at T = 32769 and 65536).  Every word is a value that
// carries its own validity (all ones: not there yet; a computed NaN is never that pattern), so one relaxed agent-scope access hands
// it over, without flags or fences.  A workgroup's chain (row and channels) is
// its index's, its tile is drawn from the chain's counter as it starts: it waits only for workgroups of the chain that have started
// before it and that wait for none behind them, so every wait ends.  A wave that was off the machine all the same (a GPU shared
// between processes) waits no longer than the context's limit: it then composes the tiles before it once more from their inputs, with the
// same operations in the same order, so the limit never changes a bit of a result (the last tile of T = 65536: 32 ms, backward 61).  Every chain's
// counter has a line of its own: additions to one address take 10 ns each.
// ------------------------------------------------------------------------------------------------
#define SCAN_GROUP 8

struct ScanWs {                        // counters [chains][16] | compositions [ntile][chains][CH] | states in front of the groups [ngroup][chains][CH]
    unsigned* next;
    unsigned long long* piece;
    unsigned* state;
    unsigned long long ticks;          // of the 100 MHz clock that a wait may take; 0: nothing is waited for
};
static inline ScanWs scan_ws(void* p, long long chains, long long slots) {
    ScanWs w;
    w.next = (unsigned*)p;
    w.piece = (unsigned long long*)((char*)p + chains * 64);
    w.state = (unsigned*)(w.piece + slots);
    return w;
}

__global__ __launch_bounds__(256) void scan_ws_kernel(uint4* ws, long long zeros, long long n16) {
    const uint4 ones = {~0u, ~0u, ~0u, ~0u}, zero = {0u, 0u, 0u, 0u};
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n16; i += (long long)gridDim.x * 256) ws[i] = i < zeros ? zero : ones;
}

__device__ __forceinline__ unsigned valid_bits(float v) { return v != v ? 0x7FC00000u : __builtin_bit_cast(unsigned, v); }
__device__ __forceinline__ void publish(unsigned long long* p, float A, float B) {
    __hip_atomic_store(p, ((unsigned long long)valid_bits(B) << 32) | valid_bits(A), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish(unsigned* p, float v) { __hip_atomic_store(p, valid_bits(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The value that enters the i-th tile of a chain (i = 0: `first`), for one channel a lane.  slot: the tile's place among the
// compositions (of the workgroup: the same for all lanes); hop: from one tile of the chain to the next; row: the group's place among
// the states, row_hop: to the group before; again(): the same value without the other workgroups.
template <typename Again>
__device__ __forceinline__ float look_back(const ScanWs& w, int i, float first, unsigned lane, long long slot, long long hop, long long row, long long row_hop, Again again) {
    if (i == 0) return first;
    const bool head = i % SCAN_GROUP == 0;             // the first tile of a group folds the whole group before it
    const int m = head ? SCAN_GROUP : i % SCAN_GROUP, group = i / SCAN_GROUP - (head ? 1 : 0);
    const unsigned* start = w.state + (head ? row - row_hop : row);
    const unsigned long long* from = w.piece + (slot - hop * m);
    const unsigned long long t0 = __builtin_amdgcn_s_memrealtime();
    unsigned st = 0;
    unsigned long long pc[SCAN_GROUP];
    bool all = false, late = false;                    // late: one more look at everything, then no more
    while (w.ticks > 0) {
        // all of it at once, each address a scalar base and the lane
        if (group > 0) st = __hip_atomic_load(start + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int k = 0; k < SCAN_GROUP; ++k) {
            const unsigned long long* at = from + hop * (k < m ? k : m - 1);
            asm("" : "+s"(at));
            pc[k] = __hip_atomic_load(at + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        bool there = st != ~0u;
#pragma unroll
        for (int k = 0; k < SCAN_GROUP; ++k) there = there && pc[k] != ~0ull;
        all = __all(there);
        if (all || late) break;
        // not yet: wait for the tile before, then for the state, one word a lane at a time (waves that wait would otherwise read as
        // much as waves that work)
        const unsigned long long* before = w.piece + (slot - hop);
        bool wait = true;
        while (wait && !late) {
            __builtin_amdgcn_s_sleep(1);
            const unsigned long long v = __hip_atomic_load(before + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            wait = !__all(v != ~0ull);
            if (!wait && group > 0) wait = !__all(__hip_atomic_load(start + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != ~0u);
            late = __builtin_amdgcn_s_memrealtime() - t0 > w.ticks;
        }
    }
    float h = group > 0 ? __builtin_bit_cast(float, st) : first;
    if (all) {
#pragma unroll
        for (int k = 0; k < SCAN_GROUP; ++k)
            if (k < m) h = fmaf(__builtin_bit_cast(float, (unsigned)pc[k]), h, __builtin_bit_cast(float, (unsigned)(pc[k] >> 32)));
    } else {
        h = again();
    }
    if (head) publish(w.state + row + lane, h);
    return h;
}

// the next tile of a chain (the first where there is but one)
__device__ __forceinline__ int draw_tile(const ScanWs& w, unsigned chain, int ntile) {
    __shared__ unsigned s_tile;
    if (ntile < 2) return 0;
    if (threadIdx.x == 0) s_tile = atomicAdd(w.next + (size_t)chain * 16, 1u);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane((int)s_tile);
}

// zeros at the positions of the tile that lie behind the row's length
template <typename E, bool BUF, int L, int C>
__device__ __forceinline__ void zero_rows(const t2_seq& q, int b, int first, int tg, int c, int nc, bool on, int len, int T) {
    const int rows = T - first < C ? T - first : C;
    const SeqRows<E, BUF> r(q, b, first, rows, len, false);
#pragma unroll
    for (int l = 0; l < L; ++l) {
        const int i = tg * L + l;
        r.template store<false>(i, c, nc, on && first + i >= len && i < rows, 0.f, 0.f, 0.f, 0.f);
    }
}

// The channels of a thread: four from c on.  BUF: the last four of the row for threads beyond its end (they repeat another thread's
// work; `mine`: whether any of them is this thread's to write).  Otherwise nc of them are there.
struct Channels { int c, nc; bool mine; };
template <bool BUF>
__device__ __forceinline__ Channels channels(int c, int H) {
    Channels r;
    r.mine = c < H;
    r.c = BUF ? (c < H - 4 ? c : H - 4) : c;
    r.nc = BUF ? 4 : c >= H ? 0 : H - c < 4 ? H - c : 4;
    return r;
}
// the channel behind slot `lane` of the tile's channels, or -1
template <bool BUF>
__device__ __forceinline__ int channel_of(int c0, unsigned lane_, int H) {
    const int lane = (int)lane_;
    if (BUF) { const int c = c0 + (lane & ~3); return (c < H - 4 ? c : H - 4) + (lane & 3); }
    return c0 + lane < H ? c0 + lane : -1;
}

// A workgroup's place: its row, channels and length, and each thread's channels and first step in a tile.
template <bool BUF, int LANES, int L>
struct Place {
    int b, c0, len, tg, i0;
    Channels me;
    __device__ __forceinline__ Place(const t2_scan_args& a, unsigned chain) {
        const unsigned ncb = (a.H + 4 * LANES - 1) / (4 * LANES);
        b = (int)(chain / ncb);
        c0 = (int)(chain - (unsigned)b * ncb) * 4 * LANES;
        len = row_length(a.lens, b, a.T);
        tg = threadIdx.x / LANES;
        i0 = tg * L;
        me = channels<BUF>(c0 + (threadIdx.x % LANES) * 4, a.H);
    }
    // the steps of the tile from step `first` on that are there (at most C)
    __device__ __forceinline__ int rows(int first, int C) const { return len - first < C ? len - first : C; }
    template <typename E>
    __device__ __forceinline__ void load(typename E::Raw* r, const t2_seq& q, int first, int rows, bool reverse) const {
        const SeqRows<E, BUF> s(q, b, first, rows, len, reverse);
#pragma unroll
        for (int l = 0; l < L; ++l) r[l] = s.load(i0 + l, me.c, me.nc, i0 + l < rows);
    }
    template <typename E, int C>
    __device__ __forceinline__ void zeros(const t2_seq& q, int first, int T) const { zero_rows<E, BUF, L, C>(q, b, first, tg, me.c, me.nc, me.mine, len, T); }
};

// Workgroups of neighbouring channels on one XCD (workgroups go round the eight of them): lines that two tiles share are fetched once.
// Long sequences 4 % faster, rows that start inside a line 6 %.
__device__ __forceinline__ unsigned chain_of(unsigned index, unsigned chains) {
    const unsigned c = index % chains;
    return chains % 8 == 0 ? c % 8 * (chains / 8) + c / 8 : c;
}

// A product of gates in fp32 reaches zero where the gates do not, and zero times an infinite h would be NaN: the smallest number instead
// keeps h infinite, as every single step does, and is nothing beside any other h.
__device__ __forceinline__ float product(float A) { return fmaxf(A, 0x1p-149f); }

// the composition of all TG pieces of a channel, in the order of the steps or against it
template <int TG, int CH, bool BACK>
__device__ __forceinline__ void compose(const float2 (*piece)[CH], unsigned lane, float& A, float& B) {
    A = 1.f; B = 0.f;
#pragma unroll
    for (int k = 0; k < TG; ++k) {
        const float2 p = piece[BACK ? TG - 1 - k : k][lane];
        B = fmaf(p.x, B, p.y);
        A *= p.x;
    }
    A = product(A);
    asm volatile("" ::: "memory");                         // distribute() reads the pieces again: 2 TG registers otherwise
}
// v, which enters the tile, taken through the pieces: what enters each of them goes to `in`; returns what leaves
template <int TG, int CH, bool BACK>
__device__ __forceinline__ float distribute(const float2 (*piece)[CH], f32v4 (*in)[CH / 4], unsigned lane, float v) {
#pragma unroll
    for (int k = 0; k < TG; ++k) {
        const int i = BACK ? TG - 1 - k : k;
        const float2 p = piece[i][lane];
        ((float*)in[i])[lane] = v;
        v = fmaf(p.x, v, p.y);
    }
    return v;
}

// ---- forward: what a thread does with its L steps of a tile ----
template <typename E, int L> struct Inputs { typename E::Raw z[L], f[L]; };
template <int L> struct Steps { float a[L][4], x[L][4]; };          // h' = a h + x

template <typename E, int L>
__device__ __forceinline__ void steps_of(const Inputs<E, L>& in, int i0, int rows, int C, Steps<L>& s, float2 (&piece)[4]) {
    float A[4] = {1.f, 1.f, 1.f, 1.f}, B[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float b;
            gate(E::at(in.f[l], j), s.a[l][j], b);
            s.x[l][j] = b * E::at(in.z[l], j);
        }
    if (rows < C) {                                          // padding: h stays
#pragma unroll
        for (int l = 0; l < L; ++l)
#pragma unroll
            for (int j = 0; j < 4; ++j) if (i0 + l >= rows) { s.a[l][j] = 1.f; s.x[l][j] = 0.f; }
    }
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            B[j] = fmaf(s.a[l][j], B[j], s.x[l][j]);
            A[j] *= s.a[l][j];
        }
#pragma unroll
    for (int j = 0; j < 4; ++j) piece[j] = make_float2(product(A[j]), B[j]);
}

// The kernel's arguments out of their memory, for code that hardly ever runs: nothing of it is held in scalar registers before.
typedef const __attribute__((address_space(4))) t2_scan_args* ArgsAgain;
__device__ __forceinline__ ArgsAgain args_again() {
    ArgsAgain a = (ArgsAgain)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return a;
}

// The state in front of the tile `tile` of channel cc: the pieces and compositions of the tiles before it, as those tiles make them.
template <typename E, int TG, int L>
__device__ __forceinline__ float states_again(int b, int len, int cc, int tile, float h) {
    if (cc < 0) return h;
    const ArgsAgain a = args_again();
    const long long zs = a->reverse ? -a->z.stride_t : a->z.stride_t, fs = a->reverse ? -a->f.stride_t : a->f.stride_t;
    long long z = b * a->z.stride_b + cc + (a->reverse ? len - 1 : 0) * a->z.stride_t, f = b * a->f.stride_b + cc + (a->reverse ? len - 1 : 0) * a->f.stride_t;
#pragma unroll 1
    for (int t = 0; t < tile; ++t) {
        float At = 1.f, Bt = 0.f;
#pragma unroll 1
        for (int k = 0; k < TG; ++k) {
            float A = 1.f, B = 0.f;
#pragma unroll 1
            for (int l = 0; l < L; ++l, z += zs, f += fs) {
                float g, x;
                gate(E::get(a->f.ptr, f), g, x);
                x = x * E::get(a->z.ptr, z);
                B = fmaf(g, B, x);
                A *= g;
            }
            A = product(A);
            Bt = fmaf(A, Bt, B);
            At *= A;
        }
        h = fmaf(product(At), h, Bt);
    }
    return h;
}

template <typename E, bool GATE, bool BUF, bool NT, int LANES, int L, int C>
__device__ __forceinline__ void finish(const t2_scan_args& a, const Place<BUF, LANES, L>& t, int first, int rows, const Steps<L>& s, const typename E::Raw* o, f32v4 hin) {
    float h[4] = {hin[0], hin[1], hin[2], hin[3]};
    const int s0 = first + t.i0;
    if (a.tape && t.i0 < rows && s0 % T2_SCAN_SPAN == 0 && t.me.mine) {
        float* q = a.tape + ((long long)t.b * ((a.T + T2_SCAN_SPAN - 1) / T2_SCAN_SPAN) + s0 / T2_SCAN_SPAN) * a.H + t.me.c;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (j < t.me.nc) q[j] = h[j];
    }
    const SeqRows<E, BUF> out(a.y, t.b, first, rows, t.len, a.reverse);
#pragma unroll
    for (int l = 0; l < L; ++l) {
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = fmaf(s.a[l][j], h[j], s.x[l][j]);
            y[j] = GATE ? h[j] * sigmoid1(E::at(o[l], j)) : h[j];
        }
        out.template store<NT>(t.i0 + l, t.me.c, t.me.nc, t.i0 + l < rows && t.me.mine, y[0], y[1], y[2], y[3]);
    }
    if (rows < C) t.template zeros<E, C>(a.y, first, a.T);
}

template <typename E, bool GATE, bool BUF, bool NT, int LANES, int TG, int L, int WAVES>
__global__ __launch_bounds__(LANES* TG, WAVES) void scan_tile_kernel(t2_scan_args a, ScanWs w, int ntile) {
    constexpr int C = TG * L, CH = 4 * LANES;
    __shared__ float2 s_piece[TG][CH];
    __shared__ f32v4 s_in[TG][LANES];
    const unsigned chains = gridDim.x / (unsigned)ntile, chain = chain_of(blockIdx.x, chains);
    const Place<BUF, LANES, L> t(a, chain);
    const int tile = draw_tile(w, chain, ntile), first = tile * C;
    if (first >= t.len && tile > 0) { t.template zeros<E, C>(a.y, first, a.T); return; }
    const int rows = t.rows(first, C);
    Inputs<E, L> in;
    typename E::Raw o[L];
    t.template load<E>(in.f, a.f, first, rows, a.reverse);
    t.template load<E>(in.z, a.z, first, rows, a.reverse);
    if (GATE) t.template load<E>(o, a.o, first, rows, a.reverse);
    Steps<L> s;
    float2 piece[4];
    steps_of<E, L>(in, t.i0, rows, C, s, piece);
#pragma unroll
    for (int j = 0; j < 4; ++j) s_piece[t.tg][(threadIdx.x % LANES) * 4 + j] = piece[j];
    __syncthreads();
    if (threadIdx.x < CH) {
        const unsigned lane = threadIdx.x;
        const int cc = channel_of<BUF>(t.c0, lane, a.H);
        float At, Bt;
        compose<TG, CH, false>(s_piece, lane, At, Bt);
        const long long line = (long long)chains * CH, place = (long long)chain * CH, slot = tile * line + place;
        const bool more = first + C < t.len;                     // a tile behind this one will look back
        if (more) publish(w.piece + slot + lane, At, Bt);
        const float h0 = a.state && cc >= 0 ? a.state[(long long)t.b * a.H + cc] : 0.f;
        const float h = look_back(w, tile, h0, lane, slot, line, tile / SCAN_GROUP * line + place, line,
                                  [&] { return states_again<E, TG, L>(t.b, t.len, cc, tile, h0); });
        if (!more && a.final_state && cc >= 0) a.final_state[(long long)t.b * a.H + cc] = fmaf(At, h, Bt);
        distribute<TG, CH, false>(s_piece, s_in, lane, h);
    }
    __syncthreads();
    finish<E, GATE, BUF, NT, LANES, L, C>(a, t, first, rows, s, o, s_in[t.tg][threadIdx.x % LANES]);
}

// ---- backward ----
// l_t, the gradient that leaves step t for the state in front of it, obeys l_t = a_t (l_{t+1} + g_t), g = dy sigmoid(o): the same
// recurrence from the other end; tiles are drawn from the last to the first and look back at the tiles behind them.  The states
// inside a tile come from the tape's, which needs no other tile.
template <typename E, int L> struct Grads { typename E::Raw z[L], f[L], o[L], d[L]; };
template <int L> struct BackSteps { float a[L][4], b[L][4]; };

template <typename E, bool GATE, int L>
__device__ __forceinline__ void back_steps_of(const Grads<E, L>& in, int i0, int rows, int C, BackSteps<L>& s, float2 (&fwd)[4], float2 (&bwd)[4]) {
    float A[4] = {1.f, 1.f, 1.f, 1.f}, B[4] = {0.f, 0.f, 0.f, 0.f}, Q[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
        for (int j = 0; j < 4; ++j) gate(E::at(in.f[l], j), s.a[l][j], s.b[l][j]);
    if (rows < C) {
#pragma unroll
        for (int l = 0; l < L; ++l)
#pragma unroll
            for (int j = 0; j < 4; ++j) if (i0 + l >= rows) { s.a[l][j] = 1.f; s.b[l][j] = 0.f; }
    }
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            B[j] = fmaf(s.a[l][j], B[j], s.b[l][j] * E::at(in.z[l], j));
            A[j] *= s.a[l][j];
        }
#pragma unroll
    for (int l = L - 1; l >= 0; --l)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float dy = E::at(in.d[l], j);                    // rows that are not there were read as zeros
            Q[j] = s.a[l][j] * (GATE ? fmaf(dy, sigmoid1(E::at(in.o[l], j)), Q[j]) : Q[j] + dy);
        }
#pragma unroll
    for (int j = 0; j < 4; ++j) { fwd[j] = make_float2(product(A[j]), B[j]); bwd[j] = make_float2(fwd[j].x, Q[j]); }
}

// The gradient that enters the tile `tile` of channel cc from behind, out of the tiles behind it (the last of them may end early).
template <typename E, bool GATE, int TG, int L>
__device__ __forceinline__ float gradients_again(int b, int len, int cc, int last, int tile, float v) {
    if (cc < 0) return v;
    const ArgsAgain a = args_again();
    const bool reverse = a->reverse;
    auto place = [&](auto& q, int s) { return b * q.stride_b + (reverse ? len - 1 - s : s) * q.stride_t + cc; };
#pragma unroll 1
    for (int t = last; t > tile; --t) {
        float At = 1.f, Qt = 0.f;
#pragma unroll 1
        for (int k = TG - 1; k >= 0; --k) {
            const int first = (t * TG + k) * L, rows = len - first < L ? len - first : L;
            float A = 1.f, Q = 0.f;
#pragma unroll 1
            for (int l = 0; l < rows; ++l) {
                float g, x;
                gate(E::get(a->f.ptr, place(a->f, first + l)), g, x);
                A *= g;
            }
#pragma unroll 1
            for (int l = rows - 1; l >= 0; --l) {
                float g, x;
                gate(E::get(a->f.ptr, place(a->f, first + l)), g, x);
                const float dy = E::get(a->dy.ptr, place(a->dy, first + l));
                Q = g * (GATE ? fmaf(dy, sigmoid1(E::get(a->o.ptr, place(a->o, first + l))), Q) : Q + dy);
            }
            A = product(A);
            Qt = fmaf(A, Qt, Q);
            At *= A;
        }
        v = fmaf(product(At), v, Qt);
    }
    return v;
}

// the states in front of the pieces, from the tape's
__device__ __forceinline__ float tape_state(const t2_scan_args& a, int b, int first, int rows, int cc, int k) {
    const int ntape = (a.T + T2_SCAN_SPAN - 1) / T2_SCAN_SPAN;
    return cc >= 0 && k * T2_SCAN_SPAN < rows ? a.tape[((long long)b * ntape + first / T2_SCAN_SPAN + k) * a.H + cc] : 0.f;
}
template <int TG, int L, int CH>
__device__ __forceinline__ void distribute_states(const t2_scan_args& a, int b, int first, int rows, int cc, const float2 (*piece)[CH], f32v4 (*in)[CH / 4], unsigned lane) {
    float h = 0.f;
#pragma unroll
    for (int i = 0; i < TG; ++i) {
        if (i * L % T2_SCAN_SPAN == 0) h = tape_state(a, b, first, rows, cc, i * L / T2_SCAN_SPAN);
        const float2 p = piece[i][lane];
        ((float*)in[i])[lane] = h;
        h = fmaf(p.x, h, p.y);
    }
}

// Returns the gradient that leaves the thread's first step for the state in front of it.
template <typename E, bool GATE, bool BUF, bool NT, int LANES, int L, int C>
__device__ __forceinline__ f32v4 back_finish(const t2_scan_args& a, const Place<BUF, LANES, L>& t, int first, int rows, const BackSteps<L>& s, const typename E::Raw* zr,
                                            const typename E::Raw* orr, const typename E::Raw* dr, f32v4 hin, f32v4 lin) {
    float h[4] = {hin[0], hin[1], hin[2], hin[3]}, d[4] = {lin[0], lin[1], lin[2], lin[3]};
    float wf[L][4], g[L][4];                                       // wf: df but for the gradient of h
    const SeqRows<E, BUF> dz(a.dz, t.b, first, rows, t.len, a.reverse), df(a.df, t.b, first, rows, t.len, a.reverse);
    const SeqRows<E, BUF> dout(GATE ? a.do_ : a.dz, t.b, first, rows, t.len, a.reverse);
#pragma unroll
    for (int l = 0; l < L; ++l) {
        float o4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float z = E::at(zr[l], j);
            wf[l][j] = (h[j] - z) * (s.a[l][j] * s.b[l][j]);
            h[j] = fmaf(s.a[l][j], h[j], s.b[l][j] * z);
            g[l][j] = E::at(dr[l], j);
            if (GATE) {                                            // again: 2 L registers to keep it cost more (odd: 285 us, 273 so)
                float so, sn;
                gate(E::at(orr[l], j), so, sn);
                g[l][j] *= so;
                o4[j] = g[l][j] * sn * h[j];
            }
        }
        if (GATE) dout.template store<NT>(t.i0 + l, t.me.c, t.me.nc, t.i0 + l < rows && t.me.mine, o4[0], o4[1], o4[2], o4[3]);
    }
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
        float z4[4], f4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            d[j] += g[l][j];
            z4[j] = s.b[l][j] * d[j];
            f4[j] = wf[l][j] * d[j];
            d[j] *= s.a[l][j];
        }
        dz.template store<NT>(t.i0 + l, t.me.c, t.me.nc, t.i0 + l < rows && t.me.mine, z4[0], z4[1], z4[2], z4[3]);
        df.template store<NT>(t.i0 + l, t.me.c, t.me.nc, t.i0 + l < rows && t.me.mine, f4[0], f4[1], f4[2], f4[3]);
    }
    return f32v4{d[0], d[1], d[2], d[3]};
}

template <typename E, bool GATE, bool BUF, int LANES, int L, int C>
__device__ __forceinline__ void back_zeros(const t2_scan_args& a, const Place<BUF, LANES, L>& t, int first) {
    t.template zeros<E, C>(a.dz, first, a.T);
    t.template zeros<E, C>(a.df, first, a.T);
    if (GATE) t.template zeros<E, C>(a.do_, first, a.T);
}

// ONE: a sequence has one tile; nothing is drawn, published or looked back at, and the registers of that are free (B=64, T=250, H=2048 bf16:
// 137 us with it, 129 so).  The forward kernel loses by the same cut (62 to 126: the compiler spills).
template <typename E, bool GATE, bool BUF, bool NT, bool ONE, int LANES, int TG, int L, int WAVES>
__global__ __launch_bounds__(LANES* TG, WAVES) void scan_tile_backward_kernel(t2_scan_args a, ScanWs w, int ntile) {
    constexpr int C = TG * L, CH = 4 * LANES;
    static_assert(C % T2_SCAN_SPAN == 0 && T2_SCAN_SPAN % L == 0, "tiles start where the tape has a state");
    static_assert(TG >= 8, "two sets of waves, one for the states and one for the gradients");
    __shared__ float2 s_fwd[TG][CH], s_bwd[TG][CH];
    __shared__ f32v4 s_h[TG][LANES], s_l[TG][LANES];
    const unsigned chains = gridDim.x / (unsigned)ntile, chain = chain_of(blockIdx.x, chains);
    const Place<BUF, LANES, L> t(a, chain);
    const int tile = ONE ? 0 : ntile - 1 - draw_tile(w, chain, ntile), first = tile * C;
    if (first >= t.len && tile > 0) { back_zeros<E, GATE, BUF, LANES, L, C>(a, t, first); return; }
    const int rows = t.rows(first, C);
    Grads<E, L> in;
    t.template load<E>(in.f, a.f, first, rows, a.reverse);
    if (GATE) t.template load<E>(in.o, a.o, first, rows, a.reverse);
    t.template load<E>(in.d, a.dy, first, rows, a.reverse);
    t.template load<E>(in.z, a.z, first, rows, a.reverse);
    BackSteps<L> s;
    float2 fwd[4], bwd[4];
    back_steps_of<E, GATE, L>(in, t.i0, rows, C, s, fwd, bwd);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = (threadIdx.x % LANES) * 4 + j;
        s_fwd[t.tg][k] = fwd[j];
        s_bwd[t.tg][k] = bwd[j];
    }
    __syncthreads();
    if (threadIdx.x < CH) {
        distribute_states<TG, L, CH>(a, t.b, first, rows, channel_of<BUF>(t.c0, threadIdx.x, a.H), s_fwd, s_h, threadIdx.x);
    } else if (threadIdx.x < 2 * CH) {
        const unsigned lane = threadIdx.x - CH;
        const int cc = channel_of<BUF>(t.c0, lane, a.H);
        const float l0 = a.dfinal && cc >= 0 ? a.dfinal[(long long)t.b * a.H + cc] : 0.f;
        float l = l0;
        if constexpr (!ONE) {
            float At, Qt;
            compose<TG, CH, true>(s_bwd, lane, At, Qt);
            const int last = t.len > 0 ? (t.len - 1) / C : 0, at = last - tile;     // the last tile that is not all padding comes first
            const long long line = (long long)chains * CH, place = (long long)chain * CH, slot = tile * line + place;
            if (tile > 0) publish(w.piece + slot + lane, At, Qt);
            l = look_back(w, at, l0, lane, slot, -line, at / SCAN_GROUP * line + place, line,
                          [&] { return gradients_again<E, GATE, TG, L>(t.b, t.len, cc, last, tile, l0); });
        }
        distribute<TG, CH, true>(s_bwd, s_l, lane, l);
    }
    __syncthreads();
    const f32v4 d = back_finish<E, GATE, BUF, NT, LANES, L, C>(a, t, first, rows, s, in.z, in.o, in.d, s_h[t.tg][threadIdx.x % LANES], s_l[t.tg][threadIdx.x % LANES]);
    // out of the steps themselves: where dfinal and dy cancel, the tile's composition has rounded its part already
    if (tile == 0 && t.tg == 0 && a.dstate && t.me.mine) {
        float* q = a.dstate + (long long)t.b * a.H + t.me.c;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (j < t.me.nc) q[j] = d[j];
    }
    if (rows < C) back_zeros<E, GATE, BUF, LANES, L, C>(a, t, first);
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
    const int64_t rows = (int64_t)B * ((T + T2_SCAN_SPAN - 1) / T2_SCAN_SPAN);
    if (rows > (INT64_MAX >> 3) / H) return fail(T2_EINVAL, "[%d,%d,%d] is too large", B, T, H);      // bytes of it are counted in 64 bits too
    return rows * H;
}

// The tile of a call, by its sizes (kernel times in us; frames: B=32, T=800, H=512 bf16; long: B=2, T=65536, H=1024 bf16; odd: B=2,
// T=32769, H=1001 fp16).  A sequence that one tile covers needs no workspace, no look back and one launch: tiles of 64 and of 256
// steps (B=32, T=140, H=256 fp32: a call of 14 us, 18.6 with two tiles); where 64 channels a workgroup would leave compute units
// idle, 32 (the same sizes: forward 7.6 -> 6.7, backward 10.0 -> 8.8; B=64, T=250, H=2048 bf16: 62 -> 64, 126 -> 132).  Otherwise
// 64 channels a tile, which gives more and smaller workgroups, and 128 (256 bytes of a 16-bit row) where there are enough of those
// for 12 and more on every compute unit: forward 20.4 narrow / 24.0 wide at frames, 241 / 225 at long, 148 / 141 at odd; backward
// 38.6 / 41.2 at frames, 271 / 262 at odd.  256 channels: 286 at long, 177 and 266 to 274 at odd.
// (One workgroup for all tiles of a row, the next tile's inputs in flight, needs no workspace either: at frames without lengths 24.5
// against 25.3 forward and 58 to 64 against 47 backward, elsewhere slower both ways; not taken.)
struct Tile {
    int lanes, tg, l;
    constexpr int steps() const { return tg * l; }
    constexpr int channels() const { return 4 * lanes; }
};
enum Shape { SHORT, MEDIUM, NARROW, WIDE, FEW };
static constexpr Tile forward_tile[] = {{16, 8, 8}, {16, 32, 8}, {16, 16, 8}, {32, 8, 16}, {8, 32, 8}};
static constexpr Tile backward_tile[] = {{16, 16, 4}, {16, 32, 8}, {16, 16, 4}, {32, 8, 8}, {8, 32, 8}};
static constexpr int forward_waves[] = {4, 4, 4, 2, 4}, backward_waves[] = {3, 2, 3, 2, 2};     // a SIMD: registers for the tile without spills (but for 24 to 32 bytes a thread of forward fp32 tiles with an output gate)

static Shape shape_of(bool backward, int B, int T, int H, bool buf) {
    const Tile* tiles = backward ? backward_tile : forward_tile;
    if (T <= tiles[SHORT].steps() && buf) return SHORT;
    if (T <= tiles[MEDIUM].steps()) return buf && (int64_t)B * ((H + 63) / 64) < 256 ? FEW : MEDIUM;
    if (!buf) return NARROW;
    const Tile& w = tiles[WIDE];
    const int64_t blocks = (int64_t)B * ((H + w.channels() - 1) / w.channels()) * ((T + w.steps() - 1) / w.steps());
    return blocks >= 12 * 256 ? WIDE : NARROW;
}

static int64_t ws_bytes(int B, int T, int H, Tile t) {
    const int64_t ntile = (T + t.steps() - 1) / t.steps(), chains = (int64_t)B * ((H + t.channels() - 1) / t.channels());
    if (ntile * chains > 0xFFFFFFFFLL / (t.lanes * t.tg)) return fail(T2_EINVAL, "[%d,%d,%d] is too large for one call", B, T, H);
    return ntile < 2 ? 0 : chains * 64 + (ntile * 8 + (ntile + SCAN_GROUP - 1) / SCAN_GROUP * 4) * chains * t.channels();
}

extern "C" int64_t t2_gated_scan_ws(int B, int T, int H) {
    if (!sizes_ok(B, T, H)) return fail(T2_EINVAL, "bad shape [%d,%d,%d]", B, T, H);
    int64_t most = 0;
    for (int backward = 0; backward < 2; ++backward)
        for (int buf = 0; buf < 2; ++buf) {
            const int64_t n = ws_bytes(B, T, H, (backward ? backward_tile : forward_tile)[shape_of(backward, B, T, H, buf)]);
            if (n < 0) return n;
            most = n > most ? n : most;
        }
    return most;
}

// The bytes of a tensor: rows of `row` bytes, n_hi by n_lo of them, hi and lo bytes from one to the next (hi >= lo, from the lowest on).
struct Places { int64_t at, hi, lo, n_hi, n_lo, row; };
static Places places(const void* ptr, int64_t stride_b, int64_t stride_t, int64_t B, int64_t T, int64_t row) {      // strides in bytes
    if (B == 1) stride_b = 0;
    if (T == 1) stride_t = 0;
    int64_t at = (int64_t)ptr;
    if (stride_b < 0) { at += stride_b * (B - 1); stride_b = -stride_b; }
    if (stride_t < 0) { at += stride_t * (T - 1); stride_t = -stride_t; }
    if (stride_b == 0) B = 1;                              // all in one place
    if (stride_t == 0) T = 1;
    return stride_b >= stride_t ? Places{at, stride_b, stride_t, B, T, row} : Places{at, stride_t, stride_b, T, B, row};
}
static Places block(const void* ptr, int64_t bytes) { return {(int64_t)ptr, 0, 0, 1, 1, bytes}; }
static int64_t length(const Places& p) { return p.hi * (p.n_hi - 1) + p.lo * (p.n_lo - 1) + p.row; }
// every run of n_lo rows ends before the next begins
static bool nested(const Places& p, int64_t row) { return p.n_hi == 1 || p.hi >= p.lo * (p.n_lo - 1) + row; }

// Whether a row of q meets the n bytes from x on: i hi + j lo lies in [from, to].  One run is looked up by a division; there are more than a
// few runs to look at only where those of q reach into each other (inputs that are windows of one signal).
static bool meets_block(int64_t x, int64_t n, const Places& q) {
    const int64_t from = x - q.row + 1 - q.at, to = x + n - 1 - q.at, run = q.lo * (q.n_lo - 1);
    if (to < 0) return false;
    const int64_t first = q.hi && from > run ? (from - run + q.hi - 1) / q.hi : 0, last = q.hi && to / q.hi < q.n_hi - 1 ? to / q.hi : q.n_hi - 1;
    for (int64_t i = first; i <= last; ++i) {
        const int64_t a = from - i * q.hi, j = a <= 0 ? 0 : q.lo ? (a + q.lo - 1) / q.lo : q.n_lo;
        if (j < q.n_lo && j * q.lo <= to - i * q.hi) return true;
    }
    return false;
}
static bool meet(const Places& p, const Places& q) {
    if (!p.at || !q.at || q.at >= p.at + length(p) || p.at >= q.at + length(q)) return false;
    if (p.hi == q.hi && p.lo == q.lo && p.n_hi == q.n_hi && p.n_lo == q.n_lo && nested(p, p.row > q.row ? p.row : q.row)) {
        // the same pattern: two rows kh and kl apart, one of the nine next to the quotients
        const int64_t d = q.at - p.at;
        for (int64_t i = -1; i <= 1; ++i)
            for (int64_t j = -1; j <= 1; ++j) {
                const int64_t kh = p.hi ? d / p.hi + i : 0, r = d - kh * p.hi, kl = p.lo ? r / p.lo + j : 0, e = r - kl * p.lo;
                if (kh > -p.n_hi && kh < p.n_hi && kl > -p.n_lo && kl < p.n_lo && e < p.row && e > -q.row) return true;
            }
        return false;
    }
    const bool fewer = p.n_hi * p.n_lo <= q.n_hi * q.n_lo;         // row by row of the one that has fewer
    const Places &s = fewer ? p : q, &m = fewer ? q : p;
    for (int64_t i = 0; i < s.n_hi; ++i)
        for (int64_t j = 0; j < s.n_lo; ++j)
            if (meets_block(s.at + i * s.hi + j * s.lo, s.row, m)) return true;
    return false;
}
// a tensor whose rows go round memory more than once is none
static bool reaches(const t2_seq& s, int B, int T) {
    const __int128 b = B > 1 ? s.stride_b : 0, t = T > 1 ? s.stride_t : 0;
    return (b < 0 ? -b : b) * (B - 1) + (t < 0 ? -t : t) * (T - 1) < (1LL << 52);
}
static bool meets_itself(const t2_seq& s, const Places& p, int B, int T) {
    return (B > 1 && s.stride_b == 0) || (T > 1 && s.stride_t == 0) || (p.n_lo > 1 && p.lo < p.row) || !nested(p, p.row);
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
    // what is written against what is read and what else is written; the tape is written by the forward call and read by the other
    const int64_t size = a->dtype == T2_F32 ? 4 : 2, row = a->H * size, states = (int64_t)a->B * a->H * 4;
    const t2_seq none = {nullptr, 0, 0}, seq_in[] = {a->z, a->f, a->o, backward ? a->dy : none};
    const t2_seq seq_out[] = {backward ? a->dz : a->y, backward ? a->df : none, backward && a->o.ptr ? a->do_ : none};
    Places in[7], out[6];
    int n_in = 0, n_out = 0;
    auto seq = [&](const t2_seq& s) { return places(s.ptr, s.stride_b * size, s.stride_t * size, a->B, a->T, row); };
    for (const t2_seq& s : seq_in) {
        if (!s.ptr) continue;
        if (!reaches(s, a->B, a->T)) return fail(T2_EINVAL, "strides of %lld and %lld elements", (long long)s.stride_b, (long long)s.stride_t);
        in[n_in++] = seq(s);
    }
    for (const t2_seq& s : seq_out) {
        if (!s.ptr) continue;
        if (!reaches(s, a->B, a->T)) return fail(T2_EINVAL, "strides of %lld and %lld elements", (long long)s.stride_b, (long long)s.stride_t);
        out[n_out++] = seq(s);
        if (meets_itself(s, out[n_out - 1], a->B, a->T)) return fail(T2_EINVAL, "the elements of an output overlap (strides %lld, %lld)", (long long)s.stride_b, (long long)s.stride_t);
    }
    const Places tape = block(a->tape, t2_gated_scan_tape(a->B, a->T, a->H) * 4);
    in[n_in++] = block(a->lens, (int64_t)a->B * 8);
    in[n_in++] = block(backward ? a->dfinal : a->state, states);
    if (backward) in[n_in++] = tape;
    else out[n_out++] = tape;
    out[n_out++] = block(backward ? a->dstate : a->final_state, states);
    if (ws > 0) out[n_out++] = block(a->ws, ws);
    for (int i = 0; i < n_out; ++i) {
        for (int j = 0; j < n_in; ++j) if (meet(out[i], in[j])) return fail(T2_EINVAL, "an output overlaps an input");
        for (int j = 0; j < i; ++j) if (meet(out[i], out[j])) return fail(T2_EINVAL, "two outputs overlap");
    }
    if (a->ws_bytes < ws || (ws > 0 && (!a->ws || ((uintptr_t)a->ws & 15)))) return fail(T2_EINVAL, "workspace of %lld bytes, 16-byte aligned, needed", (long long)ws);
    return T2_OK;
}

// Buffer descriptors and four channels at a time, but for rows of fewer channels and for strides whose tile leaves the range of an offset.
static bool buffers(const t2_scan_args* a, int steps, const t2_seq* const* q, int n) {
    const int64_t size = a->dtype == T2_F32 ? 4 : 2, most = SEQ_RANGE / size / (steps + 1);
    if (a->H < 4 || a->H > most) return false;
    for (int i = 0; i < n; ++i)
        if (q[i]->ptr && (q[i]->stride_t > most || q[i]->stride_t < -most)) return false;
    return true;
}

template <typename E, bool GATE, bool BUF, bool NT, bool BACKWARD, Shape S>
static int launch(t2_ctx* ctx, const t2_scan_args* a) {
    constexpr Tile tile = BACKWARD ? backward_tile[S] : forward_tile[S];
    constexpr int CH = tile.channels(), WAVES = BACKWARD ? backward_waves[S] : forward_waves[S];
    const int ntile = (a->T + tile.steps() - 1) / tile.steps();
    const int64_t blocks = (int64_t)ntile * a->B * ((a->H + CH - 1) / CH);
    ScanWs w = {};
    if (ntile > 1) {
        w = scan_ws(a->ws, blocks / ntile, blocks * CH);
        w.ticks = ctx->scan_wait_ticks;
        const long long n16 = ws_bytes(a->B, a->T, a->H, tile) / 16, nb = (n16 + 1023) / 1024;
        hipLaunchKernelGGL(scan_ws_kernel, dim3((unsigned)(nb < 2048 ? nb : 2048)), dim3(256), 0, ctx->stream, (uint4*)a->ws, blocks / ntile * 4, n16);
    }
    const dim3 grid((unsigned)blocks), threads(tile.lanes * tile.tg);
    if constexpr (BACKWARD) hipLaunchKernelGGL((scan_tile_backward_kernel<E, GATE, BUF, NT, S != NARROW && S != WIDE, tile.lanes, tile.tg, tile.l, WAVES>), grid, threads, 0, ctx->stream, *a, w, ntile);
    else hipLaunchKernelGGL((scan_tile_kernel<E, GATE, BUF, NT, tile.lanes, tile.tg, tile.l, WAVES>), grid, threads, 0, ctx->stream, *a, w, ntile);
    HIP_TRY(hipGetLastError());
    return T2_OK;
}

template <typename E, bool GATE, bool BACKWARD>
static int launch_shape(t2_ctx* ctx, const t2_scan_args* a, Shape s, bool buf, bool nt) {
    if (!buf) return s == MEDIUM ? launch<E, GATE, false, false, BACKWARD, MEDIUM>(ctx, a) : launch<E, GATE, false, false, BACKWARD, NARROW>(ctx, a);
    if (s == SHORT) return launch<E, GATE, true, false, BACKWARD, SHORT>(ctx, a);
    if (s == MEDIUM) return launch<E, GATE, true, false, BACKWARD, MEDIUM>(ctx, a);
    if (s == FEW) return launch<E, GATE, true, false, BACKWARD, FEW>(ctx, a);
    if (s == NARROW) return nt ? launch<E, GATE, true, true, BACKWARD, NARROW>(ctx, a) : launch<E, GATE, true, false, BACKWARD, NARROW>(ctx, a);
    return nt ? launch<E, GATE, true, true, BACKWARD, WIDE>(ctx, a) : launch<E, GATE, true, false, BACKWARD, WIDE>(ctx, a);
}

template <bool BACKWARD>
static int launch_any(t2_ctx* ctx, const t2_scan_args* a, const t2_seq* const* in, int n_in, const t2_seq* const* out, int n_out) {
    DeviceScope dev(ctx->device);
    HIP_TRY(dev.err);
    // a tile of every shape fits the range of its offsets, or none of this call uses them
    const Tile& most = (BACKWARD ? backward_tile : forward_tile)[MEDIUM];
    const bool buf = buffers(a, most.steps(), in, n_in) && buffers(a, most.steps(), out, n_out);
    const Shape s = shape_of(BACKWARD, a->B, a->T, a->H, buf);
    // Stores past L2 where they fill whole 128-byte lines (frames: forward 20.9 -> 19.7 us, backward 36.7 -> 32.8); rows that start
    // inside a line lose by it (odd: backward 290 -> 324).
    bool nt = true;
    const int64_t size = a->dtype == T2_F32 ? 4 : 2;
    for (int i = 0; i < n_out; ++i)
        if (out[i]->ptr && ((((uintptr_t)out[i]->ptr) | (uintptr_t)(out[i]->stride_b * size) | (uintptr_t)(out[i]->stride_t * size)) & 127)) nt = false;
    const bool gated = a->o.ptr != nullptr;
#define SCAN_CASE(E) (gated ? launch_shape<E, true, BACKWARD>(ctx, a, s, buf, nt) : launch_shape<E, false, BACKWARD>(ctx, a, s, buf, nt))
    return a->dtype == T2_F32 ? SCAN_CASE(ElemF32) : a->dtype == T2_BF16 ? SCAN_CASE(ElemBF16) : SCAN_CASE(ElemF16);
#undef SCAN_CASE
}

extern "C" int t2_gated_scan(t2_ctx* ctx, const t2_scan_args* a) {
    T2_TRY(check_args(ctx, a, false));
    const t2_seq *in[] = {&a->z, &a->f, &a->o}, *out[] = {&a->y};
    return launch_any<false>(ctx, a, in, 3, out, 1);
}

extern "C" int t2_gated_scan_backward(t2_ctx* ctx, const t2_scan_args* a) {
    T2_TRY(check_args(ctx, a, true));
    const t2_seq *in[] = {&a->z, &a->f, &a->o, &a->dy}, *out[] = {&a->dz, &a->df, &a->do_};
    return launch_any<true>(ctx, a, in, 4, out, a->o.ptr ? 3 : 2);
}

extern "C" int t2_gated_scan_step(t2_ctx* ctx, int dtype, int B, int H, const void* z, int64_t z_stride, const void* f, int64_t f_stride, const void* o,
                                  int64_t o_stride, float* state, int64_t state_stride, const uint8_t* active, void* y, int64_t y_stride) {
    if (!ctx || !z || !f || !state || !y) return fail(T2_EINVAL, "null argument");
    if (dtype < T2_F32 || dtype > T2_F16) return fail(T2_EINVAL, "unknown type %d", dtype);
    if (!sizes_ok(B, 1, H)) return fail(T2_EINVAL, "bad shape [%d,%d]", B, H);
    if (B > 1 && (state_stride < H || y_stride < H)) return fail(T2_EINVAL, "rows of the state or of y overlap");
    // y may be z, f or o itself: a thread reads its channel before it writes it
    const int64_t size = dtype == T2_F32 ? 4 : 2, row = H * size, in_stride[] = {z_stride, f_stride, o_stride};
    const void* const in[] = {z, f, o};
    for (int64_t s : {z_stride, f_stride, o_stride, state_stride, y_stride})
        if (!reaches({nullptr, s, 0}, B, 1)) return fail(T2_EINVAL, "a stride of %lld elements", (long long)s);
    const Places py = places(y, y_stride * size, 0, B, 1, row), ps = places(state, state_stride * 4, 0, B, 1, (int64_t)H * 4), pa = block(active, B);
    if (meet(py, ps)) return fail(T2_EINVAL, "y overlaps the state");
    if (meet(py, pa) || meet(ps, pa)) return fail(T2_EINVAL, "an output overlaps active");
    for (int i = 0; i < 3; ++i) {
        const Places q = places(in[i], in_stride[i] * size, 0, B, 1, row);
        if (meet(ps, q)) return fail(T2_EINVAL, "the state overlaps an input");
        if (!(q.at == py.at && q.hi == py.hi) && meet(py, q)) return fail(T2_EINVAL, "y overlaps an input");
    }
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
