// Micro-benchmark of the conv GEMM fast path at PostNetV2's shape (not part of the library).
// Build: hipcc --offload-arch=gfx950 -O3 -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops tools/conv_bench.hip -o /tmp/conv_bench
#include "../tacotron2_amd/csrc/kernels.h"
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>
#define CK(x) do { hipError_t e = (x); if (e != hipSuccess) { printf("%s: %s\n", #x, hipGetErrorString(e)); exit(1); } } while (0)
int main(int argc, char** argv) {
    const int B = 64, T = 800, Cin = argc > 1 ? atoi(argv[1]) : 512, N = 512, ktaps = 5, Mtot = B * T;
    float *x, *w, *sc, *sh, *y, *y2;
    CK(hipMalloc(&x, (size_t)Mtot * Cin * 4)); CK(hipMalloc(&w, (size_t)ktaps * Cin * N * 4)); CK(hipMalloc(&sc, N * 4)); CK(hipMalloc(&sh, N * 4));
    CK(hipMalloc(&y, (size_t)Mtot * N * 4)); CK(hipMalloc(&y2, (size_t)Mtot * N * 4));
    std::vector<float> hx((size_t)Mtot * Cin), hw((size_t)ktaps * Cin * N), hs(N, 1.f);
    for (auto& v : hx) v = rand() / (float)RAND_MAX - 0.5f;
    for (auto& v : hw) v = (rand() / (float)RAND_MAX - 0.5f) * 0.05f;
    CK(hipMemcpy(x, hx.data(), hx.size() * 4, hipMemcpyHostToDevice)); CK(hipMemcpy(w, hw.data(), hw.size() * 4, hipMemcpyHostToDevice));
    CK(hipMemcpy(sc, hs.data(), N * 4, hipMemcpyHostToDevice)); CK(hipMemset(sh, 0, N * 4));
    ConvArgs a{};
    a.x = x; a.ldx = Cin; a.w = w; a.scale = sc; a.shift = sh; a.y = y; a.ldy = N; a.Mtot = Mtot; a.T = T; a.Cin = Cin; a.N = N; a.ktaps = ktaps;
    a.pad_l = 2; a.act = 2; a.vec_a = 1; a.vec_b = 1;
    hipEvent_t e0, e1; CK(hipEventCreate(&e0)); CK(hipEventCreate(&e1));
    const dim3 grid(N / CG_BN, (Mtot + CG_BM - 1) / CG_BM);
    // reference: the generic kernel (same summation order: the results must be bit-identical)
    ConvArgs r = a; r.y = y2;
    hipLaunchKernelGGL(conv_gemm_kernel, grid, dim3(256), 0, 0, r);
    float best = 1e9;
    for (int it = 0; it < 12; ++it) {
        CK(hipEventRecord(e0));
        hipLaunchKernelGGL(conv_gemm_fast_kernel<2>, grid, dim3(256), 0, 0, a);
        CK(hipEventRecord(e1)); CK(hipEventSynchronize(e1));
        float ms; CK(hipEventElapsedTime(&ms, e0, e1));
        if (it > 1 && ms < best) best = ms;
    }
    CK(hipGetLastError());
    std::vector<float> h1((size_t)Mtot * N), h2((size_t)Mtot * N);
    CK(hipMemcpy(h1.data(), y, h1.size() * 4, hipMemcpyDeviceToHost)); CK(hipMemcpy(h2.data(), y2, h2.size() * 4, hipMemcpyDeviceToHost));
    const bool same = memcmp(h1.data(), h2.data(), h1.size() * 4) == 0;
    const double fl = 2.0 * Mtot * (double)ktaps * Cin * N;
    printf("conv_gemm_fast_kernel<2> M=%d K=%d N=%d: %.3f ms = %.1f TFLOP/s (%.3f of 157.3); bit-identical to the generic kernel: %s\n", Mtot, ktaps * Cin, N,
           best, fl / best / 1e9, fl / best / 1e9 / 157.3, same ? "yes" : "NO");
    return same ? 0 : 2;
}
