// Products of one 4-bit matrix with n tokens: argument checks and the choice of the kernel.
#include <algorithm>
#include <cstdio>
#include <cstdlib>

#include "w4_kernels.cuh"

namespace mlk {

int launch_w4_dense(const W4DenseParams& p, cudaStream_t s) {
    if (p.m <= 0 || p.m % 16 != 0) return fail(kInvalidArg, "gemm_layoutA_w4: m must be a positive multiple of 16 (got %d)", p.m);
    if (p.k <= 0) return fail(kInvalidArg, "gemm_layoutA_w4: k must be positive");
    if (p.n < 0) return fail(kInvalidArg, "gemm_layoutA_w4: n must not be negative");
    if (p.w.group != 32 && p.w.group != 64 && p.w.group != 128)
        return fail(kInvalidArg, "gemm_layoutA_w4: groups of 32, 64 or 128 (got %d)", p.w.group);
    if (p.k % p.w.group != 0) return fail(kInvalidArg, "gemm_layoutA_w4: k = %d is not whole groups of %d", p.k, p.w.group);
    if (p.dtype != kBF16 && p.dtype != kFP16) return fail(kInvalidArg, "gemm_layoutA_w4: activations must be bf16 or fp16");
    if (!p.w.q || !p.w.s || (p.n > 0 && (!p.X || !p.C))) return fail(kInvalidArg, "gemm_layoutA_w4: null pointer");
    if (((uintptr_t)p.w.q | (uintptr_t)p.w.s | (uintptr_t)p.w.z | (uintptr_t)p.X | (uintptr_t)p.C) & 15)
        return fail(kInvalidArg, "gemm_layoutA_w4: A, scales, zeros, B and C must be 16-byte aligned");
    if ((uintptr_t)p.bias & 1) return fail(kInvalidArg, "gemm_layoutA_w4: bias is not aligned");
    if (p.n == 0) return kOk;

    W4KernelParams g{};
    g.alpha = p.alpha;
    g.bias = p.bias;
    g.out_tiles = g.mat_tiles = p.m / 16;
    g.k = p.k;
    g.X = p.X;
    g.C = p.C;
    g.n = p.n;
    int np = p.n <= 32 ? 32 : (p.n <= 64 ? 64 : (p.n <= 128 ? 128 : 256)), sk = 0, lim = 16;
    if (const char* v = getenv("W4_U")) sscanf(v, "%d,%d,%d", &lim, &np, &sk);
    if (p.n > lim) {
        const int tokens = (p.n + np - 1) / np, tiles = (g.out_tiles + 7) / 8, stages = (p.k + 127) / 128;
        if (sk == 0) { sk = 1; while (sk < 8 && np <= 128 && tiles * tokens * sk < sm_count() && stages / sk >= 4) ++sk; }
        return launch_w4_umma(0, p.dtype, g, p.w, 1, p.n, np, sk, tokens, p.status, s);
    }
    const int nt = p.n <= 8 ? 1 : 2, items = (p.n + 8 * nt - 1) / (8 * nt);
    return launch_w4_mma(0, p.dtype, g, p.w, items, items, nt, s);
}

}  // namespace mlk
