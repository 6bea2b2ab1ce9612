// Products of one 4-bit matrix with n tokens: argument checks and the choice of the kernel.
#include <algorithm>

#include "w4_kernels.cuh"

namespace mlk {

int launch_w4_dense(const W4DenseParams& p, cudaStream_t s) {
    if (p.m <= 0 || p.m % 16 != 0) return fail(kInvalidArg, "gemm_layoutA_w4: m must be a positive multiple of 16 (got %d)", p.m);
    if (p.k <= 0) return fail(kInvalidArg, "gemm_layoutA_w4: k must be positive");
    if (p.m > kW4MaxDim || p.k > kW4MaxDim) return fail(kUnsupported, "gemm_layoutA_w4: more than 2^28 rows or k");
    if (p.n < 0) return fail(kInvalidArg, "gemm_layoutA_w4: n must not be negative");
    if (p.w.group != 32 && p.w.group != 64 && p.w.group != 128)
        return fail(kInvalidArg, "gemm_layoutA_w4: groups of 32, 64 or 128 (got %d)", p.w.group);
    if (p.k % p.w.group != 0) return fail(kInvalidArg, "gemm_layoutA_w4: k = %d is not whole groups of %d", p.k, p.w.group);
    if (p.dtype != kBF16 && p.dtype != kFP16) return fail(kInvalidArg, "gemm_layoutA_w4: activations must be bf16 or fp16");
    if (!p.w.q || !p.w.s || (p.n > 0 && (!p.X || !p.C))) return fail(kInvalidArg, "gemm_layoutA_w4: null pointer");
    if (((uintptr_t)p.w.q | (uintptr_t)p.w.s | (uintptr_t)p.w.z | (uintptr_t)p.X | (uintptr_t)p.C) & 15)
        return fail(kInvalidArg, "gemm_layoutA_w4: A, scales, zeros, B and C must be 16-byte aligned");
    if (((uintptr_t)p.bias & 1) || ((uintptr_t)p.status & 3)) return fail(kInvalidArg, "gemm_layoutA_w4: bias or status is not aligned");
    if (p.n == 0) return kOk;

    W4KernelParams g{};
    g.alpha = p.alpha;
    g.bias = p.bias;
    g.out_tiles = g.mat_tiles = p.m / 16;
    g.k = p.k;
    g.X = p.X;
    g.C = p.C;
    g.n = p.n;
    // Up to 16 tokens the streaming kernel, above it tcgen05, whose decode and hand-offs cost the same for any token count.
    // By time the border would be near 8: 28672 x 8192 at 8 tokens 30 us against 36; from 9 tokens on (9 / 12 / 16 tokens)
    // 46 / 48 / 51 against 36.5, 4096 x 14336 17.0 / 17.2 / 17.6 against 15.7, 14336 x 4096 17.9 / 18.9 / 20.3 against 16.1,
    // 8192 x 8192 15.5 / 15.7 / 16.7 against 16.2, 4096 x 4096 7.3 / 7.4 / 7.7 against 7.3, 1040 x 2080 5.5 / 5.5 / 5.9 against
    // 4.9.  It stays at 16 because the streaming kernel keeps the weights exact, which a decode batch of that size is
    // promised.  14336 x 4096 at 61 tokens: 65 against 16.8.
    if (p.n <= 16) return launch_w4_mma(0, p.dtype, g, p.w, 1, 1, p.n <= 8 ? 1 : 2, s);
    const W4UmmaPlan q = w4_umma_plan(g.out_tiles, p.n, p.k);
    const int tokens = (p.n + q.np - 1) / q.np;
    // a launch holds at most 65535 token tiles
    for (int t0 = 0; t0 < tokens; t0 += 65535) {
        const long long n0 = (long long)t0 * q.np;
        g.X = reinterpret_cast<const uint8_t*>(p.X) + n0 * p.k * 2;
        g.C = reinterpret_cast<uint8_t*>(p.C) + n0 * p.m * 2;
        g.n = (int)std::min<long long>(p.n - n0, 65535LL * q.np);
        if (int st = launch_w4_umma(0, p.dtype, g, p.w, 1, g.n, q.np, q.sk, 1, std::min(tokens - t0, 65535), p.status, s)) return st;
    }
    return kOk;
}

}  // namespace mlk
