// 4-bit weights, few tokens: streaming products on the warp-level tensor cores (dense, and the experts of a mixture).
//
//   C[n, m] = alpha * sum_k W[m, k] x[n, k] (+ bias),   W = (q - z) s per group of 32, 64 or 128 k
//
// What bounds it: the packed weights, read once.  At 6.5 TB/s that is 46 weights per SM and cycle, so the work per weight
// has to stay small: a word of eight weights becomes the 16-row operand of one m16n8k16 step with two ANDs, half a shift
// and one packed FMA per two weights (w4.cuh), the zero point subtracted exactly on the way, and the scale multiplies the
// fp32 sums of a group, not the weights.  Measured on the arithmetic alone (operands from shared memory, no other
// traffic): 16.8 T weights/s with one column tile of 8 tokens, 11 T with two; HBM delivers 13 T.  More than 16 tokens go
// to the tcgen05 kernel.
//
// A warp owns R tiles of 16 rows and every W-th block of 64 k; the activation fragment of a block (column operand, one
// 8-byte load per step and 8 tokens) serves all R tiles.  Weights travel through a private ring of each warp in shared
// memory filled by 16-byte cp.async: a lane copies exactly the bytes that it will read itself, so the ring needs no
// barrier, costs no registers and keeps 2 to 4 KB per warp in flight.  The warps' partial sums meet in shared memory, the
// k parts of a cluster in distributed shared memory, both in a fixed order: results do not depend on timing.
#include <algorithm>

#include "umma_common.cuh"
#include "w4.cuh"
#include "w4_kernels.cuh"

namespace mlk {

namespace {

constexpr int kWarps = 8;
constexpr int kTokStride = 20;   // floats between two tokens' 16 rows in the reduction buffer: conflict-free fragments

__device__ __forceinline__ uint2 ld_x(const uint8_t* p) {
    uint2 v;
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

__device__ __forceinline__ void cp_async16_hint(uint32_t dst, const void* src, uint64_t pol) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(pol) : "memory");
}

// first step of a group: the accumulator starts at zero
template <int WT>
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint2 b) {
    d[0] = d[1] = d[2] = d[3] = 0.f;
    mma16816<WT>(d, a[0], a[1], a[2], a[3], b.x, b.y);
}

// NT: column tiles of 8 tokens; RT: 16-row tiles of a CTA (MODE 1: half gate, half up); DI: ring depth in k blocks;
// G32: groups of 32 k (two per block), else a block lies inside one group.
template <int WT, int NT, int RT, int DI, bool G32, bool ZP, int MODE>
__global__ void __launch_bounds__(kWarps * 32) w4_mma_kernel(const W4KernelParams p, const int static_weights) {
    extern __shared__ __align__(128) uint8_t smem[];
    using D = W4Decode<WT>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, t = lane & 3;
    const int rank = blockIdx.y, SK = gridDim.y;
    constexpr int RO = MODE == 1 ? RT / 2 : RT;          // output tiles of this CTA
    const int tile0 = blockIdx.x * RO;

    if constexpr (MODE != 0) {
        pdl_wait();                                      // the work list comes from the kernel before
        pdl_launch_dependents();
    } else if (!static_weights) {
        pdl_wait();
        pdl_launch_dependents();
    }

    int n0 = 0, ntok = 0, mat = 0, pos0 = 0, cpos0 = 0;
    if constexpr (MODE == 0) {
        n0 = blockIdx.z * NT * 8;
        ntok = min(NT * 8, p.n - n0);
    } else {
        const int items = p.worklist[0].x;
        if ((int)blockIdx.z >= items) return;            // uniform over the cluster
        const int4 item = p.worklist[1 + blockIdx.z];
        mat = item.x; pos0 = item.y; ntok = item.z; cpos0 = item.w;
    }

    // the row tiles of this CTA; tiles past the end repeat the last one and are not stored
    const uint8_t* wbase[RT];
    size_t sbase[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        int tile = min(tile0 + (MODE == 1 ? i % RO : i), p.out_tiles - 1);
        if (MODE == 1 && i >= RO) tile += p.out_tiles;
        const size_t at = (size_t)mat * p.mat_tiles + tile;
        wbase[i] = p.q + at * p.kc * kW4BlockBytes + lane * 16;
        sbase[i] = at * p.groups * 8 + r;
    }
    const int cb = (int)((long long)p.kc * rank / SK), ce = (int)((long long)p.kc * (rank + 1) / SK);
    const int nit = (ce - cb - warp + kWarps - 1) / kWarps;
    const uint32_t ring = smem_u32(smem) + warp * (DI * RT * kW4BlockBytes) + lane * 16;
    const uint64_t pol = l2_policy_evict_first();

    auto fetch = [&](int i) {
        if (i < nit) {
            const size_t off = (size_t)(cb + warp + i * kWarps) * kW4BlockBytes;
            const uint32_t slot = ring + (i % DI) * (RT * kW4BlockBytes);
#pragma unroll
            for (int j = 0; j < RT; ++j) cp_async16_hint(slot + j * kW4BlockBytes, wbase[j] + off, pol);
        }
        cp_async_commit();                               // an empty group keeps the count
    };
#pragma unroll
    for (int i = 0; i < DI; ++i) fetch(i);
    if constexpr (MODE == 0) {
        if (static_weights) {
            pdl_launch_dependents();
            pdl_wait();
        }
    }

    const uint8_t* xrow[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int c = nt * 8 + r;
        xrow[nt] = nullptr;
        if (c < ntok) {
            long long row;
            if constexpr (MODE == 0) row = n0 + c;
            else if constexpr (MODE == 1) row = p.sorted[pos0 + c] / p.topk;
            else row = cpos0 + c;
            xrow[nt] = reinterpret_cast<const uint8_t*>(p.X) + row * (2LL * p.k) + 8 * t;
        }
    }

    float tot[RT][NT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) tot[i][nt][e] = 0.f;

    for (int it = 0; it < nit; ++it) {
        const int c = cb + warp + it * kWarps;
        const bool half_only = G32 && c * kW4BlockK + 32 >= p.k;     // k ends in the middle of the block
        uint2 x[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[nt][j] = make_uint2(0u, 0u);
                if (xrow[nt] != nullptr && !(half_only && j >= 2)) x[nt][j] = ld_x(xrow[nt] + (size_t)c * (kW4BlockK * 2) + j * 32);
            }
        constexpr int NG = G32 ? 2 : 1;
        const int g0 = G32 ? 2 * c : (c * kW4BlockK) >> p.group_shift;
        uint32_t sc[RT][NG], zp[RT][NG];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const size_t at = sbase[i] + (size_t)((G32 && g == 1 && half_only) ? g0 : g0 + g) * 8;
                sc[i][g] = __ldg(p.s + at);
                zp[i][g] = ZP ? (uint32_t)__ldg(p.z + at) : 0x0808u;
            }
        cp_async_wait<DI - 1>();
        const uint32_t slot = ring + (it % DI) * (RT * kW4BlockBytes);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const uint4 w = lds16(slot + i * kW4BlockBytes);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t zl, zh;
                D::zero(zp[i][g], zl, zh);
                float acc[NT][4];
#pragma unroll
                for (int j = g * (4 / NG); j < (g + 1) * (4 / NG); ++j) {
                    uint32_t a[4];
                    D::word(words[j], zl, zh, a);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (j == g * (4 / NG)) mma_first<WT>(acc[nt], a, x[nt][j]);
                        else mma16816<WT>(acc[nt], a[0], a[1], a[2], a[3], x[nt][j].x, x[nt][j].y);
                    }
                }
                if (G32 && g == 1 && half_only) continue;
                const float2 s2 = unpack2<WT>(sc[i][g]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    tot[i][nt][0] = fmaf(s2.x, acc[nt][0], tot[i][nt][0]);
                    tot[i][nt][1] = fmaf(s2.x, acc[nt][1], tot[i][nt][1]);
                    tot[i][nt][2] = fmaf(s2.y, acc[nt][2], tot[i][nt][2]);
                    tot[i][nt][3] = fmaf(s2.y, acc[nt][3], tot[i][nt][3]);
                }
            }
        }
        fetch(it + DI);
    }

    // ---- partial sums of the warps, then of the cluster ----
    cp_async_wait<0>();
    __syncthreads();
    float* const red = reinterpret_cast<float*>(smem);
    constexpr int kPerWarp = RT * NT * 8 * kTokStride;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float* const d = red + warp * kPerWarp + (i * NT * 8 + nt * 8 + 2 * t) * kTokStride + r;
            d[0] = D::kFactorLow * tot[i][nt][0];
            d[kTokStride] = D::kFactorLow * tot[i][nt][1];
            d[8] = D::kFactorHigh * tot[i][nt][2];
            d[kTokStride + 8] = D::kFactorHigh * tot[i][nt][3];
        }
    __syncthreads();
    auto place = [&](int i, int tok, int row) { return (i * NT * 8 + tok) * kTokStride + row; };
    for (int e = tid; e < RT * 16 * ntok; e += kWarps * 32) {
        const int row = e & 15, i = (e >> 4) % RT, tok = (e >> 4) / RT;
        const int at = place(i, tok, row);
        float v = red[at];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) v += red[w * kPerWarp + at];
        red[at] = v;
    }
    uint32_t remote[8];
    __syncwarp();
    if (SK > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
#pragma unroll
        for (int q = 0; q < 8; ++q)
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote[q]) : "r"(smem_u32(smem)), "r"(q < SK ? q : 0));
    } else {
        __syncthreads();
    }
    auto total = [&](int at) {
        if (SK == 1) return red[at];
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (q < SK) {
                float u;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u) : "r"(remote[q] + 4u * at) : "memory");
                v += u;
            }
        return v;
    };
    const int outs = RO * 16 * ntok;
    for (int e = outs * rank / SK + tid; e < outs * (rank + 1) / SK; e += kWarps * 32) {
        const int row16 = e & 15, i = (e >> 4) % RO, tok = (e >> 4) / RO;
        if (tile0 + i >= p.out_tiles) continue;
        const int row = (tile0 + i) * 16 + row16;
        const size_t ld = (size_t)p.out_tiles * 16;
        const float v = total(place(i, tok, row16));
        if constexpr (MODE == 0) {
            const float b = p.bias ? load_scalar16<WT>(p.bias, row) : 0.f;
            store16<WT>(p.C, (size_t)(n0 + tok) * ld + row, fmaf(p.alpha, v, b));
        } else if constexpr (MODE == 1) {
            const float up = total(place(i + RO, tok, row16));
            store16<WT>(p.C, (size_t)(cpos0 + tok) * ld + row, v / (1.f + __expf(-v)) * up);
        } else {
            const int slot = p.sorted[pos0 + tok];
            reinterpret_cast<float*>(p.C)[(size_t)slot * ld + row] = load_scalar16<WT>(p.topk_weights, slot) * v;
        }
    }
    __syncwarp();
    if (SK > 1)     // nobody leaves while its shared memory may still be read
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int WT, int NT, int RT, int DI, int MODE>
const void* pick(bool g32, bool zp) {
    if (g32) return zp ? reinterpret_cast<const void*>(w4_mma_kernel<WT, NT, RT, DI, true, true, MODE>)
                       : reinterpret_cast<const void*>(w4_mma_kernel<WT, NT, RT, DI, true, false, MODE>);
    return zp ? reinterpret_cast<const void*>(w4_mma_kernel<WT, NT, RT, DI, false, true, MODE>)
              : reinterpret_cast<const void*>(w4_mma_kernel<WT, NT, RT, DI, false, false, MODE>);
}
template <int NT, int RT, int DI, int MODE>
const void* pick(int wt, bool g32, bool zp) {
    return wt == kFP16 ? pick<kFP16, NT, RT, DI, MODE>(g32, zp) : pick<kBF16, NT, RT, DI, MODE>(g32, zp);
}

}  // namespace

int launch_w4_mma(int mode, int wt, W4KernelParams p, const W4Weights& w, int token_blocks, int nt, int sk, cudaStream_t s) {
    constexpr int RT = 2, DI = 4;
    const bool g32 = w.group == 32, zp = w.z != nullptr;
    const void* kern = nullptr;
    if (mode == 0) kern = nt == 1 ? pick<1, RT, DI, 0>(wt, g32, zp) : pick<2, RT, DI, 0>(wt, g32, zp);
    else if (mode == 1) kern = nt == 1 ? pick<1, RT, DI, 1>(wt, g32, zp) : pick<2, RT, DI, 1>(wt, g32, zp);
    else kern = nt == 1 ? pick<1, RT, DI, 2>(wt, g32, zp) : pick<2, RT, DI, 2>(wt, g32, zp);
    const int ro = mode == 1 ? RT / 2 : RT;
    const size_t smem = std::max((size_t)kWarps * DI * RT * kW4BlockBytes, (size_t)kWarps * RT * nt * 8 * kTokStride * 4);
    const size_t launch_smem = umma::prepare_kernel(kern, kWarps * 32, smem, 0);
    if (launch_smem == 0) return fail(kCudaError, "w4: the streaming kernel cannot be launched on this device");
    if (token_blocks > 65535) return fail(kUnsupported, "w4: %d token blocks exceed one launch", token_blocks);
    p.q = w.q;
    p.s = reinterpret_cast<const uint32_t*>(w.s);
    p.z = reinterpret_cast<const uint16_t*>(w.z);
    p.kc = (p.k + kW4BlockK - 1) / kW4BlockK;
    p.groups = p.k / w.group;
    p.group_shift = w.group == 128 ? 7 : (w.group == 64 ? 6 : 5);
    int static_weights = option(kOptStaticWeights);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.out_tiles + ro - 1) / ro), (unsigned)sk, (unsigned)token_blocks);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = launch_smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    cfg.numAttrs = launch_attrs(attr, sk);
    void* args[2] = {&p, &static_weights};
    const cudaError_t e = cudaLaunchKernelExC(&cfg, kern, args);
    if (e != cudaSuccess) return fail(kCudaError, "w4 launch: %s", cudaGetErrorString(e));
    return kOk;
}

// k parts: enough warps for the whole chip to have its loads in flight at once, at least two k blocks per warp.
int w4_mma_split(long long row_ctas, int kc) {
    int sk = 1;
    while (sk < 8 && row_ctas * sk < 3LL * sm_count() && kc / (kWarps * sk * 2) >= 2) sk *= 2;
    return sk;
}

}  // namespace mlk
