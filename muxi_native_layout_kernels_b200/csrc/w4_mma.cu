// 4-bit weights, few tokens: streaming products on the warp-level tensor cores (dense, and the experts of a mixture).
//
//   C[n, m] = alpha * sum_k W[m, k] x[n, k] (+ bias),   W = (q - z) s per group of 32, 64 or 128 k
//
// What bounds it: the packed weights, read once, and the instructions on them.  At 6.5 TB/s that is 46 weights per SM and
// cycle, so the work per weight has to stay small: a word of eight weights becomes the 16-row operand of one m16n8k16 step
// with four ANDs, a shift and four packed FMAs (w4.cuh), the zero point subtracted exactly on the way, and the scale
// multiplies the fp32 sums of a group, not the weights.  Measured on the arithmetic alone (operands from shared memory, no
// other traffic): 16.8 T weights/s with one column tile of 8 tokens, 11 T with two; HBM delivers 13 T; a copy of the
// weights into shared memory alone takes 21 us for the 117 MB of 28672 x 8192, with the arithmetic 25.
// Measured (us, and of the time that the bytes take at the copy bandwidth): 4096 x 4096 at 1 token 5.8 (1.3: one wave of
// CTAs, latency), 28672 x 8192 at 8 tokens 31 (18.6), 4096 x 14336 fp16 with zero points at 16 tokens 17.5 (5.0), 8 of 128 experts of 2048 x 768 for one token 15.3 (3.0: two
// kernels of latency), 33 tokens on them 63 (42), 5 tokens on 8 experts of 4096 x 14336 123 (85).  At 28672 x 8192 and 8 tokens a word takes 16
// warp instructions in all, and the issue slots are 54 % busy, the ALU pipe 45 %, the tensor pipe 27 %: the warps wait for
// one another's pipes, not for memory.  More than 16 tokens go to the tcgen05 kernel.
//
// A warp owns RT tiles of 16 rows and every WK-th unit of 128 k; WR x WK = 8 warps share the rows and the k range of a CTA.
// The CTA's activations and scales are staged in shared memory once, so that a unit costs one 8-byte shared load per step
// and 8 tokens for the column operand of all RT tiles.  Weights travel through a private ring of each warp filled by
// 16-byte cp.async: a lane copies exactly the bytes that it will read itself, so the ring needs no barrier and costs no
// registers.  The warps' partial sums meet in shared memory, the k parts of a cluster in distributed shared memory, both
// in a fixed order: results do not depend on timing.
// Measured and not used: activations and scales fetched by each warp from global memory (28672 x 8192 at 8 tokens 37
// instead of 31 us); a persistent grid with an equal run of tiles per SM (31 us there, but 80 instead of 64 us for 33
// tokens on 128 small experts); activations kept in registers with the rows streaming past (33 and 85 us: every few tiles
// all warps have to meet); rings one unit deep (37 and 70 us); two row tiles per warp with rings of two / three units (31 / 34 us
// there, 19 / 25 instead of 17.7 us at 16 tokens of 4096 x 14336, 61 / 62 us for 33 tokens on the experts).
#include <algorithm>
#include <array>
#include <cmath>
#include <map>

#include "umma_common.cuh"
#include "w4.cuh"
#include "w4_kernels.cuh"

namespace mlk {

namespace {

constexpr int kTokStride = 20;   // floats between two tokens' 16 rows in the reduction buffer: conflict-free fragments

__device__ __forceinline__ uint2 lds8(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t lds2(uint32_t addr) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
    return v;
}

__device__ __forceinline__ void cp_async16_hint(uint32_t dst, const void* src, uint64_t pol) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(pol) : "memory");
}

// first step of a group: D = A * B
template <int WT>
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint2 b) {
    if constexpr (WT == kFP16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "f"(0.f));
}

constexpr int kWarps = 8, kRT = 4, kDI = 2;     // warps of a CTA, row tiles of a warp, ring depth in units

// Local expert of a slot of the single token, -1 = none here.
__device__ __forceinline__ int expert_of(const W4KernelParams& p, int slot) {
    int e = p.ids[slot];
    if (p.experts_map != nullptr) e = e >= 0 && e < p.experts_map_len ? p.experts_map[e] : -1;
    return e >= 0 && e < p.experts ? e : -1;
}

// NT: column tiles of 8 tokens; RT: 16-row tiles of a warp (MODE 1: half gate, half up); DI: ring depth in units of 128 k;
// G: group size; ZP: zero points given.
template <int WT, int NT, int RT, int DI, int G, bool ZP, int MODE>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) w4_mma_kernel(const W4KernelParams p, const int static_weights) {
    extern __shared__ __align__(128) uint8_t smem[];
    using D = W4Decode<WT>;
    constexpr int RO = MODE == 1 ? RT / 2 : RT;          // output tiles of a warp
    constexpr int NG = 128 / G, SG = G / 16;             // groups of a unit, 16-k steps of a group
    constexpr uint32_t kSlot = RT * 2 * kW4BlockBytes;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, t = lane & 3;
    const bool single = MODE != 0 && p.ids != nullptr;   // one token: items are its slots
    const bool gathered = MODE == 2 && single;           // the cluster's CTAs are the slots, not parts of k
    const int rank = blockIdx.y, SK = gridDim.y;
    const int krank = gathered ? 0 : rank, KSK = gathered ? 1 : SK;
    const int WR = p.row_warps, WK = kWarps / WR, wr = warp / WK, wk = warp - wr * WK;
    const int tile0 = blockIdx.x * RO * WR;

    const bool early = MODE == 0 && static_weights;      // weights may be read before the kernel in front has finished
    if (!early) {
        pdl_wait();
        pdl_launch_dependents();
    }

    int n0 = 0, ntok = 0, mat = 0, pos0 = 0, cpos0 = 0;
    if constexpr (MODE == 0) {
        n0 = blockIdx.z * NT * 8;
        ntok = min(NT * 8, p.n - n0);
    } else if (single) {
        cpos0 = gathered ? rank : blockIdx.z;            // the slot
        mat = expert_of(p, cpos0);
        ntok = 1;
        if (mat < 0) {
            if (!gathered) return;                       // uniform over the cluster: its row is not read either
            mat = ntok = 0;                              // nothing of this slot: zeros for the sum
        }
    } else {
        const int items = p.worklist[0].x;
        const int4 item = p.worklist[1 + blockIdx.z];
        if ((int)blockIdx.z >= items) return;            // uniform over the cluster
        mat = item.x; pos0 = item.y; ntok = item.z; cpos0 = item.w;
    }

    // tile j of row warp w; tiles past the end repeat the last one and are not stored
    auto tile_of = [&](int w, int j) {
        const int tile = min(tile0 + w * RO + (MODE == 1 ? j % RO : j), p.out_tiles - 1);
        return MODE == 1 && j >= RO ? tile + p.out_tiles : tile;
    };
    const int units = (p.kc + 1) >> 1;                   // two blocks (128 k) each; the last one of an odd number is half
    const int ub = (int)((long long)units * krank / KSK), ue = ntok == 0 ? ub : (int)((long long)units * (krank + 1) / KSK);
    const size_t tile_bytes = (size_t)p.kc * kW4BlockBytes;
    const uint8_t* wnext[RT];                            // the unit that is fetched next
#pragma unroll
    for (int i = 0; i < RT; ++i)
        wnext[i] = p.q + ((size_t)mat * p.mat_tiles + tile_of(wr, i)) * tile_bytes + (size_t)(ub + wk) * 1024 + lane * 16;
    const uint32_t smem0 = smem_u32(smem);
    const uint32_t ring0 = smem0 + warp * (DI * kSlot) + lane * 16, ring1 = ring0 + DI * kSlot;
    const uint64_t pol = l2_policy_evict_first();

    int fu = ub + wk;
    uint32_t put = ring0, get = ring0;
    auto fetch = [&]() {
        if (fu < ue) {
            const bool second = fu * 2 + 1 < p.kc;
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                cp_async16_hint(put + j * 1024, wnext[j], pol);
                if (second) cp_async16_hint(put + j * 1024 + kW4BlockBytes, wnext[j] + kW4BlockBytes, pol);
                wnext[j] += WK * 1024;
            }
            put = put + kSlot == ring1 ? ring0 : put + kSlot;
            fu += WK;
        }
        cp_async_commit();                               // an empty group keeps the count
    };

    // staging area: activations [token][pitch], scales [row tile][group][8][2], zero points likewise.  Tokens behind the
    // last one, k behind the end, and the groups there are zeros: the loop below needs no case for them.
    const uint32_t xs = smem0 + kWarps * DI * kSlot;
    const uint32_t pitch = (uint32_t)p.seg_units * 256 + 32;     // 32 bytes off a multiple of 128: no bank conflicts
    const int sg = p.seg_units * NG;
    const uint32_t ss = xs + NT * 8 * pitch, zs = ss + (uint32_t)(WR * RT) * sg * 32;
    auto stage = [&](int u0, int u1) {
        const int k0 = u0 * 128, v = (min(u1 * 128, p.k) - k0) / 8, all = (u1 - u0) * 16;     // 16-byte pieces of a row
        for (int i = tid; i < all * NT * 8; i += kWarps * 32) {
            const int c = i / all, o = i - c * all;
            const bool in = c < ntok && o < v;
            const uint8_t* src = reinterpret_cast<const uint8_t*>(p.X);
            if (in) {
                long long row;
                if constexpr (MODE == 0) row = n0 + c;
                else if constexpr (MODE == 1) row = single ? 0 : p.sorted[pos0 + c] / p.topk;
                else row = cpos0 + c;
                src += (row * p.k + k0) * 2 + o * 16;
            }
            cp_async16(xs + c * pitch + o * 16, src, in ? 16 : 0);
        }
        const int g0 = u0 * NG, sv = (u1 - u0) * NG * 2;
        for (int i = tid; i < WR * RT * sv; i += kWarps * 32) {
            const int j = i / sv, o = i - j * sv;
            const bool in = g0 + o / 2 < p.groups;
            const size_t at = ((size_t)mat * p.mat_tiles + tile_of(j / RT, j % RT)) * p.groups + g0;
            cp_async16(ss + (j * sg * 2 + o) * 16, reinterpret_cast<const uint8_t*>(p.s) + (in ? at * 32 + o * 16 : 0), in ? 16 : 0);
            if (ZP && !(o & 1))
                cp_async16(zs + (j * sg * 2 + o) * 8, reinterpret_cast<const uint8_t*>(p.z) + (in ? at * 16 + o * 8 : 0), in ? 16 : 0);
        }
    };

    if (early) {
#pragma unroll
        for (int i = 0; i < DI; ++i) fetch();
        pdl_launch_dependents();
        pdl_wait();
        stage(ub, min(ub + p.seg_units, ue));
        cp_async_commit();
        cp_async_wait<0>();
    } else {
        stage(ub, min(ub + p.seg_units, ue));
        cp_async_commit();
#pragma unroll
        for (int i = 0; i < DI; ++i) fetch();
        cp_async_wait<DI>();
    }
    __syncthreads();

    float tot[RT][NT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) tot[i][nt][e] = 0.f;

    int u = ub + wk;
    for (int u0 = ub; u0 < ue; u0 += p.seg_units) {
        const int u1 = min(u0 + p.seg_units, ue);
        if (u0 > ub) {                                   // the next segment of activations and scales
            __syncthreads();
            stage(u0, u1);
            cp_async_commit();
            cp_async_wait<0>();
            __syncthreads();
        }
        uint32_t xa = xs + r * pitch + (u - u0) * 256 + 8 * t;
        uint32_t sa = ss + (uint32_t)(wr * RT * sg + (u - u0) * NG) * 32 + 4 * r;
        uint32_t za = zs + (uint32_t)(wr * RT * sg + (u - u0) * NG) * 16 + 2 * r;
        for (; u < u1; u += WK) {
            uint2 x[NT][8];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[nt][j] = lds8(xa + nt * 8 * pitch + 32 * j);
            cp_async_wait<DI - 1>();
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const uint4 w0 = lds16(get + i * 1024), w1 = lds16(get + i * 1024 + kW4BlockBytes);
                const uint32_t words[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    uint32_t zl, zh;
                    D::zero(ZP ? lds2(za + (i * sg + g) * 16) : 0x0808u, zl, zh);
                    const float2 s2 = unpack2<WT>(lds4(sa + (i * sg + g) * 32));
                    float acc[NT][4];
#pragma unroll
                    for (int j = g * SG; j < (g + 1) * SG; ++j) {
                        uint32_t a[4];
                        D::word(words[j], zl, zh, a);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            if (j == g * SG) mma_first<WT>(acc[nt], a, x[nt][j]);
                            else mma16816<WT>(acc[nt], a[0], a[1], a[2], a[3], x[nt][j].x, x[nt][j].y);
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        tot[i][nt][0] = fmaf(s2.x, acc[nt][0], tot[i][nt][0]);
                        tot[i][nt][1] = fmaf(s2.x, acc[nt][1], tot[i][nt][1]);
                        tot[i][nt][2] = fmaf(s2.y, acc[nt][2], tot[i][nt][2]);
                        tot[i][nt][3] = fmaf(s2.y, acc[nt][3], tot[i][nt][3]);
                    }
                }
            }
            get = get + kSlot == ring1 ? ring0 : get + kSlot;
            xa += WK * 256;
            sa += WK * NG * 32;
            za += WK * NG * 16;
            fetch();
        }
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
    // four rows at a time: the sums of row warp w's tile i, token tok, rows 4 q .. of 16
    auto place = [&](int w, int i, int tok, int q) { return w * WK * kPerWarp + (i * NT * 8 + tok) * kTokStride + 4 * q; };
    auto add = [](float4& v, float4 o) { v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w; };
    auto warps_sum = [&](int at) {
        float4 v = *reinterpret_cast<const float4*>(red + at);
        for (int q = 1; q < WK; ++q) add(v, *reinterpret_cast<const float4*>(red + q * kPerWarp + at));
        return v;
    };
    const int cols = gathered ? 1 : ntok;                // a skipped slot of a single token adds zeros
    if (SK > 1 || gathered) {
        if (WK > 1) {
            for (int e = tid; e < WR * RT * 4 * cols; e += kWarps * 32) {
                const int q = e & 3, i = (e >> 2) % RT, rest = (e >> 2) / RT, w = rest % WR, tok = rest / WR;
                const int at = place(w, i, tok, q);
                *reinterpret_cast<float4*>(red + at) = warps_sum(at);
            }
        }
        __syncwarp();
        if (SK > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        else __syncthreads();
    }
    auto part = [&](int q, int at) {                     // rank q's sums
        if (SK == 1) return *reinterpret_cast<const float4*>(red + at);
        uint32_t a;
        float4 o;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem0 + 4u * at), "r"(q));
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(o.x), "=f"(o.y), "=f"(o.z), "=f"(o.w) : "r"(a) : "memory");
        return o;
    };
    auto total = [&](int at) {
        if (SK == 1) return warps_sum(at);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int q = 0; q < SK; ++q) add(v, part(q, at));
        return v;
    };
    const int outs = WR * RO * 4 * cols;
    const size_t ld = (size_t)p.out_tiles * 16;
    for (int e = outs * rank / SK + tid; e < outs * (rank + 1) / SK; e += kWarps * 32) {
        const int q = e & 3, i = (e >> 2) % RO, rest = (e >> 2) / RO, w = rest % WR, tok = rest / WR;
        const int tile = tile0 + w * RO + i;
        if (tile >= p.out_tiles) continue;
        const int row = tile * 16 + 4 * q;
        if (MODE == 2 && single) {
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);  // the token's slots in order, in fp32, rounded once
            for (int j = 0; j < SK; ++j) {
                if (expert_of(p, j) < 0) continue;
                const float f = load_scalar16<WT>(p.topk_weights, j);
                const float4 v = part(j, place(w, i, tok, q));
                y.x += f * v.x; y.y += f * v.y; y.z += f * v.z; y.w += f * v.w;
            }
            if (p.y_fp32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.C) + row) = y;
            else *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.C) + row) = make_uint2(pack2<WT>(y.x, y.y), pack2<WT>(y.z, y.w));
            continue;
        }
        const float4 v = total(place(w, i, tok, q));
        if constexpr (MODE == 0) {
            float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p.bias) b = make_float4(load_scalar16<WT>(p.bias, row), load_scalar16<WT>(p.bias, row + 1), load_scalar16<WT>(p.bias, row + 2), load_scalar16<WT>(p.bias, row + 3));
            uint2 o;
            o.x = pack2<WT>(fmaf(p.alpha, v.x, b.x), fmaf(p.alpha, v.y, b.y));
            o.y = pack2<WT>(fmaf(p.alpha, v.z, b.z), fmaf(p.alpha, v.w, b.w));
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.C) + (size_t)(n0 + tok) * ld + row) = o;
        } else if constexpr (MODE == 1) {
            const float4 up = total(place(w, i + RO, tok, q));
            auto act = [](float g, float h) { return g / (1.f + __expf(-g)) * h; };
            uint2 o;
            o.x = pack2<WT>(act(v.x, up.x), act(v.y, up.y));
            o.y = pack2<WT>(act(v.z, up.z), act(v.w, up.w));
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.C) + (size_t)(cpos0 + tok) * ld + row) = o;
        } else {
            const int slot = p.sorted[pos0 + tok];
            const float f = load_scalar16<WT>(p.topk_weights, slot);
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.C) + (size_t)slot * ld + row) = make_float4(f * v.x, f * v.y, f * v.z, f * v.w);
        }
    }
    if (SK > 1) {                                        // nobody leaves while its shared memory may still be read
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

template <int WT, int NT, int MODE>
const void* pick(int group, bool zp) {
    if (group == 128) return zp ? reinterpret_cast<const void*>(w4_mma_kernel<WT, NT, kRT, kDI, 128, true, MODE>)
                                : reinterpret_cast<const void*>(w4_mma_kernel<WT, NT, kRT, kDI, 128, false, MODE>);
    if (group == 64) return zp ? reinterpret_cast<const void*>(w4_mma_kernel<WT, NT, kRT, kDI, 64, true, MODE>)
                               : reinterpret_cast<const void*>(w4_mma_kernel<WT, NT, kRT, kDI, 64, false, MODE>);
    return zp ? reinterpret_cast<const void*>(w4_mma_kernel<WT, NT, kRT, kDI, 32, true, MODE>)
              : reinterpret_cast<const void*>(w4_mma_kernel<WT, NT, kRT, kDI, 32, false, MODE>);
}
template <int WT>
const void* pick(int mode, int nt, int group, bool zp) {     // more than 8 slots per item of an expert go to tcgen05
    if (mode == 0) return nt == 1 ? pick<WT, 1, 0>(group, zp) : pick<WT, 2, 0>(group, zp);
    if (nt != 1) return nullptr;
    return mode == 1 ? pick<WT, 1, 1>(group, zp) : pick<WT, 1, 2>(group, zp);
}

// Clusters of sk CTAs that the device holds at once.  A cluster sits inside one group of SMs, so for sk > 2 this is less
// than the SMs suggest, and a launch that exceeds it by one cluster takes another round.
int active_clusters(const void* kern, size_t smem, int sk, int resident) {
    if (sk == 1) return resident * sm_count();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, (unsigned)sk);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = (unsigned)sk;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) n = 0;
    cudaGetLastError();
    return n;
}

struct Plan {
    int wr, sk, seg;
    size_t smem;                // launch size, 0 = the kernel cannot run here
};

// Row warps, cluster size and staging of a launch, by an estimate of its time that knows four things: a CTA costs 2.5 us
// to start, stage and reduce; a CTA alone on an SM takes 0.95 us for an iteration of its warps (32 KB of weights) with 8
// tokens, 2.0 with 16; several on an SM share the memory at 0.87 and 1.1 us per CTA; and rounds are whole.  (Fitted to
// sweeps over 4096 x 4096 .. 28672 x 8192 and the expert shapes; the best and the chosen split differ by at most 8 % there.)
// `slots` > 0: the cluster is that many CTAs, each over the whole k (the second product of a single token).
Plan make_plan(const void* kern, int mode, int nt, int group, bool zp, int tiles, int units, int items, int slots) {
    Plan best{1, 1, 1, 0};
    double best_us = 1e30;
    const size_t ring = (size_t)kWarps * kDI * kRT * 1024;
    for (int wr = 1; wr <= kWarps; wr *= 2)
        for (int sk = slots > 0 ? slots : 1; sk <= (slots > 0 ? slots : std::min(8, units)); ++sk) {
            const int ro = (mode == 1 ? kRT / 2 : kRT) * wr, wk = kWarps / wr;
            if (wr > 1 && ro / 2 >= tiles) continue;                    // half of the row warps would have nothing to do
            auto staged = [&](int n) { return (size_t)nt * 8 * (n * 256 + 32) + (size_t)wr * kRT * n * (128 / group) * (zp ? 48 : 32); };
            // a segment: the CTA's whole k range where it fits beside the ring, else as many units as do
            const int per_rank = slots > 0 ? units : (units + sk - 1) / sk;
            int seg = per_rank;
            while (ring + staged(seg) > 200 * 1024) seg = (seg + 1) / 2;
            const size_t smem = std::max(ring + staged(seg), (size_t)kWarps * kRT * nt * 8 * kTokStride * 4);
            int resident = 0;
            const size_t launch_smem = umma::prepare_kernel(kern, kWarps * 32, smem, 0, false, &resident);
            if (launch_smem == 0) continue;
            const int room = active_clusters(kern, launch_smem, sk, resident);
            if (room < 1) continue;
            const double clusters = (double)((tiles + ro - 1) / ro) * items, iters = (per_rank + wk - 1) / wk;
            const double rounds = std::ceil(clusters / room), share = std::min<double>(resident, std::ceil(clusters * sk / sm_count()));
            const double iter_us = nt == 1 ? std::max(0.95, 0.87 * share) : std::max(2.0, 1.1 * share);
            const double us = rounds * (2.5 * ((per_rank + seg - 1) / seg) + iters * iter_us) + (sk > 1 ? 0.5 : 0.0);
            if (us < best_us) {
                best_us = us;
                best = Plan{wr, sk, seg, launch_smem};
            }
        }
    return best;
}

Plan cached_plan(const void* kern, int mode, int nt, int group, bool zp, int tiles, int units, int items, int slots) {
    static std::mutex mu;
    static std::map<std::array<long long, 6>, Plan> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return Plan{1, 1, 1, 0};
    const std::array<long long, 6> key{(long long)(uintptr_t)kern, dev, tiles, units, items, slots};
    std::lock_guard<std::mutex> lock(mu);
    auto it = known.find(key);
    if (it != known.end()) return it->second;
    if (known.size() > 4096) known.clear();              // a server sees a few hundred shapes
    return known[key] = make_plan(kern, mode, nt, group, zp, tiles, units, items, slots);
}

}  // namespace

int launch_w4_mma(int mode, int wt, W4KernelParams p, const W4Weights& w, int items, int likely_items, int nt, cudaStream_t s) {
    const bool zp = w.z != nullptr;
    p.kc = (p.k + kW4BlockK - 1) / kW4BlockK;
    p.groups = p.k / w.group;
    p.q = w.q;
    p.s = reinterpret_cast<const uint32_t*>(w.s);
    p.z = reinterpret_cast<const uint16_t*>(w.z);
    if (items > 65535) return fail(kUnsupported, "w4: %d work items exceed one launch", items);
    const void* kern = wt == kFP16 ? pick<kFP16>(mode, nt, w.group, zp) : pick<kBF16>(mode, nt, w.group, zp);
    if (kern == nullptr) return fail(kInvalidArg, "w4: %d tokens per item are not built", 8 * nt);
    const Plan q = cached_plan(kern, mode, nt, w.group, zp, p.out_tiles, (p.kc + 1) / 2, mode == 2 && p.ids ? 1 : likely_items,
                               mode == 2 && p.ids ? p.topk : 0);
    if (q.smem == 0) return fail(kCudaError, "w4: the streaming kernel cannot be launched on this device");
    p.seg_units = q.seg;
    p.row_warps = q.wr;
    const int ro = (mode == 1 ? kRT / 2 : kRT) * q.wr;
    int static_weights = option(kOptStaticWeights);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.out_tiles + ro - 1) / ro), (unsigned)q.sk, (unsigned)(mode == 2 && p.ids ? 1 : items));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = q.smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    cfg.numAttrs = launch_attrs(attr, q.sk);
    void* args[2] = {&p, &static_weights};
    const cudaError_t e = cudaLaunchKernelExC(&cfg, kern, args);
    if (e != cudaSuccess) return fail(kCudaError, "w4 launch: %s", cudaGetErrorString(e));
    return kOk;
}

}  // namespace mlk
