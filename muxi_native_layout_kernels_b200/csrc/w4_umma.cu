// 4-bit weights, more than a few tokens: products on the 5th-generation tensor cores (dense, and the experts of a mixture).
//
// A CTA computes 128 weight rows x NP tokens (swap-AB: rows are the M dimension of the MMA), fp32 accumulator in tensor
// memory.  Per stage of 128 k:
//   TMA (one thread)     packed blocks, scales and zero points of the rows -> raw ring; token tile (128-byte swizzle) -> ring
//   8 converter warps    raw block -> registers -> tensor memory.  A lane's 16 bytes of a block are, word by word, the
//                        16-lane x 256-bit fragment of a tensor-memory store (w4.cuh), so a row group's 128 k are two
//                        16-byte shared loads, the decode, and one tcgen05.st of 32 registers.  Two sets of four warps
//                        take the stages in turn, or, where a CTA holds a gate and an up tile, one tile each
//   MMA (one thread)     tcgen05.mma with the weights in tensor memory and the token tile in shared memory
// The decoded weight is (q - z) s rounded once to the activation type, the value a dequantised checkpoint holds: scaling
// the fp32 sums instead would take one accumulator pass per group.  In bf16 the decode leaves a constant factor of the row
// (w4.cuh) that is put back on the accumulator.
// What bounds it: up to about 64 tokens the decode (13 packed instructions per word of eight weights) and the hand-offs
// between the roles, at NP = 256 the tensor pipe.  Small grids split k over a cluster; partial tiles are added through
// distributed shared memory in a fixed order.
// Measured (us, and the floor by bytes or by the tensor peak): 14336 x 4096 with zero points per 32 at 61 tokens 17.2 (5.7;
// issue slots 49 % busy, tensor pipe 27 %), 8192 x 8192 at 500 tokens 53 at full clocks, 62 under the power cap (40.6; tensor pipe
// 62 %), 512 tokens x 8 on 128 experts of 2048 x 768 in fp16 with zero points 151, under the power cap 165-173 (51).
// The parts of a stage overlap only in part: at 37888 x 8192 and 64 tokens (45 us) a copy without the stores to tensor memory
// took 41, without the MMAs 36, without the decode 38, with none of them 30.  An MMA with its rows in tensor memory takes
// 20 / 32 / 64 / 128 cycles at 32 / 64 / 128 / 256 tokens.  Three slots, six raw stages, or one CTA per SM with all of the
// tensor memory (142 -> 167 us for 512 tokens on the experts in bf16) were no better.
// A store to tensor memory in the 16 x 256-bit shape moves 254 bytes per SM and cycle (16 x 128 bit 455, 32 x 32 bit 372):
// that shape is taken because it needs no exchange between lanes, and the stores are not what a stage waits for.
#include <algorithm>
#include <cmath>

#include "umma_common.cuh"
#include "w4_kernels.cuh"

namespace mlk {

namespace {

using namespace umma;

constexpr int kStageK = 128;
constexpr int kRaw = 8 * 2 * kW4BlockBytes;        // packed bytes of 128 rows x 128 k
constexpr int kConv = 8;                           // converter warps
constexpr int kThreads = 64 + kConv * 32;
constexpr uint32_t kAll = 0xFFFFFFFFu;             // a whole warp

// Tensor memory: accumulators, then decoded tiles of 64 columns per weight tile.  With one weight tile per CTA the two
// converter sets take the stages in turn, and the number of slots (and of raw stages) is even: a set that shares its
// barriers with the other one would miss phases of them.
constexpr int tmem_columns(int na, int np) { return na == 1 ? (np <= 128 ? 256 : 512) : (np <= 64 ? 256 : 512); }
constexpr int conv_slots(int na, int np) {
    const int fit = (tmem_columns(na, np) - na * np) / (na * 64);
    return na == 2 ? fit : fit / 2 * 2;
}
constexpr int raw_stages(int na) { return na == 2 ? 3 : 4; }
// Dense products with small grids split k over a cluster: the partial tiles fit into the rings up to 128 tokens.
constexpr bool can_split(int mode, int np) { return mode == 0 && np <= 128; }
constexpr int token_stages(int np) { return np >= 256 ? 2 : (np >= 128 ? 2 : 3); }

struct UmmaParams {
    W4KernelParams k;
    int stages;                 // stages of 128 k
    int run;                    // consecutive row tiles of a CTA (1 where a cluster splits k)
    int* status;
};

__device__ __forceinline__ void tmem_st_16x256b_x8(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
          "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
          "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
          "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}

// One lane of a converged warp.  The role loops run with the whole warp, so that ring positions, descriptors and tensor-memory
// addresses stay in uniform registers, and only the issuing instructions sit behind this predicate (in a branch on the
// lane number each tcgen05.mma cost some 80 cycles of register moves, 1300 for a stage with its waits).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

template <int WT>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    if constexpr (WT == kBF16) return mul_bf16x2(a, b);
    else {
        uint32_t r;
        asm("mul.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
}

// G: group size; ZP: zero points given; MODE as in the streaming kernel.
template <int WT, int NP, int G, bool ZP, int MODE>
__global__ void __launch_bounds__(kThreads, tmem_columns(MODE == 1 ? 2 : 1, NP) == 512 ? 1 : 2)
    w4_umma_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_s,
                   const __grid_constant__ CUtensorMap map_z, const __grid_constant__ CUtensorMap map_x,
                   const UmmaParams u, const int static_weights) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    using D = W4Decode<WT>;
    constexpr int NA = MODE == 1 ? 2 : 1;
    constexpr int NG = kStageK / G;
    constexpr int S2 = conv_slots(NA, NP), RS = raw_stages(NA), SB = token_stages(NP);
    static_assert(S2 >= 1 && (NA == 2 || (S2 % 2 == 0 && RS % 2 == 0)), "a converter set has to see every phase of its barriers");
    constexpr uint32_t kTmemCols = tmem_columns(NA, NP);
    constexpr int kTile = kRaw + 256 * NG + (ZP ? 128 * NG : 0);      // raw stage of one weight tile
    constexpr int kB = NP * 256;                                     // token tile of a stage: two 64-k halves
    __shared__ __align__(8) uint64_t bars[2 * RS + 2 * S2 + 2 * SB + 2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    // MODE 2: slot and routing weight of every token of the item.  (Fetched where they are used, each column of the read-out
    // waits for two dependent loads behind the stores of the one before: 181 instead of 153 us for 512 tokens x 8 on 128
    // experts of 2048 x 768, both products.)
    __shared__ int slot_of[MODE == 2 ? NP : 1];
    __shared__ float weight_of[MODE == 2 ? NP : 1];

    const W4KernelParams& p = u.k;
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const int row_tiles = (p.out_tiles + 7) / 8, tile = blockIdx.x * u.run, rank = can_split(MODE, NP) ? blockIdx.y : 0, SK = can_split(MODE, NP) ? gridDim.y : 1;
    const int run = min(u.run, row_tiles - tile);

    const bool early = MODE == 0 && static_weights;  // weights may be fetched before the kernel in front has finished
    if (!early) pdl_wait();
    int mat = 0, pos0 = 0, row0 = 0, ntok;       // row0: first row of the token tile
    if constexpr (MODE == 0) {
        row0 = blockIdx.z * NP;
        ntok = min(NP, p.n - row0);
    } else {
        const int items = p.worklist[0].x;
        const int4 item = p.worklist[1 + blockIdx.z];
        if ((int)blockIdx.z >= items) return;
        mat = item.x; pos0 = item.y; ntok = item.z; row0 = item.w;
    }
    if constexpr (MODE == 2) {
        for (int c = tid; c < ntok; c += kThreads) {
            const int slot = p.sorted[pos0 + c];
            slot_of[c] = slot;
            weight_of[c] = load_scalar16<WT>(p.topk_weights, slot);
        }
    }
    const int st0 = (int)((long long)u.stages * rank / SK), n = (int)((long long)u.stages * (rank + 1) / SK) - st0;
    const int total = n * run;                   // stages of all row tiles, one after the other

    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t x_base = base, r_base = base + SB * kB;
    const uint32_t bar0 = smem_u32(bars);
    auto raw_full = [&](int s) { return bar0 + 8u * s; };
    auto raw_empty = [&](int s) { return bar0 + 8u * (RS + s); };
    auto cv_full = [&](int s) { return bar0 + 8u * (2 * RS + s); };
    auto cv_empty = [&](int s) { return bar0 + 8u * (2 * RS + S2 + s); };
    auto x_full = [&](int s) { return bar0 + 8u * (2 * RS + 2 * S2 + s); };
    auto x_empty = [&](int s) { return bar0 + 8u * (2 * RS + 2 * S2 + SB + s); };
    const uint32_t acc_full = bar0 + 8u * (2 * RS + 2 * S2 + 2 * SB), acc_empty = acc_full + 8u;

    if (tid == 0) {
        for (int s = 0; s < RS; ++s) {
            mbar_init(raw_full(s), 1);
            mbar_init(raw_empty(s), 4 * NA);     // one arrival per converter warp that reads the stage
        }
        for (int s = 0; s < S2; ++s) {
            mbar_init(cv_full(s), 4 * NA);
            mbar_init(cv_empty(s), 1);           // tcgen05.commit
        }
        for (int s = 0; s < SB; ++s) {
            mbar_init(x_full(s), 1);
            mbar_init(x_empty(s), 1);            // tcgen05.commit
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, kConv);             // one arrival per warp that has read its part
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }

    const int g16 = mat * p.mat_tiles + tile * 8;                      // first 16-row group
    auto load_raw = [&](int i, int t, int s) {   // stage i of row tile t of the run
        const uint64_t wpol = l2_evict_first_policy();
        if (elect_one()) {
            mbar_expect_tx(raw_full(s), NA * kTile);
#pragma unroll
            for (int w = 0; w < NA; ++w) {
                const uint32_t dst = r_base + (s * NA + w) * kTile;
                const int g = g16 + t * 8 + (w == 1 ? p.out_tiles : 0);
                tma_load_3d_hint(dst, &map_q, raw_full(s), 0, (st0 + i) * 2, g, wpol);
                tma_load_3d(dst + kRaw, &map_s, raw_full(s), 0, (st0 + i) * NG, g);
                if constexpr (ZP) tma_load_3d(dst + kRaw + 256 * NG, &map_z, raw_full(s), 0, (st0 + i) * NG, g);
            }
        }
        __syncwarp();
    };
    int ri = 0, rs = 0, rk = 0, rt = 0;          // the producer's next raw stage, its ring slot, and as (stage, row tile)
    uint32_t rpar = 1;                           // parity that says the slot is free: the first round finds it so
    if (early) {
        if (warp == 0) {
            __syncwarp();
            for (; ri < min(total, RS); ++ri) {
                load_raw(rk, rt, ri);
                if (++rk == n) { rk = 0; ++rt; }
            }
            if (ri == RS) rpar ^= 1u;
            rs = ri % RS;
        }
        pdl_wait();
    }
    // Tensor memory is taken when the kernel in front has finished, and the next kernel is let in when it has been: a CTA
    // never holds columns while it waits for a kernel that may still be asking for them.
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, tmem_slot, 0);
    pdl_launch_dependents();

    // ---- read-out of one row tile where this CTA has the whole sums: set 0 the lower half of the tokens, set 1 the upper,
    // straight from tensor memory, a thread has one row, neighbouring lanes neighbouring rows ----
    const size_t ld = (size_t)p.out_tiles * 16;
    auto silu_mul = [](float g, float h) { return g / (1.f + __expf(-g)) * h; };
    auto read_out = [&](int rt, int quad, int set) {
        const int lrow = quad * 32 + lane, row = rt * kTileM + lrow;
        const float f = (lrow & 8) ? D::kFactorHigh : D::kFactorLow;   // the decode's constant factor of this row
        const uint32_t at = tmem + ((uint32_t)(quad * 32) << 16);
        const bool mine = row < p.out_tiles * 16;
        const float alpha = MODE == 0 ? f * p.alpha : f;
        const float bias = MODE == 0 && mine && p.bias ? load_scalar16<WT>(p.bias, row) : 0.f;
        uint16_t* out = reinterpret_cast<uint16_t*>(p.C) + (size_t)(row0 + set * (NP / 2)) * ld + row;
#pragma unroll 1
        for (int c0 = set * (NP / 2); c0 < (set + 1) * (NP / 2) && c0 < ntok; c0 += 16) {
            uint32_t a[16], b[16];
            tmem_ld16(at + c0, a);
            if constexpr (NA == 2) tmem_ld16(at + NP + c0, b);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            const int left = mine ? ntok - c0 : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (i < left) {
                    const float v = __uint_as_float(a[i]);
                    if constexpr (MODE == 0) {
                        store16<WT>(out, 0, fmaf(alpha, v, bias));
                    } else if constexpr (MODE == 1) {
                        store16<WT>(out, 0, silu_mul(f * v, f * __uint_as_float(b[i])));
                    } else {
                        reinterpret_cast<float*>(p.C)[(size_t)slot_of[c0 + i] * ld + row] = weight_of[c0 + i] * (f * v);
                    }
                }
                out += ld;
            }
        }
    };

    int raw_issued = 0, x_issued = 0;
    if (warp == 0) {
        // ---- TMA producer: raw weights and token tiles are two independent streams, polled without blocking ----
        int xi = 0, xs = 0, xk = 0;              // the next token tile, its ring slot, its stage within a row tile
        uint32_t xpar = 1;
        uint32_t idle = 0;
        while ((xi < total || ri < total) && !__any_sync(kAll, abort_flag)) {
            bool progressed = false;
            if (ri < total && __any_sync(kAll, mbar_test_wait(raw_empty(rs), rpar))) {
                load_raw(rk, rt, rs);
                ++ri;
                if (++rk == n) { rk = 0; ++rt; }
                if (++rs == RS) { rs = 0; rpar ^= 1u; }
                progressed = true;
            }
            if (xi < total && __any_sync(kAll, mbar_test_wait(x_empty(xs), xpar))) {
                if (elect_one()) {
                    mbar_expect_tx(x_full(xs), kB);
                    tma_load_2d(x_base + xs * kB, &map_x, x_full(xs), (st0 + xk) * kStageK, row0);
                    tma_load_2d(x_base + xs * kB + NP * 128, &map_x, x_full(xs), (st0 + xk) * kStageK + 64, row0);
                }
                __syncwarp();
                ++xi;
                if (++xk == n) xk = 0;
                if (++xs == SB) { xs = 0; xpar ^= 1u; }
                progressed = true;
            }
            if (progressed) {
                idle = 0;
            } else if (++idle > 4 * kSpinLimit) {
                if (u.status && lane == 0) atomicExch(u.status, 1);
                abort_flag = 1;
            } else {
                __nanosleep(40);
            }
            __syncwarp();
        }
        raw_issued = ri;
        x_issued = xi;
    } else if (warp == 1) {
        // ---- MMA issuer ----
        constexpr uint32_t idesc = instr_desc<WT, NP>();
        const uint64_t d0 = smem_desc(x_base, 16, 1024, 2);
        const uint32_t a0 = tmem + NA * NP;
        int s2 = 0, sb = 0;
        uint32_t par2 = 0, parb = 0, para = 1;   // para: the parity that says the accumulator is free
        for (int f = 0, i = 0; f < total; ++f) {
            bool ready = mbar_wait(x_full(sb), parb) && mbar_wait(cv_full(s2), par2);
            if (i == 0) {
                ready = ready && mbar_wait(acc_empty, para);
                para ^= 1u;
            }
            if (__any_sync(kAll, !ready || abort_flag)) {
                if (!abort_flag && u.status && lane == 0) atomicExch(u.status, 2);
                abort_flag = 1;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t db = d0 + (uint32_t)(sb * (kB >> 4));
            const uint32_t da = a0 + s2 * (NA * 64);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < kStageK / 16; ++kk)
#pragma unroll
                    for (int w = 0; w < NA; ++w)
                        umma_f16_ts(tmem + w * NP, da + w * 64 + kk * 8, db + ((kk >> 2) * (NP * 128 >> 4) + (kk & 3) * 2), idesc,
                                    kk > 0 ? 1u : (uint32_t)(i > 0));
                umma_commit(cv_empty(s2));
                umma_commit(x_empty(sb));
                if (i == n - 1) umma_commit(acc_full);
            }
            __syncwarp();
            if (++i == n) i = 0;
            if (++s2 == S2) { s2 = 0; par2 ^= 1u; }
            if (++sb == SB) { sb = 0; parb ^= 1u; }
        }
    } else if (warp >= 2) {
        // ---- converter warps ----
        const int quad = warp & 3, set = (warp - 2) >> 2, r = lane >> 2;
        constexpr int kStep = NA == 2 ? 1 : 2;   // stages of a set
        int s = NA == 2 ? 0 : set, s2 = s % S2;
        uint32_t parr = 0, par2 = 1, para = 0;   // par2: the parity that says the slot is free
        int f = s;
        for (int t = 0; t < run; ++t) {
          for (; f < (t + 1) * n; f += kStep) {
            bool ok = mbar_wait(raw_full(s), parr) && !abort_flag;
            uint32_t v[32];
#pragma unroll
            for (int h = 0; h < 2; ++h) {                              // the two 16-row groups of this warp's 32 lanes
                const int w = NA == 2 ? set : 0, rg = 2 * quad + h;
                if (ok) {
                    const uint8_t* const t = base_ptr + SB * kB + (s * NA + w) * kTile;
                    const uint4 b0 = *reinterpret_cast<const uint4*>(t + rg * 1024 + lane * 16);
                    const uint4 b1 = *reinterpret_cast<const uint4*>(t + rg * 1024 + kW4BlockBytes + lane * 16);
                    const uint32_t words[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const uint32_t sc = *reinterpret_cast<const uint32_t*>(t + kRaw + (rg * NG + g) * 32 + 4 * r);
                        const uint32_t sl = __byte_perm(sc, 0u, 0x1010), sh = __byte_perm(sc, 0u, 0x3232);
                        uint32_t zl, zh;
                        D::zero(ZP ? *reinterpret_cast<const uint16_t*>(t + kRaw + 256 * NG + (rg * NG + g) * 16 + 2 * r) : 0x0808u, zl, zh);
#pragma unroll
                        for (int j = g * (8 / NG); j < (g + 1) * (8 / NG); ++j) {
                            uint32_t a[4];
                            D::word(words[j], zl, zh, a);
                            v[4 * j + 0] = mul2<WT>(a[0], sl);         // row r, columns 2t and 2t + 1
                            v[4 * j + 1] = mul2<WT>(a[2], sl);
                            v[4 * j + 2] = mul2<WT>(a[1], sh);         // row r + 8
                            v[4 * j + 3] = mul2<WT>(a[3], sh);
                        }
                    }
                }
                if (h == 0) {                                          // the slot's previous MMAs are complete
                    ok = __all_sync(kAll, ok && mbar_wait(cv_empty(s2), par2));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                tmem_st_16x256b_x8(tmem + ((uint32_t)(quad * 32 + h * 16) << 16) + NA * NP + (s2 * NA + w) * 64, v);
            }
            if (!ok) {
                if (!abort_flag && u.status && lane == 0) atomicExch(u.status, 8);
                abort_flag = 1;
                break;
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(cv_full(s2)) : "memory");
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(raw_empty(s)) : "memory");
            }
            s += kStep;
            if (s >= RS) { s -= RS; parr ^= 1u; }
            s2 += kStep;
            if (s2 >= S2) { s2 -= S2; par2 ^= 1u; }
          }
            // the row tile's accumulator is complete
            if (__any_sync(kAll, abort_flag || !mbar_wait(acc_full, para))) {
                if (!abort_flag && u.status && lane == 0) atomicExch(u.status, 3);
                abort_flag = 1;
                break;
            }
            para ^= 1u;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (SK > 1) break;                   // read out below, with the cluster
            read_out(tile + t, quad, set);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(acc_empty) : "memory");
        }
    }
    __syncwarp();

    // ---- cluster: partial tiles over the k parts ----
    if constexpr (can_split(MODE, NP)) {
        if (SK > 1) {
            const int rows_left = p.out_tiles * 16 - tile * kTileM;        // rows of the matrix in this tile
            constexpr int kChunk = NP < 64 ? NP : 64;                      // tokens of one pass through shared memory
            // [token][row] of a chunk of tokens in the (idle) rings, added over the cluster in rank order
            float* const red = reinterpret_cast<float*>(base_ptr);
            uint32_t remote[8];
#pragma unroll
            for (int q = 0; q < 8; ++q)
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote[q]) : "r"(base), "r"(q < SK ? q : 0));
#pragma unroll 1
            for (int cb = 0; cb < NP; cb += kChunk) {
                if (warp >= 2 && !abort_flag) {
                    const int quad = warp & 3, set = (warp - 2) >> 2, lrow = quad * 32 + lane;
                    const float f = (lrow & 8) ? D::kFactorHigh : D::kFactorLow;
#pragma unroll
                    for (int c0 = 0; c0 < kChunk / 2; c0 += 16) {
                        const int c = set * (kChunk / 2) + c0;
                        uint32_t a[16];
                        tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + cb + c, a);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int i = 0; i < 16; ++i) red[(c + i) * kTileM + lrow] = f * __uint_as_float(a[i]);
                    }
                }
                __syncwarp();
                asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
                // this rank's share of the tokens, four rows of one token per thread and step
                const int left = max(0, min(kChunk, ntok - cb));
                for (int e = left * rank / SK * 32 + tid; e < left * (rank + 1) / SK * 32; e += kThreads) {
                    const int c = e >> 5, lrow = (e & 31) * 4, row = tile * kTileM + lrow;
                    const uint32_t off = 4u * (c * kTileM + lrow);
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (q < SK) {
                            float4 o;
                            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(o.x), "=f"(o.y), "=f"(o.z), "=f"(o.w) : "r"(remote[q] + off) : "memory");
                            v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
                        }
                    if (lrow >= rows_left) continue;                       // whole 16-row groups are in or out
                    float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (p.bias) b = make_float4(load_scalar16<WT>(p.bias, row), load_scalar16<WT>(p.bias, row + 1), load_scalar16<WT>(p.bias, row + 2), load_scalar16<WT>(p.bias, row + 3));
                    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.C) + (size_t)(row0 + cb + c) * ld + row) =
                        make_uint2(pack2<WT>(fmaf(p.alpha, v.x, b.x), fmaf(p.alpha, v.y, b.y)),
                                   pack2<WT>(fmaf(p.alpha, v.z, b.z), fmaf(p.alpha, v.w, b.w)));
                }
                __syncwarp();
                asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            }
        }
    }

    // ---- teardown: if the pipeline stopped early, wait (bounded) for the TMA copies still in flight ----
    if (warp == 0 && lane == 0 && abort_flag) {
        for (int i = max(0, raw_issued - RS); i < raw_issued; ++i) mbar_wait(raw_full(i % RS), (i / RS) & 1);
        for (int i = max(0, x_issued - SB); i < x_issued; ++i) mbar_wait(x_full(i % SB), (i / SB) & 1);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

template <int WT, int NP, int MODE>
const void* pick(int group, bool zp) {
    if (group == 128) return zp ? reinterpret_cast<const void*>(w4_umma_kernel<WT, NP, 128, true, MODE>)
                                : reinterpret_cast<const void*>(w4_umma_kernel<WT, NP, 128, false, MODE>);
    if (group == 64) return zp ? reinterpret_cast<const void*>(w4_umma_kernel<WT, NP, 64, true, MODE>)
                               : reinterpret_cast<const void*>(w4_umma_kernel<WT, NP, 64, false, MODE>);
    return zp ? reinterpret_cast<const void*>(w4_umma_kernel<WT, NP, 32, true, MODE>)
              : reinterpret_cast<const void*>(w4_umma_kernel<WT, NP, 32, false, MODE>);
}
template <int WT>
const void* pick(int mode, int np, int group, bool zp) {
    if (mode == 0) {
        switch (np) {
            case 32: return pick<WT, 32, 0>(group, zp);
            case 64: return pick<WT, 64, 0>(group, zp);
            case 128: return pick<WT, 128, 0>(group, zp);
            case 256: return pick<WT, 256, 0>(group, zp);
        }
    } else if (mode == 1) {
        switch (np) {
            case 32: return pick<WT, 32, 1>(group, zp);
            case 64: return pick<WT, 64, 1>(group, zp);
            case 128: return pick<WT, 128, 1>(group, zp);
        }
    } else {
        switch (np) {
            case 32: return pick<WT, 32, 2>(group, zp);
            case 64: return pick<WT, 64, 2>(group, zp);
            case 128: return pick<WT, 128, 2>(group, zp);
        }
    }
    return nullptr;
}

// Tensor maps over 16-row groups: packed blocks [groups16][kc][128 words], scales [groups16][groups][16], zero points alike;
// and over the token rows.  Encoded for every launch.
bool map_packed(CUtensorMap* m, const void* q, long long groups16, int kc) {
    const cuuint64_t dims[3] = {128, (cuuint64_t)kc, (cuuint64_t)groups16};
    const cuuint64_t strides[2] = {kW4BlockBytes, (cuuint64_t)kc * kW4BlockBytes};
    const cuuint32_t box[3] = {128, 2, 8}, estr[3] = {1, 1, 1};
    return encode_fn()(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(q), dims, strides, box, estr,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool map_groups(CUtensorMap* m, const void* v, long long groups16, int groups, int group, int elem) {
    const cuuint64_t dims[3] = {16, (cuuint64_t)groups, (cuuint64_t)groups16};
    const cuuint64_t strides[2] = {(cuuint64_t)16 * elem, (cuuint64_t)groups * 16 * elem};
    const cuuint32_t box[3] = {16, (cuuint32_t)(kStageK / group), 8}, estr[3] = {1, 1, 1};
    return encode_fn()(m, elem == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(v), dims,
                       strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool map_tokens(CUtensorMap* m, const void* X, int n, int k, int wt, int np) {
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)n};
    const cuuint64_t strides[1] = {(cuuint64_t)k * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)np}, estr[2] = {1, 1};
    return encode_fn()(m, wt == kFP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(X),
                       dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Estimated time (us) of a product: a CTA costs 5 us to start and to read out (1 more with a cluster), a stage of 128 k on an
// SM the time below, whatever the number of CTAs that share it, and rounds are whole.  (Fitted to sweeps over 4096 x 4096 ..
// 28672 x 8192 at 8 to 500 tokens; within 15 % there.)
double stage_us(int np) { return np == 32 ? 0.33 : (np == 64 ? 0.37 : (np == 128 ? 0.51 : 0.70)); }
double estimate(int tiles, int tokens, int stages, int np, int sk) {
    const double ctas = (double)tiles * tokens * sk, resident = np == 256 ? 1.0 : 2.0;
    const double slots = sm_count() * resident * (sk > 2 ? 0.9 : 1.0);     // clusters of more than two do not fill every SM
    const double rounds = std::ceil(ctas / slots), share = std::min(resident, std::ceil(ctas / sm_count()));
    return rounds * (5.0 + (sk > 1 ? 1.0 : 0.0) + std::ceil((double)stages / sk) * stage_us(np) * share);
}

}  // namespace

W4UmmaPlan w4_umma_plan(int rows16, int n, int k) {
    const int tiles = (rows16 + 7) / 8, stages = (k + kStageK - 1) / kStageK;
    W4UmmaPlan best{32, 1, 1e30};
    for (int np = 32; np <= 256; np *= 2) {
        const int tokens = (n + np - 1) / np;
        for (int sk = 1; sk <= (can_split(0, np) ? 8 : 1) && sk <= stages; ++sk) {
            const double us = estimate(tiles, tokens, stages, np, sk);
            if (us < best.us) best = W4UmmaPlan{np, sk, us};
        }
        if (tokens == 1) break;                  // a wider tile would only compute more columns that nobody reads
    }
    return best;
}

// One product.  mode 0: X = tokens [n, k]; mode 1: X = gathered tokens [x_rows, k]; mode 2: X = activations [x_rows, k].
// np: token tile; sk: CTAs of a cluster along k; run: consecutive row tiles of a CTA; items: token tiles (mode 0) or an upper bound of the work items.
int launch_w4_umma(int mode, int wt, const W4KernelParams& kp, const W4Weights& w, long long matrices, int x_rows, int np, int sk, int run,
                   int items, int* status, cudaStream_t s) {
    const bool zp = w.z != nullptr;
    UmmaParams u{};
    u.k = kp;
    u.k.kc = (kp.k + kW4BlockK - 1) / kW4BlockK;
    u.k.groups = kp.k / w.group;
    u.stages = (u.k.kc + 1) / 2;
    u.run = std::max(1, std::min(run, (kp.out_tiles + 7) / 8));
    u.status = status;
    const void* kern = wt == kFP16 ? pick<kFP16>(mode, np, w.group, zp) : pick<kBF16>(mode, np, w.group, zp);
    if (kern == nullptr) return fail(kInvalidArg, "w4 (tcgen05): token tile %d is not built", np);
    if (sk < 1 || sk > 8 || sk > u.stages) return fail(kInvalidArg, "w4 (tcgen05): cluster size %d out of range", sk);
    if (sk > 1 && u.run > 1) return fail(kInvalidArg, "w4 (tcgen05): a cluster takes one row tile");
    if (sk > 1 && !can_split(mode, np)) return fail(kInvalidArg, "w4 (tcgen05): k is not split in mode %d with %d tokens per tile", mode, np);
    if (encode_fn() == nullptr) return fail(kUnsupported, "w4 (tcgen05): cuTensorMapEncodeTiled is not available");
    if (items > 65535) return fail(kUnsupported, "w4 (tcgen05): %d work items exceed one launch", items);
    const int na = mode == 1 ? 2 : 1, ng = kStageK / w.group;
    const long long groups16 = matrices * kp.mat_tiles;
    if (groups16 > 0x7FFFFFFF) return fail(kUnsupported, "w4 (tcgen05): too many rows");
    CUtensorMap mq, ms, mz, mx;
    if (!map_packed(&mq, w.q, groups16, u.k.kc)) return fail(kUnsupported, "w4 (tcgen05): weight tensor map rejected");
    if (!map_groups(&ms, w.s, groups16, u.k.groups, w.group, 2)) return fail(kUnsupported, "w4 (tcgen05): scale tensor map rejected");
    if (zp) {
        if (!map_groups(&mz, w.z, groups16, u.k.groups, w.group, 1)) return fail(kUnsupported, "w4 (tcgen05): zero-point tensor map rejected");
    } else {
        mz = ms;
    }
    if (!map_tokens(&mx, kp.X, x_rows, kp.k, wt, np)) return fail(kUnsupported, "w4 (tcgen05): activation tensor map rejected");
    const size_t tile = kRaw + 256 * ng + (zp ? 128 * ng : 0);
    const size_t rings = (size_t)token_stages(np) * np * 256 + (size_t)raw_stages(na) * na * tile;
    const size_t partial = sk > 1 ? (size_t)std::min(np, 64) * kTileM * 4 : 0;
    const size_t smem = prepare_kernel(kern, kThreads, std::max(rings, partial) + 1024, tmem_columns(na, np));
    if (smem == 0) return fail(kCudaError, "w4 (tcgen05): a CTA with %d tokens does not fit on this device", np);
    int static_weights = option(kOptStaticWeights);
    cudaLaunchConfig_t cfg = {};
    const int row_tiles = (kp.out_tiles + 7) / 8;
    cfg.gridDim = dim3((unsigned)((row_tiles + u.run - 1) / u.run), (unsigned)sk, (unsigned)items);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    cfg.numAttrs = launch_attrs(attr, sk);
    void* args[6] = {&mq, &ms, &mz, &mx, &u, &static_weights};
    const cudaError_t e = cudaLaunchKernelExC(&cfg, kern, args);
    if (e != cudaSuccess) return fail(kCudaError, "w4 (tcgen05) launch: %s", cudaGetErrorString(e));
    return kOk;
}

}  // namespace mlk
