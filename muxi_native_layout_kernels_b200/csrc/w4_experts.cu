// The experts of a mixture layer with 4-bit weights: y[t] = sum_j p[t, j] W2_e (silu(Wg_e x_t) * (Wu_e x_t)), e = ids[t, j].
//
// Sequence: alignment (routed slots grouped by expert, one work item per expert and up to 8, 32, 64 or 128 slots) -> with
// more than a few slots per expert the token rows in slot order -> gate/up product with SiLU on the fp32 sums -> down
// product, weighted, into one fp32 row per slot -> sum of a token's rows in slot order with one rounding.  A single token takes two
// launches instead: its slots are the work items, and clusters of them sum the result.  The activation between the two
// products is rounded to the 16-bit activation type, as in the 16-bit and e4m3 expert kernels.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "moe.cuh"
#include "w4_kernels.cuh"

namespace mlk {

namespace {

// Experts: what the alignment takes.  Slots: the work items of a launch are its grid's z dimension, and from 80 slots an
// expert on they hold 128 slots each, with one unfilled per expert at worst.
constexpr int kMaxExperts = 1024;
constexpr int kMaxSlots = (65535 - kMaxExperts) * 128;

constexpr long long align256(long long b) { return (b + 255) / 256 * 256; }

struct Layout {
    long long sorted, cumsum, nblocks, block_expert, worklist, act, scratch, bytes;
};

// Work items of at least `block` slots' capacity: no expert's last item is full, at worst.
long long max_items(long long slots, int E, int block) { return std::min<long long>(slots, slots / block + E); }

Layout layout(int T, int E, int topk, int H, int I) {
    const long long slots = (long long)T * topk;
    Layout l{};
    long long at = 0;
    auto take = [&](long long bytes) { const long long here = at; at += align256(bytes); return here; };
    l.sorted = take(slots * 4);
    l.cumsum = take(((long long)E + 1) * 4);
    l.nblocks = take(4);
    l.block_expert = take(slots * 4);
    l.worklist = take((1 + max_items(slots, E, 8)) * 16);
    l.act = take(slots * I * 2);
    l.scratch = take(slots * H * 4);
    l.bytes = at;
    return l;
}

int check_weights(const W4Weights& w, long long k, const char* name) {
    if (!w.q || !w.s) return fail(kInvalidArg, "fused_experts_compute_w4: %s: null pointer", name);
    if (w.group != 32 && w.group != 64 && w.group != 128)
        return fail(kInvalidArg, "fused_experts_compute_w4: %s: groups of 32, 64 or 128 (got %d)", name, w.group);
    if (k % w.group != 0) return fail(kInvalidArg, "fused_experts_compute_w4: %s: k = %lld is not whole groups of %d", name, k, w.group);
    if (((uintptr_t)w.q | (uintptr_t)w.s | (uintptr_t)w.z) & 15)
        return fail(kInvalidArg, "fused_experts_compute_w4: %s, its scales and zeros must be 16-byte aligned", name);
    return kOk;
}

// Token row of every routed slot in position order, one warp per row (the slots behind the last routed one hold no row).
__global__ void __launch_bounds__(256) w4_gather_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ sorted, const int4* __restrict__ worklist,
                                                        int topk, int h8, uint4* __restrict__ xg) {
    pdl_wait();
    pdl_launch_dependents();
    const int pos = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (pos >= worklist[0].y) return;                    // routed slots on this rank
    const uint4* const src = x + (size_t)(sorted[pos] / topk) * h8;
    uint4* const dst = xg + (size_t)pos * h8;
#pragma unroll 4
    for (int i = lane; i < h8; i += 32) dst[i] = src[i];
}

int launch_gather(const void* x, const int32_t* sorted, const int4* worklist, int topk, int H, void* xg, long long slots, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((slots + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    cfg.numAttrs = launch_attrs(attr, 1);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, w4_gather_kernel, reinterpret_cast<const uint4*>(x), sorted, worklist, topk, H / 8,
                                             reinterpret_cast<uint4*>(xg));
    if (e != cudaSuccess) return fail(kCudaError, "fused_experts_compute_w4: gather launch: %s", cudaGetErrorString(e));
    return kOk;
}

}  // namespace

long long w4_experts_workspace_bytes(int T, int E, int topk, int H, int I) {
    if (T <= 0 || E <= 0 || topk <= 0 || H <= 0 || I <= 0) return 0;
    return layout(T, E, topk, H, I).bytes;
}

int launch_w4_experts(const W4ExpertsParams& p, cudaStream_t s) {
    if (p.T < 0 || p.E <= 0 || p.topk <= 0 || p.H <= 0 || p.I <= 0) return fail(kInvalidArg, "fused_experts_compute_w4: bad sizes");
    if (p.dtype != kBF16 && p.dtype != kFP16) return fail(kInvalidArg, "fused_experts_compute_w4: activations must be bf16 or fp16");
    if (p.H > kW4MaxDim || p.I > kW4MaxDim / 2) return fail(kUnsupported, "fused_experts_compute_w4: more than 2^28 rows or k");
    if (p.H % 32 != 0 || p.I % 32 != 0)
        return fail(kInvalidArg, "fused_experts_compute_w4: hidden and intermediate sizes must be multiples of 32 (got %d, %d)", p.H, p.I);
    if (int st = check_weights(p.w1, p.H, "w1")) return st;
    if (int st = check_weights(p.w2, p.I, "w2")) return st;
    if (p.T == 0) return kOk;
    if (!p.x || !p.topk_ids || !p.topk_weights || !p.y || !p.workspace) return fail(kInvalidArg, "fused_experts_compute_w4: null pointer");
    if (((uintptr_t)p.x | (uintptr_t)p.y | (uintptr_t)p.workspace) & 15)
        return fail(kInvalidArg, "fused_experts_compute_w4: activations, result and workspace must be 16-byte aligned");
    if ((((uintptr_t)p.topk_ids | (uintptr_t)p.experts_map | (uintptr_t)p.status) & 3) || ((uintptr_t)p.topk_weights & 1))
        return fail(kInvalidArg, "fused_experts_compute_w4: topk_ids, topk_weights, experts_map or status is not aligned");
    if (p.experts_map != nullptr && p.experts_map_len <= 0) return fail(kInvalidArg, "fused_experts_compute_w4: experts_map needs its length");
    const long long slots = (long long)p.T * p.topk;
    if (p.E > kMaxExperts) return fail(kUnsupported, "fused_experts_compute_w4: at most %d experts (got %d)", kMaxExperts, p.E);
    if (slots > kMaxSlots) return fail(kUnsupported, "fused_experts_compute_w4: at most %d routed slots (got %lld)", kMaxSlots, slots);
    const Layout l = layout(p.T, p.E, p.topk, p.H, p.I);
    if (p.workspace_bytes < l.bytes)
        return fail(kInvalidArg, "fused_experts_compute_w4: workspace holds %lld bytes, needs %lld", p.workspace_bytes, l.bytes);
    uint8_t* const ws = reinterpret_cast<uint8_t*>(p.workspace);
    int32_t* const sorted = reinterpret_cast<int32_t*>(ws + l.sorted);
    int4* const worklist = reinterpret_cast<int4*>(ws + l.worklist);
    void* const act = ws + l.act;
    float* const scratch = reinterpret_cast<float*>(ws + l.scratch);

    W4KernelParams g{};
    g.topk_weights = p.topk_weights;
    g.topk = p.topk;
    if (p.T == 1 && p.topk <= 8) {
        // a single token: its slots are the work items, and a cluster of them sums the result: two launches, no work list
        g.ids = p.topk_ids;
        g.experts_map = p.experts_map;
        g.experts_map_len = p.experts_map_len;
        g.experts = p.E;
        g.y_fp32 = p.y_fp32;
        g.X = p.x;
        g.C = act;
        g.k = p.H;
        g.out_tiles = p.I / 16;
        g.mat_tiles = 2 * p.I / 16;
        if (int st = launch_w4_mma(1, p.dtype, g, p.w1, p.topk, p.topk, 1, s)) return st;
        g.X = act;
        g.C = p.y;
        g.k = p.I;
        g.out_tiles = g.mat_tiles = p.H / 16;
        return launch_w4_mma(2, p.dtype, g, p.w2, p.topk, p.topk, 1, s);
    }

    // Slots of a work item, by the slots an expert gets (all routed slots over the experts here: with an experts_map the slots
    // of other ranks count too, since only the device knows them): the streaming kernel up to 4, above it tcgen05 with 32, 64 or 128.
    // Measured (us): 2 slots 63 against 81, 4 slots 82 / 174 against 98 / 176, 8 slots 130 / 230 against 109 / 186 (128 experts of
    // 2048 x 768 / 8 of 4096 x 14336); 32 against 64 slots a tile: 127 / 190 against 142 / 215 at 16 slots, 173 / 273
    // against 170 / 231 at 32; 128 slots a tile: 497 against 542 at 128.
    const int np = slots <= 4LL * p.E ? 0 : (slots <= 24LL * p.E ? 32 : (slots <= 80LL * p.E ? 64 : 128));
    const int block = np > 0 ? np : 8;
    const int items = (int)max_items(slots, p.E, block);
    // experts that get a slot when all are as likely, and the further items of full ones: what the grid is planned for
    const int likely = std::min(items, std::max(1, (int)(p.E * (1.0 - std::exp(-(double)slots / p.E)) + (double)slots / block * 0.5)));
    if (int st = launch_moe_align(p.T, p.E, p.topk, 1, p.topk_ids, sorted, reinterpret_cast<int32_t*>(ws + l.cumsum),
                                  reinterpret_cast<int32_t*>(ws + l.nblocks), reinterpret_cast<int32_t*>(ws + l.block_expert),
                                  p.experts_map, p.experts_map_len, s, worklist, block))
        return st;

    g.worklist = worklist;
    g.sorted = sorted;
    g.X = p.x;
    g.C = act;
    g.k = p.H;
    g.out_tiles = p.I / 16;
    g.mat_tiles = 2 * p.I / 16;
    MoeParams m{};
    m.scratch = scratch; m.topk_ids = p.topk_ids; m.experts_map = p.experts_map; m.experts_map_len = p.experts_map_len;
    m.E = p.E; m.T = p.T; m.topk = p.topk; m.H = p.H; m.y = p.y; m.y_fp32 = p.y_fp32;
    if (np > 0) {
        // consecutive row tiles of a CTA of the second product: up to four where k is short and two rounds of two CTAs per SM
        // are left (128 experts of 2048 x 768, us with 1 / 2 / 4 / 8: 113 / 107 / 106 / 106 at 128 tokens, 152 / 144 / 141 / 141
        // at 512; 60 of 2048 x 1408 at 512 tokens 119 / 116 / 116).  Where k is longer it costs: 16 experts, 256 tokens, us with 1 / 2
        // / 4: 49 / 54 / 71 at 2048 x 2048 (the second bound keeps it at 1 there), 111 / 110 / 123 at 4096 x 2816, 90 / 96 / 122 at
        // 2048 x 4096; 8 of 4096 x 8192 155 / 166 / 213, of 4096 x 14336 193 / 220 / 303.  Nor does it pay for the first product
        const int run = p.I > 2048 ? 1 : std::max(1, std::min(4, (int)((p.H + 127) / 128 * (long long)likely / (4LL * sm_count()))));
        // the token rows of a work item have to be contiguous for the tile copy; the gathered rows borrow the scratch
        if (int st = launch_gather(p.x, sorted, worklist, p.topk, p.H, scratch, slots, s)) return st;
        g.X = scratch;
        if (int st = launch_w4_umma(1, p.dtype, g, p.w1, p.E, (int)slots, np, 1, 1, items, p.status, s)) return st;
        g.X = act;
        g.C = scratch;
        g.k = p.I;
        g.out_tiles = g.mat_tiles = p.H / 16;
        if (int st = launch_w4_umma(2, p.dtype, g, p.w2, p.E, (int)slots, np, 1, run, items, p.status, s)) return st;
        return launch_moe_combine(m, p.dtype, s);
    }
    if (int st = launch_w4_mma(1, p.dtype, g, p.w1, items, likely, 1, s)) return st;
    g.X = act;
    g.C = scratch;
    g.k = p.I;
    g.out_tiles = g.mat_tiles = p.H / 16;
    if (int st = launch_w4_mma(2, p.dtype, g, p.w2, items, likely, 1, s)) return st;

    return launch_moe_combine(m, p.dtype, s);
}

}  // namespace mlk
