// The experts of a mixture layer with 4-bit weights: y[t] = sum_j p[t, j] W2_e (silu(Wg_e x_t) * (Wu_e x_t)), e = ids[t, j].
//
// Sequence: alignment (routed slots grouped by expert, one work item per expert and up to 8 or 16 slots) -> gate/up
// product with SiLU on the fp32 sums -> down product, weighted, into one fp32 row per slot -> sum of a token's rows in
// slot order with one rounding.  The activation between the two products is rounded to the 16-bit activation type, as in
// the 16-bit and e4m3 expert kernels.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>

#include "moe.cuh"
#include "w4_kernels.cuh"

namespace mlk {

namespace {

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

}  // namespace

long long w4_experts_workspace_bytes(int T, int E, int topk, int H, int I) {
    if (T <= 0 || E <= 0 || topk <= 0 || H <= 0 || I <= 0) return 0;
    return layout(T, E, topk, H, I).bytes;
}

int launch_w4_experts(const W4ExpertsParams& p, cudaStream_t s) {
    if (p.T < 0 || p.E <= 0 || p.topk <= 0 || p.H <= 0 || p.I <= 0) return fail(kInvalidArg, "fused_experts_compute_w4: bad sizes");
    if (p.dtype != kBF16 && p.dtype != kFP16) return fail(kInvalidArg, "fused_experts_compute_w4: activations must be bf16 or fp16");
    if (p.H % 32 != 0 || p.I % 32 != 0)
        return fail(kInvalidArg, "fused_experts_compute_w4: hidden and intermediate sizes must be multiples of 32 (got %d, %d)", p.H, p.I);
    if (int st = check_weights(p.w1, p.H, "w1")) return st;
    if (int st = check_weights(p.w2, p.I, "w2")) return st;
    if (p.T == 0) return kOk;
    if (!p.x || !p.topk_ids || !p.topk_weights || !p.y || !p.workspace) return fail(kInvalidArg, "fused_experts_compute_w4: null pointer");
    if (((uintptr_t)p.x | (uintptr_t)p.y | (uintptr_t)p.workspace) & 15)
        return fail(kInvalidArg, "fused_experts_compute_w4: activations, result and workspace must be 16-byte aligned");
    if (p.experts_map != nullptr && p.experts_map_len <= 0) return fail(kInvalidArg, "fused_experts_compute_w4: experts_map needs its length");
    const long long slots = (long long)p.T * p.topk;
    if (slots > (1 << 24)) return fail(kUnsupported, "fused_experts_compute_w4: more than 2^24 routed slots");
    const Layout l = layout(p.T, p.E, p.topk, p.H, p.I);
    if (p.workspace_bytes < l.bytes)
        return fail(kInvalidArg, "fused_experts_compute_w4: workspace holds %lld bytes, needs %lld", p.workspace_bytes, l.bytes);
    uint8_t* const ws = reinterpret_cast<uint8_t*>(p.workspace);
    int32_t* const sorted = reinterpret_cast<int32_t*>(ws + l.sorted);
    int4* const worklist = reinterpret_cast<int4*>(ws + l.worklist);
    void* const act = ws + l.act;
    float* const scratch = reinterpret_cast<float*>(ws + l.scratch);

    int np = 0, sk1 = 1, sk2 = 1;
    if (slots > 8LL * p.E) np = slots > 48LL * p.E ? 128 : (slots > 24LL * p.E ? 64 : 32);
    if (const char* v = getenv("W4_X")) sscanf(v, "%d,%d,%d", &np, &sk1, &sk2);
    const int nt = slots <= 4LL * p.E ? 1 : 2, block = np > 0 ? np : 8 * nt;
    const int items = (int)max_items(slots, p.E, block);
    // experts that get a slot when all are as likely, and the further items of full ones: what the grid is planned for
    const int likely = std::min(items, std::max(1, (int)(p.E * (1.0 - std::exp(-(double)slots / p.E)) + (double)slots / block * 0.5)));
    if (int st = launch_moe_align(p.T, p.E, p.topk, 1, p.topk_ids, sorted, reinterpret_cast<int32_t*>(ws + l.cumsum),
                                  reinterpret_cast<int32_t*>(ws + l.nblocks), reinterpret_cast<int32_t*>(ws + l.block_expert),
                                  p.experts_map, p.experts_map_len, s, worklist, block))
        return st;

    W4KernelParams g{};
    g.worklist = worklist;
    g.sorted = sorted;
    g.topk_weights = p.topk_weights;
    g.topk = p.topk;
    g.X = p.x;
    g.C = act;
    g.k = p.H;
    g.out_tiles = p.I / 16;
    g.mat_tiles = 2 * p.I / 16;
    MoeParams m{};
    m.scratch = scratch; m.topk_ids = p.topk_ids; m.experts_map = p.experts_map; m.experts_map_len = p.experts_map_len;
    m.E = p.E; m.T = p.T; m.topk = p.topk; m.H = p.H; m.y = p.y; m.y_fp32 = p.y_fp32;
    if (np > 0) {
        // the token rows of a work item have to be contiguous for the tile copy; the gathered rows borrow the scratch
        if (int st = launch_moe_gather_positions(p.x, sorted, worklist, p.topk, p.H, scratch, items, s)) return st;
        g.X = scratch;
        if (int st = launch_w4_umma(1, p.dtype, g, p.w1, p.E, (int)slots, np, sk1, items, p.status, s)) return st;
        g.X = act;
        g.C = scratch;
        g.k = p.I;
        g.out_tiles = g.mat_tiles = p.H / 16;
        if (int st = launch_w4_umma(2, p.dtype, g, p.w2, p.E, (int)slots, np, sk2, items, p.status, s)) return st;
        return launch_moe_combine(m, p.dtype, s);
    }
    if (int st = launch_w4_mma(1, p.dtype, g, p.w1, items, likely, nt, s)) return st;
    g.X = act;
    g.C = scratch;
    g.k = p.I;
    g.out_tiles = g.mat_tiles = p.H / 16;
    if (int st = launch_w4_mma(2, p.dtype, g, p.w2, items, likely, nt, s)) return st;

    return launch_moe_combine(m, p.dtype, s);
}

}  // namespace mlk
