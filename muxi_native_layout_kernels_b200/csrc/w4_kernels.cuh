// Kernel parameters and launch interface shared by the 4-bit weight kernels.
#pragma once

#include "w4.cuh"

namespace mlk {

struct W4KernelParams {
    const uint8_t* q;
    const uint32_t* s;          // scales, two rows per word
    const uint16_t* z;          // zero points, two rows per half word
    const void* X;
    void* C;
    const void* bias;
    float alpha;
    int out_tiles;              // 16-row tiles of the output (MODE 1: of the gate half)
    int mat_tiles;              // 16-row tiles of one expert's matrix
    int n, k, kc, groups;
    int row_warps;              // warps of a CTA side by side in the rows; the others split k
    int seg_units;              // units of 128 k of one staging of activations and scales
    // experts
    const int4* worklist;       // [0] = {items,..}; then {expert, first position, slots, first compact position}
    const int32_t* sorted;      // slot id of every position
    const void* topk_weights;
    int topk;
    // a single token: work item = slot, no work list.  The first product leaves row `slot` of the activation; the CTAs of a
    // cluster of the second are the token's slots, and their weighted sum is the result.
    const int32_t* ids;         // [topk], or null
    const int32_t* experts_map;
    int experts_map_len, experts;
    int y_fp32;
};

template <int WT>
__device__ __forceinline__ void store16(void* base, size_t i, float v) {
    if constexpr (WT == kFP16) reinterpret_cast<__half*>(base)[i] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
}

// MODE of both forms: 0 = dense product, 1 = the experts' gate/up product with SiLU, 2 = their down product.
// items: work items (exact for the dense products, an upper bound for the experts, whose number the device knows).
// tcgen05 form: np = tokens per tile (32, 64, 128; 256 in mode 0), sk = CTAs of a cluster along k, run = consecutive
// row tiles of a CTA, matrices = experts (1 in mode 0), x_rows = rows of X.
int launch_w4_umma(int mode, int wt, const W4KernelParams& p, const W4Weights& w, long long matrices, int x_rows, int np, int sk,
                   int run, int items, int* status, cudaStream_t s);
struct W4UmmaPlan {
    int np, sk;
    double us;                  // estimated time
};
W4UmmaPlan w4_umma_plan(int rows16, int n, int k);
// Streaming form: nt = 8-token column tiles, likely_items = what the split over k is chosen for.  With p.ids the experts'
// modes take a single token's slots (at most 8) as their items.
int launch_w4_mma(int mode, int wt, W4KernelParams p, const W4Weights& w, int items, int likely_items, int nt, cudaStream_t s);

}  // namespace mlk
