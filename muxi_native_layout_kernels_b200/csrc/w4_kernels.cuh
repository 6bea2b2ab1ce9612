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
    int n, k, kc, groups, group_shift;
    // experts
    const int4* worklist;       // [0] = {items,..}; then {expert, first position, slots, first compact position}
    const int32_t* sorted;      // slot id of every position
    const void* topk_weights;
    int topk;
};

template <int WT>
__device__ __forceinline__ void store16(void* base, size_t i, float v) {
    if constexpr (WT == kFP16) reinterpret_cast<__half*>(base)[i] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
}

int launch_w4_mma(int mode, int wt, W4KernelParams p, const W4Weights& w, int token_blocks, int nt, int sk, cudaStream_t s);
int w4_mma_split(long long row_ctas, int kc);

}  // namespace mlk
