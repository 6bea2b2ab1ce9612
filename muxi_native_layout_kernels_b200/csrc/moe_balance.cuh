// Host-side launch interface of the router's balance loss and per-expert counts.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace mlk {

constexpr int kBalanceMaxExperts = 1024;

struct BalanceParams {
    const void* logits;          // [T, E]
    const int32_t* ids;          // [T, topk]
    const uint8_t* mask;         // [T], 0 = the token is not counted, or null
    const int32_t* cu_seqlens;   // [B + 1] or null
    int T, E, topk, B, score_fun, dtype;   // dtype 0 / 1 / 3 = bf16 / fp16 / fp32
    float coef;
    float* loss;
    int32_t* counts;             // [E]
    float* u;                    // [B, E]: d loss / d p of every token of a sequence
    const float* grad_loss;      // scalar on the device, or null = 1
    void* grad;                  // [T, E] in the logits' type
};

long long balance_workspace_bytes(int T, int E, int B);
int launch_balance_loss(const BalanceParams& b, void* workspace, long long workspace_bytes, cudaStream_t s);
int launch_balance_grad(const BalanceParams& b, cudaStream_t s);
int launch_expert_counts(const int32_t* ids, const uint8_t* mask, int T, int topk, int E, int32_t* counts, cudaStream_t s);

}  // namespace mlk
