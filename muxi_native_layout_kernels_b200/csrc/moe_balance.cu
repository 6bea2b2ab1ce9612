// Balance loss of a mixture layer's router, per-expert counts, and the gradient with respect to the router logits.
//
//   p[t, e]  = softmax(l_t)_e, or sigmoid(l_te) / sum_f sigmoid(l_tf)
//   c[b, e]  = picks of expert e by the counted tokens of sequence b (ids[t, j] == e),   n_b = counted tokens of b
//   loss     = coef / B * sum_b E / (topk n_b^2) * sum_e c[b, e] * sum_{t in b} p[t, e]      (n_b = 0 adds nothing)
//   u[b, e]  = coef E c[b, e] / (B topk n_b^2)                                               = d loss / d p[t, e]
//   d loss / d l_te = p_te (u_be - sum_f p_tf u_bf)           (times 1 - sigmoid(l_te) for the sigmoid scores)
//
// The counts are known only when every token has been seen, so the logits are read twice: three kernels,
//   partial   blocks over runs of R tokens; a run crosses sequence borders freely, each (run i, sequence b) that meet
//             leaves one record (sums of p in fp32, counts, tokens) at index i + b, which is unique because both only
//             grow along the tokens: no buffer has to be cleared and no float is added by an atomic
//   finish    one cluster of eight CTAs, a slice of the experts each: records -> counts, u, loss, in a fixed order
//   grad      the runs again: p recomputed, u in, gradient out
// and for small batches one launch, a CTA or a cluster of eight that keeps p in shared memory and does all three steps.
// What bounds it: latency, of a row (load, two reductions over its lanes) and of the launches; the logits' traffic (two
// reads, one write) is a few microseconds at the largest sizes.  A row's 16-byte loads are spread over as few lanes as
// cover it (8 experts in bf16: one lane per token), so that a warp holds up to 32 tokens.  Rows are overlapped by warps, not
// inside a warp: with four row groups unrolled the code of these kernels, run once per launch, waited for its own
// instructions (192 x 8 in one CTA: 8.6 us against 4.0).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "moe_balance.cuh"
#include "status.h"
#include "umma_common.cuh"

namespace mlk {

namespace {

constexpr int kThreads = 512;
constexpr int kFinishThreads = 1024;
constexpr int kSmallThreads = 512;
constexpr int kSmallElems = 16384;   // scores of a CTA's tokens in a small batch, in shared memory
constexpr int kSmallSums = 1024;     // (sequence, expert) pairs of a small batch
constexpr int kSmallCluster = 8;
constexpr int kFinishCtas = 8;
constexpr int kF32 = 3;          // dtype code of fp32 logits in this file

struct Params {
    const void* logits;
    const int32_t* ids;          // [T, topk]
    const uint8_t* mask;         // [T] or null
    const int32_t* cu;           // [B + 1] or null (one sequence, all tokens)
    int T, E, topk, B, score_fun;
    int R;                       // tokens per run
    int lpr;                     // lanes per row
    int cw, parts, per;          // finish: experts per CTA, threads per expert, threads per expert and sequence
    float coef;
    float* P;                    // records
    int32_t* C;
    int32_t* N;
    float* u;                    // [B, E]
    float* loss;
    int32_t* counts;             // [E]
    const float* grad_loss;      // scalar or null = 1
    void* grad;                  // [T, E]
};

__device__ __forceinline__ int seq_start(const Params& p, int b) {
    return p.cu == nullptr ? (b == 0 ? 0 : p.T) : min(max(p.cu[b], 0), p.T);
}

// First sequence that ends behind token t (B: none), found by the whole block: the sequences that end at or before t.
__device__ __forceinline__ int block_seq_of(const Params& p, int t) {
    if (p.cu == nullptr) return 0;
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += blockDim.x) {
        const int b = b0 + (int)threadIdx.x;
        before += __syncthreads_count(b < p.B && seq_start(p, b + 1) <= t);
    }
    return before;
}

template <int T>
struct Elem;
template <> struct Elem<kBF16> { using type = uint16_t; };
template <> struct Elem<kFP16> { using type = uint16_t; };
template <> struct Elem<kF32> { using type = float; };

template <int DT>
__device__ __forceinline__ float as_float(typename Elem<DT>::type v) {
    if constexpr (DT == kF32) return v;
    else if constexpr (DT == kBF16) return __uint_as_float((uint32_t)v << 16);
    else return __half2float(__ushort_as_half(v));
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::type from_float(float v) {
    if constexpr (DT == kF32) return v;
    else if constexpr (DT == kBF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
    else return __half_as_ushort(__float2half_rn(v));
}

__device__ __forceinline__ float group_sum(float v, int lpr) {
    for (int o = lpr >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
__device__ __forceinline__ float group_max(float v, int lpr) {
    for (int o = lpr >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

// Column of value i of a lane: J vectors of V neighbouring experts, lpr * V apart.
template <int V>
__device__ __forceinline__ int column(int i, int sub, int lpr) { return (i / V) * (lpr * V) + sub * V + i % V; }

template <int DT, int V, int J>
__device__ __forceinline__ void load_row(const Params& p, long long row, int sub, bool live, float (&x)[V * J]) {
    using E = typename Elem<DT>::type;
    const E* base = reinterpret_cast<const E*>(p.logits) + row * p.E;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int c = j * (p.lpr * V) + sub * V;
        E v[V];
        if (live && c < p.E) {                  // V divides E: a vector is in or out as a whole
            if constexpr (V * sizeof(E) == 16) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(base + c);
            else if constexpr (V * sizeof(E) == 8) *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(base + c);
            else {
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = base[c + i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) x[j * V + i] = as_float<DT>(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) x[j * V + i] = -INFINITY;     // exp and sigmoid give 0
        }
    }
}

// Scores of a row in place; `one_minus`: 1 - sigmoid for the gradient (sigmoid scores).  A row whose logits are all -inf
// has no distribution: its scores are 0.
template <int N, bool GRAD>
__device__ __forceinline__ void scores(const Params& p, float (&x)[N], float (&one_minus)[GRAD ? N : 1]) {
    float s = 0.f;
    if (p.score_fun == 0) {
        float m = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
        m = group_max(m, p.lpr);
        if (m == -INFINITY) m = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s += x[i] = expf(x[i] - m);
    } else {
        // sigmoid(x) = e^min(x,0) / (1 + e^-|x|), taken here over e^m, m the row's largest min(x,0): the factor cancels in p, no
        // term overflows and the sum is at least 1/2, where the sigmoids themselves end below about -88 - ln E.  With a
        // logit of 0 or more in the row m is 0 and one exponential does: a warp whose rows all have one, or nothing but -inf,
        // skips the maximum and the second exponential (16384 x 128: 31 us the three kernels, with them in every row 33).
        bool high = false, some = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            high |= x[i] >= 0.f;
            some |= x[i] > -INFINITY;
        }
        const uint32_t row = (0xFFFFFFFFu >> (32 - p.lpr)) << (threadIdx.x & 31 & ~(p.lpr - 1));
        const uint32_t highs = __ballot_sync(0xFFFFFFFFu, high) & row, somes = __ballot_sync(0xFFFFFFFFu, some) & row;
        float m = 0.f;
        if (!__all_sync(0xFFFFFFFFu, highs != 0u || somes == 0u)) {
            m = fminf(x[0], 0.f);
#pragma unroll
            for (int i = 1; i < N; ++i) m = fmaxf(m, fminf(x[i], 0.f));
            m = group_max(m, p.lpr);
            if (m == -INFINITY) m = 0.f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float lo = fminf(x[i], 0.f), e = expf(-fabsf(x[i])), d = 1.f / (1.f + e);
            if constexpr (GRAD) one_minus[i] = x[i] >= 0.f ? e * d : d;
            float f = x[i] >= 0.f ? 1.f : e;
            if (m != 0.f) f = expf(lo - m);
            s += x[i] = f * d;                                   // NaN stays NaN through d
        }
    }
    s = group_sum(s, p.lpr);
    const float inv = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= inv;
}

template <int DT, int V, int J>
__global__ void __launch_bounds__(kThreads) balance_partial_kernel(const Params p) {
    constexpr int N = V * J;
    extern __shared__ __align__(16) uint8_t smem[];
    float* const sP = reinterpret_cast<float*>(smem);                       // [warps][E]
    int32_t* const sC = reinterpret_cast<int32_t*>(sP + (kThreads / 32) * p.E);
    __shared__ int sN[kThreads / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane & (p.lpr - 1);
    const int rows_per_warp = 32 / p.lpr, group = lane / p.lpr;
    pdl_wait();
    pdl_launch_dependents();
    const int begin = blockIdx.x * p.R, end = min(begin + p.R, p.T);
    for (int b = block_seq_of(p, begin); b < p.B; ++b) {
        const int s0 = seq_start(p, b), s1 = seq_start(p, b + 1);
        if (s0 >= end) break;
        const int a = max(s0, begin), z = min(s1, end);
        if (a >= z) continue;                                               // an empty sequence has no record
        for (int e = tid; e < p.E; e += kThreads) sC[e] = 0;
        __syncthreads();
        float acc[N];
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.f;
        int n = 0;
        for (int r0 = a + warp * rows_per_warp; r0 < z; r0 += (kThreads / 32) * rows_per_warp) {
            // logits, mask and picks on their way before the first is used; what is not counted becomes -inf
            const int row = r0 + group;
            bool live = row < z;
            float x[N], unused[1];
            load_row<DT, V, J>(p, row, sub, live, x);
            const int pick = live && sub < p.topk ? p.ids[(long long)row * p.topk + sub] : -1;
            if (p.mask != nullptr && live) live = p.mask[row] != 0;
            if (live) {
                if (pick >= 0 && pick < p.E) atomicAdd(&sC[pick], 1);
                for (int j = sub + p.lpr; j < p.topk; j += p.lpr) {
                    const int e = p.ids[(long long)row * p.topk + j];
                    if (e >= 0 && e < p.E) atomicAdd(&sC[e], 1);
                }
                n += sub == 0;
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] = -INFINITY;
            }
            scores<N, false>(p, x, unused);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] += x[i];
        }
        // the warp's rows, then the warps, in a fixed order
        for (int o = 16; o >= p.lpr; o >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] += __shfl_xor_sync(0xFFFFFFFFu, acc[i], o);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
        if (group == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = column<V>(i, sub, p.lpr);
                if (c < p.E) sP[warp * p.E + c] = acc[i];
            }
        if (lane == 0) sN[warp] = n;
        __syncthreads();
        const long long rec = (long long)blockIdx.x + b;
        for (int e = tid; e < p.E; e += kThreads) {
            float v = sP[e];
#pragma unroll
            for (int w = 1; w < kThreads / 32; ++w) v += sP[w * p.E + e];
            p.P[rec * p.E + e] = v;
            p.C[rec * p.E + e] = sC[e];
        }
        if (tid == 0) {
            int v = 0;
            for (int w = 0; w < kThreads / 32; ++w) v += sN[w];
            p.N[rec] = v;
        }
        __syncthreads();
    }
}

// One cluster: CTA r owns the experts [r * cw, (r + 1) * cw).  A thread is (expert column, part): `per` parts share the
// records of a sequence, parts / per sequences make a round (all powers of two).
__global__ void __cluster_dims__(kFinishCtas, 1, 1) __launch_bounds__(kFinishThreads) balance_finish_kernel(const Params p) {
    const int cw = p.cw, parts = p.parts, per = p.per;
    __shared__ float sP[kFinishThreads];
    __shared__ int sC[kFinishThreads], sN[kFinishThreads];
    __shared__ float total;
    const int tid = threadIdx.x, r = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    const int col = tid % cw, part = tid / cw;
    const int e = r * cw + col;
    const bool mine = part < parts && e < p.E;
    const int round = parts / per, sub = part % per, which = part / per;
    float loss = 0.f;
    int count = 0;
    for (int b0 = 0; b0 < p.B; b0 += round) {
        const int b = b0 + which;
        float P = 0.f;
        int C = 0, n = 0;
        if (mine && b < p.B) {
            const int s0 = seq_start(p, b), s1 = seq_start(p, b + 1);
            if (s0 < s1) {
                const int i1 = (s1 - 1) / p.R;
#pragma unroll 4
                for (int i = s0 / p.R + sub; i <= i1; i += per) {
                    const long long rec = (long long)i + b;
                    P += p.P[rec * p.E + e];
                    C += p.C[rec * p.E + e];
                    n += p.N[rec];
                }
            }
        }
        // the parts of a sequence, halved step by step: a fixed order
        for (int h = per >> 1; h > 0; h >>= 1) {
            sP[tid] = P; sC[tid] = C; sN[tid] = n;
            __syncthreads();
            if (mine && sub < h) {
                P += sP[tid + h * cw];
                C += sC[tid + h * cw];
                n += sN[tid + h * cw];
            }
            __syncthreads();
        }
        if (mine && b < p.B && sub == 0) {
            // n_b * n_b in fp32: 24 bits are enough for a scale factor
            const float u = n > 0 ? p.coef * (float)p.E * (float)C / ((float)p.B * (float)p.topk * (float)n * (float)n) : 0.f;
            p.u[(long long)b * p.E + e] = u;
            loss += u * P;
            count += C;
        }
    }
    sP[tid] = loss;
    sC[tid] = count;
    __syncthreads();
    for (int h = parts >> 1; h > 0; h >>= 1) {
        if (part < h) {
            sP[tid] += sP[tid + h * cw];
            sC[tid] += sC[tid + h * cw];
        }
        __syncthreads();
    }
    if (tid < cw && e < p.E) p.counts[e] = sC[tid];
    if (tid < 32) {                                                         // the columns of this CTA
        float v = 0.f;
        for (int c = tid; c < cw; c += 32) v += sP[c];
        v = warp_sum(v);
        if (tid == 0) total = v;
    }
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (r == 0 && tid < 32) {
        float x = 0.f;
        if (tid < kFinishCtas) {
            uint32_t at;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&total)), "r"(tid));
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
        }
        x = warp_sum(x);
        if (tid == 0) p.loss[0] = x;
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The gradient of one row from its logits (x), given u of its sequence.
template <int DT, int V, int J>
__device__ __forceinline__ void grad_row(const Params& p, int row, int sub, bool live, float g, float (&x)[V * J], const float (&u)[V * J]) {
    constexpr int N = V * J;
    using E = typename Elem<DT>::type;
    float one_minus[N], dot = 0.f;
    scores<N, true>(p, x, one_minus);
#pragma unroll
    for (int i = 0; i < N; ++i) dot += x[i] * u[i];
    dot = group_sum(dot, p.lpr);
    if (row < 0) return;
    E* const out = reinterpret_cast<E*>(p.grad) + (long long)row * p.E;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int c = j * (p.lpr * V) + sub * V;
        if (c >= p.E) continue;
        E v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float d = live ? g * (x[j * V + i] * (u[j * V + i] - dot)) : 0.f;
            if (p.score_fun == 1 && live) d *= one_minus[j * V + i];
            v[i] = from_float<DT>(d);
        }
        if constexpr (V * sizeof(E) == 16) *reinterpret_cast<uint4*>(out + c) = *reinterpret_cast<uint4*>(v);
        else if constexpr (V * sizeof(E) == 8) *reinterpret_cast<uint2*>(out + c) = *reinterpret_cast<uint2*>(v);
        else {
#pragma unroll
            for (int i = 0; i < V; ++i) out[c + i] = v[i];
        }
    }
}

template <int DT, int V, int J>
__global__ void __launch_bounds__(kThreads) balance_grad_kernel(const Params p) {
    constexpr int N = V * J;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane & (p.lpr - 1);
    const int rows_per_warp = 32 / p.lpr, group = lane / p.lpr, step = (kThreads / 32) * rows_per_warp;
    pdl_wait();
    pdl_launch_dependents();
    const float g = p.grad_loss ? *p.grad_loss : 1.f;
    const int begin = blockIdx.x * p.R, end = min(begin + p.R, p.T);
    // segments of the run: one per sequence in it, and what lies before, between and behind them (in no sequence)
    int b = block_seq_of(p, begin);
    for (int a = begin; a < end;) {
        while (b < p.B && seq_start(p, b + 1) <= a) ++b;                    // empty ones
        const int s0 = b < p.B ? seq_start(p, b) : p.T, s1 = b < p.B ? seq_start(p, b + 1) : p.T;
        const bool inside = b < p.B && s0 <= a;
        const int z = min(inside ? s1 : max(s0, a + 1), end);
        float u[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = column<V>(i, sub, p.lpr);
            u[i] = inside && c < p.E ? p.u[(long long)b * p.E + c] : 0.f;
        }
        for (int r0 = a + warp * rows_per_warp; r0 < z; r0 += step) {
            const int row = r0 + group;
            bool live = inside && row < z;
            float x[N];
            load_row<DT, V, J>(p, row, sub, live, x);
            if (p.mask != nullptr && live) live = p.mask[row] != 0;
            if (!live)
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] = -INFINITY;
            grad_row<DT, V, J>(p, row < z ? row : -1, sub, live, g, x, u);
        }
        a = z;
    }
}

// A small batch in one launch, by one CTA or a cluster of eight that share the tokens: scores in shared memory, counts and
// sums of p per (sequence, expert) of the own tokens, then, over the cluster in rank order, u, the loss and the counts, and
// the gradient of the own tokens if it is wanted.
template <int DT, int V, int J>
__global__ void __launch_bounds__(kSmallThreads) balance_small_kernel(const Params p) {
    constexpr int N = V * J;
    extern __shared__ __align__(16) uint8_t smem[];
    const int sums = p.B * p.E;
    int CL, rank;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(CL));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int t0 = (int)((long long)p.T * rank / CL), t1 = (int)((long long)p.T * (rank + 1) / CL);
    int* const sc = reinterpret_cast<int*>(smem);                           // [B][E] counts of the own tokens
    float* const sP = reinterpret_cast<float*>(sc + sums);                  // [B][E] sums of p of the own tokens
    float* const su = sP + sums;                                            // [B][E] u
    int* const sn = reinterpret_cast<int*>(su + sums);                      // [B] own tokens counted
    float* const sp = reinterpret_cast<float*>(sn + p.B);                   // [own tokens][E] scores
    __shared__ float red[kSmallThreads];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane & (p.lpr - 1);
    const int rows_per_warp = 32 / p.lpr, group = lane / p.lpr, step = (kSmallThreads / 32) * rows_per_warp;
    for (int i = tid; i < sums; i += kSmallThreads) sc[i] = 0;
    for (int i = tid; i < p.B; i += kSmallThreads) sn[i] = 0;
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    // sequence of a row (-1: none)
    auto seq_of = [&](int row) {
        if (p.cu == nullptr) return 0;
        int lo = 0, hi = p.B;                                               // first sequence that ends behind the row
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (seq_start(p, mid + 1) > row) hi = mid;
            else lo = mid + 1;
        }
        return lo < p.B && seq_start(p, lo) <= row ? lo : -1;
    };
    for (int r0 = t0 + warp * rows_per_warp; r0 < t1; r0 += step) {
        const int row = r0 + group;
        float x[N], unused[1];
        load_row<DT, V, J>(p, row, sub, row < t1, x);
        const int b = row < t1 && (p.mask == nullptr || p.mask[row] != 0) ? seq_of(row) : -1;
        if (b >= 0) {
            for (int j = sub; j < p.topk; j += p.lpr) {
                const int e = p.ids[(long long)row * p.topk + j];
                if (e >= 0 && e < p.E) atomicAdd(&sc[b * p.E + e], 1);
            }
            if (sub == 0) atomicAdd(&sn[b], 1);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = -INFINITY;
        }
        scores<N, false>(p, x, unused);
        if (row < t1)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = column<V>(i, sub, p.lpr);
                if (c < p.E) sp[(row - t0) * p.E + c] = x[i];
            }
    }
    __syncthreads();
    // sums of p: thread = (pair, part); the parts of a pair are neighbours in a warp
    int parts = 1;
    while (parts * 2 * sums <= kSmallThreads && parts < 32) parts *= 2;
    const int pairs = kSmallThreads / parts;                                // pairs of one round
    for (int q0 = 0; q0 < sums; q0 += pairs) {
        const int q = q0 + tid / parts, sub_part = tid % parts;
        float P = 0.f;
        if (q < sums) {
            const int sb = q / p.E, e = q - sb * p.E, s0 = max(seq_start(p, sb), t0), s1 = min(seq_start(p, sb + 1), t1);
            for (int t = s0 + sub_part; t < s1; t += parts) P += sp[(t - t0) * p.E + e];
        }
        for (int h = parts >> 1; h > 0; h >>= 1) P += __shfl_xor_sync(0xFFFFFFFFu, P, h);
        if (q < sums && sub_part == 0) sP[q] = P;
    }
    __syncthreads();
    if (CL > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    auto over_cluster = [&](const void* at, auto zero) {
        using T = decltype(zero);
        if (CL == 1) return *reinterpret_cast<const T*>(at);
        T v[kSmallCluster];                                                 // all on their way at once: a remote load takes 0.3 us
#pragma unroll
        for (int r = 0; r < kSmallCluster; ++r) {
            uint32_t a, w;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(at)), "r"(r));
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w) : "r"(a) : "memory");
            if constexpr (std::is_same<T, float>::value) v[r] = __uint_as_float(w);
            else v[r] = (T)w;
        }
        T t = v[0];
#pragma unroll
        for (int r = 1; r < kSmallCluster; ++r) t += v[r];
        return t;
    };
    float loss = 0.f;
    for (int q = tid; q < sums; q += kSmallThreads) {
        const int n = over_cluster(sn + q / p.E, 0), C = over_cluster(sc + q, 0);
        const float u = n > 0 ? p.coef * (float)p.E * (float)C / ((float)p.B * (float)p.topk * (float)n * (float)n) : 0.f;
        su[q] = u;
        if (rank == 0) {
            loss += u * over_cluster(sP + q, 0.f);
            if (p.u) p.u[q] = u;
        }
    }
    if (rank == 0) {
        red[tid] = loss;
        __syncthreads();
        for (int h = kSmallThreads / 2; h > 0; h >>= 1) {
            if (tid < h) red[tid] += red[tid + h];
            __syncthreads();
        }
        if (tid == 0) p.loss[0] = red[0];
        for (int e = tid; e < p.E; e += kSmallThreads) {
            int c = 0;
            for (int q = 0; q < p.B; ++q) c += over_cluster(sc + q * p.E + e, 0);
            p.counts[e] = c;
        }
    }
    __syncthreads();
    // nobody leaves, or writes its sums, while they may still be read
    if (CL > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (p.grad == nullptr) return;
    for (int r0 = t0 + warp * rows_per_warp; r0 < t1; r0 += step) {
        const int row = r0 + group;
        float x[N], u[N];
        load_row<DT, V, J>(p, row, sub, row < t1, x);
        const int b = row < t1 && (p.mask == nullptr || p.mask[row] != 0) ? seq_of(row) : -1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = column<V>(i, sub, p.lpr);
            u[i] = b >= 0 && c < p.E ? su[b * p.E + c] : 0.f;
            if (b < 0) x[i] = -INFINITY;
        }
        grad_row<DT, V, J>(p, row < t1 ? row : -1, sub, b >= 0, 1.f, x, u);
    }
}

// Counts alone: one counter block per CTA in shared memory, integer atomics into the cleared result.
__global__ void __launch_bounds__(kThreads) expert_counts_kernel(const int32_t* __restrict__ ids, const uint8_t* __restrict__ mask,
                                                                long long n, int topk, int E, int32_t* __restrict__ counts) {
    extern __shared__ int32_t c[];
    for (int e = threadIdx.x; e < E; e += kThreads) c[e] = 0;
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kThreads) {
        const int e = ids[i];
        if (e >= 0 && e < E && (mask == nullptr || mask[i / topk] != 0)) atomicAdd(&c[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kThreads)
        if (c[e] != 0) atomicAdd(&counts[e], c[e]);
}

struct Plan {
    int v, j, lpr, runs, R;
};

Plan plan(int T, int E, int elem, bool aligned) {
    Plan q{};
    q.v = elem == 2 && E % 8 == 0 ? 8 : (E % 4 == 0 ? 4 : 1);
    if (!aligned) q.v = 1;
    const int vectors = (E + q.v - 1) / q.v;
    q.lpr = 1;
    while (q.lpr < 32 && q.lpr < vectors) q.lpr *= 2;
    q.j = (vectors + q.lpr - 1) / q.lpr;
    // up to two runs per SM, at least one pass of a block's warps each
    const int rows = (kThreads / 32) * (32 / q.lpr);
    const int want = 2 * sm_count();
    q.R = std::max(rows, ((T + want - 1) / want + rows - 1) / rows * rows);
    q.runs = (T + q.R - 1) / q.R;
    return q;
}

using Kern = void (*)(Params);
enum Kind { kPartial, kGrad, kSmall };
template <int DT, int KIND, int V, int J>
constexpr Kern kernel() {
    if constexpr (KIND == kGrad) return balance_grad_kernel<DT, V, J>;
    else if constexpr (KIND == kPartial) return balance_partial_kernel<DT, V, J>;
    else return balance_small_kernel<DT, V, J>;
}
template <int DT, int KIND>
Kern pick(int v, int j) {
    if (DT != kF32 && v == 8) return j == 1 ? kernel<DT, KIND, DT == kF32 ? 4 : 8, 1>() : kernel<DT, KIND, DT == kF32 ? 4 : 8, 4>();
    if (v == 4) return j == 1 ? kernel<DT, KIND, 4, 1>() : (j == 2 ? kernel<DT, KIND, 4, 2>() : kernel<DT, KIND, 4, 8>());
    return j <= 2 ? kernel<DT, KIND, 1, 2>() : kernel<DT, KIND, 1, 32>();
}
template <int KIND>
Kern pick(int dt, int v, int j) {
    return dt == kF32 ? pick<kF32, KIND>(v, j) : (dt == kFP16 ? pick<kFP16, KIND>(v, j) : pick<kBF16, KIND>(v, j));
}

int launch(const char* what, Kern kern, int grid, int threads, size_t smem, cudaStream_t s, const Params& p, int cluster = 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[3];
    cfg.attrs = attr;
    cfg.numAttrs = launch_attrs(attr, 1);
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return fail(kCudaError, "%s launch: %s", what, cudaGetErrorString(e));
    return kOk;
}

int check(const BalanceParams& b, const char* who) {
    if (b.T < 0 || b.B < 1 || b.topk < 1) return fail(kInvalidArg, "%s: bad sizes", who);
    if (b.E < 1 || b.E > kBalanceMaxExperts) return fail(kUnsupported, "%s: 1 <= experts <= %d (got %d)", who, kBalanceMaxExperts, b.E);
    if (b.dtype < 0 || b.dtype > 3 || b.dtype == kE4M3) return fail(kInvalidArg, "%s: logits must be bf16, fp16 or fp32", who);
    if (b.score_fun != 0 && b.score_fun != 1) return fail(kInvalidArg, "%s: score_fun must be 0 (softmax) or 1 (sigmoid)", who);
    if (b.B > 1 && !b.cu_seqlens) return fail(kInvalidArg, "%s: more than one sequence needs cu_seqlens", who);
    if (b.T > 0 && !b.logits) return fail(kInvalidArg, "%s: null pointer", who);
    if ((long long)b.B + b.T > 0x3FFFFFFF) return fail(kUnsupported, "%s: too many tokens or sequences", who);
    if ((long long)b.T * b.topk > 0x7FFFFFFF) return fail(kUnsupported, "%s: counts of more than 2^31 - 1 picks", who);
    const uintptr_t elem = b.dtype == kF32 ? 3 : 1;
    if ((((uintptr_t)b.logits | (uintptr_t)b.grad) & elem) || (((uintptr_t)b.ids | (uintptr_t)b.cu_seqlens) & 3))
        return fail(kInvalidArg, "%s: logits, grad, topk_ids or cu_seqlens is not aligned", who);
    if (((uintptr_t)b.loss | (uintptr_t)b.counts | (uintptr_t)b.u | (uintptr_t)b.grad_loss) & 3)
        return fail(kInvalidArg, "%s: loss, counts, dprob or grad_loss is not aligned", who);
    return kOk;
}

Params params(const BalanceParams& b, const Plan& q) {
    Params p{};
    p.logits = b.logits; p.ids = b.ids; p.mask = b.mask; p.cu = b.cu_seqlens;
    p.T = b.T; p.E = b.E; p.topk = b.topk; p.B = b.B; p.score_fun = b.score_fun; p.coef = b.coef;
    p.R = q.R; p.lpr = q.lpr;
    p.u = b.u; p.loss = b.loss; p.counts = b.counts; p.grad_loss = b.grad_loss; p.grad = b.grad;
    return p;
}

Plan plan_of(const BalanceParams& b) {
    const bool aligned = (((uintptr_t)b.logits | (uintptr_t)b.grad) & 15) == 0;
    return plan(b.T, b.E, b.dtype == kF32 ? 4 : 2, aligned);
}

}  // namespace

// CTAs of the one-launch form, 0 = the batch is too large for it.
static int small_batch(int T, int E, int B) {
    if ((long long)B * E > kSmallSums || B > 1024) return 0;
    if ((long long)T * E <= kSmallElems / 8) return 1;
    return (long long)((T + kSmallCluster - 1) / kSmallCluster) * E <= kSmallElems ? kSmallCluster : 0;
}

long long balance_workspace_bytes(int T, int E, int B) {
    if (T < 0 || E < 1 || B < 1 || small_batch(T, E, B)) return 0;
    // the most runs any plan makes: 2 per SM, and never more than tokens
    const long long records = (long long)std::min(T, 2 * sm_count() + 1) + B;
    return (records * E * 2 + records) * 4;
}

int launch_balance_loss(const BalanceParams& b, void* workspace, long long workspace_bytes, cudaStream_t s) {
    if (int st = check(b, "router_balance_loss")) return st;
    const int small = small_batch(b.T, b.E, b.B);
    if (!b.loss || !b.counts || (b.T > 0 && !b.ids)) return fail(kInvalidArg, "router_balance_loss: null pointer");
    if (!small && (!b.u || !workspace)) return fail(kInvalidArg, "router_balance_loss: null pointer (dprob, workspace)");
    const Plan q = plan_of(b);
    Params p = params(b, q);
    if (small) {
        const size_t most = (kSmallElems + 3 * kSmallSums + 1024) * 4;
        const Kern kern = pick<kSmall>(b.dtype, q.v, q.j);
        if (umma::prepare_kernel(reinterpret_cast<const void*>(kern), kSmallThreads, most, 0) == 0)
            return fail(kCudaError, "router_balance_loss: the kernel cannot be launched on this device");
        const size_t rows = (b.T + small - 1) / small;
        return launch("router_balance_loss", kern, small, kSmallThreads, (rows * b.E + 3 * (size_t)b.B * b.E + b.B) * 4, s, p, small);
    }
    const long long records = (long long)q.runs + b.B;
    if ((uintptr_t)workspace & 3) return fail(kInvalidArg, "router_balance_loss: workspace is not aligned");
    if (workspace_bytes < (records * b.E * 2 + records) * 4)
        return fail(kInvalidArg, "router_balance_loss: workspace holds %lld bytes, needs %lld", workspace_bytes, (records * b.E * 2 + records) * 4);
    p.P = reinterpret_cast<float*>(workspace);
    p.C = reinterpret_cast<int32_t*>(p.P + records * b.E);
    p.N = p.C + records * b.E;
    if (b.T > 0) {
        const size_t smem = (size_t)(kThreads / 32 + 1) * b.E * 4;
        const Kern kern = pick<kPartial>(b.dtype, q.v, q.j);
        if (smem > 40 * 1024 && umma::prepare_kernel(reinterpret_cast<const void*>(kern), kThreads, (kThreads / 32 + 1) * kBalanceMaxExperts * 4, 0) == 0)
            return fail(kCudaError, "router_balance_loss: the kernel cannot be launched on this device");
        if (int st = launch("router_balance_loss", kern, q.runs, kThreads, smem, s, p)) return st;
    }
    const int cw = (b.E + kFinishCtas - 1) / kFinishCtas;
    int parts = 1, per = 1;
    while (parts * 2 * cw <= kFinishThreads) parts *= 2;
    while (per * 2 <= parts && per * 2 * b.B <= parts) per *= 2;
    p.cw = cw; p.parts = parts; p.per = per;
    if (int st = launch("router_balance_loss (finish)", balance_finish_kernel, kFinishCtas, kFinishThreads, 0, s, p)) return st;
    return b.grad ? launch_balance_grad(b, s) : (int)kOk;
}

int launch_balance_grad(const BalanceParams& b, cudaStream_t s) {
    if (int st = check(b, "router_balance_grad")) return st;
    if (b.T == 0) return kOk;
    if (!b.u || !b.grad) return fail(kInvalidArg, "router_balance_grad: null pointer");
    const Plan q = plan_of(b);
    return launch("router_balance_grad", pick<kGrad>(b.dtype, q.v, q.j), q.runs, kThreads, 0, s, params(b, q));
}

int launch_expert_counts(const int32_t* ids, const uint8_t* mask, int T, int topk, int E, int32_t* counts, cudaStream_t s) {
    if (T < 0 || topk < 1) return fail(kInvalidArg, "expert_counts: bad sizes");
    if (E < 1 || E > kBalanceMaxExperts) return fail(kUnsupported, "expert_counts: 1 <= experts <= %d (got %d)", kBalanceMaxExperts, E);
    if ((long long)T * topk > 0x7FFFFFFF) return fail(kUnsupported, "expert_counts: counts of more than 2^31 - 1 picks");
    if (!counts || (T > 0 && !ids)) return fail(kInvalidArg, "expert_counts: null pointer");
    if (((uintptr_t)ids | (uintptr_t)counts) & 3) return fail(kInvalidArg, "expert_counts: topk_ids or counts is not aligned");
    cudaError_t e = cudaMemsetAsync(counts, 0, (size_t)E * 4, s);
    if (e != cudaSuccess) return fail(kCudaError, "expert_counts: %s", cudaGetErrorString(e));
    if (T == 0) return kOk;
    const long long n = (long long)T * topk;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<long long>((n + 4 * kThreads - 1) / (4 * kThreads), 2LL * sm_count()));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)E * 4;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    cfg.numAttrs = launch_attrs(attr, 1);
    e = cudaLaunchKernelEx(&cfg, expert_counts_kernel, ids, mask, n, topk, E, counts);
    if (e != cudaSuccess) return fail(kCudaError, "expert_counts launch: %s", cudaGetErrorString(e));
    return kOk;
}

}  // namespace mlk
