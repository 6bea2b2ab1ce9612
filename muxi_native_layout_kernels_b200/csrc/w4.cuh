// 4-bit weights with group scales: format, decode, and the host-side launch interface.
//
//   W[row, k] = (q[row, k] - z[row, k / group]) * s[row, k / group],  q, z in 0..15, s in the activation type
//
// Packed weights ("layout A, 4 bits"): [m/16][ceil(k/64)][32 lanes][16 bytes].  One block of 512 bytes holds 16 rows x
// 64 k.  Lane (r = lane / 4, t = lane % 4) owns rows r and r + 8; of its 32-bit word j (0..3) the nibble pair p (0..3) at
// bits 4p and 16 + 4p is row r + 8 * (p & 1), k = 16 j + 4 t + 2 * (p >> 1) and the k after it.  Word j is therefore the
// whole 16-row operand of one m16n8k16 tensor-core step over k = 16 j .. 16 j + 15, in the register order (a0, a1, a2,
// a3) of that instruction with the contraction index permuted so that lane t owns four consecutive k (one 8-byte load of
// the activation row is the matching column operand).  It is also the 16-lane x 256-bit fragment of a tensor-memory
// store: column 2t + (p >> 1) of the eight 32-bit columns a step fills is the pair k = 16 j + 2 (2t + (p >> 1)), +1: natural
// k order.  k beyond the matrix inside the last block is stored as 0 and never multiplied by anything but 0.
// Scales and zero points: [m/16][k/group][8][2], entry (r, h) = row r + 8 h of the 16-row group, so that a lane fetches
// the values of its two rows with one load.
#pragma once

#include "common.cuh"
#include "status.h"

namespace mlk {

constexpr int kW4BlockK = 64;        // k per 512-byte block
constexpr int kW4BlockBytes = 512;
constexpr int kW4MaxDim = 1 << 28;   // rows of a matrix and k: keeps 32-bit row and byte-in-row arithmetic exact

struct W4Weights {
    const uint8_t* q;      // packed blocks
    const void* s;         // 16-bit scales in pair order
    const uint8_t* z;      // zero points in pair order, or null = 8 everywhere
    int group;             // 32, 64 or 128
};

// Decode of one word into the four operand registers.
//   bf16  The nibble bits, left where they are in a 16-bit half, are a subnormal (or first-binade) bf16 number: bits 0..3
//         hold q * 2^-133, bits 4..7 q * 2^-129, both exactly.  One packed fused multiply-add by 2^127 normalises them
//         and subtracts the zero point: (q - z) / 64 for the low nibble, (q - z) / 4 for the high one, exact.  The low
//         nibbles are rows r, the high ones rows r + 8: the factor is a constant of the row and is put back on the fp32
//         sums (kFactorLow, kFactorHigh).  Two rows' pairs cost two ANDs and half a shift this way, where placing all four nibbles
//         at the same position takes three shifts.
//   fp16  The nibble is or-ed under the exponent of 1024: 1024 + q (low) or 1024 + 16 q (high); one packed fused
//         multiply-add turns that into q - z, exact.  (The method of Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't
//         Run: Bringing Large Scale MoE Models into Cloud Scale Production", 2022.)
// `zl`, `zh`: the packed subtrahends of rows r and r + 8, made by zero() from a pair of zero-point bytes of which the low
// four bits count.
template <int WT>
struct W4Decode;

template <>
struct W4Decode<kBF16> {
    static constexpr float kFactorLow = 64.f, kFactorHigh = 4.f;
    static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) { return fma_bf16x2(a, b, c); }
    static __device__ __forceinline__ void zero(uint32_t z, uint32_t& zl, uint32_t& zh) {
        // z as raw bits q * 2^-133: times -2^127 is -z / 64; times 16 (bits 4..7) is -z / 4
        const uint32_t l = (z & 0xFu) * 0x00010001u, h = ((z >> 8) & 0xFu) * 0x00100010u;
        zl = mul_bf16x2(l, 0xFF00FF00u);
        zh = mul_bf16x2(h, 0xFF00FF00u);
    }
    static __device__ __forceinline__ void word(uint32_t w, uint32_t zl, uint32_t zh, uint32_t (&a)[4]) {
        const uint32_t v = w >> 8;
        a[0] = fma2(w & 0x000F000Fu, 0x7F007F00u, zl);
        a[1] = fma2(w & 0x00F000F0u, 0x7F007F00u, zh);
        a[2] = fma2(v & 0x000F000Fu, 0x7F007F00u, zl);
        a[3] = fma2(v & 0x00F000F0u, 0x7F007F00u, zh);
    }
};

template <>
struct W4Decode<kFP16> {
    static constexpr float kFactorLow = 1.f, kFactorHigh = 1.f;
    static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
        uint32_t r;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
        return r;
    }
    static __device__ __forceinline__ void zero(uint32_t z, uint32_t& zl, uint32_t& zh) {
        // -(1024 + z): its low mantissa bits are z; -(64 + z): a mantissa step is 1/16
        zl = 0xE400E400u + (z & 0xFu) * 0x00010001u;
        zh = 0xD400D400u + ((z >> 8) & 0xFu) * 0x00100010u;
    }
    static __device__ __forceinline__ void word(uint32_t w, uint32_t zl, uint32_t zh, uint32_t (&a)[4]) {
        const uint32_t v = w >> 8;
        a[0] = fma2((w & 0x000F000Fu) | 0x64006400u, 0x3C003C00u, zl);
        a[1] = fma2((w & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, zh);
        a[2] = fma2((v & 0x000F000Fu) | 0x64006400u, 0x3C003C00u, zl);
        a[3] = fma2((v & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, zh);
    }
};

// ---- host side ------------------------------------------------------------------------------------------------

// Row-major packed nibbles [m, k/2] (low nibble = even k) <-> the blocks above.
int launch_w4_pack(const void* src, void* dst, long long m, int k, int inverse, cudaStream_t s);
// [m, groups] -> [m/16][groups][8][2], elements of 1 or 2 bytes.
int launch_w4_groups(const void* src, void* dst, long long m, int groups, int elem, cudaStream_t s);

struct W4DenseParams {
    W4Weights w;
    const void* X;         // [n, k]
    void* C;               // [n, m]
    const void* bias;      // [m] or null
    float alpha;
    int m, n, k;
    int dtype;             // kBF16 or kFP16
    int* status;
};
int launch_w4_dense(const W4DenseParams& p, cudaStream_t s);

struct W4ExpertsParams {
    W4Weights w1, w2;      // [E, 2I, H] and [E, H, I]
    const void* x;         // [T, H]
    const int32_t* topk_ids;
    const void* topk_weights;
    void* y;               // [T, H]
    int T, E, topk, H, I, dtype, y_fp32;
    const int32_t* experts_map;
    int experts_map_len;
    void* workspace;
    long long workspace_bytes;
    int* status;
};
long long w4_experts_workspace_bytes(int T, int E, int topk, int H, int I);
int launch_w4_experts(const W4ExpertsParams& p, cudaStream_t s);

}  // namespace mlk
