// Prepack of 4-bit weights (format in w4.cuh): row-major nibbles <-> 512-byte blocks, and the pair order of scales and
// zero points.  Run once per matrix at load time; a thread moves one lane's 16 bytes of a block (eight 2-byte reads, one
// 16-byte store).  What bounds it: the 2-byte accesses to the row-major side.  28672 x 8192 (117 MB in, 117 MB out; 36 us at the
// copy bandwidth) takes 60 us, the way back, with 2-byte stores, 118 us; the scales of that matrix in groups of 32 (29 MB in all,
// 4.5 us) 21 us.  Not made faster: 100 GB of packed weights take 50 ms, once.
#include "w4.cuh"

namespace mlk {

namespace {

// Four k of one row as they sit in the packed word: bits 0, 16, 8, 24 (pairs 0 and 2 of a row r; a row r + 8 is 4 higher).
__device__ __forceinline__ uint32_t spread(uint32_t v) {
    return (v & 0xFu) | ((v & 0xF0u) << 12) | (v & 0xF00u) | ((v & 0xF000u) << 12);
}
__device__ __forceinline__ uint16_t gather(uint32_t w) {
    return (uint16_t)((w & 0xFu) | ((w >> 12) & 0xF0u) | (w & 0xF00u) | ((w >> 12) & 0xF000u));
}

__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* __restrict__ src, uint8_t* __restrict__ dst,
                                                     long long lanes, int k, int kc, int inverse) {
    pdl_wait();
    pdl_launch_dependents();
    const uint8_t* const rowmajor = inverse ? dst : src;
    const uint8_t* const blocks = inverse ? src : dst;
    const long long ld = k / 2;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < lanes; i += (long long)gridDim.x * blockDim.x) {
        const int lane = (int)(i & 31), r = lane >> 2, t = lane & 3;
        const long long block = i >> 5, R = block / kc;
        const int C = (int)(block - R * kc);
        const long long lo = (R * 16 + r) * ld, hi = lo + 8 * ld;
        uint4 out = make_uint4(0u, 0u, 0u, 0u);
        uint32_t* const w = reinterpret_cast<uint32_t*>(&out);
        if (inverse) out = *reinterpret_cast<const uint4*>(blocks + i * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k0 = C * kW4BlockK + 16 * j + 4 * t;
            if (k0 < k) {                                       // k is a multiple of 32: four k are in or out together
                uint16_t* const a = reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(rowmajor) + lo + k0 / 2);
                uint16_t* const b = reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(rowmajor) + hi + k0 / 2);
                if (inverse) {
                    *a = gather(w[j]);
                    *b = gather(w[j] >> 4);
                } else {
                    w[j] = spread(*a) | (spread(*b) << 4);
                }
            }
        }
        if (!inverse) *reinterpret_cast<uint4*>(const_cast<uint8_t*>(blocks) + i * 16) = out;
    }
}

template <class T>
__global__ void __launch_bounds__(256) w4_groups_kernel(const T* __restrict__ src, T* __restrict__ dst, long long n, int groups) {
    pdl_wait();
    pdl_launch_dependents();
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const int h = (int)(i & 1), r = (int)((i >> 1) & 7);
        const long long rest = i >> 4, R = rest / groups;
        dst[i] = src[(R * 16 + h * 8 + r) * groups + (rest - R * groups)];
    }
}

template <class... KArgs, class... Args>
int launch_grid_stride(const char* what, void (*kern)(KArgs...), long long n, cudaStream_t s, Args... args) {
    if (n == 0) return kOk;
    cudaLaunchConfig_t cfg = {};
    const long long blocks = (n + 255) / 256, most = 16LL * sm_count();
    cfg.gridDim = dim3((unsigned)(blocks < most ? blocks : most));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    cfg.numAttrs = launch_attrs(attr, 1);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) return fail(kCudaError, "%s launch: %s", what, cudaGetErrorString(e));
    return kOk;
}

}  // namespace

int launch_w4_pack(const void* src, void* dst, long long m, int k, int inverse, cudaStream_t s) {
    if (m < 0 || m % 16 != 0) return fail(kInvalidArg, "layoutA_w4: m must be a multiple of 16 (got %lld)", m);
    if (k <= 0 || k % 32 != 0) return fail(kInvalidArg, "layoutA_w4: k must be a positive multiple of 32 (got %d)", k);
    if (k > kW4MaxDim) return fail(kUnsupported, "layoutA_w4: more than 2^28 k");
    if (m > 0 && (!src || !dst)) return fail(kInvalidArg, "layoutA_w4: null pointer");
    if (((uintptr_t)src | (uintptr_t)dst) & 15) return fail(kInvalidArg, "layoutA_w4: pointers must be 16-byte aligned");
    const int kc = (k + kW4BlockK - 1) / kW4BlockK;
    const long long lanes = m / 16 * kc * 32;
    return launch_grid_stride("layoutA_w4", w4_pack_kernel, lanes, s, reinterpret_cast<const uint8_t*>(src),
                              reinterpret_cast<uint8_t*>(dst), lanes, k, kc, inverse);
}

int launch_w4_groups(const void* src, void* dst, long long m, int groups, int elem, cudaStream_t s) {
    if (m < 0 || m % 16 != 0) return fail(kInvalidArg, "layoutA_w4_groups: m must be a multiple of 16 (got %lld)", m);
    if (groups <= 0) return fail(kInvalidArg, "layoutA_w4_groups: there must be at least one group");
    if (m > 0 && (!src || !dst)) return fail(kInvalidArg, "layoutA_w4_groups: null pointer");
    if (elem == 2 && (((uintptr_t)src | (uintptr_t)dst) & 1)) return fail(kInvalidArg, "layoutA_w4_groups: pointers are not aligned");
    const long long n = m * groups;
    if (elem == 1)
        return launch_grid_stride("layoutA_w4_groups", w4_groups_kernel<uint8_t>, n, s, reinterpret_cast<const uint8_t*>(src),
                                  reinterpret_cast<uint8_t*>(dst), n, groups);
    if (elem == 2)
        return launch_grid_stride("layoutA_w4_groups", w4_groups_kernel<uint16_t>, n, s, reinterpret_cast<const uint16_t*>(src),
                                  reinterpret_cast<uint16_t*>(dst), n, groups);
    return fail(kInvalidArg, "layoutA_w4_groups: elements of 1 or 2 bytes (got %d)", elem);
}

}  // namespace mlk
