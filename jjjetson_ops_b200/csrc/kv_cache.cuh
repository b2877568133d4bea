// The paged cache on the device: checks of the descriptor, element types, and the fault that a bad page number sets.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "../../include/jq_kv_cache.h"
#include "jq_common.cuh"
#include "kv_index.h"

namespace jq {

constexpr int FAULT_BAD_PAGE = 4;
constexpr int64_t KV_MAX_DIM = 256;

// Checks the descriptor and fills the kernels' indices.
int check_kv_cache(const jq_kv_cache *c, KvIndex *ix);

inline int kv_element_bytes(int type) { return type == JQ_KV_E4M3 ? 1 : 2; }

#ifdef __CUDACC__

__device__ __forceinline__ void report_bad_page(int *fault) {
    report_fault(fault, FAULT_BAD_PAGE);
}

struct KvF16 {
    using Element = __half;
    static constexpr float LARGEST = 65504.f;
};
struct KvBf16 {
    using Element = __nv_bfloat16;
    static constexpr float LARGEST = 3.3895313892515355e38f;
};
struct KvE4m3 {
    using Element = __nv_fp8_storage_t;
    static constexpr float LARGEST = 448.f;
};

// to the largest finite value; NaN stays NaN (fminf and fmaxf would lose it)
template <typename T>
__device__ __forceinline__ float saturated(float x) {
    return x > T::LARGEST ? T::LARGEST : (x < -T::LARGEST ? -T::LARGEST : x);
}
__device__ __forceinline__ uint32_t pack2(KvF16, float a, float b) {
    const __half2 h = __floats2half2_rn(saturated<KvF16>(a), saturated<KvF16>(b));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(KvBf16, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(saturated<KvBf16>(a), saturated<KvBf16>(b));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(KvE4m3, float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// N consecutive elements (2, 4 or 8), at an address aligned to all of them
template <typename T, int N>
__device__ __forceinline__ void store_elements(typename T::Element *p, const float *x) {
    constexpr int BYTES = N * (int)sizeof(typename T::Element);
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = pack2(T{}, x[2 * i], x[2 * i + 1]);
    if constexpr (sizeof(typename T::Element) == 1) {
#pragma unroll
        for (int i = 0; i + 1 < N / 2; i += 2) w[i / 2] = w[i] | w[i + 1] << 16;
    }
    if constexpr (BYTES == 2) *reinterpret_cast<uint16_t *>(p) = (uint16_t)w[0];
    if constexpr (BYTES == 4) *reinterpret_cast<uint32_t *>(p) = w[0];
    if constexpr (BYTES == 8) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    if constexpr (BYTES == 16) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

#endif  // __CUDACC__

}  // namespace jq
