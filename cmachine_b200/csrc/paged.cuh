// Device helpers of the paged K/V cache kernels: stored rows as FP32 values.
#pragma once
#include "common.cuh"
#include "paged_index.h"

namespace tcm {

constexpr int kPagedBf16 = 2, kPagedBytes = 3;  // TcmPagedCache.kind

__device__ __forceinline__ void paged_report(int *status, int bits) {
    if (bits && status) atomicOr(status, bits);
}

// Four consecutive elements of a stored row at element offset `at`, unscaled.
template <int KIND> __device__ __forceinline__ float4 paged_load4(const void *base, int64_t at) {
    if constexpr (KIND == kPagedBf16) {
        const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + at);
        return make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
    } else {
        const char4 c = *reinterpret_cast<const char4 *>(static_cast<const int8_t *>(base) + at);
        return make_float4((float)c.x, (float)c.y, (float)c.z, (float)c.w);
    }
}

}  // namespace tcm
