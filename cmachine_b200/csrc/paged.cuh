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

// What the pool can hold of a value of magnitude m: BF16 rounds from 2^128 - 2^119 on to infinity; 127 times FP32's
// largest number over 127 is one too.
template <int KIND> __device__ __forceinline__ bool paged_holds(float m) {
    return m < (KIND == kPagedBytes ? 0x1.fffffep127f : 0x1.ffp127f);
}

// Codes of elements of a row whose scale is max|x| / 127. A row so small that this underflows stands for zeros (scale 0,
// codes 0). The quotient by a reciprocal is within 5e-5 of the divided one; only where it comes near a half does the
// division decide (all of them by division: 26 us instead of 20 for 42,000 rows). The largest scale, 2^128 / 127, still
// has a reciprocal.
template <int E> __device__ __forceinline__ void paged_codes(const float (&y)[E], float scale, int8_t (&q)[E]) {
    const float up = __fdividef(1.f, scale);
    bool near_half = false;
#pragma unroll
    for (int c = 0; c < E; c++) {
        const float quotient = y[c] * up, code = rintf(quotient);
        near_half |= !(fabsf(quotient - code) <= 0.4999f);
        q[c] = (int8_t)fminf(127.f, fmaxf(-127.f, code));
    }
    if (near_half)
#pragma unroll
        for (int c = 0; c < E; c++)
            q[c] = scale > 0.f ? (int8_t)fminf(127.f, fmaxf(-127.f, roundf(__fdiv_rn(y[c], scale)))) : (int8_t)0;
}

}  // namespace tcm
