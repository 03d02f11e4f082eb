// Attention of few query rows over a paged K/V cache: single tokens and short
// drafted runs, at most R = 8 or 16 query rows of one KV head at a time.
//
// Work items are (sequence, KV head, row tile, split of the visible rows); the
// four warps of a CTA take the item's 16-row steps in turn, each with its own
// online softmax, and merge at the end. Memory bound: a cached row is read once
// from HBM (row tiles of one sequence are neighbours in the grid and meet in L2)
// and never staged: every lane loads 16-byte pieces of K and V rows straight into
// the registers it needs as tensor-core fragments (mma.sync m16n8k16; a tile of 8
// rows cannot fill a tcgen05 tile of 128), one step ahead of their use.
//
// Fragments. The order of the dims inside a k-step and of the output columns is
// free as long as both operands agree, so it follows the memory layout: lane
// (g = lane / 4, t = lane % 4) holds 16-byte pieces of key g's row for Q K^T, and
// dims [g DIM / 8, (g + 1) DIM / 8) of keys 2t, 2t + 1, 8 + 2t, 9 + 2t for P V, whose
// pairs of keys meet by byte permutes.
//
// Precision. FP32 queries and weights enter as sums of 16-bit parts whose products
// with the stored rows are exact: byte codes are FP16 integers, and two FP16 parts
// of a value scaled into FP16's range carry 22 bits; BF16 rows take three BF16
// parts (24 bits). With R = 8 the A tile of 16 rows is [first parts; second parts],
// so one MMA forms both. Sums in the tensor core truncate (about 4e-8 of the sum a
// step): chains stay as short as one warp's share of an item.
#pragma once
#include "paged.cuh"
#include <cuda_fp16.h>

namespace tcm {

constexpr int kPdWarps = 4, kPdThreads = kPdWarps * 32;
constexpr int kPdSplitsMax = 128;  // splits of one (sequence, KV head, row tile)

struct PagedDecodeArgs {
    PagedView v;
    float *out;
    const float *q;
    long long out_stride, q_stride;
    int group, window, sinks;
    int few;              // sequences of at most this many new rows are this kernel's
    int row_tiles, splits, tiles_per_item;
    float scale2;         // log2(e) / sqrt(dim): base-2 scores
    float *part;          // [item][R][DIM]
    float2 *ml;           // [item][R]: running maximum and sum
    unsigned *counters;   // [sequence][KV head][row tile], zero between calls
    int *status;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int KIND>
__device__ __forceinline__ void mma_kind(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (KIND == kPagedBytes) mma_f16(c, a0, a1, a2, a3, b0, b1);
    else mma_bf16(c, a0, a1, a2, a3, b0, b1);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two values as the parts of a pair of 16-bit operands: parts[0] + parts[1] (+ parts[2])
// is the value to 22 (FP16) or 24 (BF16) bits.
template <int KIND> constexpr int kPdParts = KIND == kPagedBytes ? 2 : 3;
template <int KIND> __device__ __forceinline__ void split_pair(float x, float y, uint32_t (&parts)[kPdParts<KIND>]) {
    if constexpr (KIND == kPagedBytes) {
        parts[0] = pack_f16(x, y);
        const float2 h = __half22float2(*reinterpret_cast<__half2 *>(&parts[0]));
        parts[1] = pack_f16(x - h.x, y - h.y);
    } else {
        parts[0] = pack_bf16(x, y);
        x -= bf16_lo(parts[0]);
        y -= bf16_hi(parts[0]);
        parts[1] = pack_bf16(x, y);
        parts[2] = pack_bf16(x - bf16_lo(parts[1]), y - bf16_hi(parts[1]));
    }
}

// Four signed bytes with their sign bits flipped -> two pairs of exact FP16 integers:
// 0x6400 | u is 1024 + u, so subtracting 1024 + 128 leaves the code.
__device__ __forceinline__ uint32_t codes_f16(uint32_t w, uint32_t select) {
    const uint32_t p = __byte_perm(w, 0x64646464u, select);
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(0x64806480u));
    return r;
}

// floor(log2 |x|) of a normal number; 0 for 0, subnormals, infinities and NaN.
__device__ __forceinline__ int exponent_of(float x) {
    const int e = (int)((__float_as_uint(x) >> 23) & 0xff);
    return e == 0 || e == 0xff ? 0 : e - 127;
}
__device__ __forceinline__ float power_of_two(int e) {
    e = e < -126 ? -126 : (e > 127 ? 127 : e);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Rows are read past L1, which keeps nothing that an append may have changed.
__device__ __forceinline__ uint4 ld_row16(const void *p) { return __ldcg(static_cast<const uint4 *>(p)); }
__device__ __forceinline__ float quad_max(float x) {  // over the four lanes of a fragment row
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
// A pair of BF16 values with non-finite ones replaced by 0.
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
    return w;
}
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

constexpr float kPdWeightTop = 14.f;  // byte rows' weights are scaled to at most 2^14

template <int KIND, int DIM, int R>
__global__ void __launch_bounds__(kPdThreads, (KIND == kPagedBytes ? 4 : 3)) paged_decode_kernel(const PagedDecodeArgs a) {
    constexpr bool kBytes = KIND == kPagedBytes;
    constexpr int ES = kBytes ? 1 : 2;              // bytes an element
    constexpr int KP = DIM * ES / 64;               // 16-byte pieces of a key a lane holds for Q K^T
    constexpr int KS = DIM / 16;                    // k-steps of Q K^T
    constexpr int DV = DIM / 8;                     // dims of a key a lane holds for P V
    constexpr int VW = DV * ES / 4;                 // the same in words
    constexpr int P = kPdParts<KIND>;
    constexpr int NA = R == 8 ? (P + 1) / 2 : P;    // A tiles a product takes
    constexpr int RW = R / 8;                       // query rows a lane holds scores of
    __shared__ __align__(16) uint4 qf[NA][KS][32];  // Q's fragments
    __shared__ float qs[R];                         // scale2 times the row's power of two
    __shared__ __align__(16) float wo[kPdWarps][R][DIM];
    __shared__ float2 wml[kPdWarps][R];
    __shared__ int last_s;
    const PagedView &v = a.v;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int s = blockIdx.z, h = blockIdx.y, rt = blockIdx.x % a.row_tiles, sp = blockIdx.x / a.row_tiles;
    pdl_wait();
    PagedExtent e;
    const int bad_extent = paged_extent(&v, s, &e);
    if (e.count > a.few || !e.count) {
        if (bad_extent && !blockIdx.x && !h && !tid) paged_report(a.status, bad_extent);
        return;
    }
    const int rows = e.count * a.group, r0 = rt * R;  // row r of the KV head: new row r / group, head r % group
    if (r0 >= rows) return;
    const int first = e.length - e.count + r0 / a.group;
    const int last = e.length - e.count + (min(rows, r0 + R) - 1) / a.group;
    const PagedTiles tiles = paged_tiles(first, last, a.window, a.sinks, 4);
    const int splits = max(1, (tiles.count + a.tiles_per_item - 1) / a.tiles_per_item);
    if (sp >= splits) return;
    const int k0 = sp * a.tiles_per_item, k1 = min(tiles.count, k0 + a.tiles_per_item);

    // ---- this item's queries as fragments: warp w prepares rows w, w + 4, ...
    for (int r = warp; r < R; r += kPdWarps) {
        float x[DIM / 32], m = 0.f;
        const bool on = r0 + r < rows;
        if (on) {
            const float *src = a.q + (long long)(e.start + (r0 + r) / a.group) * a.q_stride +
                               (h * a.group + (r0 + r) % a.group) * DIM;
            if constexpr (DIM == 128) {
                const float4 f = reinterpret_cast<const float4 *>(src)[lane];
                x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
            } else {
                const float2 f = reinterpret_cast<const float2 *>(src)[lane];
                x[0] = f.x, x[1] = f.y;
            }
        } else {
#pragma unroll
            for (int c = 0; c < DIM / 32; c++) x[c] = 0.f;
        }
        float up = 1.f, down = 1.f;
        if constexpr (kBytes) {  // into FP16's range: the largest element in [2^14, 2^15)
#pragma unroll
            for (int c = 0; c < DIM / 32; c++) m = fmaxf(m, fabsf(x[c]));
            const int ex = exponent_of(warp_max(m)) - 14;
            up = power_of_two(-ex);
            down = power_of_two(ex);
        }
        if (lane == 0) qs[r] = a.scale2 * down;
#pragma unroll
        for (int c = 0; c < DIM / 32; c += 2) {
            uint32_t parts[P];
            split_pair<KIND>(x[c] * up, x[c + 1] * up, parts);
            // Dims d, d + 1 -> k-step, lane and half of the fragment.
            const int d = lane * (DIM / 32) + c;
            int ks, ft, fh;
            if constexpr (kBytes) ks = (d / 64) * 4 + (d % 16) / 4, ft = (d % 64) / 16, fh = (d % 4) / 2;
            else ks = (d / 32) * 2 + (d % 8) / 4, ft = (d % 32) / 8, fh = (d % 4) / 2;
#pragma unroll
            for (int p = 0; p < P; p++) {
                // R = 8: part p is rows 8 (p % 2) + r of tile p / 2; R = 16: row r of tile p.
                const int tile = R == 8 ? p / 2 : p, row = R == 8 ? (p % 2) * 8 + r : r;
                reinterpret_cast<uint32_t *>(&qf[tile][ks][(row % 8) * 4 + ft])[2 * fh + row / 8] = parts[p];
            }
            if (R == 8 && P % 2) reinterpret_cast<uint32_t *>(&qf[NA - 1][ks][r * 4 + ft])[2 * fh + 1] = 0u;
        }
    }
    __syncthreads();

    // ---- the loop over this warp's 16-row steps
    const bool whole = v.page % 16 == 0;  // a step lies inside one page
    const int64_t half = (int64_t)v.pages * v.kvheads * v.page;
    float o[DV][4], m[RW], mu[RW], l[RW], sc[RW];
#pragma unroll
    for (int j = 0; j < DV; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[j][c] = 0.f;
#pragma unroll
    for (int r = 0; r < RW; r++) m[r] = mu[r] = -INFINITY, l[r] = 0.f, sc[r] = qs[g + 8 * r];

    int bad = 0;
    // The row of place j; -1 where there is none (behind the last query, or no page).
    auto page_of = [&](int k) -> int {  // the page id of lane % 16's row of step k
        if (k >= k1) return -1;
        const int j = min(paged_tile(tiles, k) * 16 + (whole ? 0 : lane & 15), last);
        return v.table[(int64_t)s * v.table_stride + paged_div(&v, j)];
    };
    auto row_of = [&](int k, int id) -> int64_t {  // of lane % 16's place
        if (k >= k1) return -1;
        const int j = paged_tile(tiles, k) * 16 + (lane & 15);
        const int64_t row = j <= last ? paged_row(&v, id, j, paged_div(&v, j), h) : -1;
        // A page that no query of the sequence needs may be missing; one that holds a visible row may not.
        if (row < 0 && j <= last && (a.window == 0 || j < a.sinks || (int64_t)j > (int64_t)first - a.window)) bad |= kPagedBadPage;
        return row;
    };
    uint4 kr[2][KP];
    uint4 vr[4][VW / 4 > 0 ? VW / 4 : 1];  // DIM 64 bytes: half a piece is used
    float scales = 0.f;                    // lanes 0-15: the K scale of the lane's row, 16-31 V's
    auto load_k = [&](int64_t row) {
#pragma unroll
        for (int gr = 0; gr < 2; gr++) {
            const int64_t rk = __shfl_sync(0xffffffffu, row, gr * 8 + g);
            const char *p = static_cast<const char *>(v.keys) + rk * (DIM * ES) + t * 16;
#pragma unroll
            for (int c = 0; c < KP; c++) kr[gr][c] = rk >= 0 ? ld_row16(p + c * 64) : make_uint4(0, 0, 0, 0);
        }
        if constexpr (kBytes) scales = row >= 0 ? __ldcg(v.scales + (lane >= 16 ? half : 0) + row) : 1.f;
    };
    auto load_v = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t rv = __shfl_sync(0xffffffffu, row, (i >> 1) * 8 + 2 * t + (i & 1));
            const char *p = static_cast<const char *>(v.values) + rv * (DIM * ES) + g * (DV * ES);
            if constexpr (VW == 2) {
                const uint2 w = rv >= 0 ? __ldcg(reinterpret_cast<const uint2 *>(p)) : make_uint2(0, 0);
                vr[i][0] = make_uint4(w.x, w.y, 0, 0);
            } else {
#pragma unroll
                for (int c = 0; c < VW / 4; c++) vr[i][c] = rv >= 0 ? ld_row16(p + c * 16) : make_uint4(0, 0, 0, 0);
            }
        }
    };

    int k = k0 + warp;
    int64_t row = row_of(k, page_of(k));
    int id_next = page_of(k + kPdWarps);
    load_k(row);
    load_v(row);
    for (; k < k1; k += kPdWarps) {
        const int64_t next = row_of(k + kPdWarps, id_next);
        const unsigned there = __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
        id_next = page_of(k + 2 * kPdWarps);
        // Scores of 16 places: S[gr] columns 2t, 2t + 1 are places base + 8 gr + 2t, + 1.
        float sf[2][4];
#pragma unroll
        for (int gr = 0; gr < 2; gr++)
#pragma unroll
            for (int c = 0; c < 4; c++) sf[gr][c] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            uint32_t b0[2], b1[2];
#pragma unroll
            for (int gr = 0; gr < 2; gr++) {
                if constexpr (kBytes) {
                    const uint32_t w = word(kr[gr][ks / 4], ks % 4) ^ 0x80808080u;
                    b0[gr] = codes_f16(w, 0x4140);
                    b1[gr] = codes_f16(w, 0x4342);
                } else {
                    b0[gr] = word(kr[gr][ks / 2], (ks % 2) * 2);
                    b1[gr] = word(kr[gr][ks / 2], (ks % 2) * 2 + 1);
                }
            }
#pragma unroll
            for (int n = NA - 1; n >= 0; n--) {
                const uint4 f = qf[n][ks][lane];
#pragma unroll
                for (int gr = 0; gr < 2; gr++) mma_kind<KIND>(sf[gr], f.x, f.y, f.z, f.w, b0[gr], b1[gr]);
            }
        }
        float ks4[4], vs4[4];
        if constexpr (kBytes) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = (i >> 1) * 8 + 2 * t + (i & 1);
                ks4[i] = __shfl_sync(0xffffffffu, scales, at);
                vs4[i] = __shfl_sync(0xffffffffu, scales, 16 + at);
            }
        }
        load_k(next);

        const int base = paged_tile(tiles, k) * 16;
        // Every query of the tile sees every place of the step?
        const bool full = there == 0xffffu && base + 15 <= first &&
                          (a.window == 0 || base + 15 < a.sinks || (int64_t)base > (int64_t)last - a.window);
        uint32_t pa[RW][2][P];  // weights as fragments' parts: [row][group of 8 places][part]
        float keep[RW];         // what this step's new reference leaves of the sums so far
        bool moved = false;
#pragma unroll
        for (int r = 0; r < RW; r++) {
            float x[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[i] = R == 8 ? sf[i >> 1][i & 1] + sf[i >> 1][2 + (i & 1)] : sf[i >> 1][2 * r + (i & 1)];
                if constexpr (kBytes) x[i] *= ks4[i];
                x[i] *= sc[r];
            }
            if (!full) {
                const int at = e.length - e.count + min(r0 + g + 8 * r, rows - 1) / a.group;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int c = (i >> 1) * 8 + 2 * t + (i & 1);
                    if (!((there >> c) & 1) || !paged_sees(at, base + c, a.window, a.sinks)) x[i] = -INFINITY;
                }
            }
            const float m_new = fmaxf(m[r], quad_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))));
            const float mr = m_new == -INFINITY ? 0.f : m_new;
            l[r] *= m[r] == -INFINITY ? 0.f : exp2f(m[r] - mr);
            m[r] = m_new;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                w[i] = exp2f(x[i] - mr);
                l[r] += w[i];
            }
            float mu_new = m_new;
            if constexpr (kBytes) {
                // The weight of a row is p_j s_j. mu follows log2 of the largest, so that 2^14 of the
                // FP16 range goes to whatever carries the sum, however unlike the rows' scales are;
                // at most 2^113 from m, so that the factor is a number.
                float u = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; i++) u = fmaxf(u, x[i] + __log2f(vs4[i]));
                mu_new = fmaxf(fmaxf(mu[r], quad_max(u)), m_new - 113.f);
                const float f = mu_new == -INFINITY ? 0.f : exp2f(mr - mu_new + kPdWeightTop);
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = x[i] == -INFINITY ? 0.f : w[i] * (vs4[i] * f);
            }
            keep[r] = mu[r] == -INFINITY ? 0.f : exp2f(mu[r] - mu_new);
            moved |= mu_new != mu[r];
            mu[r] = mu_new;
            split_pair<KIND>(w[0], w[1], pa[r][0]);
            split_pair<KIND>(w[2], w[3], pa[r][1]);
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int j = 0; j < DV; j++) {
                o[j][0] *= keep[0];
                o[j][1] *= keep[0];
                o[j][2] *= keep[RW - 1];
                o[j][3] *= keep[RW - 1];
            }
        }
        if constexpr (!kBytes) {
            // A weight of 0 times a non-finite value would spoil queries that do not see it.
            if (!full) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int c = 0; c < VW / 4; c++)
                        vr[i][c] = make_uint4(finite_pair(vr[i][c].x), finite_pair(vr[i][c].y), finite_pair(vr[i][c].z),
                                              finite_pair(vr[i][c].w));
            }
        }
        auto pv = [&](float(&acc)[4], uint32_t b0, uint32_t b1) {
            if constexpr (R == 8) {
                if constexpr (P == 3) mma_kind<KIND>(acc, pa[0][0][2], 0u, pa[0][1][2], 0u, b0, b1);
                mma_kind<KIND>(acc, pa[0][0][0], pa[0][0][1], pa[0][1][0], pa[0][1][1], b0, b1);
            } else {
#pragma unroll
                for (int p = P - 1; p >= 0; p--)
                    mma_kind<KIND>(acc, pa[0][0][p], pa[RW - 1][0][p], pa[0][1][p], pa[RW - 1][1][p], b0, b1);
            }
        };
#pragma unroll
        for (int c = 0; c < VW; c++) {
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = word(vr[i][c / 4], c % 4);
            if constexpr (kBytes) {
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] ^= 0x80808080u;
                const uint32_t lo0 = __byte_perm(x[0], x[1], 0x5140), hi0 = __byte_perm(x[0], x[1], 0x7362);
                const uint32_t lo1 = __byte_perm(x[2], x[3], 0x5140), hi1 = __byte_perm(x[2], x[3], 0x7362);
                pv(o[4 * c], codes_f16(lo0, 0x4140), codes_f16(lo1, 0x4140));
                pv(o[4 * c + 1], codes_f16(lo0, 0x4342), codes_f16(lo1, 0x4342));
                pv(o[4 * c + 2], codes_f16(hi0, 0x4140), codes_f16(hi1, 0x4140));
                pv(o[4 * c + 3], codes_f16(hi0, 0x4342), codes_f16(hi1, 0x4342));
            } else {
                pv(o[2 * c], __byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410));
                pv(o[2 * c + 1], __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
            }
        }
        load_v(next);
        row = next;
    }
    if (bad || bad_extent) paged_report(a.status, bad | bad_extent);

    // ---- the four warps' states: lane (g, t) holds dims [2 t DV, (2 t + 2) DV) of row g (+ 8)
#pragma unroll
    for (int r = 0; r < RW; r++) {
        float sum = l[r];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (t == 0) wml[warp][g + 8 * r] = make_float2(m[r], sum);
        const float f = kBytes ? (mu[r] == -INFINITY ? 0.f : exp2f(mu[r] - m[r] - kPdWeightTop)) : 1.f;
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float *dst = &wo[warp][g + 8 * r][(2 * t + c) * DV];
#pragma unroll
            for (int j = 0; j < DV; j += 4) {
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = f * (R == 8 ? o[j + i][c] + o[j + i][2 + c] : o[j + i][2 * r + c]);
                *reinterpret_cast<float4 *>(dst + j) = make_float4(y[0], y[1], y[2], y[3]);
            }
        }
    }
    __syncthreads();
    auto store_out = [&](int r, int d, float4 y, float sum) {
        const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);  // nothing seen: zeros
        *reinterpret_cast<float4 *>(a.out + (long long)(e.start + (r0 + r) / a.group) * a.out_stride +
                                    (h * a.group + (r0 + r) % a.group) * DIM + d) =
            make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
    };
    const int64_t base_item = (((int64_t)s * v.kvheads + h) * a.row_tiles + rt) * a.splits;
    const int live = min(R, rows - r0);
    for (int i = tid; i < live * (DIM / 4); i += kPdThreads) {
        const int r = i / (DIM / 4), d = i % (DIM / 4) * 4;
        float top = -INFINITY, sum = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kPdWarps; w++) top = fmaxf(top, wml[w][r].x);
#pragma unroll
        for (int w = 0; w < kPdWarps; w++) {
            const float2 ml = wml[w][r];
            const float f = ml.x == -INFINITY ? (ml.y == ml.y ? 0.f : ml.y) : exp2f(ml.x - top);
            const float4 x = *reinterpret_cast<const float4 *>(&wo[w][r][d]);
            sum = fmaf(ml.y, f, sum);
            y.x = fmaf(x.x, f, y.x);
            y.y = fmaf(x.y, f, y.y);
            y.z = fmaf(x.z, f, y.z);
            y.w = fmaf(x.w, f, y.w);
        }
        if (splits == 1) {
            store_out(r, d, y, sum);
        } else {
            *reinterpret_cast<float4 *>(a.part + ((base_item + sp) * R + r) * DIM + d) = y;
            if (d == 0) a.ml[(base_item + sp) * R + r] = make_float2(top, sum);
        }
    }
    if (splits == 1) return;

    // ---- the last split of the row tile to arrive adds all of them, in order
    __threadfence();
    __syncthreads();
    unsigned *counter = &a.counters[((int64_t)s * v.kvheads + h) * a.row_tiles + rt];
    if (tid == 0) last_s = atomicAdd(counter, 1u) == (unsigned)(splits - 1);
    __syncthreads();
    if (!last_s) return;
    __threadfence();
    if (tid == 0) *counter = 0u;
    float *factor = &wo[0][0][0];  // [row][split]
    static_assert(R * kPdSplitsMax <= kPdWarps * R * DIM, "factors fit the merge buffer");
    __shared__ float total[R];
    for (int r = warp; r < live; r += kPdWarps) {
        float top = -INFINITY, sum = 0.f;
        for (int i = lane; i < splits; i += 32) top = fmaxf(top, __ldcg(&a.ml[(base_item + i) * R + r]).x);
        top = warp_max(top);
        for (int i = lane; i < splits; i += 32) {
            const float2 ml = __ldcg(&a.ml[(base_item + i) * R + r]);
            const float f = ml.x == -INFINITY ? (ml.y == ml.y ? 0.f : ml.y) : exp2f(ml.x - top);
            factor[r * kPdSplitsMax + i] = f;
            sum = fmaf(ml.y, f, sum);
        }
        sum = warp_sum(sum);
        if (lane == 0) total[r] = sum;
    }
    __syncthreads();
    for (int i = tid; i < live * (DIM / 4); i += kPdThreads) {
        const int r = i / (DIM / 4), d = i % (DIM / 4) * 4;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int w = 0; w < splits; w++) {
            const float f = factor[r * kPdSplitsMax + w];
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(a.part + ((base_item + w) * R + r) * DIM + d));
            y.x = fmaf(x.x, f, y.x);
            y.y = fmaf(x.y, f, y.y);
            y.z = fmaf(x.z, f, y.z);
            y.w = fmaf(x.w, f, y.w);
        }
        store_out(r, d, y, total[r]);
    }
}

}  // namespace tcm
