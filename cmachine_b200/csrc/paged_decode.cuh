// Attention of few query rows over a paged K/V cache: single tokens and short
// drafted runs, at most R = 8 or 16 query rows of one KV head at a time.
//
// The work is a line of steps: 16 cached rows against one row tile, ordered by
// sequence, KV head, row tile and place. Every CTA of a grid that fills the GPU once
// counts the steps of all sequences (their lengths are on the device), takes an equal
// stretch of the line, and works through the one to few (sequence, KV head, row tile)
// segments in it; its warps take a segment's steps in turn, each with its own online
// softmax, and merge at the segment's end. A segment that began or goes on in another CTA
// leaves a partial result, and the last of its CTAs to arrive adds the partials in order.
// Memory bound: a cached row is read once from HBM (row tiles of one KV head meet in L2).
// Every warp copies its own steps into its own ring of three stages (cp.async, 16 bytes a
// lane, rows found by address), two steps ahead, and waits for no other warp; the products
// are mma.sync m16n8k16 (a tile of 8 rows cannot fill a tcgen05 tile of 128). Loading
// straight into registers instead left the compiler spilling loads in flight, which made
// every one of them a wait: 64 sessions of up to 8192 byte rows took 66 us so.
//
// Fragments. The order of the dims inside a k-step and of the output columns is
// free as long as both operands agree, so it follows the memory layout: lane
// (g = lane / 4, t = lane % 4) reads 16-byte pieces of key g's row for Q K^T, and
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
#include "stream.cuh"
#include <cuda_fp16.h>

namespace tcm {

constexpr int kPdSequences = 512;  // sequences a launch counts in shared memory

struct PagedDecodeArgs {
    PagedView v;
    float *out;
    const float *q;
    long long out_stride, q_stride;
    int group, window, sinks;
    int few;              // sequences of at most this many new rows are this kernel's
    float scale2;         // log2(e) / sqrt(dim): base-2 scores
    float *part;          // [CTA][2][R][DIM]: the first and the last segment of a CTA's stretch
    float2 *ml;           // [CTA][2][R]: running maximum and sum
    unsigned *counters;   // [CTA], of the segment that begins there and goes on; zero between calls
    int *status;
};

// Eight warps a CTA; two CTAs an SM where their rings fit.
constexpr int kPdWarps = 8, kPdThreads = kPdWarps * 32, kPdStages = 3;
template <int KIND, int DIM> struct PdGeo {
    static constexpr int kRow = DIM * (KIND == kPagedBytes ? 1 : 2);          // bytes a stored row
    static constexpr int kStage = 32 * kRow + (KIND == kPagedBytes ? 128 : 0);  // 16 K rows, 16 V rows, their scales
    static constexpr int kCtas = kRow <= 128 ? 2 : 1;
    static constexpr size_t kRing = (size_t)kPdWarps * kPdStages * kStage;
};
// The warps' outputs meet in the rings' memory.
template <int KIND, int DIM, int R> constexpr size_t kPdSmem =
    PdGeo<KIND, DIM>::kRing > (size_t)kPdWarps * R * DIM * 4 ? PdGeo<KIND, DIM>::kRing : (size_t)kPdWarps * R * DIM * 4;

// The 16-byte piece of a stored row of ROW bytes where its piece `piece` lies in a stage: the
// eight lanes that read together (keys 2j, 2j + 1 and four pieces; or four even or odd keys
// and two pieces) meet eight bank groups.
template <int ROW> __device__ __forceinline__ int pd_swizzle(int row, int piece) {
    if (ROW == 64) return piece ^ ((row >> 1) & 3);
    const int far = (((row >> 2) ^ row) & 1) << 2;
    return piece ^ (ROW == 128 ? (row & 2) | far : ((row >> 1) & 1) | far);
}
__device__ __forceinline__ void pd_copy16(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pd_copy4(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}

// Where the 16-byte piece d4 of merge row r lies, in pieces of the row: the eight lanes that
// store together (two rows, four stretches of dims) meet eight different bank groups.
template <int DIM> __device__ __forceinline__ int pd_piece(int r, int d4) {
    return DIM == 128 ? d4 ^ ((d4 >> 3) + 4 * (r & 1)) : d4 ^ ((d4 >> 3) | ((r & 1) << 1));
}

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
__device__ __forceinline__ float ex2(float x) {  // results below 2^-126 are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// What a partial result with maximum and sum ml counts for under the maximum `top`; NaN stays NaN.
__device__ __forceinline__ float pd_factor(float2 ml, float top) {
    return ml.x == -INFINITY ? (ml.y == ml.y ? 0.f : ml.y) : ex2(ml.x - top);
}
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

// A CTA's present segment; read again after the loop, so that the loop keeps its registers.
struct PdSegment {
    PagedExtent e;
    PagedTiles tiles;
    int s, h, r0;
    int k0;        // the segment's first step of the row tile's
    int from, to;  // all of the row tile's steps in the line
};

template <int KIND, int DIM, int R>
__global__ void __launch_bounds__(kPdThreads, (PdGeo<KIND, DIM>::kCtas)) paged_decode_kernel(const PagedDecodeArgs a) {
    constexpr bool kBytes = KIND == kPagedBytes;
    using G = PdGeo<KIND, DIM>;
    constexpr int W = kPdWarps, T = kPdThreads;
    constexpr int ES = kBytes ? 1 : 2;              // bytes an element
    constexpr int KP = DIM * ES / 64;               // 16-byte pieces of a key a lane holds for Q K^T
    constexpr int KS = DIM / 16;                    // k-steps of Q K^T
    constexpr int DV = DIM / 8;                     // dims of a key a lane holds for P V
    constexpr int VW = DV * ES / 4;                 // the same in words
    constexpr int P = kPdParts<KIND>;
    constexpr int NA = R == 8 ? (P + 1) / 2 : P;    // A tiles a product takes
    constexpr int RW = R / 8;                       // query rows a lane holds scores of
    extern __shared__ __align__(1024) unsigned char pc_smem[];
    float4(*wo)[R][DIM / 4] = reinterpret_cast<float4(*)[R][DIM / 4]>(pc_smem);  // the warps' outputs
    __shared__ __align__(16) uint4 qf[NA][KS][32];  // Q's fragments
    __shared__ float qs[R];                         // scale2 times the row's power of two
    __shared__ float2 wml[W][R];
    __shared__ int upto[kPdSequences + 1];    // steps before each sequence
    __shared__ int last_s;
    __shared__ PdSegment seg;
    const PagedView &v = a.v;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();

    // ---- this CTA's stretch of the line of steps
    auto tiles_of = [&](const PagedExtent &e, int rt) {
        const int origin = e.length - e.count, r0 = rt * R, r1 = min(e.count * a.group, r0 + R) - 1;
        return paged_tiles(origin + r0 / a.group, origin + r1 / a.group, a.window, a.sinks, 4);
    };
    for (int i = tid; i < v.sequences; i += T) {
        PagedExtent e;
        const int bad = paged_extent(&v, i, &e);
        if (bad && !blockIdx.x) paged_report(a.status, bad);
        int steps = 0;  // the host keeps a launch's sum below 2^31
        if (e.count <= a.few)
            for (int rt = 0; rt * R < e.count * a.group; rt++) steps += max(1, tiles_of(e, rt).count);
        upto[i + 1] = steps * v.kvheads;
    }
    __syncthreads();
    if (warp == 0) {
        int before = 0;
        for (int i0 = 0; i0 < v.sequences; i0 += 32) {
            int x = i0 + lane < v.sequences ? upto[i0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (i0 + lane < v.sequences) upto[i0 + lane + 1] = before + x;
            before += __shfl_sync(0xffffffffu, x, 31);
        }
        if (lane == 0) upto[0] = 0;
    }
    __syncthreads();
    const int steps = upto[v.sequences];
    const int share = (int)(((unsigned)steps + gridDim.x - 1) / gridDim.x + W - 1) / W * W;
    const int begin = (int)min((long long)steps, (long long)share * blockIdx.x), end = (int)min((long long)steps, begin + (long long)share);
    const int64_t half = (int64_t)v.pages * v.kvheads * v.page;
    int bad = 0;
    for (int pos = begin; pos < end;) {
    // ---- the segment at pos
    if (tid == 0) {
        PdSegment z;
        z.s = 0;
        for (int top = v.sequences - 1; z.s < top;) {  // the last sequence that begins at or before pos
            const int mid = (z.s + top + 1) >> 1;
            if (upto[mid] <= pos) z.s = mid;
            else top = mid - 1;
        }
        paged_extent(&v, z.s, &z.e);
        const int in_seq = pos - upto[z.s], a_head = (upto[z.s + 1] - upto[z.s]) / v.kvheads;
        z.h = in_seq / a_head;
        int in_tile = in_seq - z.h * a_head, rt = 0;
        z.tiles = tiles_of(z.e, 0);
        while (in_tile >= max(1, z.tiles.count)) {
            in_tile -= max(1, z.tiles.count);
            z.tiles = tiles_of(z.e, ++rt);
        }
        z.r0 = rt * R;
        z.k0 = in_tile;
        z.from = pos - in_tile;
        z.to = z.from + max(1, z.tiles.count);
        seg = z;
    }
    __syncthreads();
    const int s = seg.s, h = seg.h;
    const PagedExtent e = seg.e;
    const PagedTiles tiles = seg.tiles;
    const int k0 = seg.k0, k1 = min(tiles.count, k0 + (end - pos)), r0 = seg.r0;
    const int rows = e.count * a.group;  // row r of the KV head: new row r / group, head r % group
    const int first = e.length - e.count + r0 / a.group;
    const int last = e.length - e.count + (min(rows, r0 + R) - 1) / a.group;

    // ---- its queries as fragments: warp w prepares rows w, w + W, ...
    for (int r = warp; r < R; r += W) {
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
    float o[DV][4], m[RW], mu[RW], l[RW], sc[RW];
#pragma unroll
    for (int j = 0; j < DV; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[j][c] = 0.f;
#pragma unroll
    for (int r = 0; r < RW; r++) m[r] = mu[r] = -INFINITY, l[r] = 0.f, sc[r] = qs[g + 8 * r];

    auto page_of = [&](int k) -> int {  // the page id of lane % 16's row of step k
        if (k >= k1) return -1;
        const int j = min(paged_tile(tiles, k) * 16 + (whole ? 0 : lane & 15), last);
        return v.table[(int64_t)s * v.table_stride + paged_div(&v, j)];
    };
    // Copies step k into its stage; returns which of its 16 places have a row. One copy group a
    // call, empty behind the last step.
    const uint32_t ring = smem_addr(pc_smem) + (uint32_t)warp * kPdStages * G::kStage;
    auto fetch = [&](int k, int id, int stage) -> unsigned {
        int64_t row = -1;  // lane % 16's
        if (k < k1) {
            const int j = paged_tile(tiles, k) * 16 + (lane & 15);
            if (j <= last) {
                row = paged_row(&v, id, j, paged_div(&v, j), h);
                // A page that no query of the sequence needs may be missing; one that holds a visible row may not.
                if (row < 0 && (a.window == 0 || j < a.sinks || (int64_t)j > (int64_t)first - a.window)) bad |= kPagedBadPage;
            }
            const uint32_t dst = ring + (uint32_t)stage * G::kStage;
            constexpr int LPR = G::kRow / 16, RPL = 32 / LPR;  // lanes a row, rows at a time
#pragma unroll
            for (int i = 0; i < 16 / RPL; i++) {
                const int rr = i * RPL + lane / LPR, piece = lane % LPR;
                const int64_t r = __shfl_sync(0xffffffffu, row, rr);
                const int64_t at = r < 0 ? 0 : r * G::kRow + piece * 16;
                const uint32_t to = dst + (uint32_t)(rr * G::kRow + pd_swizzle<G::kRow>(rr, piece) * 16);
                pd_copy16(to, static_cast<const char *>(v.keys) + at, r >= 0);
                pd_copy16(to + 16 * G::kRow, static_cast<const char *>(v.values) + at, r >= 0);
            }
            if constexpr (kBytes)
                pd_copy4(dst + 32 * G::kRow + lane * 4, v.scales + (row < 0 ? 0 : (lane >= 16 ? half : 0) + row), row >= 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
    };

    int k = k0 + warp;
    unsigned there = fetch(k, page_of(k), 0), there1 = fetch(k + W, page_of(k + W), 1);
    int id_next = page_of(k + 2 * W);
    for (int stage = 0; k < k1; k += W, stage = stage == kPdStages - 1 ? 0 : stage + 1) {
        const int ahead = stage == 0 ? kPdStages - 1 : stage - 1;  // the stage read in the step before
        const unsigned there2 = fetch(k + 2 * W, id_next, ahead);
        id_next = page_of(k + 3 * W);
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        __syncwarp();
        const unsigned char *st = pc_smem + (size_t)warp * kPdStages * G::kStage + (size_t)stage * G::kStage;
        // Scores of 16 places: S[gr] columns 2t, 2t + 1 are places base + 8 gr + 2t, + 1.
        float sf[2][4];
#pragma unroll
        for (int gr = 0; gr < 2; gr++)
#pragma unroll
            for (int c = 0; c < 4; c++) sf[gr][c] = 0.f;
        uint4 kr[2];
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            constexpr int KPP = KS / KP;  // k-steps a 16-byte piece of a key feeds
            if (ks % KPP == 0)
#pragma unroll
                for (int gr = 0; gr < 2; gr++) {
                    const int key = gr * 8 + g;
                    kr[gr] = *reinterpret_cast<const uint4 *>(st + key * G::kRow + pd_swizzle<G::kRow>(key, (ks / KPP) * 4 + t) * 16);
                }
            uint32_t b0[2], b1[2];
#pragma unroll
            for (int gr = 0; gr < 2; gr++) {
                if constexpr (kBytes) {
                    const uint32_t w = word(kr[gr], ks % 4) ^ 0x80808080u;
                    b0[gr] = codes_f16(w, 0x4140);
                    b1[gr] = codes_f16(w, 0x4342);
                } else {
                    b0[gr] = word(kr[gr], (ks % 2) * 2);
                    b1[gr] = word(kr[gr], (ks % 2) * 2 + 1);
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
                const float *sc4 = reinterpret_cast<const float *>(st + 32 * G::kRow) + (i >> 1) * 8 + 2 * t + (i & 1);
                ks4[i] = sc4[0];
                vs4[i] = sc4[16];
            }
        }

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
            l[r] *= m[r] == -INFINITY ? 0.f : ex2(m[r] - mr);
            m[r] = m_new;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                w[i] = ex2(x[i] - mr);
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
                const float f = mu_new == -INFINITY ? 0.f : ex2(mr - mu_new + kPdWeightTop);
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = x[i] == -INFINITY ? 0.f : w[i] * (vs4[i] * f);
            }
            keep[r] = mu[r] == -INFINITY ? 0.f : ex2(mu[r] - mu_new);
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
        uint4 vr[4];
#pragma unroll
        for (int c = 0; c < VW; c++) {
            if (c % 4 == 0)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int key = (i >> 1) * 8 + 2 * t + (i & 1), byte = g * (DV * ES) + c * 4;
                    const unsigned char *p = st + (16 + key) * G::kRow + pd_swizzle<G::kRow>(key, byte / 16) * 16;
                    if constexpr (VW == 2) {
                        const uint2 w = *reinterpret_cast<const uint2 *>(p + byte % 16);
                        vr[i] = make_uint4(w.x, w.y, 0, 0);
                    } else {
                        vr[i] = *reinterpret_cast<const uint4 *>(p);
                    }
                    // A weight of 0 times a non-finite value would spoil queries that do not see it.
                    if (!kBytes && !full)
                        vr[i] = make_uint4(finite_pair(vr[i].x), finite_pair(vr[i].y), finite_pair(vr[i].z), finite_pair(vr[i].w));
                }
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = word(vr[i], c % 4);
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
        there = there1;
        there1 = there2;
        __syncwarp();  // every lane has read the stage before it is copied into again
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // no copy is left in flight, and the rings' memory is free for the outputs

    // ---- the warps' states: lane (g, t) holds dims [2 t DV, (2 t + 2) DV) of row g (+ 8)
#pragma unroll
    for (int r = 0; r < RW; r++) {
        float sum = l[r];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (t == 0) wml[warp][g + 8 * r] = make_float2(m[r], sum);
        const float f = kBytes ? (mu[r] == -INFINITY ? 0.f : ex2(mu[r] - m[r] - kPdWeightTop)) : 1.f;
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int j = 0; j < DV; j += 4) {
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = f * (R == 8 ? o[j + i][c] + o[j + i][2 + c] : o[j + i][2 * r + c]);
                wo[warp][g + 8 * r][pd_piece<DIM>(g + 8 * r, ((2 * t + c) * DV + j) / 4)] = make_float4(y[0], y[1], y[2], y[3]);
            }
    }
    __syncthreads();
    {
    const volatile PdSegment &z = seg;
    const int from = z.from, to = z.to, r0 = z.r0, rows = z.e.count * a.group, start = z.e.start, h = z.h;
    auto store_out = [&](int r, int d4, float4 y, float sum) {
        const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);  // nothing seen: zeros
        *reinterpret_cast<float4 *>(a.out + (long long)(start + (r0 + r) / a.group) * a.out_stride +
                                    (h * a.group + (r0 + r) % a.group) * DIM + d4 * 4) =
            make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
    };
    const int live = min(R, rows - r0);
    const bool alone = from >= begin && to <= end;
    const int slot = 2 * blockIdx.x + (pos == begin ? 0 : 1);
    for (int i = tid; i < live * (DIM / 4); i += T) {
        const int r = i / (DIM / 4), d4 = i % (DIM / 4);
        float top = -INFINITY, sum = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; w++) top = fmaxf(top, wml[w][r].x);
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float2 ml = wml[w][r];
            const float f = pd_factor(ml, top);
            const float4 x = wo[w][r][pd_piece<DIM>(r, d4)];
            sum = fmaf(ml.y, f, sum);
            y.x = fmaf(x.x, f, y.x);
            y.y = fmaf(x.y, f, y.y);
            y.z = fmaf(x.z, f, y.z);
            y.w = fmaf(x.w, f, y.w);
        }
        if (alone) {
            store_out(r, d4, y, sum);
        } else {
            reinterpret_cast<float4 *>(a.part)[((int64_t)slot * R + r) * (DIM / 4) + d4] = y;
            if (d4 == 0) a.ml[slot * R + r] = make_float2(top, sum);
        }
    }
    pos += to <= end ? to - pos : end - pos;
    if (!alone) {
        // ---- the last CTA of the row tile to arrive adds all their partials, in order
        const int c0 = (int)(from / share), pieces = (int)((to - 1) / share) - c0 + 1;
        auto slot_of = [&](int i) { return 2 * (c0 + i) + (i == 0 && from != c0 * share ? 1 : 0); };
        __threadfence();
        __syncthreads();
        if (tid == 0) last_s = atomicAdd(&a.counters[c0], 1u) == (unsigned)(pieces - 1);
        __syncthreads();
        if (last_s) {
            __threadfence();
            if (tid == 0) a.counters[c0] = 0u;
            // Warp w sums pieces w, w + W, ... of every row; then the warps are added as above.
            constexpr int L = DIM / 4, PR = 32 / L;  // lanes a row, rows at a time
            for (int rb = 0; rb < live; rb += PR) {
                const int r = rb + lane / L, d4 = lane % L;
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                float top = -INFINITY, sum = 0.f;
                if (r < live)
                    for (int i0 = warp; i0 < pieces; i0 += 8 * W) {
                        float2 ml[8];
                        float4 x[8];
#pragma unroll
                        for (int u = 0; u < 8; u++) {
                            const int i = i0 + u * W, sl = slot_of(min(i, pieces - 1));
                            ml[u] = i < pieces ? __ldcg(&a.ml[sl * R + r]) : make_float2(-INFINITY, 0.f);
                            x[u] = __ldcg(reinterpret_cast<const float4 *>(a.part) + ((int64_t)sl * R + r) * (DIM / 4) + d4);
                        }
                        float now = top;
#pragma unroll
                        for (int u = 0; u < 8; u++) now = fmaxf(now, ml[u].x);
                        const float keep = pd_factor(make_float2(top, sum), now);
                        y = make_float4(y.x * keep, y.y * keep, y.z * keep, y.w * keep);
                        sum *= keep;
                        top = now;
#pragma unroll
                        for (int u = 0; u < 8; u++)
                            if (i0 + u * W < pieces) {
                                const float f = pd_factor(ml[u], now);
                                sum = fmaf(ml[u].y, f, sum);
                                y.x = fmaf(x[u].x, f, y.x);
                                y.y = fmaf(x[u].y, f, y.y);
                                y.z = fmaf(x[u].z, f, y.z);
                                y.w = fmaf(x[u].w, f, y.w);
                            }
                    }
                if (r < live) {
                    wo[warp][r][pd_piece<DIM>(r, d4)] = y;
                    if (d4 == 0) wml[warp][r] = make_float2(top, sum);
                }
            }
            __syncthreads();
            for (int i = tid; i < live * (DIM / 4); i += T) {
                const int r = i / (DIM / 4), d4 = i % (DIM / 4);
                float top = -INFINITY, sum = 0.f;
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < W; w++) top = fmaxf(top, wml[w][r].x);
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const float2 ml = wml[w][r];
                    const float f = pd_factor(ml, top);
                    const float4 x = wo[w][r][pd_piece<DIM>(r, d4)];
                    sum = fmaf(ml.y, f, sum);
                    y.x = fmaf(x.x, f, y.x);
                    y.y = fmaf(x.y, f, y.y);
                    y.z = fmaf(x.z, f, y.z);
                    y.w = fmaf(x.w, f, y.w);
                }
                store_out(r, d4, y, sum);
            }
        }
    }
    }
    __syncthreads();  // the merge buffer, the fragments and the segment are free for the next
    }
    if (bad) paged_report(a.status, bad);
}

}  // namespace tcm
