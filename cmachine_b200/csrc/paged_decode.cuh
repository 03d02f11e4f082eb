// Attention of few query rows over a paged K/V cache: single tokens and short
// drafted runs, R = 8, 16 or 32 query rows of one KV head at a time.
//
// The work is a line of steps: 16 cached rows against one row tile, ordered by
// sequence, KV head, row tile and place. Every CTA of a grid that fills the GPU once
// counts the steps of all sequences (their lengths are on the device), takes an equal
// stretch of the line, and works through the one to few (sequence, KV head, row tile)
// segments in it; its warps take a segment's steps in turn, each with its own online
// softmax, and merge at the segment's end. A segment's start and end take as long as
// kPdSegmentCost steps, so each has that many empty steps before its own: without them a
// CTA that met seven short sequences took 20 us longer than the others. A segment that
// began or goes on in another CTA leaves a partial result, and the last of its CTAs to
// arrive adds the partials in order.
// Memory bound: a cached row is read once from HBM (row tiles of one KV head meet in L2).
// Every warp copies its own steps into its own ring of three stages (cp.async, 16 bytes a
// lane, rows found by address), two steps ahead, and waits for no other warp; the products
// are mma.sync m16n8k16 (a tile of 8 rows cannot fill a tcgen05 tile of 128). Loading
// straight into registers instead left the compiler spilling loads in flight, which made
// every one of them a wait: 64 sessions of up to 8192 byte rows took 66 us so.
//
// Measured (attention alone): 63 sessions of up to 8192 byte rows, 70 MB, 26 us; 16 of 20,000 to
// 32,768 BF16 rows, 443 MB, 83 us (84 % of copy bandwidth); one of 32,749 byte rows, 17 MB, 21 us.
// Of the first, the loop takes 12 us at about the memory's rate; the rest is the start (finding the
// stretch, the first rows and queries: 4 us), the merges (2 us) and the launch.
//
// Fragments. The order of the dims inside a k-step and of the output columns is
// free as long as both operands agree, so it follows the memory layout: lane
// (g = lane / 4, t = lane % 4) reads 16-byte pieces of key g's row for Q K^T, and
// dims [g DIM / 8, (g + 1) DIM / 8) of keys 2t, 2t + 1, 8 + 2t, 9 + 2t for P V, whose
// pairs of keys meet by byte permutes.
//
// Precision. FP32 queries and weights enter as sums of parts whose products with the stored
// rows are exact. Byte rows meet the queries as integers: a query scaled to 23 bits and its
// sign is three signed bytes, the products are exact in 32-bit integers, and codes need no
// conversion (as FP16 they took 84 of a step's 600 instructions); weights meet them in
// FP16, two parts of 22 bits together. BF16 rows take three BF16 parts (24 bits) both times.
// With R = 8 a tile of 16 rows is [first parts; second parts], so one MMA forms both.
// Floating-point sums in the tensor cores truncate: long ones are taken apart (kPdChain).
#pragma once
#include "paged.cuh"
#include "stream.cuh"
#include <cuda_fp16.h>
#include <type_traits>

namespace tcm {

// Empty steps a segment counts for. Measured with 16, 32 and 56: 64 ragged sessions of BF16 rows 34.6,
// 32.8 and 35.1 us, of byte rows 26.0, 25.6 and 27.1; 64 of 20 to 600 rows 11.9, 13.4 and 13.8.
constexpr int kPdSegmentCost = 32;
// Steps that a warp may sum inside the tensor cores. They truncate: about 2e-8 of a sum a step, 1e-7 where all values
// have one sign, so 3e-6 at most after these, what FP32 products summed in FP32 may err too. In a longer segment every
// step is summed from zero and added in FP32. Measured of doing so always: 16 BF16 sessions of 46 steps a warp 75.2 ->
// 78.2 us, 5 tokens of 4 heads over 900 to 4100 BF16 rows 105 -> 113, 64 sessions of up to 8192 byte rows 29.9 -> 30.8.
constexpr int kPdChain = 32;
constexpr int kPdSequences = 128;  // sequences a launch counts in shared memory (two CTAs an SM still fit)

struct PagedDecodeArgs {
    PagedView v;
    float *out;
    const float *q;
    long long out_stride, q_stride;
    int group, window, sinks;
    int head0, heads;     // the KV heads of this launch
    int few;              // sequences of at most this many new rows are this kernel's
    float scale2;         // log2(e) / sqrt(dim): base-2 scores
    float *part;          // [CTA][2][R][DIM]: the first and the last segment of a CTA's stretch
    float2 *ml;           // [CTA][2][R]: running maximum and sum
    unsigned *counters;   // [CTA], of the segment that begins there and goes on; zero between calls
    int *status;
    int beside;           // the launch right behind the chunk kernel of the same call, which has waited for what came
                          // before and shares no scratch with this one: no wait until the end
};

// Eight warps a CTA; two CTAs an SM where their rings fit.
constexpr int kPdWarps = 8, kPdThreads = kPdWarps * 32, kPdStages = 3;
template <int KIND, int DIM> struct PdGeo {
    static constexpr int kRow = DIM * (KIND == kPagedBytes ? 1 : 2);          // bytes a stored row
    static constexpr int kStage = 32 * kRow + (KIND == kPagedBytes ? 128 : 0);  // 16 K rows, 16 V rows, their scales
    static constexpr size_t kRing = (size_t)kPdWarps * kPdStages * kStage;
};
// With 32 rows a thread holds 128 sums: one CTA an SM.
template <int KIND, int DIM, int R> constexpr int kPdCtas = PdGeo<KIND, DIM>::kRow <= 128 && R <= 16 ? 2 : 1;
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
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
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
// Two weights as the parts of a pair of 16-bit operands: parts[0] + parts[1] (+ parts[2])
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

// floor(log2 |x|) of a normal number; -127 for 0 and subnormals, 0 for infinities and NaN.
__device__ __forceinline__ int exponent_of(float x) {
    const int e = (int)((__float_as_uint(x) >> 23) & 0xff);
    return e == 0xff ? 0 : e - 127;
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

constexpr float kPdSlack = 3.f;   // log2 of how far a row's weights may pass 1 before its reference moves
// log2 of how far the V scales of the rows at hand may lie apart while their weights share one: 2^-28 of a
// row's size is left as the weights' step. Real caches stay inside; beyond it every query row scales its weights
// for itself, at the cost of another pass over them (a chunk's tile) or some 40 instructions a step.
constexpr int kPagedSpread = 8;
constexpr int kPdWeightTop = 12;  // log2 of the largest byte row's weight at 1: 2^15 with the slack, inside FP16

// A CTA's present segment, kept by thread 0; read again after the loop, so that the loop
// keeps its registers.
struct PdSegment {
    PagedExtent e;
    PagedTiles tiles;
    int s, h, rt;
    int from;  // the row tile's first own step in the line
    int n;     // its own steps: one at least, so that queries that see nothing get their zeros
};

template <int KIND, int DIM, int R>
__global__ void __launch_bounds__(kPdThreads, (kPdCtas<KIND, DIM, R>)) paged_decode_kernel(const PagedDecodeArgs a) {
    constexpr bool kBytes = KIND == kPagedBytes;
    using G = PdGeo<KIND, DIM>;
    constexpr int W = kPdWarps, T = kPdThreads;
    constexpr int ES = kBytes ? 1 : 2;         // bytes an element
    constexpr int KS = DIM * ES / 32;          // k-steps of Q K^T: 8 bytes of a key a lane
    constexpr int DV = DIM / 8;                // dims of a key a lane holds for P V
    constexpr int VW = DV * ES / 4;            // the same in words
    constexpr int P = kPdParts<KIND>;          // parts of a weight; a query has three
    constexpr int M = R == 32 ? 2 : 1;         // tiles of 16 MMA rows
    constexpr int NA = R == 8 ? 2 : 3;         // of each, the A operands a query product takes
    constexpr int RL = R == 8 ? 1 : 2;         // query rows of a tile a lane holds scores of
    extern __shared__ __align__(1024) unsigned char pc_smem[];
    float4(*wo)[R][DIM / 4] = reinterpret_cast<float4(*)[R][DIM / 4]>(pc_smem);  // the warps' outputs
    __shared__ __align__(16) uint4 qf[M * NA][KS][32];  // Q's fragments
    __shared__ float qs[R];                             // scale2 times what the row was multiplied down by
    __shared__ float2 wml[W][R];
    // Of a warp's row whose weights have a scale of their own (`wide` below): its log2, and log2 of the largest
    // weight times V scale so far, times the running maximum's power.
    __shared__ float2 own_scale[kBytes ? W : 1][R];
    __shared__ __align__(16) int units[kPdSequences];  // each sequence's stretch of the line
    __shared__ int longest;
    __shared__ PagedExtent extents[kPdSequences];
    __shared__ int last_s;
    __shared__ PdSegment seg;
    const PagedView &v = a.v;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

    // ---- this CTA's stretch of the line of steps. Nothing is read before the dependency wait: whatever runs before
    // may have written the extents. (Reading them during an append saved 0.25 us.) Beside the chunk kernel, which
    // has waited itself before it lets this one start, every CTA waits at its end: this kernel must not be over
    // before its predecessor is.
    if (!a.beside) pdl_wait();
    auto tiles_of = [&](const PagedExtent &e, int rt) {
        const int origin = e.length - e.count, r0 = rt * R, r1 = min(e.count * a.group, r0 + R) - 1;
        return paged_tiles(origin + r0 / a.group, origin + r1 / a.group, a.window, a.sinks, 4);
    };
    static_assert(T >= kPdSequences && kPdSequences == 128, "a thread a sequence, four sequences a lane");
    if (tid == 0) longest = 0;
    __syncthreads();
    if (tid < kPdSequences) {
        PagedExtent e = {0, 0, 0};
        int steps = 0, most = 0;  // the host keeps a launch's sum below 2^31
        if (tid < v.sequences) {
            const int bad = paged_extent(&v, tid, &e);
            if (bad && !blockIdx.x) paged_report(a.status, bad);
            if (e.count <= a.few)
                for (int rt = 0; rt * R < e.count * a.group; rt++) {
                    const int n = max(1, tiles_of(e, rt).count);
                    steps += kPdSegmentCost + n;
                    most = max(most, n);
                }
        }
        extents[tid] = e;
        units[tid] = steps * a.heads;
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) atomicMax(&longest, most);
    }
    __syncthreads();
    // Every warp adds the stretches up, four sequences a lane.
    const int4 u4 = *reinterpret_cast<const int4 *>(&units[4 * lane]);
    int mine = u4.x + u4.y + u4.z + u4.w, upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    const int steps = __shfl_sync(0xffffffffu, upto, 31);
    // An equal share, in whole rounds of the warps. A share of s steps ends after s / W rounds of
    // about 1000 cycles, and a row tile of n steps then has n / s partials to add, 16 in about 800
    // cycles: the sum is least at s = sqrt(0.4 n).
    int share = max((int)(((unsigned)steps + gridDim.x - 1) / gridDim.x), (int)sqrtf(0.4f * (float)longest));
    share = (share + W - 1) / W * W;
    const int begin = (int)min((long long)steps, (long long)share * blockIdx.x), end = (int)min((long long)steps, begin + (long long)share);
    if (begin >= end) {
        if (a.beside) pdl_wait();
        return;
    }
    // The sequence, and by thread 0 the segment, that `begin` lies in.
    {
        const int holder = __ffs(__ballot_sync(0xffffffffu, upto > begin)) - 1;
        int s = 4 * holder, before = __shfl_sync(0xffffffffu, upto - mine, holder);
        if (tid == 0) {
            while (before + units[s] <= begin) before += units[s++];
            PdSegment z;
            z.s = s;
            z.e = extents[s];
            const int a_head = units[s] / a.heads;
            z.h = a.head0 + (begin - before) / a_head;
            z.rt = 0;
            z.tiles = tiles_of(z.e, 0);
            z.n = max(1, z.tiles.count);
            z.from = before + (z.h - a.head0) * a_head + kPdSegmentCost;
            while (z.from + z.n <= begin && (z.rt + 1) * R < z.e.count * a.group) {
                z.tiles = tiles_of(z.e, ++z.rt);
                z.from += z.n + kPdSegmentCost;
                z.n = max(1, z.tiles.count);
            }
            seg = z;
        }
    }
    __syncthreads();
    const int64_t half = (int64_t)v.pages * v.kvheads * v.page;
    int bad = 0;
    for (;;) {
        const int s = seg.s, h = seg.h;
        const PagedExtent e = seg.e;
        const PagedTiles tiles = seg.tiles;
        const int r0 = seg.rt * R, rows = e.count * a.group;  // row r of the KV head: new row r / group, head r % group
        const int first = e.length - e.count + r0 / a.group;
        const int last = e.length - e.count + (min(rows, r0 + R) - 1) / a.group;
        const int k0 = max(0, begin - seg.from), k1 = min(tiles.count, end - seg.from);
        if (seg.from < end && seg.from + seg.n > begin) {

            // ---- the copies of this warp's steps
            const bool whole = v.page % 16 == 0;  // a step lies inside one page, 16 rows of one stretch of memory
            auto page_of = [&](int k) -> int {    // the page id of step k, or (pages that end inside steps) of lane % 16's row
                if (k >= k1) return -1;
                const int j = min(paged_tile(tiles, k) * 16 + (whole ? 0 : lane & 15), last);
                return v.table[(int64_t)s * v.table_stride + paged_div(&v, j)];
            };
            // Copies step k into its stage; returns which of its 16 places have a row. One copy group a
            // call, empty behind the last step.
            const uint32_t ring = smem_addr(pc_smem) + (uint32_t)warp * kPdStages * G::kStage;
            auto fetch = [&](int k, int id, int stage) -> unsigned {
                constexpr int LPR = G::kRow / 16, RPL = 32 / LPR;  // lanes a row, rows at a time
                unsigned there = 0;
                if (k < k1) {
                    const int j0 = paged_tile(tiles, k) * 16;
                    const uint32_t dst = ring + (uint32_t)stage * G::kStage;
                    // A page that no query of the sequence needs may be missing; one that holds a visible row may not.
                    auto needed = [&](int j) { return a.window == 0 || j < a.sinks || (int64_t)j > (int64_t)first - a.window; };
                    if (whole) {
                        const int64_t row = paged_row(&v, id, j0, paged_div(&v, j0), h);
                        const int rows_there = row < 0 ? 0 : min(16, last - j0 + 1);
                        if (row < 0)
                            for (int j = j0; j < j0 + 16; j++)
                                if (j <= last && needed(j)) bad |= kPagedBadPage;
                        there = (1u << rows_there) - 1u;
                        const int64_t at = (row < 0 ? 0 : row) * G::kRow + lane * 16;
#pragma unroll
                        for (int i = 0; i < 16 / RPL; i++) {
                            const int rr = i * RPL + lane / LPR;
                            const uint32_t to = dst + (uint32_t)(rr * G::kRow + pd_swizzle<G::kRow>(rr, lane % LPR) * 16);
                            pd_copy16(to, static_cast<const char *>(v.keys) + at + i * 512, rr < rows_there);
                            pd_copy16(to + 16 * G::kRow, static_cast<const char *>(v.values) + at + i * 512, rr < rows_there);
                        }
                        if constexpr (kBytes)
                            pd_copy4(dst + 32 * G::kRow + lane * 4, v.scales + ((lane & 15) < rows_there ? (lane >= 16 ? half : 0) + row + (lane & 15) : 0),
                                     (lane & 15) < rows_there);
                    } else {
                        const int j = j0 + (lane & 15);
                        int64_t row = -1;  // lane % 16's
                        if (j <= last) {
                            row = paged_row(&v, id, j, paged_div(&v, j), h);
                            if (row < 0 && needed(j)) bad |= kPagedBadPage;
                        }
                        there = __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
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
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                return there;
            };
            // Page ids and queries are asked for together, before the first copy waits for an id. Warp w
            // prepares query rows w, w + W, ...
            int k = k0 + warp;
            const int id0 = page_of(k), id1 = page_of(k + W);
            int id_next = page_of(k + 2 * W);
            constexpr int E = DIM / 32;
            float qx[R / W][E];
#pragma unroll
            for (int i = 0; i < R / W; i++) {
                const int r = r0 + warp + i * W;
#pragma unroll
                for (int c = 0; c < E; c++) qx[i][c] = 0.f;
                if (r < rows) {
                    const float *src = a.q + (long long)(e.start + r / a.group) * a.q_stride + (h * a.group + r % a.group) * DIM;
                    if constexpr (E == 4) {
                        const float4 f = reinterpret_cast<const float4 *>(src)[lane];
                        qx[i][0] = f.x, qx[i][1] = f.y, qx[i][2] = f.z, qx[i][3] = f.w;
                    } else {
                        const float2 f = reinterpret_cast<const float2 *>(src)[lane];
                        qx[i][0] = f.x, qx[i][1] = f.y;
                    }
                }
            }
            unsigned there = 0, there1 = 0;
#pragma unroll 1  // one copy of the code: a cold instruction cache shows in short calls
            for (int i = 0; i < 2; i++) {
                there = there1;
                there1 = fetch(k + i * W, i ? id1 : id0, i);
            }

            // ---- the queries as fragments
#pragma unroll
            for (int i = 0; i < R / W; i++) {
                const int r = warp + i * W;
                float(&x)[E] = qx[i];
                // R = 8: part p is rows 8 (p % 2) + r of operand p / 2; else row r % 16 of operand 3 (r / 16) + p. BF16's
                // third part goes below the second: only first parts meet in the sums that truncate noticeably.
                auto place = [&](int p, int ks, int ft, int fh) {
                    const int tile = R == 8 ? p / 2 : r / 16 * 3 + p, row = R == 8 ? (p % 2 ^ (!kBytes && p > 1)) * 8 + r : r % 16;
                    return &reinterpret_cast<uint32_t *>(&qf[tile][ks][(row % 8) * 4 + ft])[2 * fh + row / 8];
                };
                const int d = lane * E;
                if constexpr (kBytes) {
                    // The row as integers up to 127 x 65536, each three signed bytes: 65536 a + 256 b + c, off by at
                    // most half of 2^-23 of the row's largest element.
                    constexpr float kMost = 127.f * 65536.f;
                    float m = 0.f;
                    bool finite = true;
#pragma unroll
                    for (int c = 0; c < E; c++) m = fmaxf(m, fabsf(x[c])), finite &= isfinite(x[c]);
                    finite = __all_sync(0xffffffffu, finite);
                    m = warp_max(m);
                    const bool any = finite && m > 0.f;
                    const float lift = m < 0x1p-60f ? 0x1p100f : 1.f;  // exact, and up stays finite
                    const float up = any ? kMost / (m * lift) : 0.f;
                    // The integers enter the scores times 2^-24, so that neither they times a row's scale nor this
                    // leaves FP32's range before the two meet.
                    if (lane == 0) qs[r] = finite ? (a.scale2 * m) * (0x1p24f / kMost) : __uint_as_float(0x7fc00000u);
                    uint32_t w[3] = {0, 0, 0};
#pragma unroll
                    for (int c = 0; c < E; c++) {
                        int n = any ? __float2int_rn(x[c] * lift * up) : 0;
                        const int lo = (int)(signed char)n;
                        n = (n - lo) >> 8;
                        const int mid = (int)(signed char)n;
                        n = (n - mid) >> 8;
                        w[0] |= (uint32_t)(n & 0xff) << (8 * c);
                        w[1] |= (uint32_t)(mid & 0xff) << (8 * c);
                        w[2] |= (uint32_t)(lo & 0xff) << (8 * c);
                    }
                    // Dims 4n .. 4n + 3 of a 16-dim piece: k-step n / 2 of the piece's two, half n % 2.
                    const int ks = (d / 64) * 2 + (d % 16) / 8, ft = (d % 64) / 16, fh = (d % 8) / 4;
#pragma unroll
                    for (int p = 0; p < 3; p++) {
                        if constexpr (E == 4) *place(p, ks, ft, fh) = w[p];
                        else reinterpret_cast<uint16_t *>(place(p, ks, ft, fh))[(d % 4) / 2] = (uint16_t)w[p];
                    }
                    if (R == 8) *place(3, ks, ft, fh) = 0u;
                } else {
                    if (lane == 0) qs[r] = a.scale2;
#pragma unroll
                    for (int c = 0; c < E; c += 2) {
                        uint32_t w[3];
                        split_pair<kPagedBf16>(x[c], x[c + 1], w);
                        const int dd = d + c, ks = (dd / 32) * 2 + (dd % 8) / 4, ft = (dd % 32) / 8, fh = (dd % 4) / 2;
#pragma unroll
                        for (int p = 0; p < 3; p++) *place(p, ks, ft, fh) = w[p];
                        if (R == 8) *place(3, ks, ft, fh) = 0u;
                    }
                }
            }
            __syncthreads();

            // ---- the loop over this warp's 16-row steps
            float o[M][DV][4], m[M][RL], l[M][RL], sc[M][RL];
#pragma unroll
            for (int mt = 0; mt < M; mt++) {
#pragma unroll
                for (int j = 0; j < DV; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[mt][j][c] = 0.f;
#pragma unroll
                for (int r = 0; r < RL; r++) m[mt][r] = -INFINITY, l[mt][r] = 0.f, sc[mt][r] = qs[16 * mt + 8 * r + g];
            }
            // Byte rows: weights carry the rows' scales, times 2^12 over a power of two above the largest
            // scale so far (v_top, exponent v_exp).
            // Rows share it until scales far apart meet (v_low is the smallest so far): then a row that it does
            // not see, or that hardly counts for it, must not push a query's weights below FP16.
            float v_top = 0.f, v_factor = 0.f, v_low = INFINITY;
            int v_exp = 0;
            bool wide = false;
            constexpr float kNear = 1.f / (1 << kPagedSpread);
            const bool long_sum = k1 - k0 > kPdChain * W;
            const int see_all = a.window == 0 || a.window > last ? 0 : last - a.window + 1;  // every query sees from here to `first`
            for (int stage = 0; k < k1; k += W, stage = stage == kPdStages - 1 ? 0 : stage + 1) {
                const int ahead = stage == 0 ? kPdStages - 1 : stage - 1;  // the stage read in the step before
                const unsigned there2 = fetch(k + 2 * W, id_next, ahead);
                id_next = page_of(k + 3 * W);
                asm volatile("cp.async.wait_group 2;" ::: "memory");
                __syncwarp();
                const unsigned char *st = pc_smem + ((size_t)warp * kPdStages + stage) * G::kStage;
                const int base = paged_tile(tiles, k) * 16;
                const bool full = there == 0xffffu && base + 15 <= first && (base >= see_all || base + 15 < a.sinks);

                // ---- scores of 16 places: x[..][i] is place base + 8 (i / 2) + 2t + i % 2
                float x[M][RL][4];
                {
                    int ci[kBytes ? M * NA : 1][2][4];
                    float cf[kBytes ? 1 : M][2][4];
#pragma unroll
                    for (int gr = 0; gr < 2; gr++)
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            if constexpr (kBytes)
#pragma unroll
                                for (int n = 0; n < M * NA; n++) ci[n][gr][c] = 0;
                            else
#pragma unroll
                                for (int mt = 0; mt < M; mt++) cf[mt][gr][c] = 0.f;
                        }
                    uint4 kr[2];
                    // BF16 rows meet the queries' smaller parts first: the tensor cores truncate a sum as large as the
                    // first parts' at every step that adds to it.
                    constexpr int kPasses = kBytes || R == 8 ? 1 : 2;
#pragma unroll
                    for (int pass = 0; pass < kPasses; pass++)
#pragma unroll
                        for (int ks = 0; ks < KS; ks++) {
                            if (ks % 2 == 0)
#pragma unroll
                                for (int gr = 0; gr < 2; gr++) {
                                    const int key = gr * 8 + g;
                                    kr[gr] = *reinterpret_cast<const uint4 *>(st + key * G::kRow + pd_swizzle<G::kRow>(key, (ks / 2) * 4 + t) * 16);
                                }
#pragma unroll
                            for (int n = M * NA - 1; n >= 0; n--) {
                                if (kPasses == 2 && (n % NA == 0) != (pass == 1)) continue;
                                const uint4 f = qf[n][ks][lane];
#pragma unroll
                                for (int gr = 0; gr < 2; gr++) {
                                    const uint32_t b0 = ks % 2 ? kr[gr].z : kr[gr].x, b1 = ks % 2 ? kr[gr].w : kr[gr].y;
                                    if constexpr (kBytes) mma_s8(ci[n][gr], f, b0, b1);
                                    else mma_bf16(cf[n / NA][gr], f.x, f.y, f.z, f.w, b0, b1);
                                }
                            }
                        }
#pragma unroll
                    for (int mt = 0; mt < M; mt++)
#pragma unroll
                        for (int r = 0; r < RL; r++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int gr = i >> 1, c = i & 1;
                                if constexpr (kBytes) {
                                    // Each sum is below 2^21, the lower two together below 2^30.
                                    const int top = R == 8 ? ci[0][gr][c] : ci[mt * NA][gr][2 * r + c];
                                    const int mid = R == 8 ? ci[0][gr][2 + c] : ci[mt * NA + 1][gr][2 * r + c];
                                    const int low = R == 8 ? ci[1][gr][c] : ci[mt * NA + NA - 1][gr][2 * r + c];
                                    x[mt][r][i] = fmaf((float)top, 0x1p-8f, (float)(mid * 256 + low) * 0x1p-24f);
                                } else {
                                    x[mt][r][i] = R == 8 ? cf[0][gr][c] + cf[0][gr][2 + c] : cf[mt][gr][2 * r + c];
                                }
                            }
                }
                float vs[4];
                if constexpr (kBytes) {
                    const float *ks4 = reinterpret_cast<const float *>(st + 32 * G::kRow);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int at = (i >> 1) * 8 + 2 * t + (i & 1);
                        vs[i] = ks4[16 + at];
#pragma unroll
                        for (int mt = 0; mt < M; mt++)
#pragma unroll
                            for (int r = 0; r < RL; r++) x[mt][r][i] *= ks4[at];
                    }
                }
                bool moves = false;
                float top[M][RL];
#pragma unroll
                for (int mt = 0; mt < M; mt++)
#pragma unroll
                    for (int r = 0; r < RL; r++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) x[mt][r][i] *= sc[mt][r];
                        if (!full) {
                            const int at = e.length - e.count + min(r0 + 16 * mt + 8 * r + g, rows - 1) / a.group;
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int c = (i >> 1) * 8 + 2 * t + (i & 1);
                                if (!((there >> c) & 1) || !paged_sees(at, base + c, a.window, a.sinks)) x[mt][r][i] = -INFINITY;
                            }
                        }
                        top[mt][r] = quad_max(fmaxf(fmaxf(x[mt][r][0], x[mt][r][1]), fmaxf(x[mt][r][2], x[mt][r][3])));
                        moves |= top[mt][r] > m[mt][r] + kPdSlack;
                    }
                float v_most = 0.f;
                if constexpr (kBytes) {
                    v_most = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
                    float least = fminf(fminf(vs[0], vs[1]), fminf(vs[2], vs[3]));
                    if (!full) {  // a row that no query of the tile sees may have any scale
                        v_most = 0.f, least = INFINITY;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int c = (i >> 1) * 8 + 2 * t + (i & 1);
                            const bool seen = a.window == 0 || base + c < a.sinks || (int64_t)base + c > (int64_t)first - a.window;
                            v_most = fmaxf(v_most, seen && vs[i] < INFINITY ? vs[i] : 0.f);
                            least = fminf(least, seen && vs[i] > 0.f ? vs[i] : INFINITY);
                        }
                    }
                    v_low = fminf(v_low, least);
                    v_most = quad_max(v_most);
                    moves |= !wide && (v_most > v_top || v_low < kNear * v_top);
                }
                // References move rarely: a row's when its maximum has passed it by 2^3 (weights have that
                // much room), the scale's when a larger one turns up.
                if (__any_sync(0xffffffffu, moves)) {
                    float shrink = 1.f;
                    if constexpr (kBytes) {
                        const int was = v_exp;
                        const bool first_rows = v_top == 0.f;
                        if (!wide && v_most > v_top) {  // the same in every lane
                            v_exp = max(-100, exponent_of(v_most) + 1);
                            shrink = first_rows ? 0.f : power_of_two(was - v_exp);
                            v_top = power_of_two(v_exp);
                            v_factor = power_of_two(kPdWeightTop - v_exp);
                        }
                        if (!wide && __any_sync(0xffffffffu, v_low < kNear * v_top)) {
                            wide = true;
                            v_factor = 1.f;
                            if (t == 0)
#pragma unroll
                                for (int mt = 0; mt < M; mt++)
#pragma unroll
                                    for (int r = 0; r < RL; r++)  // the steps before this one were bounded by the scale before it
                                        own_scale[warp][16 * mt + 8 * r + g] =
                                            make_float2((float)v_exp, first_rows ? -INFINITY : m[mt][r] + ((float)was + kPdSlack));
                            __syncwarp();
                        }
                    }
#pragma unroll
                    for (int mt = 0; mt < M; mt++) {
                        float keep[RL];
#pragma unroll
                        for (int r = 0; r < RL; r++) {
                            keep[r] = shrink;
                            if (top[mt][r] > m[mt][r] + kPdSlack) {
                                const float c = m[mt][r] == -INFINITY ? 0.f : ex2(m[mt][r] - top[mt][r]);
                                m[mt][r] = top[mt][r];
                                l[mt][r] *= c;
                                keep[r] *= c;
                            }
                        }
#pragma unroll
                        for (int j = 0; j < DV; j++) {
                            o[mt][j][0] *= keep[0];
                            o[mt][j][1] *= keep[0];
                            o[mt][j][2] *= keep[RL - 1];
                            o[mt][j][3] *= keep[RL - 1];
                        }
                    }
                }
                if constexpr (kBytes) {
#pragma unroll
                    for (int i = 0; i < 4; i++) vs[i] *= v_factor;
                }
                uint32_t pa[M][RL][2][P];  // weights as fragments' parts: [tile][row][group of 8 places][part]
#pragma unroll
                for (int mt = 0; mt < M; mt++)
#pragma unroll
                    for (int r = 0; r < RL; r++) {
                        float w[4];
                        const float mr = m[mt][r] == -INFINITY ? 0.f : m[mt][r];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            w[i] = ex2(x[mt][r][i] - mr);
                            l[mt][r] += w[i];
                            if constexpr (kBytes) w[i] *= vs[i];
                            if (kBytes && !full && x[mt][r][i] == -INFINITY) w[i] = 0.f;
                        }
                        if (kBytes && wide) {
                            const int row = 16 * mt + 8 * r + g;
                            const float2 own = own_scale[warp][row];
                            const float most = quad_max(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])));
                            const float bound = most > 0.f ? fmaxf(own.y, m[mt][r] + (float)(exponent_of(most) + 1)) : own.y;
                            const int was = (int)own.x;  // falls by at most 2^120 at a time, which FP32 can scale by
                            const int now = bound == -INFINITY ? was : max(max(-100, was - 120), (int)ceilf(fminf(bound - m[mt][r], 127.f)));
                            if (t == 0) own_scale[warp][row] = make_float2((float)now, bound);
                            if (now != was) {
                                const float keep = power_of_two(was - now);
#pragma unroll
                                for (int j = 0; j < DV; j++)
#pragma unroll
                                    for (int c = 0; c < 4; c++)
                                        if (RL == 1 || c / 2 == r) o[mt][j][c] *= keep;
                            }
                            const float up = power_of_two(kPdWeightTop - now);
#pragma unroll
                            for (int i = 0; i < 4; i++) w[i] *= up;
                        }
                        split_pair<KIND>(w[0], w[1], pa[mt][r][0]);
                        split_pair<KIND>(w[2], w[3], pa[mt][r][1]);
                    }
                auto pv = [&](int j, uint32_t b0, uint32_t b1, auto apart) {
#pragma unroll
                    for (int mt = 0; mt < M; mt++) {
                        float sum[4] = {0.f, 0.f, 0.f, 0.f};
                        float(&acc)[4] = decltype(apart)::value ? sum : o[mt][j];
                        const auto &w = pa[mt];
                        if constexpr (kBytes) {
                            if constexpr (R == 8) mma_f16(acc, w[0][0][0], w[0][0][1], w[0][1][0], w[0][1][1], b0, b1);
                            else
#pragma unroll
                                for (int p = 1; p >= 0; p--) mma_f16(acc, w[0][0][p], w[RL - 1][0][p], w[0][1][p], w[RL - 1][1][p], b0, b1);
                        } else if constexpr (R == 8) {
                            mma_bf16(acc, 0u, w[0][0][P - 1], 0u, w[0][1][P - 1], b0, b1);
                            mma_bf16(acc, w[0][0][0], w[0][0][1], w[0][1][0], w[0][1][1], b0, b1);
                        } else {
#pragma unroll
                            for (int p = P - 1; p >= 0; p--) mma_bf16(acc, w[0][0][p], w[RL - 1][0][p], w[0][1][p], w[RL - 1][1][p], b0, b1);
                        }
                        if constexpr (decltype(apart)::value)
#pragma unroll
                            for (int i = 0; i < 4; i++) o[mt][j][i] += sum[i];
                    }
                };
                auto add_values = [&](auto apart) {
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
                        uint32_t y[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) y[i] = word(vr[i], c % 4);
                        if constexpr (kBytes) {
                            const uint32_t lo0 = __byte_perm(y[0], y[1], 0x5140) ^ 0x80808080u, hi0 = __byte_perm(y[0], y[1], 0x7362) ^ 0x80808080u;
                            const uint32_t lo1 = __byte_perm(y[2], y[3], 0x5140) ^ 0x80808080u, hi1 = __byte_perm(y[2], y[3], 0x7362) ^ 0x80808080u;
                            pv(4 * c, codes_f16(lo0, 0x4140), codes_f16(lo1, 0x4140), apart);
                            pv(4 * c + 1, codes_f16(lo0, 0x4342), codes_f16(lo1, 0x4342), apart);
                            pv(4 * c + 2, codes_f16(hi0, 0x4140), codes_f16(hi1, 0x4140), apart);
                            pv(4 * c + 3, codes_f16(hi0, 0x4342), codes_f16(hi1, 0x4342), apart);
                        } else {
                            pv(2 * c, __byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410), apart);
                            pv(2 * c + 1, __byte_perm(y[0], y[1], 0x7632), __byte_perm(y[2], y[3], 0x7632), apart);
                        }
                    }
                };
                if (long_sum) add_values(std::true_type{});
                else add_values(std::false_type{});
                there = there1;
                there1 = there2;
                __syncwarp();  // every lane has read the stage before it is copied into again
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncthreads();  // no copy is left in flight, and the rings' memory is free for the outputs

            // ---- the warps' states: lane (g, t) holds dims [2 t DV, (2 t + 2) DV) of row g (+ 8)
#pragma unroll
            for (int mt = 0; mt < M; mt++)
#pragma unroll
                for (int r = 0; r < RL; r++) {
                    float sum = l[mt][r];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    const int row = 16 * mt + 8 * r + g;
                    if (t == 0) wml[warp][row] = make_float2(m[mt][r], sum);
                    const float unscale = kBytes ? power_of_two((wide ? (int)own_scale[warp][row].x : v_exp) - kPdWeightTop) : 1.f;
#pragma unroll
                    for (int c = 0; c < 2; c++)
#pragma unroll
                        for (int j = 0; j < DV; j += 4) {
                            float y[4];
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                y[i] = unscale * (R == 8 ? o[mt][j + i][c] + o[mt][j + i][2 + c] : o[mt][j + i][2 * r + c]);
                            wo[warp][row][pd_piece<DIM>(row, ((2 * t + c) * DV + j) / 4)] = make_float4(y[0], y[1], y[2], y[3]);
                        }
                }
            __syncthreads();
            {
                const volatile PdSegment &z = seg;
                const int from = z.from, n = z.n, r0 = z.rt * R, rows = z.e.count * a.group, start = z.e.start, h = z.h;
                auto store_out = [&](int r, int d4, float4 y, float sum) {
                    const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);  // nothing seen: zeros
                    *reinterpret_cast<float4 *>(a.out + (long long)(start + (r0 + r) / a.group) * a.out_stride +
                                                (h * a.group + (r0 + r) % a.group) * DIM + d4 * 4) =
                        make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
                };
                const int live = min(R, rows - r0);
                const bool alone = from >= begin && from + n <= end;
                const int slot = 2 * blockIdx.x + (from >= begin ? 1 : 0);
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
                if (!alone) {
                    // ---- the last CTA of the row tile to arrive adds all their partials, in order
                    const int c0 = from / share, pieces = (from + n - 1) / share - c0 + 1;
                    auto slot_of = [&](int i) { return 2 * (c0 + i) + (i == 0 ? 1 : 0); };
                    __threadfence();
                    __syncthreads();
                    if (tid == 0) last_s = atomicAdd(&a.counters[c0], 1u) == (unsigned)(pieces - 1);
                    __syncthreads();
                    if (last_s) {
                        __threadfence();
                        if (tid == 0) a.counters[c0] = 0u;
                        if (pieces <= 8) {  // a thread's share of the row from each at once
                            for (int i = tid; i < live * (DIM / 4); i += T) {
                                const int r = i / (DIM / 4), d4 = i % (DIM / 4);
                                float2 ml[8];
                                float4 x[8], y = make_float4(0.f, 0.f, 0.f, 0.f);
                                float top = -INFINITY, sum = 0.f;
#pragma unroll
                                for (int w = 0; w < 8; w++) {
                                    const int64_t at = (int64_t)slot_of(min(w, pieces - 1)) * R + r;
                                    ml[w] = __ldcg(&a.ml[at]);
                                    x[w] = __ldcg(reinterpret_cast<const float4 *>(a.part) + at * (DIM / 4) + d4);
                                }
#pragma unroll
                                for (int w = 0; w < 8; w++) top = fmaxf(top, ml[w].x);
#pragma unroll
                                for (int w = 0; w < 8; w++)
                                    if (w < pieces) {
                                        const float f = pd_factor(ml[w], top);
                                        sum = fmaf(ml[w].y, f, sum);
                                        y = make_float4(fmaf(x[w].x, f, y.x), fmaf(x[w].y, f, y.y), fmaf(x[w].z, f, y.z), fmaf(x[w].w, f, y.w));
                                    }
                                store_out(r, d4, y, sum);
                            }
                        } else {
                            // Warp w sums pieces w, w + W, ..., eight rows' loads in flight; then the warps are added
                            // as above.
                            constexpr int L = DIM / 4, PR = 32 / L, B = 8;  // lanes a row, rows a load, loads in flight
                            for (int rb = 0; rb < live; rb += PR * B) {
                                const int d4 = lane % L;
                                float4 y[B];
                                float2 state[B];
#pragma unroll
                                for (int u = 0; u < B; u++) y[u] = make_float4(0.f, 0.f, 0.f, 0.f), state[u] = make_float2(-INFINITY, 0.f);
                                for (int i = warp; i < pieces; i += W) {
                                    const int64_t at = (int64_t)slot_of(i) * R;
                                    float2 ml[B];
                                    float4 x[B];
#pragma unroll
                                    for (int u = 0; u < B; u++) {
                                        const int r = min(rb + u * PR + lane / L, live - 1);
                                        ml[u] = __ldcg(&a.ml[at + r]);
                                        x[u] = __ldcg(reinterpret_cast<const float4 *>(a.part) + (at + r) * L + d4);
                                    }
#pragma unroll
                                    for (int u = 0; u < B; u++) {
                                        const float now = fmaxf(state[u].x, ml[u].x), keep = pd_factor(state[u], now), f = pd_factor(ml[u], now);
                                        state[u] = make_float2(now, fmaf(ml[u].y, f, state[u].y * keep));
                                        y[u] = make_float4(fmaf(x[u].x, f, y[u].x * keep), fmaf(x[u].y, f, y[u].y * keep),
                                                           fmaf(x[u].z, f, y[u].z * keep), fmaf(x[u].w, f, y[u].w * keep));
                                    }
                                }
#pragma unroll
                                for (int u = 0; u < B; u++) {
                                    const int r = rb + u * PR + lane / L;
                                    if (r < live) {
                                        wo[warp][r][pd_piece<DIM>(r, d4)] = y[u];
                                        if (d4 == 0) wml[warp][r] = state[u];
                                    }
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
            }
        }
        __syncthreads();  // the merge buffer, the fragments and the segment are free for the next
        if (tid == 0) {
            PdSegment z = seg;
            z.from += z.n;
            if (++z.rt * R >= z.e.count * a.group) {
                z.rt = 0;
                if (++z.h == a.head0 + a.heads) {
                    z.h = a.head0;
                    do z.s++;
                    while (z.s < v.sequences && !units[z.s]);
                    if (z.s < v.sequences) z.e = extents[z.s];
                }
            }
            z.from += kPdSegmentCost;
            z.tiles = tiles_of(z.e, z.rt);
            z.n = max(1, z.tiles.count);
            if (z.s >= v.sequences) z.from = end;
            seg = z;
        }
        __syncthreads();
        if (seg.from >= end) break;
    }
    if (a.beside) pdl_wait();
    if (bad) paged_report(a.status, bad);
}

}  // namespace tcm
