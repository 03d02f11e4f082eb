// Attention of chunks of new rows over a paged K/V cache on the tcgen05 tensor
// cores: prompts and long drafted runs, 256 query rows of one KV head a CTA.
//
// Row r of the KV head's chunk is new row r / group, query head r % group, so grouped
// heads fill the tile whatever the group. Per tile of 128 cached rows
//   S = Q K^T (tcgen05.mma, M = 128 twice, N = 128), P = exp2(S - m) (registers),
//   O_t = P V (P from tensor memory), O = O c + O_t (registers).
//
// Four warpgroups: two for the softmax, one per 128 query rows (one row a thread, with
// its output row in registers), one that turns stored rows into FP16 operand tiles in
// shared memory (pages end anywhere, so rows are fetched by address), and one of which
// a single thread issues the MMAs. While one warpgroup computes weights
// the tensor cores run the other's products. A ring of three operand tiles holds
// K(t + 1), V(t) and the next.
//
// Measured: 4096 new rows over 32,768 byte rows (12 query heads, 2 KV heads) in 1.53 ms, 504 TFLOP/s
// of result and 1.01 PFLOP/s of products; 512 over 4,609 in 48 us. A tile takes 7,400 cycles, of
// which the MMAs are 4,100: the chain of one half (its maximum 700, its weights 3,700, the rest of
// P V 900, Q K^T 1,450) bounds it. The weights' 128 exponentials alone are 1,024 cycles of the
// special-function unit, and their broadcast reads of the row scales from shared memory wait behind
// the MMAs' operands. Tried and slower: two threads a row (1.78 ms), scales through L1 (2.03 ms), the
// exponentials of 16 columns beside the splitting of the 16 before (1.67 ms).
//
// Precision. Results are FP32, so a 16-bit rounding of Q or P would be visible:
// both enter as two FP16 parts (22 bits) after scaling into FP16's range by powers
// of two, against operands that are exact: a byte row is its codes, with the row's
// scale applied to the column of S and to the weight; a BF16 row is the row divided
// by the power of two below its largest element (2^-39 of that element at worst).
// That doubles the products: half of the FP16 rate is the ceiling. The tensor cores
// truncate when they add (measured: 4e-8 of the sum a step, 9e-6 after 8192
// products), so every tile's P V starts from zero and is added in FP32 registers,
// smaller parts first, instead of one long accumulation in tensor memory.
#pragma once
#include "paged_decode.cuh"
#include "stream.cuh"
#include "tc_gemm.cuh"

namespace tcm {

constexpr int kPcRows = 256, kPcTile = 128;   // query rows a CTA, cached rows a tile
constexpr int kPcThreads = 512;
constexpr int kPcSlots = 3;
constexpr int kPcSplitsMax = 32;
// Registers: four warpgroups are launched with 128 a thread; what the converters and the
// issuing warp's group give away lets the softmax threads hold an output row. Each of the
// SM's four register files holds one warp of each group: 200 + 200 + 64 + 48 = 4 x 128.
constexpr int kPcRegs = 128, kPcSoftmaxRegs = 200, kPcConvertRegs = 64, kPcIssueRegs = 48;
static_assert(2 * kPcSoftmaxRegs + kPcConvertRegs + kPcIssueRegs <= 4 * kPcRegs, "register split");
constexpr float kPcSlack = 3.f;   // log2 of how far a row's weights may pass 1 before its reference moves
constexpr int kPcWeightTop = 12;  // log2 of the largest weight times V scale at 1: 2^15 with the slack, inside FP16
constexpr unsigned kPagedWaitRanOut = 8u;     // status bit

struct PagedChunkArgs {
    PagedView v;
    float *out;
    const float *q;
    long long out_stride, q_stride;
    int group, window, sinks, few;
    int sms, slots;          // CTAs that have a place for a part
    float scale2;
    float *part;             // [CTA][256][DIM], of items that are split
    float2 *ml;              // [CTA][256]
    int4 *plan;              // [0] the row tiles and their splits, then each tile's first row, query rows, number and splits
    int *status;
    unsigned *err;           // where waits that run out are recorded (status, or scratch)
    int starve;              // self-check: 1 or 2 keeps the first K or V tile from ever being ready
};

template <int DIM> struct PcGeo {
    static constexpr uint32_t kHalf = 128 * 128;                  // bytes: 128 rows of 64 FP16 in the 128-byte swizzle
    static constexpr int kHalves = DIM / 64;
    static constexpr uint32_t kOperand = kHalves * kHalf;         // one 128-row operand tile
    static constexpr uint32_t kQ = 4 * kOperand;                  // [row half][part]
    static constexpr uint32_t kScales = kQ + kPcSlots * kOperand; // float [2 K|V][2][128]
    static constexpr uint32_t kMisc = kScales + 2 * 2 * 128 * 4;
    static constexpr size_t kSmem = kMisc + 384;
    static constexpr uint32_t kIdescS = (1u << 4) | ((128u >> 3) << 17) | (8u << 24);                     // FP16, K-major
    static constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | ((uint32_t)(DIM >> 3) << 17) | (8u << 24);  // B MN-major
};
// A CTA's work, in shared memory: what the roles need of it they read there, and their loops keep their registers.
struct PcWork {
    int s, h, start, rows, origin;  // sequence, KV head, first row in the callers' buffers, query rows, place of the first
    int r0, live, splits;           // the row tile's first query row, how many it has, into how many parts it is split
    int first, last;                // the places of its first and last
    PagedTiles tiles;               // the tiles it sees, of which
    int k0, n;                      // this CTA takes n from k0
    __device__ __forceinline__ int base(int t) const volatile {
        const int k = k0 + t;
        return (k < tiles.a ? k : tiles.b + (k - tiles.a)) * kPcTile;
    }
};
struct PcMisc {  // in shared memory behind the scales
    uint64_t full[kPcSlots], empty[kPcSlots], s_full[2], p_first[2], p_full[2], o_full[2], ks_full[2], vm_full[2], vs_full[2], q_full, done;
    uint32_t there[2][4];
    float v_scale[2];
    // Not zero: the tile's V scales are too far above one of the warp's rows, or of its rows in an earlier tile, to
    // share one.
    uint4 wide[2];
    float vmax[2][4];
    uint32_t tmem;
    PcWork work;
};
static_assert(sizeof(PcMisc) <= 384, "misc area");

// Shared-memory operand descriptors, in halves: bits 0-13 the address / 16 with the stride of
// 64-dim halves above it, and for both operands 8-row groups 1024 bytes apart in the 128-byte
// swizzle. K and Q are K-major; V (rows are keys, 128 bytes of 64 dims a row) is MN-major, the
// next 64 dims one half on.
constexpr uint32_t kPcDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t pc_desc_k(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t pc_desc_v(uint32_t saddr) { return (saddr >> 4) | ((PcGeo<128>::kHalf >> 4) << 16); }
// One thread of a converged warp. MMAs issued inside `if (pc_elect())`, their descriptors built
// from 32-bit halves, go out at the tensor cores' own rate (64 cycles for 128 x 128 x 16); from
// an ordinary one-lane branch they took 87 to 130.
__device__ __forceinline__ bool pc_elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(one));
    return one != 0;
}
template <bool ACC> __device__ __forceinline__ void pc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(kPcDescHigh), "r"(idesc), "n"(ACC ? 1 : 0)
        : "memory");
}
// A from tensor memory.
template <bool ACC> __device__ __forceinline__ void pc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(kPcDescHigh), "r"(idesc), "n"(ACC ? 1 : 0)
        : "memory");
}
// 16 columns of this thread's tensor-memory lane: the load (complete after tc_wait_ld), and
// eight columns back.
__device__ __forceinline__ void tc_ld16_async(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// The registers pass through the wait, so nothing reads them before it.
__device__ __forceinline__ void tc_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tc_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]));
}
__device__ __forceinline__ float2 as_pair(uint32_t x, uint32_t y) {
    return make_float2(__uint_as_float(x), __uint_as_float(y));
}
// Bounded wait. The timer is read once in 256 tries: reading it takes longer than these
// waits usually last, and the barrier completing meanwhile would go unnoticed.
__device__ __forceinline__ bool pc_wait(uint64_t *bar, uint32_t parity, unsigned *err) {
    unsigned long long start = 0;
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 256; i++)
            if (mbar_try(bar, parity)) return true;
        const unsigned long long now = global_ns();
        if (!start) start = now;
        if (wait_expired(now - start)) {
            atomicOr(err, kPagedWaitRanOut);
            return false;
        }
    }
}
// The same of a whole warp, which leaves it converged: all lanes go on, or none.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, unsigned *err) {
    return __all_sync(0xffffffffu, pc_wait(bar, parity, err));
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Byte offset of 16-byte piece `piece` of row `row` inside a 128-byte-swizzled half tile.
__device__ __forceinline__ uint32_t pc_swizzle(int row, int piece) {
    return (uint32_t)(row * 128 + ((piece ^ (row & 7)) << 4));
}
__device__ __forceinline__ void st_smem16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void st_smem8(uint32_t a, uint32_t x, uint32_t y) {
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}
// Bits [0, n) of a word.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Eight stored elements of a BF16 row (16 bytes), scaled, as FP16 pairs.
__device__ __forceinline__ uint32_t bf16_pair_f16(uint32_t w, float scale) {
    return pack_f16(bf16_lo(w) * scale, bf16_hi(w) * scale);
}

// The converters: operand tile `which` (0 K, 1 V) of 128 rows from `base` into the
// shared-memory tile at `dst`, with its row scales. Warp w of the group takes rows
// 32 w .. 32 w + 31, LPR lanes a row.
template <int KIND, int DIM>
struct PcConvert {
    static constexpr int ES = KIND == kPagedBytes ? 1 : 2;
    static constexpr int LPR = DIM * ES / 16;   // 16-byte pieces a row
    static constexpr int RPL = 32 / LPR;        // rows a load instruction covers
    static constexpr int LOADS = 32 / RPL;
    static constexpr int BATCH = LOADS < 8 ? LOADS : 8;
};

// The largest of a row's 128 scores times their K scales; MASKED leaves out columns whose
// bit of vis is clear. Each 16 columns are loaded while the ones before are used.
template <bool MASKED> __device__ __forceinline__ float pc_row_max(uint32_t ts, const float *ks, const uint32_t (&vis)[4]) {
    uint32_t buf[2][16];
    float a = -INFINITY, b = -INFINITY;
    tc_ld16_async(ts, buf[0]);
#pragma unroll
    for (int c = 0; c < 8; c++) {
        uint32_t(&f)[16] = buf[c & 1];
        tc_wait_ld(f);
        if (c < 7) tc_ld16_async(ts + 16 * (c + 1), buf[(c + 1) & 1]);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 k4 = *reinterpret_cast<const float4 *>(ks + 16 * c + j);
            float2 y0 = __fmul2_rn(as_pair(f[j], f[j + 1]), make_float2(k4.x, k4.y));
            float2 y1 = __fmul2_rn(as_pair(f[j + 2], f[j + 3]), make_float2(k4.z, k4.w));
            if (MASKED) {
                const uint32_t seen = vis[c / 2] >> (16 * (c & 1) + j);
                y0.x = seen & 1 ? y0.x : -INFINITY;
                y0.y = seen & 2 ? y0.y : -INFINITY;
                y1.x = seen & 4 ? y1.x : -INFINITY;
                y1.y = seen & 8 ? y1.y : -INFINITY;
            }
            a = fmaxf(a, fmaxf(y0.x, y0.y));
            b = fmaxf(b, fmaxf(y1.x, y1.y));
        }
    }
    return fmaxf(a, b);
}
// The largest weight times V scale among 64 of a row's columns that it sees.
__device__ __forceinline__ float pc_row_most(uint32_t ts, const float *ks, const float *vs, float qs, float m, uint32_t vis0,
                                             uint32_t vis1) {
    float most = 0.f;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        uint32_t f[16];
        tc_ld16_async(ts + 16 * c, f);
        tc_wait_ld(f);
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const float w = ex2(fmaf(__uint_as_float(f[j]) * ks[16 * c + j], qs, -m)) * vs[16 * c + j];
            if (((c < 2 ? vis0 : vis1) >> (16 * (c & 1) + j)) & 1) most = fmaxf(most, w);
        }
    }
    return most;
}
// The weights of 64 of a row's scores, over the scores they come from, and their sum before the
// V scales: the 16 columns of an MMA k-step become eight of first parts and eight of second parts.
template <bool MASKED>
__device__ __forceinline__ float pc_row_weights(uint32_t ts, const float *ks, const float *vs, float qs, float m,
                                                uint32_t vis0, uint32_t vis1) {
    uint32_t buf[2][16];
    float2 sum = make_float2(0.f, 0.f);
    tc_ld16_async(ts, buf[0]);
#pragma unroll
    for (int c = 0; c < 4; c++) {
        uint32_t(&f)[16] = buf[c & 1];
        uint32_t hi[8], lo[8];
        tc_wait_ld(f);
        if (c < 3) tc_ld16_async(ts + 16 * (c + 1), buf[(c + 1) & 1]);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 k4 = *reinterpret_cast<const float4 *>(ks + 16 * c + j);
            const float4 v4 = *reinterpret_cast<const float4 *>(vs + 16 * c + j);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int b = j + 2 * u;
                const float2 y = __fmul2_rn(as_pair(f[b], f[b + 1]), u ? make_float2(k4.z, k4.w) : make_float2(k4.x, k4.y));
                float2 p = make_float2(ex2(fmaf(y.x, qs, -m)), ex2(fmaf(y.y, qs, -m)));
                const uint32_t seen = (c < 2 ? vis0 : vis1) >> (16 * (c & 1) + b);
                if (MASKED) {
                    p.x = seen & 1 ? p.x : 0.f;
                    p.y = seen & 2 ? p.y : 0.f;
                }
                sum = __fadd2_rn(sum, p);
                float2 w = __fmul2_rn(p, u ? make_float2(v4.z, v4.w) : make_float2(v4.x, v4.y));
                if (MASKED) {  // the scale of a row not seen may be anything
                    w.x = seen & 1 ? w.x : 0.f;
                    w.y = seen & 2 ? w.y : 0.f;
                }
                uint32_t parts[2];
                split_pair<kPagedBytes>(w.x, w.y, parts);
                hi[b / 2] = parts[0];
                lo[b / 2] = parts[1];
            }
        }
        tc_st8(ts + 16 * c, hi);
        tc_st8(ts + 16 * c + 8, lo);
    }
    return sum.x + sum.y;
}

// The tiles that the queries of row tile rt see.
__device__ __forceinline__ PagedTiles pc_tiles(const PagedChunkArgs &a, const PagedExtent &e, int rt) {
    const int origin = e.length - e.count, r0 = rt * kPcRows, live = min(kPcRows, e.count * a.group - r0);
    return paged_tiles(origin + r0 / a.group, origin + (r0 + live - 1) / a.group, a.window, a.sinks, 7);
}

// What a CTA works on: split sp of `splits` of row tile rt (the j-th of the batch) of sequence s, for KV head h.
struct PcItem {
    int s, rt, j, h, sp, splits;
    PagedExtent e;  // the sequence's
};
// Finds it, the same in every thread, or returns false. Every CTA counts the row tiles of all sequences (their
// extents are on the device) and takes the splits for what there is, not for the declared maxima: with one chunk of
// 512 rows beside 63 single tokens that had left the chunk on 24 SMs (196 us, now 95; 48 alone), and an empty CTA
// takes 3 us of an SM. `sh` is shared memory that the caller uses for nothing else before its next barrier.
__device__ __forceinline__ bool pc_item(const PagedChunkArgs &a, int *sh, PcItem &it) {
    const PagedView &v = a.v;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int W = kPcThreads / 32;
    int bad = 0, longest = 0, sum = 0;  // of this thread's sequences: the tiles of the longest row tile, and of all
    PagedExtent e;                      // of its last one
    auto row_tiles = [&](int s) {
        e.start = e.count = e.length = 0;
        if (s < v.sequences) bad |= paged_extent(&v, s, &e);
        if (e.count <= a.few) return 0;
        const int n = (e.count * a.group + kPcRows - 1) / kPcRows, most = pc_tiles(a, e, n - 1).count;
        longest = max(longest, most);
        sum += n * (v.sequences == 1 ? most : (pc_tiles(a, e, 0).count + most + 1) / 2);
        return n;
    };
    // A sequence a thread: how many row tiles it has (n), and the sequences before it (low); then `total` counts
    // those of this round too.
    int n = 0, low = 0, total = 0;
    auto round = [&](int s0) {
        n = row_tiles(s0 + tid);
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const int far = __reduce_max_sync(0xffffffffu, longest), all = __reduce_add_sync(0xffffffffu, sum);
        if (s0) __syncthreads();  // the last round's sums have been read
        if (lane == 31) sh[4 + warp] = upto, sh[4 + W + warp] = far, sh[4 + 2 * W + warp] = all;
        __syncthreads();
        const int sums = lane < W ? sh[4 + lane] : 0;
        low = total + __reduce_add_sync(0xffffffffu, lane < warp ? sums : 0) + upto - n;
        total += __reduce_add_sync(0xffffffffu, sums);
    };
    if (v.sequences == 1) {
        total = n = row_tiles(0);  // of every thread
    } else {
        for (int s0 = 0; s0 < v.sequences; s0 += kPcThreads) round(s0);
        longest = __reduce_max_sync(0xffffffffu, lane < W ? sh[4 + W + lane] : 0);
        sum = __reduce_add_sync(0xffffffffu, lane < W ? sh[4 + 2 * W + lane] : 0);
    }
    // Splits: a number a lane (paged_splits).
    static_assert(kPcSplitsMax == 32, "a lane for each number of splits");
    const int64_t items = (int64_t)total * v.kvheads;
    const int mean = v.sequences == 1 ? longest : (sum + total - 1) / max(total, 1);
    const float cost = paged_may_split(items, lane + 1, longest, a.slots) ? paged_split_cost((unsigned)items, lane + 1, mean, longest, a.sms) : INFINITY;
    const int splits = __ffs(__ballot_sync(0xffffffffu, cost <= -1.03f * warp_max(-cost)));
    if (blockIdx.x == 0) {
        if (items > gridDim.x) bad |= kPagedBadExtent;  // only where sequences share rows of the callers' buffers
        paged_report(a.status, bad);
        if (tid == 0) a.plan[0] = make_int4(total, splits, 0, 0);
    }
    const unsigned index = blockIdx.x / (unsigned)splits;
    if (index >= items) return false;
    it.splits = splits;
    it.sp = (int)(blockIdx.x - index * (unsigned)splits);
    it.j = (int)(index / (unsigned)v.kvheads);
    it.h = (int)(index - (unsigned)it.j * (unsigned)v.kvheads);
    if (v.sequences == 1) {
        it.s = 0;
        it.rt = n - 1 - it.j;
        it.e = e;
        return true;
    }
    if (tid == 0) sh[0] = -1;
    const int count = total;
    if (v.sequences > kPcThreads) {
        __syncthreads();  // every warp has read the sums
        total = 0;
    }
    for (int s0 = 0; s0 < v.sequences; s0 += kPcThreads) {  // one round's n and low are still there
        if (v.sequences > kPcThreads) round(s0);
        else __syncthreads();
        if (it.j >= low && it.j < low + n) {
            sh[0] = s0 + tid;
            sh[1] = n - 1 - (it.j - low);  // the longest row tiles (the last ones) start first
            sh[2] = e.start, sh[3] = e.count, sh[4 + 3 * W] = e.length;
        }
        if (it.j < total || total >= count) break;
    }
    __syncthreads();
    it.s = sh[0];
    it.rt = sh[1];
    it.e.start = sh[2], it.e.count = sh[3], it.e.length = sh[4 + 3 * W];
    return it.s >= 0;
}

template <int KIND, int DIM>
__global__ void __launch_bounds__(kPcThreads, 1) paged_chunk_kernel(const PagedChunkArgs a) {
    using G = PcGeo<DIM>;
    constexpr bool kBytes = KIND == kPagedBytes;
    extern __shared__ __align__(1024) unsigned char pc_smem[];
    unsigned char *smem = pc_smem;
    PcMisc &x = *reinterpret_cast<PcMisc *>(smem + G::kMisc);
    float *scales = reinterpret_cast<float *>(smem + G::kScales);  // [K|V][tile parity][128]
    const PagedView &v = a.v;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    pdl_wait();
    pdl_trigger();  // the decode kernel of the same call starts beside the last CTAs
    PcItem it;
    if (!pc_item(a, reinterpret_cast<int *>(smem), it)) return;
    const PagedExtent &extent = it.e;
    const PagedTiles tiles = pc_tiles(a, extent, it.rt);
    const int splits = max(1, min(it.splits, tiles.count));
    if (tid == 0 && it.h == 0 && it.sp == 0) a.plan[1 + it.j] = make_int4(extent.start, extent.count * a.group, it.rt, splits);
    if (it.sp >= splits) return;
    // Below 2^23 tiles, at most 32 splits.
    const int k0 = (int)((unsigned)(tiles.count * it.sp) / (unsigned)splits), n = (int)((unsigned)(tiles.count * (it.sp + 1)) / (unsigned)splits) - k0;
    const int halves = extent.count * a.group - it.rt * kPcRows > 128 ? 2 : 1;
    if (tid == 0) {
        PcWork z;
        z.s = it.s, z.h = it.h, z.start = extent.start, z.rows = extent.count * a.group;
        z.origin = extent.length - extent.count;
        z.r0 = it.rt * kPcRows, z.live = min(kPcRows, z.rows - z.r0), z.splits = splits;
        z.first = z.origin + z.r0 / a.group, z.last = z.origin + (z.r0 + z.live - 1) / a.group;
        z.tiles = tiles, z.k0 = k0, z.n = n;
        x.work = z;
    }
    const volatile PcWork &z = x.work;

    const uint32_t base_s = smem_addr(smem);
    if (base_s & 1023u) {  // the swizzled tiles need it; a launch without static shared memory starts there
        if (!tid) atomicOr(a.err, kPagedWaitRanOut);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < kPcSlots; i++) {
            mbar_init(&x.full[i], 128);
            mbar_init(&x.empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&x.s_full[i], 1);
            mbar_init(&x.p_first[i], 128);
            mbar_init(&x.p_full[i], 128);
            mbar_init(&x.o_full[i], 1);
            mbar_init(&x.ks_full[i], 128);
            mbar_init(&x.vm_full[i], 4);
            mbar_init(&x.vs_full[i], 128);
        }
        mbar_init(&x.q_full, halves * 128);
        mbar_init(&x.done, 1);
        mbar_fence_init();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&x.tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, x.tmem, 0);  // columns: S and P of half i at 128 i, O at 256 + 128 i

    if (warp < 8) {
        // ================================================================ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPcSoftmaxRegs));
        const int i = warp >> 2, row = (warp & 3) * 32 + lane, r = z.r0 + i * 128 + row;
        if (i == 0 || z.live > 128) {
            // ---- Q: this warp's 32 rows as two FP16 parts, scaled by the row's power of two
            float mine = 0.f;
            constexpr int E = DIM / 32, QB = 16;  // rows whose loads are in flight together
            const long long q_at = r < z.rows ? (long long)(z.start + r / a.group) * a.q_stride + (z.h * a.group + r % a.group) * DIM : -1;
#pragma unroll 1
            for (int first_k = 0; first_k < 32; first_k += QB) {
                float f[QB][E];
#pragma unroll
                for (int k = 0; k < QB; k++) {
                    const long long at = __shfl_sync(0xffffffffu, q_at, first_k + k);
#pragma unroll
                    for (int c = 0; c < E; c++) f[k][c] = 0.f;
                    if (at >= 0) {
                        const float *src = a.q + at + lane * E;
                        if constexpr (E == 4) {
                            const float4 t = *reinterpret_cast<const float4 *>(src);
                            f[k][0] = t.x, f[k][1] = t.y, f[k][2] = t.z, f[k][3] = t.w;
                        } else {
                            const float2 t = *reinterpret_cast<const float2 *>(src);
                            f[k][0] = t.x, f[k][1] = t.y;
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < QB; k++) {
                    float m = 0.f;
#pragma unroll
                    for (int c = 0; c < E; c++) m = fmaxf(m, fabsf(f[k][c]));
                    const int ex = max(-126, exponent_of(warp_max(m)) - 14);  // up and its inverse are both normal
                    const float up = power_of_two(-ex);
                    if (lane == first_k + k) mine = a.scale2 * power_of_two(ex);
                    uint32_t hi[E / 2], lo[E / 2];
#pragma unroll
                    for (int c = 0; c < E; c += 2) {
                        uint32_t p[2];
                        split_pair<kPagedBytes>(f[k][c] * up, f[k][c + 1] * up, p);
                        hi[c / 2] = p[0];
                        lo[c / 2] = p[1];
                    }
                    const int d = lane * E, rr = (warp & 3) * 32 + first_k + k;  // half tile, 16-byte piece, offset inside it
                    const uint32_t at = base_s + (uint32_t)(2 * i) * G::kOperand + (uint32_t)(d / 64) * G::kHalf +
                                        pc_swizzle(rr, (d % 64) / 8) + (uint32_t)(d % 8) * 2;
                    if constexpr (E == 4) {
                        st_smem8(at, hi[0], hi[1]);
                        st_smem8(at + G::kOperand, lo[0], lo[1]);
                    } else {
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(hi[0]) : "memory");
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + G::kOperand), "r"(lo[0]) : "memory");
                    }
                }
            }
            fence_async_smem();
            mbar_arrive(&x.q_full);

            const float qs = mine;
            const int at = r < z.rows ? z.origin + r / a.group : -1;  // a row behind the last sees nothing
            const int top_row = min(z.live, (i + 1) * 128) - 1;
            const int first_i = z.origin + (z.r0 + i * 128) / a.group, last_i = z.origin + (z.r0 + top_row) / a.group;
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t ts = tmem + lanes + (uint32_t)(128 * i), to = tmem + lanes + 256u + (uint32_t)(128 * i);
            float o[DIM], m = -INFINITY, l = 0.f;
#pragma unroll
            for (int c = 0; c < DIM; c++) o[c] = 0.f;
            for (int t = 0; t < z.n; t++) {
                const int base = z.base(t), par = t & 1;
                const float *ks = scales + par * 128, *vs = scales + 256 + par * 128;
                if (!warp_wait(&x.ks_full[par], (t >> 1) & 1, a.err)) break;
                if (!warp_wait(&x.s_full[i], t & 1, a.err)) break;
                tc_fence_after();
                uint32_t vis[4];
#pragma unroll
                for (int w = 0; w < 4; w++) vis[w] = x.there[par][w];
                // Every row of this half sees the whole tile?
                const bool full = (vis[0] & vis[1] & vis[2] & vis[3]) == 0xffffffffu && base + 127 <= first_i &&
                                  (a.window == 0 || base + 127 < a.sinks || base > last_i - a.window);
                if (!full) {
                    const int hi = at - base + 1, lo = a.window == 0 || a.window > at ? 0 : at - a.window - base + 1,
                              sk = a.sinks - base;
#pragma unroll
                    for (int w = 0; w < 4; w++)
                        vis[w] &= bits_below(hi - 32 * w) & (~bits_below(lo - 32 * w) | bits_below(sk - 32 * w));
                }
                const float top = full ? pc_row_max<false>(ts, ks, vis) : pc_row_max<true>(ts, ks, vis);
                // The reference moves only when the maximum has passed it by 2^3: weights have that much
                // room, and output rows whose reference stays need no rescaling.
                float keep = 1.f;
                if (top * qs > m + kPcSlack) {
                    keep = m == -INFINITY ? 0.f : ex2(m - top * qs);
                    m = top * qs;
                }
                const float mr = m == -INFINITY ? 0.f : m;
                const bool moved = __any_sync(0xffffffffu, keep != 1.f);
                if (!warp_wait(&x.vs_full[par], (t >> 1) & 1, a.err)) break;
                float v_scale = x.v_scale[par];
                const uint4 far = x.wide[par];
                l *= keep;
                // In two halves of the columns: the first half's products start while the second is computed.
                auto half_done = [&](int c) {
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    mbar_arrive(c ? &x.p_full[i] : &x.p_first[i]);
                };
                if (!(far.x | far.y | far.z | far.w)) {
#pragma unroll 1
                    for (int c = 0; c < 128; c += 64) {
                        const uint32_t v0 = c ? vis[2] : vis[0], v1 = c ? vis[3] : vis[1];
                        l += full ? pc_row_weights<false>(ts + c, ks + c, vs + c, qs, mr, 0, 0)
                                  : pc_row_weights<true>(ts + c, ks + c, vs + c, qs, mr, v0, v1);
                        half_done(c);
                    }
                } else {
                    // V scales far apart meet: the largest weight of the columns that a row sees sets its scale, so
                    // that none that it does not see or that hardly counts can push its weights below FP16. The
                    // factor 2^up goes into the exponent, and what the subtraction rounds off comes back with it.
                    float most = 0.f, sum = 0.f;
#pragma unroll 1
                    for (int c = 0; c < 128; c += 64)
                        most = fmaxf(most, pc_row_most(ts + c, ks + c, vs + c, qs, mr, c ? vis[2] : vis[0], c ? vis[3] : vis[1]));
                    const float up = (float)min(100, kPcWeightTop - exponent_of(most)), mw = __fsub_rn(mr, up);
#pragma unroll 1
                    for (int c = 0; c < 128; c += 64) {
                        sum += pc_row_weights<true>(ts + c, ks + c, vs + c, qs, mw, c ? vis[2] : vis[0], c ? vis[3] : vis[1]);
                        half_done(c);
                    }
                    const float by = __fsub_rn(mw, mr), off = __fadd_rn(__fsub_rn(mr, __fsub_rn(mw, by)), __fsub_rn(-up, by));
                    const float back = power_of_two(-(int)up) * ex2(-off);
                    l = fmaf(sum, back, l);
                    v_scale *= back;
                }
                // ---- this tile's output
                if (!warp_wait(&x.o_full[i], t & 1, a.err)) break;
                tc_fence_after();
                if (moved) {
#pragma unroll
                    for (int c = 0; c < DIM; c++) o[c] *= keep;
                }
                uint32_t buf[2][16];
                tc_ld16_async(to, buf[0]);
#pragma unroll
                for (int c = 0; c < DIM / 16; c++) {
                    uint32_t(&f)[16] = buf[c & 1];
                    tc_wait_ld(f);
                    if (c + 1 < DIM / 16) tc_ld16_async(to + 16 * (c + 1), buf[(c + 1) & 1]);
#pragma unroll
                    for (int j = 0; j < 16; j++) o[16 * c + j] = fmaf(__uint_as_float(f[j]), v_scale, o[16 * c + j]);
                }
                tc_fence_before();
            }
            // ---- rows out, through this half's part of the Q area (its products are over) so that a
            // warp writes whole rows. Every warp has written its queries there (with no tile at all nothing
            // else has made sure of that).
            warp_wait(&x.q_full, 0, a.err);
            const int parts = z.splits, rows = z.rows;
            const float f = parts > 1 ? 1.f : l > 0.f ? 1.f / l : (l == l ? 0.f : l);  // nothing seen: zeros
            const int64_t slot = blockIdx.x;
            if (parts > 1 && r < rows) a.ml[slot * kPcRows + (r - z.r0)] = make_float2(m, l);
            constexpr int PR = DIM / 4;  // 16-byte pieces a row
            const uint32_t area = base_s + (uint32_t)(2 * i) * G::kOperand + (uint32_t)((warp & 3) * 32 * DIM * 4);
#pragma unroll
            for (int c = 0; c < PR; c++)
                st_smem16(area + (uint32_t)(lane * PR + (c ^ (lane & (PR - 1)))) * 16, __float_as_uint(o[4 * c] * f),
                          __float_as_uint(o[4 * c + 1] * f), __float_as_uint(o[4 * c + 2] * f), __float_as_uint(o[4 * c + 3] * f));
            __syncwarp();
            const long long mine_at = parts > 1 ? (slot * kPcRows + (r - z.r0)) * DIM
                                                : (long long)(z.start + r / a.group) * a.out_stride + (z.h * a.group + r % a.group) * DIM;
            float *dst = parts > 1 ? a.part : a.out;
#pragma unroll 4
            for (int k = 0; k < 32; k += 32 / PR) {
                const int rr = k + lane / PR, c = lane % PR;
                const long long at_row = __shfl_sync(0xffffffffu, mine_at, rr);
                uint4 y;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                             : "r"(area + (uint32_t)(rr * PR + (c ^ (rr & (PR - 1)))) * 16));
                if (r - lane + rr < rows) *reinterpret_cast<uint4 *>(dst + at_row + c * 4) = y;
            }
        }
    } else if (warp < 12) {
        // ================================================================ stored rows -> operand tiles
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPcConvertRegs));
        using C = PcConvert<KIND, DIM>;
        const int w = warp - 8, piece = lane % C::LPR, sub = lane / C::LPR;
        const int64_t half = (int64_t)v.pages * v.kvheads * v.page;
        int bad = 0;
        bool ok = true;
        float v_low = INFINITY;  // the smallest V scale of this lane's rows so far
        for (int t = 0; t < z.n && ok; t++) {
            const int base = z.base(t), par = t & 1;
            // This lane's row: place base + 32 w + lane.
            const int j = base + 32 * w + lane;
            int64_t mine = -1;
            // Rows that no query of the tile sees are left out: they may hold anything, a scale that would
            // drown the others' too, and their page may be missing.
            if (j <= z.last && (a.window == 0 || j < a.sinks || (int64_t)j > (int64_t)z.first - a.window)) {
                const int pg = paged_div(&v, j);
                mine = paged_row(&v, v.table[(int64_t)z.s * v.table_stride + pg], j, pg, z.h);
                if (mine < 0) bad |= kPagedBadPage;
            }
            const uint32_t there = __ballot_sync(0xffffffffu, mine >= 0);
#pragma unroll 1
            for (int which = 0; which < 2; which++) {
                const char *pool = static_cast<const char *>(which ? v.values : v.keys);
                const int use = 2 * t + which, slot = use % kPcSlots;
                const uint32_t dst = base_s + G::kQ + (uint32_t)slot * G::kOperand;
                float scale = 0.f;
                if (kBytes && mine >= 0) scale = __ldcg(v.scales + (which ? half : 0) + mine);
#pragma unroll 1
                for (int b = 0; b < C::LOADS; b += C::BATCH) {
                    uint4 in[C::BATCH];
#pragma unroll
                    for (int k = 0; k < C::BATCH; k++) {
                        const int64_t rk = __shfl_sync(0xffffffffu, mine, (b + k) * C::RPL + sub);
                        in[k] = rk >= 0 ? ld_row16(pool + rk * (DIM * C::ES) + piece * 16) : make_uint4(0, 0, 0, 0);
                    }
                    if (b == 0 && use >= kPcSlots) {  // the slot's last use is over
                        ok = warp_wait(&x.empty[slot], ((use / kPcSlots) & 1) ^ 1, a.err);
                        if (!ok) break;
                    }
#pragma unroll
                    for (int k = 0; k < C::BATCH; k++) {
                        const int rl = (b + k) * C::RPL + sub, rr = 32 * w + rl;
                        uint4 y = in[k];
                        if constexpr (kBytes) {
                            // 16 codes: dims 16 piece ..: two 16-byte pieces of FP16. The lanes of a row's
                            // second 64 dims store their pieces in the other order: eight lanes, all banks.
                            const int d = piece * 16, other = d / 64;
                            const uint32_t at = dst + (uint32_t)(d / 64) * G::kHalf;
                            if (other) y = make_uint4(y.z, y.w, y.x, y.y);
                            const uint32_t q0 = y.x ^ 0x80808080u, q1 = y.y ^ 0x80808080u, q2 = y.z ^ 0x80808080u,
                                           q3 = y.w ^ 0x80808080u;
                            st_smem16(at + pc_swizzle(rr, (d % 64) / 8 + other), codes_f16(q0, 0x4140), codes_f16(q0, 0x4342),
                                      codes_f16(q1, 0x4140), codes_f16(q1, 0x4342));
                            st_smem16(at + pc_swizzle(rr, (d % 64) / 8 + 1 - other), codes_f16(q2, 0x4140),
                                      codes_f16(q2, 0x4342), codes_f16(q3, 0x4140), codes_f16(q3, 0x4342));
                        } else {
                            // The row's largest magnitude as bits, over its lanes.
                            uint32_t mb = __vmaxu2(__vmaxu2(y.x & 0x7fff7fffu, y.y & 0x7fff7fffu),
                                                   __vmaxu2(y.z & 0x7fff7fffu, y.w & 0x7fff7fffu));
                            mb = max(mb & 0xffffu, mb >> 16);
#pragma unroll
                            for (int off = C::LPR / 2; off; off >>= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, off));
                            const int ef = (int)(mb >> 7);
                            const int ex = ef == 255 ? 0 : max(-126, ef - 127 - 14);
                            const float up = power_of_two(-ex);
                            // A non-finite V row enters as zeros with a NaN weight: only who sees it is touched.
                            if (ef == 255 && which) y = make_uint4(0, 0, 0, 0);
                            const float rs = __shfl_sync(0xffffffffu, ef == 255 && which ? __uint_as_float(0x7fc00000u) : power_of_two(ex),
                                                         (lane % C::RPL) * C::LPR);
                            if (lane / C::RPL == b + k) scale = rs;  // row rl = (b + k) RPL + lane % RPL is this lane's
                            const int d = piece * 8;
                            st_smem16(dst + (uint32_t)(d / 64) * G::kHalf + pc_swizzle(rr, (d % 64) / 8),
                                      bf16_pair_f16(y.x, up), bf16_pair_f16(y.y, up), bf16_pair_f16(y.z, up),
                                      bf16_pair_f16(y.w, up));
                        }
                    }
                }
                if (!ok) break;
                fence_async_smem();
                if (t || a.starve != 1 + which) mbar_arrive(&x.full[slot]);
                if (!which) {
                    scales[par * 128 + 32 * w + lane] = mine >= 0 ? scale : 0.f;
                    if (lane == 0) x.there[par][w] = there;
                    mbar_arrive(&x.ks_full[par]);
                } else {
                    // Weights are scaled by the tile's largest V scale: s 2^12 / R < 2^12. Rows of zeros (and those
                    // below about 2^-105) say nothing about how far scales lie apart.
                    if (mine < 0) scale = 0.f;
                    const float top = warp_max(isfinite(scale) ? scale : 0.f);
                    if (scale > 0x1p-120f) v_low = fminf(v_low, scale);
                    if (lane == 0) {
                        x.vmax[par][w] = top;
                        mbar_arrive(&x.vm_full[par]);
                    }
                    ok = warp_wait(&x.vm_full[par], (t >> 1) & 1, a.err);
                    if (!ok) break;
                    const float vmax = fmaxf(fmaxf(x.vmax[par][0], x.vmax[par][1]), fmaxf(x.vmax[par][2], x.vmax[par][3]));
                    const int er = max(-100, exponent_of(vmax) + 1) - kPcWeightTop;
                    scales[256 + par * 128 + 32 * w + lane] = scale * power_of_two(-er);
                    const bool far = __any_sync(0xffffffffu, v_low < power_of_two(er + kPcWeightTop - kPagedSpread));
                    if (lane == 0) reinterpret_cast<uint32_t *>(&x.wide[par])[w] = far;
                    if (w == 0 && lane == 0) x.v_scale[par] = power_of_two(er);
                    mbar_arrive(&x.vs_full[par]);
                }
            }
        }
        if (bad) paged_report(a.status, bad);
    } else {
        // ================================================================ MMA
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPcIssueRegs));
    }
    if (warp == 12) {
        const uint32_t ring = base_s + G::kQ;
        const int n = z.n, halves = z.live > 128 ? 2 : 1;
        bool ok = warp_wait(&x.q_full, 0, a.err);
        auto scores = [&](int t, int i) {  // S_i = Q_i K(t)^T
            const int use = 2 * t, slot = use % kPcSlots;
            if (!warp_wait(&x.full[slot], (use / kPcSlots) & 1, a.err)) return false;
            // P_i(t - 1) lies in the same columns: its product must be over.
            if (t && !warp_wait(&x.o_full[i], (t - 1) & 1, a.err)) return false;
            tc_fence_after();
            if (pc_elect()) {
                const uint32_t d = tmem + (uint32_t)(128 * i), kd = pc_desc_k(ring + (uint32_t)slot * G::kOperand);
#pragma unroll
                for (int part = 1; part >= 0; part--) {
                    const uint32_t qd = pc_desc_k(base_s + (uint32_t)(2 * i + part) * G::kOperand);
#pragma unroll
                    for (int ks = 0; ks < DIM / 16; ks++) {  // 32 bytes on in a row of 128, then the next half
                        const uint32_t off = (uint32_t)(ks / 4) * (G::kHalf >> 4) + 2 * (ks % 4);
                        if (part == 1 && ks == 0) pc_mma_ss<false>(d, qd + off, kd + off, G::kIdescS);
                        else pc_mma_ss<true>(d, qd + off, kd + off, G::kIdescS);
                    }
                }
                tc_commit(&x.s_full[i]);
                if (i == halves - 1) tc_commit(&x.empty[slot]);
            }
            __syncwarp();
            return true;
        };
        for (int i = 0; i < halves && ok && n > 0; i++) ok = scores(0, i);
        for (int t = 0; t < n && ok; t++)
            for (int i = 0; i < halves && ok; i++) {
                const int use = 2 * t + 1, slot = use % kPcSlots;
                ok = warp_wait(&x.full[slot], (use / kPcSlots) & 1, a.err);
#pragma unroll
                for (int first = 0; first < 2 && ok; first++) {
                    ok = warp_wait(first ? &x.p_full[i] : &x.p_first[i], t & 1, a.err);
                    if (!ok) break;
                    tc_fence_after();
                    if (pc_elect()) {
                        const uint32_t d = tmem + 256u + (uint32_t)(128 * i), p = tmem + (uint32_t)(128 * i),
                                       vd = pc_desc_v(ring + (uint32_t)slot * G::kOperand);
#pragma unroll
                        for (int part = 1; part >= 0; part--)
#pragma unroll
                            for (int ks = 4 * first; ks < 4 * first + 4; ks++) {  // 16 keys: 2048 bytes on in V, 16 columns on in P
                                const uint32_t pa = p + 16 * ks + 8 * part, vb = vd + (uint32_t)(128 * ks);
                                if (part == 1 && ks == 0) pc_mma_ts<false>(d, pa, vb, G::kIdescO);
                                else pc_mma_ts<true>(d, pa, vb, G::kIdescO);
                            }
                        if (first) {
                            tc_commit(&x.o_full[i]);
                            if (i == halves - 1) tc_commit(&x.empty[slot]);
                        }
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (t + 1 < n) ok = scores(t + 1, i);
            }
        // Every product and arrival is over before tensor memory and the barriers are given back.
        if (pc_elect()) tc_commit(&x.done);
        __syncwarp();
        warp_wait(&x.done, 0, a.err);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// The parts of split row tiles, joined in order: a warp a query row. A kernel of its own, because
// the last of a row tile's CTAs alone took 10 us over its 256 rows.
constexpr int kPcJoinThreads = 256;
// Query row rr of a row tile (its entry of the plan) and KV head h, whose parts begin at slot `item`.
template <int DIM> __device__ __forceinline__ void pc_join_row(const PagedChunkArgs &a, int4 tile, int h, int64_t item, int rr, int lane) {
    constexpr int E = DIM / 32;
    const int start = tile.x, splits = tile.w, r = tile.z * kPcRows + rr;
    if (splits == 1 || r >= tile.y) return;
    // Lane w holds split w's maximum and sum; every lane a piece of the row of each split.
    static_assert(kPcSplitsMax <= 32, "a lane for each split");
    const float2 ml = lane < splits ? __ldcg(&a.ml[(item + lane) * kPcRows + rr]) : make_float2(-INFINITY, 0.f);
    const float top = warp_max(ml.x), mine = pd_factor(ml, top), sum = warp_sum(ml.y * mine);
    float y[E];
#pragma unroll
    for (int c = 0; c < E; c++) y[c] = 0.f;
    for (int w0 = 0; w0 < splits; w0 += 8) {
        float z[8][E];
#pragma unroll
        for (int w = 0; w < 8; w++) {
            const float *src = a.part + ((item + min(w0 + w, splits - 1)) * kPcRows + rr) * DIM + lane * E;
            if constexpr (E == 4) {
                const float4 t = __ldcg(reinterpret_cast<const float4 *>(src));
                z[w][0] = t.x, z[w][1] = t.y, z[w][2] = t.z, z[w][3] = t.w;
            } else {
                const float2 t = __ldcg(reinterpret_cast<const float2 *>(src));
                z[w][0] = t.x, z[w][1] = t.y;
            }
        }
#pragma unroll
        for (int w = 0; w < 8; w++) {
            const float f = __shfl_sync(0xffffffffu, mine, (w0 + w) & 31);
            if (w0 + w < splits)
#pragma unroll
                for (int c = 0; c < E; c++) y[c] = fmaf(z[w][c], f, y[c]);
        }
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
    float *dst = a.out + (long long)(start + r / a.group) * a.out_stride + (h * a.group + r % a.group) * DIM + lane * E;
    if constexpr (E == 4) *reinterpret_cast<float4 *>(dst) = make_float4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
    else *reinterpret_cast<float2 *>(dst) = make_float2(y[0] * inv, y[1] * inv);
}
template <int DIM>
__global__ void __launch_bounds__(kPcJoinThreads) paged_chunk_join_kernel(const PagedChunkArgs a) {
    const int kvheads = a.v.kvheads, lane = threadIdx.x & 31, step = gridDim.x * (kPcJoinThreads / 32);
    int at = (blockIdx.x * kPcJoinThreads + threadIdx.x) / 32;  // an item's query row
    pdl_wait();
    // Every warp reads these: through L1 (past it, 6144 warps met in a few lines of L2, 1 us longer).
    int4 tile = a.plan[1 + at / kPcRows / kvheads];  // the launch is no larger than the plan
    const int4 head = a.plan[0];
    if (head.y == 1) return;
    for (;;) {  // a batch that is split has no more items than there are places for parts
        const int index = at / kPcRows;
        if (index >= head.x * kvheads) return;
        pc_join_row<DIM>(a, tile, index % kvheads, (int64_t)index * head.y, at % kPcRows, lane);
        at += step;
        if (at / kPcRows < head.x * kvheads) tile = a.plan[1 + at / kPcRows / kvheads];
    }
}

}  // namespace tcm
