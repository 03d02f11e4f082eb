// Attention of single query rows over pages chosen for them, one KV head at a time (paged_sparse.cu writes the choice).
//
// An item is a query row and a KV head: up to eight query heads, a table of pages of its own, and the number of rows
// that they hold, all of them visible. A cluster of CTAs has an item and shares its rows out in steps of 16 or 32; every warp
// takes steps in turn, each with its own online softmax, and the parts meet in shared memory, the CTAs' in one
// another's. No item waits for another, and nothing is left in global memory in between.
//
// The MMAs are those of the decode kernel's tile of eight query rows (paged_decode.cuh): the queries' first and second
// parts share an operand, and 16-byte pieces of the rows are the other one as they come. A warp's copies go through a
// ring of two steps, K and V apart. Every row that a query has is visible, so nothing of a tile is ever masked but the
// places behind the last row and pages without an id, which are copied as zeros.
//
// Precision is the decode kernel's: products exact, queries as three BF16 parts or three signed bytes, weights as three
// BF16 parts, or over byte rows, whose scales they carry, as FP16 pairs: every head scales its own by a power of two
// that follows the largest weight times scale so far, and falls when the maximum rises, so that no row sets it for what
// comes after. Sums in the tensor cores truncate: no more than kPdChain steps of P V follow one another there.
//
// What bounds it: with many items the instructions of a row, 25 of bytes, at half of the issue slots, as three warps a
// scheduler wait for one another's fixed latencies (512 rows of 4096 byte rows, 2 KV heads: 213 us; four CTAs an SM at 128
// registers 222); over BF16 rows L2 (160 rows of 1280 rows, 8 KV heads: 111 us, 7.5 TB/s). With few items the chain of a
// warp, 2 us a step, behind 3 us to the first rows and before 4 of joining (64 rows of 128 to 2048 byte rows, 2 KV heads:
// 20 us; one row: 8). The same choice read by the decode kernel, a row a sequence, made whole calls of 298, 193 and 43 us
// that take 249, 131 and 47 here: its line of equal stretches serves 64 unequal items better, its tiles of one row each the
// others worse.
#pragma once
#include "paged_decode.cuh"
#include <cooperative_groups.h>

namespace tcm {

struct PagedChosenArgs {
    PagedView v;
    const float *q;
    float *out;
    long long q_stride, out_stride;
    int group, blocks, row0;
    const int *lengths;  // [rows of the slab]: rows that the pages hold; -1: no row of the batch
    const int *table;    // [rows][kvheads][blocks]
    float scale2;        // log2(e) / sqrt(dim)
    int *status;
};

constexpr int kPsWarps = 4, kPsThreads = kPsWarps * 32, kPsCtas = 3, kPsCluster = 16;
constexpr float kPsMost = 32768.f;  // of a byte row's scaled weight, inside FP16
template <int KIND, int DIM> struct PsGeo {
    static constexpr int kRow = DIM * (KIND == kPagedBytes ? 1 : 2);               // bytes of a stored row
    // Rows of a step: 32 cost a quarter fewer instructions a row than 16 (493 and 400 of byte rows, measured), but leave no
    // room for a second step in the ring beside BF16 rows of 128 (32 sequences of 5 tokens: 117 us, 111 with 16).
    static constexpr int kStep = KIND == kPagedBf16 && DIM == 128 ? 16 : 32;
    static constexpr int kUnit = kStep * kRow + (KIND == kPagedBytes ? kStep * 4 : 0) + 16;  // rows, their scales, which are there
    static constexpr int kAhead = 2;                                                      // steps in a warp's ring: three CTAs an SM fit
    static constexpr int kSteps = kRow / 32;                                       // k-steps of Q K^T
    static constexpr size_t kRing = (size_t)kPsWarps * 2 * kAhead * kUnit;
    static constexpr size_t kFrag = (size_t)2 * kSteps * 32 * 16;
    static constexpr size_t kSmem = kRing + kFrag;
};

template <int KIND, int DIM>
__global__ void __launch_bounds__(kPsThreads, kPsCtas) paged_chosen_kernel(const __grid_constant__ PagedChosenArgs a) {
    constexpr bool kBytes = KIND == kPagedBytes;
    using G = PsGeo<KIND, DIM>;
    constexpr int W = kPsWarps, T = kPsThreads, ES = kBytes ? 1 : 2, DV = DIM / 8, VW = DV * ES / 4, KS = G::kSteps;
    constexpr int P = kPdParts<KIND>, A = G::kAhead, S = G::kStep;
    constexpr unsigned kAll = S == 32 ? 0xffffffffu : 0xffffu;
    extern __shared__ __align__(16) unsigned char ps_smem[];
    uint4(*qf)[KS][32] = reinterpret_cast<uint4(*)[KS][32]>(ps_smem + G::kRing);   // the queries' fragments
    float4(*wo)[8][DIM / 4] = reinterpret_cast<float4(*)[8][DIM / 4]>(ps_smem);     // the warps' outputs, then the CTAs'
    // Behind them, of the cluster's outputs this CTA's share from each CTA, and each one's maxima and sums.
    float4 *parts = reinterpret_cast<float4 *>(ps_smem + (size_t)W * 8 * DIM * 4);
    constexpr int kParts = 8 * DIM / 4 + kPsCluster;
    float2(*parts_ml)[8] = reinterpret_cast<float2(*)[8]>(parts + kParts);
    static_assert(G::kRing >= (size_t)W * 8 * DIM * 4 + kParts * 16 + kPsCluster * 8 * 8, "outputs fit the ring");
    __shared__ float qs[8];  // log2(e) / sqrt(dim) times what a query was multiplied down by
    __shared__ float2 wml[W][8];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const PagedView &v = a.v;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int C = gridDim.x, part = blockIdx.x, h = blockIdx.y, r = blockIdx.z;
    pdl_trigger();
    pdl_wait();
    const int n = a.lengths[r];
    float *out = a.out + (long long)(a.row0 + r) * a.out_stride + (int64_t)h * a.group * DIM;
    if (n <= 0) {  // no row of the batch, or a query that sees nothing
        if (n == 0 && part == 0)
            for (int i = tid; i < a.group * (DIM / 4); i += T) reinterpret_cast<float4 *>(out)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        return;
    }
    const int *table = a.table + ((int64_t)r * v.kvheads + h) * a.blocks;
    const int steps = (n + S - 1) / S;
    const int k0 = (int)((int64_t)steps * part / C), k1 = (int)((int64_t)steps * (part + 1) / C);

    // ---- the copies of this warp's steps k0 + warp, + W, ...: unit i is K (even i) or V of the i / 2-th. A lane copies 16
    // bytes of every kRpl-th row; where they lie in a unit goes by pd_swizzle, whose change from one of its rows to the
    // next is the same in every lane.
    constexpr int kLpr = G::kRow / 16, kRpl = 32 / kLpr, kRowsCopied = S / kRpl;  // lanes a row, rows at a time, rows of a lane
    const bool whole = v.page % 16 == 0;  // 16 rows lie inside one page
    const bool wide = whole && (!kBytes || ((uintptr_t)v.scales & 15) == 0);  // scales by 16 bytes as well
    const uint32_t lane_to = (uint32_t)(lane / kLpr * G::kRow + pd_swizzle<G::kRow>(lane / kLpr, lane % kLpr) * 16);
    unsigned char *const ring = ps_smem + warp * 2 * A * G::kUnit;
    const char *const keys = static_cast<const char *>(v.keys) + lane * 16, *const values = static_cast<const char *>(v.values) + lane * 16;
    const int page_rows = v.kvheads * v.page, head_row = h * v.page;  // rows of a page, and before this head's in it
    int bad = 0;
    // The lane's place in step k: its 16 rows' first, or (pages that end inside 16 rows) its own; and the page id of it.
    auto place_of = [&](int k) { return S * k + (whole ? lane & (S - 16) : lane & (S - 1)); };
    auto id_of = [&](int k) -> int { return k < k1 ? table[paged_div(&v, min(place_of(k), n - 1))] : -1; };
    // Of the step that is copied next: its number, where its 16 rows, or the lane's one, are in the pool (-1:
    // nowhere), which are there, the unit that takes its K rows, and the page id of the step behind it.
    int ahead = k0 + warp, next_id = id_of(ahead);
    int64_t row[2] = {-1, -1};
    unsigned there = 0;
    uint32_t to = smem_addr(ring);
    const uint32_t ring_end = to + 2 * A * G::kUnit;
    auto copy = [&](const char *pool, const float *scales, uint32_t unit) {
        auto row_to = [&](int i) { return unit + (lane_to ^ (uint32_t)(pd_swizzle<G::kRow>(i * kRpl, 0) * 16)) + (uint32_t)(i * 512); };
        if (wide && there == kAll) {
#pragma unroll
            for (int half = 0; half < S / 16; half++) {
                const char *src = pool + row[half] * G::kRow;
#pragma unroll
                for (int i = 0; i < 16 / kRpl; i++)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(row_to(half * (16 / kRpl) + i)), "l"(src + i * 512) : "memory");
            }
            if constexpr (kBytes)
                if (lane < S / 4)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(unit + S * G::kRow + lane * 16),
                                 "l"(scales + (lane < 4 ? row[0] : row[1]) + lane % 4 * 4) : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < kRowsCopied; i++) {
                const int rr = i * kRpl + lane / kLpr;
                const bool has = (there >> rr) & 1;
                const int64_t from = whole ? row[i >= 16 / kRpl] + rr % 16 : __shfl_sync(0xffffffffu, row[0], rr);
                pd_copy16(row_to(i), has ? pool - lane * 16 + from * G::kRow + lane % kLpr * 16 : pool, has);
            }
            if constexpr (kBytes) {
                const bool has = (there >> lane) & 1;
                if (lane < S) pd_copy4(unit + S * G::kRow + lane * 4, scales + (!has ? 0 : whole ? (lane < 16 ? row[0] : row[1]) + lane % 16 : row[0]), has);
            }
        }
    };
    auto copy_keys = [&]() {
        if (ahead < k1) {
            const int j = place_of(ahead), p = paged_div(&v, j), last = whole ? j + (lane & 15) : j;
            int64_t mine = -1;
            if (j < n) {
                if (next_id < 0 || next_id >= v.pages) bad |= kPagedBadPage;
                else mine = (int64_t)next_id * page_rows + (head_row + j - p * v.page);
            }
            there = __ballot_sync(0xffffffffu, mine >= 0 && last < n) & kAll;
            row[0] = mine;
            if (whole) row[0] = __shfl_sync(0xffffffffu, mine, 0), row[1] = __shfl_sync(0xffffffffu, mine, S - 16);
            next_id = id_of(ahead + W);
            copy(keys, v.scales, to);
            if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + G::kUnit - 16), "r"(there) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto copy_values = [&]() {
        if (ahead < k1) copy(values, kBytes ? v.scales + (int64_t)v.pages * v.kvheads * v.page : nullptr, to + G::kUnit);
        asm volatile("cp.async.commit_group;" ::: "memory");
        ahead += W;
        to += 2 * G::kUnit;
        if (to == ring_end) to -= 2 * A * G::kUnit;
    };
#pragma unroll 1
    for (int i = 0; i < A; i++) copy_keys(), copy_values();

    // ---- the queries as fragments, two heads a warp
#pragma unroll
    for (int i = 0; i < 8 / W; i++) {
        constexpr int E = DIM / 32;
        const int head = warp + i * W, d = lane * E;
        // Part p is rows 8 (p % 2) + head of operand p / 2; BF16's third goes below the second: only first parts meet in the
        // sums that truncate noticeably.
        auto place = [&](int p, int ks, int ft, int fh) {
            return &reinterpret_cast<uint32_t *>(&qf[p / 2][ks][head * 4 + ft])[2 * fh + ((p % 2) ^ (!kBytes && p > 1))];
        };
        float x[E];
#pragma unroll
        for (int c = 0; c < E; c++) x[c] = 0.f;
        if (head < a.group) {
            const float *src = a.q + (long long)(a.row0 + r) * a.q_stride + ((int64_t)h * a.group + head) * DIM + d;
            if constexpr (E == 4) {
                const float4 f = *reinterpret_cast<const float4 *>(src);
                x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
            } else {
                const float2 f = *reinterpret_cast<const float2 *>(src);
                x[0] = f.x, x[1] = f.y;
            }
        }
        if constexpr (kBytes) {
            // The row as integers up to 127 x 65536, each three signed bytes: 65536 a + 256 b + c, off by at most half of
            // 2^-23 of the row's largest element.
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
            // The integers enter the scores times 2^-24, so that neither they times a row's scale nor this leaves FP32's
            // range before the two meet.
            if (lane == 0) qs[head] = finite ? (a.scale2 * m) * (0x1p24f / kMost) : __uint_as_float(0x7fc00000u);
            uint32_t w[3] = {0, 0, 0};
#pragma unroll
            for (int c = 0; c < E; c++) {
                int y = any ? __float2int_rn(x[c] * lift * up) : 0;
                const int lo = (int)(signed char)y;
                y = (y - lo) >> 8;
                const int mid = (int)(signed char)y;
                y = (y - mid) >> 8;
                w[0] |= (uint32_t)(y & 0xff) << (8 * c);
                w[1] |= (uint32_t)(mid & 0xff) << (8 * c);
                w[2] |= (uint32_t)(lo & 0xff) << (8 * c);
            }
            // Dims 4n .. 4n + 3 of a 16-dim piece: k-step n / 2 of the piece's two, half n % 2.
            const int ks = d / 64 * 2 + d % 16 / 8, ft = d % 64 / 16, fh = d % 8 / 4;
#pragma unroll
            for (int p = 0; p < 3; p++) {
                if constexpr (E == 4) *place(p, ks, ft, fh) = w[p];
                else reinterpret_cast<uint16_t *>(place(p, ks, ft, fh))[d % 4 / 2] = (uint16_t)w[p];
            }
            *place(3, ks, ft, fh) = 0u;
        } else {
            if (lane == 0) qs[head] = a.scale2;
#pragma unroll
            for (int c = 0; c < E; c += 2) {
                uint32_t w[3];
                split_pair<kPagedBf16>(x[c], x[c + 1], w);
                const int dd = d + c, ks = dd / 32 * 2 + dd % 8 / 4, ft = dd % 32 / 8, fh = dd % 4 / 2;
#pragma unroll
                for (int p = 0; p < 3; p++) *place(p, ks, ft, fh) = w[p];
                *place(3, ks, ft, fh) = 0u;
            }
        }
    }
    __syncthreads();

    // ---- the steps. Lane (g, t) has the scores of query head g: x[i] of place 8 (i / 2) + 2t + i % 2
    float o[DV][4], m = -INFINITY, l = 0.f, ref = 0.f;  // ref: m, 0 before the first
    int v_exp = -100;                                   // byte rows: weights times scales count in units of 2^(v_exp - 12)
    float v_up = power_of_two(kPdWeightTop + 100);
    const float sc = qs[g];
#pragma unroll
    for (int j = 0; j < DV; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[j][c] = 0.f;
    auto rescale = [&](float keep) {
#pragma unroll
        for (int j = 0; j < DV; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[j][c] *= keep;
    };
    const bool long_sum = S / 16 * (k1 - k0) > kPdChain * W;  // steps of the tensor cores are 16 rows
    // Where a lane's pieces of K rows g, g + 8, ..., and of V rows 2t, 2t + 1, 8 + 2t, 9 + 2t, ..., lie in a unit.
    const unsigned char *unit = ring;
    const int k_at = g * G::kRow + pd_swizzle<G::kRow>(g, t) * 16;
    const int v_at = 2 * t * G::kRow + pd_swizzle<G::kRow>(2 * t, g * (DV * ES) / 16) * 16 + g * (DV * ES) % 16;
    auto value_at = [&](int odd, int row8, int piece) {  // row 2t + odd + 8 row8, the piece-th 16 bytes of the lane's stretch
        return unit + G::kUnit + ((v_at ^ (odd * (pd_swizzle<G::kRow>(1, 0) * 16)) ^ (piece * 16)) + odd * G::kRow + row8 * 8 * G::kRow);
    };
    for (int k = k0 + warp; k < k1; k += W) {
        asm volatile("cp.async.wait_group %0;" ::"n"(2 * A - 1) : "memory");
        __syncwarp();
        const unsigned has = *reinterpret_cast<const unsigned *>(unit + G::kUnit - 16);
        float x[S / 4];
        {
            int ci[kBytes ? 2 : 1][S / 8][4] = {};
            float cf[S / 8][4] = {};
            uint4 kr[S / 8];
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                if (ks % 2 == 0)
#pragma unroll
                    for (int gr = 0; gr < S / 8; gr++)
                        kr[gr] = *reinterpret_cast<const uint4 *>(unit + (k_at ^ (ks / 2 * 64)) + gr * 8 * G::kRow);
#pragma unroll
                for (int p = 1; p >= 0; p--) {
                    const uint4 f = qf[p][ks][lane];
#pragma unroll
                    for (int gr = 0; gr < S / 8; gr++) {
                        const uint32_t b0 = ks % 2 ? kr[gr].z : kr[gr].x, b1 = ks % 2 ? kr[gr].w : kr[gr].y;
                        if constexpr (kBytes) mma_s8(ci[p][gr], f, b0, b1);
                        else mma_bf16(cf[gr], f.x, f.y, f.z, f.w, b0, b1);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < S / 4; i++) {
                const int gr = i >> 1, c = i & 1;
                if constexpr (kBytes)  // each sum is below 2^21, the lower two together below 2^30
                    x[i] = fmaf((float)ci[0][gr][c], 0x1p-8f, (float)(ci[0][gr][2 + c] * 256 + ci[1][gr][c]) * 0x1p-24f);
                else x[i] = cf[gr][c] + cf[gr][2 + c];
            }
        }
        if constexpr (kBytes) {
            const float *scales = reinterpret_cast<const float *>(unit + S * G::kRow) + 2 * t;
#pragma unroll
            for (int gr = 0; gr < S / 8; gr++) {
                const float2 y = *reinterpret_cast<const float2 *>(scales + 8 * gr);
                x[2 * gr] *= y.x, x[2 * gr + 1] *= y.y;
            }
        }
#pragma unroll
        for (int i = 0; i < S / 4; i++) x[i] *= sc;
        if (has != kAll)
#pragma unroll
            for (int i = 0; i < S / 4; i++)
                if (!((has >> ((i >> 1) * 8 + 2 * t + (i & 1))) & 1)) x[i] = -INFINITY;
        __syncwarp();  // every lane has read the unit before it is copied into again
        copy_keys();

        // ---- weights. The reference moves rarely: when the maximum has passed it by 2^3.
        auto most_of = [](const float (&y)[S / 4]) {
            float z = y[0];
#pragma unroll
            for (int i = 1; i < S / 4; i++) z = fmaxf(z, y[i]);
            return z;
        };
        float top = most_of(x);
        if (__any_sync(0xffffffffu, top > m + kPdSlack)) {
            top = quad_max(top);
            float keep = 1.f;
            if (top > m + kPdSlack) {
                keep = ex2(m - top);
                l *= keep;
                if constexpr (kBytes) {  // what came before is that much less
                    const int was = v_exp;
                    v_exp = max(-100, v_exp - (int)fminf(top - m, 1000.f));
                    v_up = power_of_two(kPdWeightTop - v_exp);
                    keep = ex2((m - top) + (float)(was - v_exp));
                }
                m = ref = top;
            }
            rescale(keep);
        }
        float w[S / 4];
#pragma unroll
        for (int i = 0; i < S / 4; i++) {
            w[i] = ex2(x[i] - ref);
            l += w[i];
        }

        // ---- O += P V
        asm volatile("cp.async.wait_group %0;" ::"n"(2 * A - 1) : "memory");
        __syncwarp();
        if constexpr (kBytes) {  // (rows that are not there have scale 0)
            const float *scales = reinterpret_cast<const float *>(unit + G::kUnit + S * G::kRow) + 2 * t;
#pragma unroll
            for (int gr = 0; gr < S / 8; gr++) {
                const float2 y = *reinterpret_cast<const float2 *>(scales + 8 * gr);
                w[2 * gr] *= y.x, w[2 * gr + 1] *= y.y;
            }
            const float most = most_of(w);
            if (__any_sync(0xffffffffu, most * v_up > kPsMost)) {
                const float all = quad_max(most);
                float keep = 1.f;
                if (all * v_up > kPsMost) {
                    const int was = v_exp;
                    v_exp = exponent_of(all) + 1;
                    v_up = power_of_two(kPdWeightTop - v_exp);
                    keep = was - v_exp < -126 ? 0.f : power_of_two(was - v_exp);
                }
                rescale(keep);
            }
#pragma unroll
            for (int i = 0; i < S / 4; i++) w[i] *= v_up;
        }
        uint32_t pa[S / 8][P];
#pragma unroll
        for (int i = 0; i < S / 8; i++) split_pair<KIND>(w[2 * i], w[2 * i + 1], pa[i]);
        auto pv = [&](int j, int q, uint32_t b0, uint32_t b1, auto apart) {  // rows 16 q .. 16 q + 15
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            float(&acc)[4] = decltype(apart)::value ? sum : o[j];
            if constexpr (kBytes) mma_f16(acc, pa[2 * q][0], pa[2 * q][1], pa[2 * q + 1][0], pa[2 * q + 1][1], b0, b1);
            else {
                mma_bf16(acc, 0u, pa[2 * q][P - 1], 0u, pa[2 * q + 1][P - 1], b0, b1);
                mma_bf16(acc, pa[2 * q][0], pa[2 * q][1], pa[2 * q + 1][0], pa[2 * q + 1][1], b0, b1);
            }
            if constexpr (decltype(apart)::value)
#pragma unroll
                for (int i = 0; i < 4; i++) o[j][i] += sum[i];
        };
        auto add_values = [&](auto apart) {
            uint4 vr[4];
#pragma unroll
            for (int q = 0; q < S / 16; q++)
#pragma unroll
            for (int c = 0; c < VW; c++) {
                if (c % 4 == 0)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const unsigned char *p = value_at(i & 1, 2 * q + (i >> 1), c / 4);
                        if constexpr (VW == 2) {
                            const uint2 y = *reinterpret_cast<const uint2 *>(p);
                            vr[i] = make_uint4(y.x, y.y, 0, 0);
                        } else {
                            vr[i] = *reinterpret_cast<const uint4 *>(p);
                        }
                    }
                uint32_t y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = word(vr[i], c % 4);
                if constexpr (kBytes) {
                    const uint32_t lo0 = __byte_perm(y[0], y[1], 0x5140) ^ 0x80808080u, hi0 = __byte_perm(y[0], y[1], 0x7362) ^ 0x80808080u;
                    const uint32_t lo1 = __byte_perm(y[2], y[3], 0x5140) ^ 0x80808080u, hi1 = __byte_perm(y[2], y[3], 0x7362) ^ 0x80808080u;
                    pv(4 * c, q, codes_f16(lo0, 0x4140), codes_f16(lo1, 0x4140), apart);
                    pv(4 * c + 1, q, codes_f16(lo0, 0x4342), codes_f16(lo1, 0x4342), apart);
                    pv(4 * c + 2, q, codes_f16(hi0, 0x4140), codes_f16(hi1, 0x4140), apart);
                    pv(4 * c + 3, q, codes_f16(hi0, 0x4342), codes_f16(hi1, 0x4342), apart);
                } else {
                    pv(2 * c, q, __byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410), apart);
                    pv(2 * c + 1, q, __byte_perm(y[0], y[1], 0x7632), __byte_perm(y[2], y[3], 0x7632), apart);
                }
            }
        };
        if (long_sum) add_values(std::true_type{});
        else add_values(std::false_type{});
        __syncwarp();
        copy_values();
        unit = unit == ring + 2 * (A - 1) * G::kUnit ? ring : unit + 2 * G::kUnit;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // no copy is left in flight, and the ring's memory is free for the outputs
    if (C > 1) cluster.barrier_arrive();

    // ---- the warps' states: lane (g, t) holds dims [2 t DV, (2 t + 2) DV) of head g
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) wml[warp][g] = make_float2(m, l);
    const float unscale = kBytes ? power_of_two(v_exp - kPdWeightTop) : 1.f;
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int j = 0; j < DV; j += 4) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = unscale * (o[j + i][c] + o[j + i][2 + c]);
            wo[warp][g][pd_piece<DIM>(g, ((2 * t + c) * DV + j) / 4)] = make_float4(y[0], y[1], y[2], y[3]);
        }
    __syncthreads();
    auto store = [&](int head, int d4, float4 y, float sum) {
        const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);  // no page had rows: zeros
        reinterpret_cast<float4 *>(out)[head * (DIM / 4) + d4] = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
    };
    auto fold = [](float4 &y, float &sum, const float4 &x, float2 ml, float top) {
        const float f = pd_factor(ml, top);
        sum = fmaf(ml.y, f, sum);
        y = make_float4(fmaf(x.x, f, y.x), fmaf(x.y, f, y.y), fmaf(x.z, f, y.z), fmaf(x.w, f, y.w));
    };
    if (C > 1) cluster.barrier_wait();  // every CTA's ring is free
    const int items = a.group * (DIM / 4), share = (items + C - 1) / C;  // pieces of the outputs, and of a CTA's to fold
    for (int i = tid; i < items; i += T) {
        const int head = i / (DIM / 4), d4 = i % (DIM / 4);
        float top = -INFINITY, sum = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; w++) top = fmaxf(top, wml[w][head].x);
#pragma unroll
        for (int w = 0; w < W; w++) fold(y, sum, wo[w][head][pd_piece<DIM>(head, d4)], wml[w][head], top);
        if (C == 1) store(head, d4, y, sum);
        else {
            const int to = i / share;
            cluster.map_shared_rank(parts, to)[part * share + i % share] = y;
            if (d4 == 0)
                for (int c = 0; c < C; c++) cluster.map_shared_rank(&parts_ml[part][0], c)[head] = make_float2(top, sum);
        }
    }
    if (C > 1) {
        cluster.sync();
        const int i = part * share + tid;  // share <= 8 DIM / 4 / 2 <= T
        if (tid < share && i < items) {
            const int head = i / (DIM / 4);
            float top = -INFINITY, sum = 0.f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = 0; c < C; c++) top = fmaxf(top, parts_ml[c][head].x);
            for (int c = 0; c < C; c++) fold(y, sum, parts[c * share + tid], parts_ml[c][head], top);
            store(head, i % (DIM / 4), y, sum);
        }
    }
    if (bad) paged_report(a.status, bad);
}

}  // namespace tcm
