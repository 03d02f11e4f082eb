// Attention over few pages of a paged K/V cache: the pages' bounds, the choice of each query's pages, and the attention
// over what was chosen (paged_chosen.cuh).
//
// The choice leaves each query row and KV head a table that names the chosen pages in order, and the number of rows that
// they hold. The query's own page is the last of them and the only one that may be partly filled, so all those rows are
// visible.
#include "paged_host.cuh"
#include "paged_chosen.cuh"
#include <float.h>
#include <math.h>

namespace tcm {
namespace {

// ---------------------------------------------------------------- bounds
// Memory bound: the page's keys are read once. A thread holds eight elements of a row, the CTA's threads DIM / 8 a row;
// what they find meets over the lanes of a warp that hold the same elements, then over the warps. 8 sequences of 9,000 to
// 16,384 BF16 rows of 2 KV heads, pages of 128: 15 us, of which their 52 MB take 8; one page of bytes 7.
constexpr int kBoundThreads = 128;

template <int KIND, int DIM>
__global__ void __launch_bounds__(kBoundThreads) paged_bounds_kernel(PagedView v, uint16_t *bounds, int *status) {
    constexpr int T = DIM / 8, R = kBoundThreads / T, W = kBoundThreads / 32;  // threads a row, rows at a time, warps
    __shared__ float ends[W][2][DIM];
    const int tid = threadIdx.x, h = blockIdx.y, s = blockIdx.z, d = (tid % T) * 8;
    pdl_trigger();
    pdl_wait();
    PagedExtent e;
    int bad = paged_extent(&v, s, &e);
    const int from = e.length - e.count > 0 ? e.length - e.count : 0;
    if (e.count && e.length)
        for (int p = paged_div(&v, from) + blockIdx.x; p <= paged_div(&v, e.length - 1); p += gridDim.x) {
            const int id = v.table[(int64_t)s * v.table_stride + p], rows = min(v.page, e.length - p * v.page);
            const int64_t base = paged_row(&v, id, 0, 0, h);
            if (base < 0) {
                bad |= kPagedBadPage;
                continue;
            }
            float low[8], high[8];
#pragma unroll
            for (int i = 0; i < 8; i++) low[i] = INFINITY, high[i] = -INFINITY;
#pragma unroll 4
            for (int j = tid / T; j < rows; j += R) {
                const int64_t at = (base + j) * DIM + d;
                if constexpr (KIND == kPagedBf16) {
                    const uint4 w = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(v.keys) + at));
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float x = bf16_lo(word(w, i)), y = bf16_hi(word(w, i));
                        low[2 * i] = fminf(low[2 * i], x), high[2 * i] = fmaxf(high[2 * i], x);
                        low[2 * i + 1] = fminf(low[2 * i + 1], y), high[2 * i + 1] = fmaxf(high[2 * i + 1], y);
                    }
                } else {
                    const uint2 w = __ldcg(reinterpret_cast<const uint2 *>(static_cast<const int8_t *>(v.keys) + at));
                    const float scale = __ldcg(v.scales + base + j);
#pragma unroll
                    for (int i = 0; i < 8; i++) {  // the product of a code and a scale lies between its two roundings
                        const float code = (float)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i % 4)));
                        low[i] = fminf(low[i], __fmul_rd(code, scale)), high[i] = fmaxf(high[i], __fmul_ru(code, scale));
                    }
                }
            }
#pragma unroll
            for (int o = T; o < 32; o <<= 1)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    low[i] = fminf(low[i], __shfl_xor_sync(0xffffffffu, low[i], o));
                    high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], o));
                }
            if (tid % 32 < T)
#pragma unroll
                for (int i = 0; i < 8; i++) ends[tid / 32][0][d + i] = low[i], ends[tid / 32][1][d + i] = high[i];
            __syncthreads();
            for (int i = tid; i < 2 * DIM; i += kBoundThreads) {
                const int side = i / DIM;
                float x = ends[0][side][i % DIM];
                for (int w = 1; w < W; w++) x = side ? fmaxf(x, ends[w][1][i % DIM]) : fminf(x, ends[w][0][i % DIM]);
                // To BF16, towards its side: away from zero where bits are lost on that side of it.
                uint32_t u = __float_as_uint(x);
                if ((u & 0xffffu) && (u >> 31) != (uint32_t)side) u += 0x10000u;
                bounds[((int64_t)id * v.kvheads + h) * 2 * DIM + i] = (uint16_t)(u >> 16);
            }
            __syncthreads();
        }
    if (tid == 0) paged_report(status, bad);
}

// ---------------------------------------------------------------- the choice of pages
// A score is a product of 2 DIM elements, [q-, q+] . [low, high], so scores of 16 pages and a KV head's query heads are
// one tile of mma.sync, whose bounds go from memory to the operand as they are. The queries enter as two BF16 parts, so
// these scores are only near the exact ones, and no nearer than `slack` below; the few pages for which that leaves open
// whether they belong are summed again in 64 bits. On the CUDA cores in 64 bits alone the scores of 512 rows over 512
// pages of 2 KV heads took 239 us, of one row 60; now 49 and 17.
//
// What bounds it: few CTAs, each a chain. 16 rows over 1024 pages of 2 KV heads: 7 us for the bounds (an SM's share of
// 512 KB), 7 for extents, fragments, counts, cut, 64-bit sums and the table. Rows at a time share the bounds' loads and take
// 5 us more for each after the first.
constexpr int kChoicePages = 16384, kChoiceBins = 256, kChoiceFew = 1024;

struct PagedChoiceArgs {
    PagedView v;
    const float *q;
    long long q_stride;
    const uint16_t *bounds;
    int group, blocks, first, recent;
    int row0, rows;       // the slab
    int pages;            // scores that a row has room for
    int *lengths, *table;  // the slab's: rows chosen, -1 for no row of the batch; [rows][kvheads][blocks]
    int *selected;        // [rows][kvheads][blocks] of all rows, or null
    int *status;
};

// Sequences of more pages than a CTA holds scores of are left out, as bad extents are.
__device__ __forceinline__ int choice_extent(const PagedView &v, int s, PagedExtent *e) {
    int bad = paged_extent(&v, s, e);
    if ((int64_t)e->length > (int64_t)kChoicePages * v.page) {
        e->start = e->count = e->length = 0;
        bad = kPagedBadExtent;
    }
    return bad;
}
// Floats in the order of unsigned numbers, NaN below all.
__device__ __forceinline__ uint32_t choice_key(float x) {
    const uint32_t u = __float_as_uint(x);
    return x != x ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float choice_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// A BF16 number by its bits as a 64-bit one 2^-896 times as large: zero and subnormal numbers need no case of their own.
__device__ __forceinline__ double choice_widen(uint32_t u) {
    return __hiloint2double((int)(((u & 0x7fffu) << 13) | ((u & 0x8000u) << 16)), 0);
}

// R rows of one KV head at a time: two where there are many, by CTAs of 128 threads, four of which have an SM, as most of a
// row's time is waiting. (160 rows over 128 pages of 8 KV heads, and 512 over 512 of 2, whole calls: 131 and 248 us; four
// rows by 256 threads 138 and 248, by 128 144 and 274; two rows by 256 139 and 254.)
template <int R> constexpr int kChoiceThreads = R == 1 ? 512 : 128;
template <int DIM> constexpr int kChoiceRow = 2 * (2 * DIM / 16) * 32;  // fragments of a row: [part][k-step][lane]
constexpr size_t choice_smem(int dim, int r, long long pages) {
    return (size_t)r * (dim == 64 ? kChoiceRow<64> : kChoiceRow<128>) * 8 + (size_t)pages * (8 + 4 * r);
}

template <int T, typename V, typename F> __device__ __forceinline__ V block_fold(V x, V *shared, F f) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
    __syncthreads();
    x = shared[0];
    for (int w = 1; w < T / 32; w++) x = f(x, shared[w]);
    return x;
}

template <int DIM, int R>
__global__ void __launch_bounds__(kChoiceThreads<R>, R == 1 ? 1 : 4) paged_choice_kernel(const __grid_constant__ PagedChoiceArgs a) {
    constexpr int T = kChoiceThreads<R>, W = T / 32, P = DIM / 32;  // threads, warps, stretches of 32 elements
    extern __shared__ __align__(16) unsigned char choice_smem_bytes[];
    uint2(*frag)[2][4 * P][32] = reinterpret_cast<uint2(*)[2][4 * P][32]>(choice_smem_bytes);  // [row][part][k-step][lane]
    double *exact = reinterpret_cast<double *>(choice_smem_bytes + R * kChoiceRow<DIM> * 8);   // of the pages left open
    float *near = reinterpret_cast<float *>(exact + a.pages);                                  // [row][page]
    __shared__ double fold[W];
    __shared__ unsigned bins[4][kChoiceBins];
    __shared__ uint32_t ends[R][2], reach[R];  // of a row's scores: least and largest key; largest bound's bits
    __shared__ float weight[R];                // the queries' sum of magnitudes, of the largest head
    __shared__ int2 sums[W];
    __shared__ int found[R], sure, open_count, open_pages[kChoiceFew], cut_bin, cut_left, cut_count;
    const PagedView &v = a.v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, h = blockIdx.x;
    const int tile0 = blockIdx.y * R, tile_rows = min(R, a.rows - tile0);  // in the slab
    if (tid < R) found[tid] = 0x7fffffff;
    pdl_trigger();
    pdl_wait();
    __syncthreads();
    PagedExtent e;
    for (int s = tid; s < v.sequences; s += T) {
        const int bad = choice_extent(v, s, &e);
        if (bad && !blockIdx.x && !(a.row0 + blockIdx.y)) paged_report(a.status, bad);
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int r = a.row0 + tile0 + i;
            if (i < tile_rows && r >= e.start && r < e.start + e.count) atomicMin(&found[i], s);
        }
    }
    __syncthreads();
    for (int i0 = 0, i1; i0 < tile_rows; i0 = i1) {  // rows of one sequence
        const int s = found[i0];
        for (i1 = i0 + 1; i1 < tile_rows && found[i1] == s; i1++) {}
        const bool live = s < v.sequences;
        if (live) choice_extent(v, s, &e);
        const int at0 = live ? e.length - e.count + (a.row0 + tile0 + i0 - e.start) : 0;  // the first row's place
        if (h == 0)
            for (int i = i0 + tid; i < i1; i += T) {
                const int at = at0 + i - i0, own = at < 0 ? -1 : paged_div(&v, at);
                a.lengths[tile0 + i] = !live ? -1 : at < 0 ? 0 : (min(own + 1, a.blocks) - 1) * v.page + at - own * v.page + 1;
            }
        if (!live) continue;
        const int *ids = v.table + (int64_t)s * v.table_stride;
        const int last = at0 + i1 - i0 - 1, top = last < 0 ? -1 : paged_div(&v, last);
        const int lo = a.first, want = a.blocks - a.first - a.recent, most_hi = top + 1 - a.recent;
        if (top >= a.blocks && want) {
            // ---- the queries as fragments, a warp a row: element d0 .. d0 + 3 of head n is one lane's in a k-step. They
            // are scaled together to a largest magnitude in [1, 2), so that no score leaves FP32's range.
            for (int i = i0 + warp; i < i1; i += W) {
                float4 q[8];
                float big = 0.f, sum = 0.f;
#pragma unroll
                for (int n = 0; n < 8; n++) {
                    q[n] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (n < a.group && lane < DIM / 4)
                        q[n] = reinterpret_cast<const float4 *>(a.q + (long long)(a.row0 + tile0 + i) * a.q_stride +
                                                                ((int64_t)h * a.group + n) * DIM)[lane];
                    big = fmaxf(big, fmaxf(fmaxf(fabsf(q[n].x), fabsf(q[n].y)), fmaxf(fabsf(q[n].z), fabsf(q[n].w))));
                }
                big = warp_max(big);
                const int lift = big > 0.f && big < INFINITY ? 127 - (int)(__float_as_uint(big) >> 23) : 0;
                // In two steps, each a power of two inside FP32's range.
                const float up0 = power_of_two(lift / 2), up1 = power_of_two(lift - lift / 2);
#pragma unroll
                for (int n = 0; n < 8; n++) {
                    q[n] = make_float4(q[n].x * up0 * up1, q[n].y * up0 * up1, q[n].z * up0 * up1, q[n].w * up0 * up1);
                    const float head = warp_sum(fabsf(q[n].x) + fabsf(q[n].y) + fabsf(q[n].z) + fabsf(q[n].w));
                    sum = head > sum || head != head ? head : sum;
                }
                if (lane == 0) weight[i] = sum, reach[i] = 0, ends[i][0] = 0xffffffffu, ends[i][1] = 0;
                if (lane < DIM / 4) {
                    const int d0 = 4 * lane, ks = d0 / 32 * 2 + d0 % 8 / 4;
#pragma unroll
                    for (int n = 0; n < 8; n++) {
                        const float y[4] = {q[n].x, q[n].y, q[n].z, q[n].w};
#pragma unroll
                        for (int side = 0; side < 2; side++) {
                            float z[4];
#pragma unroll
                            for (int c = 0; c < 4; c++) z[c] = side ? fmaxf(y[c], 0.f) : fminf(y[c], 0.f);
                            const uint2 large = make_uint2(pack_bf16(z[0], z[1]), pack_bf16(z[2], z[3]));
                            const uint2 small = make_uint2(pack_bf16(z[0] - bf16_lo(large.x), z[1] - bf16_hi(large.x)),
                                                           pack_bf16(z[2] - bf16_lo(large.y), z[3] - bf16_hi(large.y)));
                            const int to = n * 4 + d0 % 32 / 8;
                            frag[i][0][side * 2 * P + ks][to] = large;
                            frag[i][1][side * 2 * P + ks][to] = small;
                        }
                    }
                }
            }
            __syncthreads();

            // ---- scores, 16 pages a warp at a time: lane (g, t) has pages g and g + 8, every fourth piece of eight elements
            const int step = W * 16;
            int p0 = lo + warp * 16;
            auto id_of = [&](int p) { return p < most_hi ? ids[p] : -1; };
            int id_a = id_of(p0 + g), id_b = id_of(p0 + g + 8);
            uint32_t widest = 0;  // pairs of magnitudes
            for (; p0 < most_hi; p0 += step) {
                const bool there_a = id_a >= 0 && id_a < v.pages, there_b = id_b >= 0 && id_b < v.pages;
                const uint4 *ba = reinterpret_cast<const uint4 *>(a.bounds + ((int64_t)(there_a ? id_a : 0) * v.kvheads + h) * 2 * DIM);
                const uint4 *bb = reinterpret_cast<const uint4 *>(a.bounds + ((int64_t)(there_b ? id_b : 0) * v.kvheads + h) * 2 * DIM);
                uint4 xa[2 * P], xb[2 * P];  // low, then high
#pragma unroll
                for (int k = 0; k < 2 * P; k++) {
                    xa[k] = xb[k] = make_uint4(0, 0, 0, 0);
                    if (there_a) xa[k] = __ldcg(ba + k * 4 + t);
                    if (there_b) xb[k] = __ldcg(bb + k * 4 + t);
                }
                id_a = id_of(p0 + step + g), id_b = id_of(p0 + step + g + 8);
#pragma unroll
                for (int k = 0; k < 2 * P; k++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        widest = __vmaxu2(widest, __vmaxu2(word(xa[k], c) & 0x7fff7fffu, word(xb[k], c) & 0x7fff7fffu));
                for (int i = i0; i < i1; i++) {
                    float c[4][4];  // four sums, so that no more than eight truncating steps follow one another
#pragma unroll
                    for (int n = 0; n < 4; n++)
#pragma unroll
                        for (int j = 0; j < 4; j++) c[n][j] = 0.f;
#pragma unroll
                    for (int part = 1; part >= 0; part--)
#pragma unroll
                        for (int k = 0; k < 4 * P; k++) {
                            const uint2 f = frag[i][part][k][lane];
                            if (k % 2) mma_bf16(c[k % 4], xa[k / 2].z, xb[k / 2].z, xa[k / 2].w, xb[k / 2].w, f.x, f.y);
                            else mma_bf16(c[k % 4], xa[k / 2].x, xb[k / 2].x, xa[k / 2].y, xb[k / 2].y, f.x, f.y);
                        }
                    float best[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) {  // page g, page g + 8: the largest of the heads
                        const float x = (c[0][2 * j] + c[1][2 * j]) + (c[2][2 * j] + c[3][2 * j]);
                        const float y = (c[0][2 * j + 1] + c[1][2 * j + 1]) + (c[2][2 * j + 1] + c[3][2 * j + 1]);
                        best[j] = quad_max(fmaxf(2 * t < a.group ? x : -INFINITY, 2 * t + 1 < a.group ? y : -INFINITY));
                    }
                    if (t < 2) {
                        const int p = p0 + g + 8 * t, at = at0 + i - i0, hi = at < 0 ? 0 : paged_div(&v, at) + 1 - a.recent;
                        const float x = t ? (there_b ? best[1] : -INFINITY) : (there_a ? best[0] : -INFINITY);
                        if (p < hi) near[(int64_t)i * a.pages + p] = x;
                    }
                }
            }
            widest = max(widest & 0xffffu, widest >> 16);
            widest = __reduce_max_sync(0xffffffffu, widest);
            if (lane == 0) atomicMax(&reach[i0], widest);
            __syncthreads();
        }
        for (int i = i0; i < i1; i++) {
            const int at = at0 + i - i0, own = at < 0 ? -1 : paged_div(&v, at), n = own + 1, count = min(n, a.blocks);
            int *table = a.table + ((int64_t)(tile0 + i) * v.kvheads + h) * a.blocks;
            int *selected = a.selected ? a.selected + ((int64_t)(a.row0 + tile0 + i) * v.kvheads + h) * a.blocks : nullptr;
            if (selected)
                for (int k = count + tid; k < a.blocks; k += T) selected[k] = -1;
            if (n <= a.blocks) {
                for (int k = tid; k < n; k += T) {
                    table[k] = ids[k];
                    if (selected) selected[k] = k;
                }
                continue;
            }
            const int hi = n - a.recent;
            const float *score = near + (int64_t)i * a.pages;
            float above = INFINITY, below = -INFINITY;  // pages with scores above are taken, pages below are not, those between are open
            double cut = INFINITY;                      // of which those with an exact score above it are taken, and `ties` at it
            int ties = 0;
            bool all_open = false;
            if (want) {
                // ---- a score that `want` pages reach and no more pass: bins over the keys' range, then over the bin it lies in
                for (int k = tid; k < 4 * kChoiceBins; k += T) bins[k / kChoiceBins][k % kChoiceBins] = 0;
                if (tid == 0) sure = open_count = 0;
                uint32_t least = 0xffffffffu, most = 0;
                for (int p = lo + tid; p < hi; p += T) {
                    const uint32_t key = choice_key(score[p]);
                    least = min(least, key), most = max(most, key);
                }
                least = __reduce_min_sync(0xffffffffu, least), most = __reduce_max_sync(0xffffffffu, most);
                if (lane == 0) atomicMin(&ends[i][0], least), atomicMax(&ends[i][1], most);
                __syncthreads();
                uint32_t base = ends[i][0], width = ends[i][1] - base;  // keys base .. base + width
                int left = want, shift = max(0, 32 - __clz(width) - 8);
                for (int pass = 0;; pass++) {
                    for (int p = lo + tid; p < hi; p += T) {
                        const uint32_t key = choice_key(score[p]) - base;
                        if (key <= width) atomicAdd(&bins[pass][key >> shift], 1u);
                    }
                    __syncthreads();
                    // Every warp finds the bin, eight bins a lane from the top.
                    unsigned c[8], mine = 0;
#pragma unroll
                    for (int k = 0; k < 8; k++) mine += c[k] = bins[pass][kChoiceBins - 1 - 8 * lane - k];
                    unsigned upto = mine;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned y = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += y;
                    }
                    const int holder = __ffs(__ballot_sync(0xffffffffu, upto >= (unsigned)left)) - 1;
                    unsigned passed = upto - mine;
                    int bin = 0;
                    unsigned in_bin = 0;
#pragma unroll
                    for (int k = 7; k >= 0; k--) {  // the first bin at which `left` are reached
                        unsigned upto_k = passed;
#pragma unroll
                        for (int m = 0; m <= k; m++) upto_k += c[m];
                        if (upto_k >= (unsigned)left) bin = kChoiceBins - 1 - 8 * lane - k, in_bin = c[k], mine = upto_k - c[k];
                    }
                    bin = __shfl_sync(0xffffffffu, bin, holder);
                    in_bin = __shfl_sync(0xffffffffu, in_bin, holder);
                    left -= (int)__shfl_sync(0xffffffffu, mine, holder);
                    base += (uint32_t)bin << shift;
                    if (shift == 0 || in_bin == (unsigned)left) break;
                    width = (1u << shift) - 1u;
                    shift = max(0, shift - 8);
                }
                // ---- what is near it. A score is off by less than 2^-16 of the sum of its terms' sizes: 2^-18 by the
                // queries' parts, and at most 8 x 17 x 2^-24 in each of the four sums, whose steps may truncate every
                // addend at 2^-24 of the largest. Twice that, as both scores of a pair are off, and 1 / 64 for this
                // arithmetic; below 2^-100 numbers that BF16 or FP32 holds no more are in the way.
                const float slack = 2.f * 0x1.04p-16f * (weight[i] * __uint_as_float(reach[i0] << 16)) + 0x1p-100f;
                const float edge = choice_value(base);
                above = edge + slack, below = edge - slack;
                if (!(slack < INFINITY)) above = INFINITY, below = -INFINITY;
                int passed = 0;
                for (int p = lo + tid; p < hi; p += T) {
                    const float x = score[p];
                    if (x > above) passed++;
                    else if (!(x < below)) {
                        const int k = atomicAdd(&open_count, 1);
                        if (k < kChoiceFew) open_pages[k] = p;
                    }
                }
                passed = __reduce_add_sync(0xffffffffu, passed);
                if (lane == 0 && passed) atomicAdd(&sure, passed);
                __syncthreads();
                const int open = open_count;
                left = want - sure;
                all_open = open == left;
                if (!all_open) {
                    // ---- exact scores of the open pages, a warp a page
                    const bool listed = open <= kChoiceFew;
                    const int from = listed ? 0 : lo, to = listed ? open : hi;
                    for (int k = from + warp; k < to; k += W) {
                        const int p = listed ? open_pages[k] : k;
                        if (!listed && (score[p] > above || score[p] < below)) {
                            if (lane == 0) exact[p] = __longlong_as_double(0x7ff8000000000000ll);
                            continue;
                        }
                        const int id = ids[p];
                        const bool there = id >= 0 && id < v.pages;
                        const uint32_t *b = reinterpret_cast<const uint32_t *>(a.bounds + ((int64_t)(there ? id : 0) * v.kvheads + h) * 2 * DIM);
                        double low[P], high[P], best = -INFINITY;
#pragma unroll
                        for (int c = 0; c < P; c++) {
                            const uint32_t l = __ldcg(b + (lane * P + c) / 2), u = __ldcg(b + DIM / 2 + (lane * P + c) / 2);
                            low[c] = choice_widen(c % 2 ? l >> 16 : l & 0xffffu), high[c] = choice_widen(c % 2 ? u >> 16 : u & 0xffffu);
                        }
                        const float *q = a.q + (long long)(a.row0 + tile0 + i) * a.q_stride + (int64_t)h * a.group * DIM + lane * P;
                        for (int m = 0; m < a.group; m++) {
                            double x = 0.0;
#pragma unroll
                            for (int c = 0; c < P; c++) {
                                const double y = (double)q[m * DIM + c] * 0x1p895;  // products of FP32 and BF16 are exact
                                x = fma(y, y < 0.0 ? low[c] : high[c], x);
                            }
#pragma unroll
                            for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                            best = fmax(best, x);
                        }
                        // Finite, so that differences are numbers.
                        if (lane == 0) exact[p] = there && best >= -1e300 ? fmin(best, 1e300) : -1e300;
                    }
                    __syncthreads();
                    if (listed) {  // by rank; the few that are taken are marked
                        bool in[kChoiceFew / T];
#pragma unroll
                        for (int c = 0; c < kChoiceFew / T; c++) {
                            const int k = tid + c * T;
                            in[c] = false;
                            if (k >= open) continue;
                            const int p = open_pages[k];
                            const double x = exact[p];
                            int rank = 0;
                            for (int m = 0; m < open; m++) {
                                const double y = exact[open_pages[m]];
                                rank += y > x || (y == x && open_pages[m] < p);
                            }
                            in[c] = rank < left;
                        }
                        __syncthreads();
#pragma unroll
                        for (int c = 0; c < kChoiceFew / T; c++)
                            if (tid + c * T < open) exact[open_pages[tid + c * T]] = in[c] ? 1e301 : -1e301;
                        cut = 1e300;
                        __syncthreads();
                    } else {  // by bins over the range of the scores that may still be the cut, then over the bin that holds it
                        double down = INFINITY, up = -INFINITY;
                        for (int p = lo + tid; p < hi; p += T) down = fmin(down, exact[p]), up = fmax(up, exact[p]);
                        down = block_fold<T>(down, fold, [](double x, double y) { return fmin(x, y); });
                        up = block_fold<T>(up, fold, [](double x, double y) { return fmax(x, y); });
                        while (down < up) {
                            const double scale = (kChoiceBins - 0.001) / (up - down);
                            auto bin_of = [&](double x) {  // 0 for `down`, the last for `up`, and not falling
                                return scale < 1e300 ? (int)((x - down) * scale) : x > down ? kChoiceBins - 1 : 0;
                            };
                            for (int k = tid; k < kChoiceBins; k += T) bins[0][k] = 0;
                            __syncthreads();
                            for (int p = lo + tid; p < hi; p += T)
                                if (exact[p] >= down && exact[p] <= up) atomicAdd(&bins[0][bin_of(exact[p])], 1u);
                            __syncthreads();
                            if (tid == 0) {
                                int k = kChoiceBins - 1, passed = 0;
                                while (passed + (int)bins[0][k] < left) passed += (int)bins[0][k--];
                                cut_bin = k, cut_left = left - passed, cut_count = (int)bins[0][k];
                            }
                            __syncthreads();
                            const int bin = cut_bin;
                            left = cut_left;
                            double next_down = INFINITY, next_up = -INFINITY;
                            for (int p = lo + tid; p < hi; p += T)
                                if (exact[p] >= down && exact[p] <= up && bin_of(exact[p]) == bin)
                                    next_down = fmin(next_down, exact[p]), next_up = fmax(next_up, exact[p]);
                            down = block_fold<T>(next_down, fold, [](double x, double y) { return fmin(x, y); });
                            up = block_fold<T>(next_up, fold, [](double x, double y) { return fmax(x, y); });
                            if (left == cut_count) up = down, left = 0x7fffffff;  // all of the bin
                            __syncthreads();
                        }
                        cut = down, ties = left;
                    }
                }
            }

            // ---- the chosen pages in ascending order: each thread has a stretch of pages
            const int stretch = (n + T - 1) / T, from = min(n, tid * stretch), to = min(n, from + stretch);
            auto kind = [&](int p) {  // 2 taken, 1 at the cut
                if (p < lo || p >= hi) return 2;
                if (!want || score[p] < below) return 0;
                if (all_open || score[p] > above) return 2;
                return exact[p] > cut ? 2 : exact[p] == cut ? 1 : 0;
            };
            int2 mine = make_int2(0, 0);
            for (int p = from; p < to; p++) {
                const int k = kind(p);
                mine.x += k == 2, mine.y += k == 1;
            }
            int2 upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto.x, o), y = __shfl_up_sync(0xffffffffu, upto.y, o);
                if (lane >= o) upto.x += x, upto.y += y;
            }
            if (lane == 31) sums[warp] = upto;
            __syncthreads();
            int taken = upto.x - mine.x, level = upto.y - mine.y;
            for (int w = 0; w < warp; w++) taken += sums[w].x, level += sums[w].y;
            int k = taken + min(level, ties);
            for (int p = from; p < to; p++) {
                const int what = kind(p);
                if (what == 2 || (what == 1 && level < ties)) {
                    table[k] = ids[p];
                    if (selected) selected[k] = p;
                    k++;
                }
                level += what == 1;
            }
            __syncthreads();  // the next row has the bins, the list and the exact scores
        }
    }
}

template <int DIM, int R> void choice_launch(const PagedChoiceArgs &a) {
    static PerDeviceOnce once;
    once.run([] {
        const size_t most = choice_smem(DIM, R, kChoicePages);
        TCM_CUDA(cudaFuncSetAttribute(paged_choice_kernel<DIM, R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)(most < 208 * 1024 ? most : 208 * 1024)));
    });
    launch(paged_choice_kernel<DIM, R>, dim3(a.v.kvheads, (a.rows + R - 1) / R), dim3(kChoiceThreads<R>), choice_smem(DIM, R, a.pages),
           stream(), true, a);
}

// CTAs an item: as many as run at once for all items while a warp has two steps, eight at most; and so that no warp sums
// more than kPdChain steps of 16 rows in the tensor cores, which needs no sums of its own for each.
template <int KIND, int DIM> void chosen_launch(const PagedChosenArgs &a, int rows, long long most_rows) {
    constexpr size_t smem = PsGeo<KIND, DIM>::kSmem;
    static PerDeviceOnce once;
    once.run([] {
        TCM_CUDA(cudaFuncSetAttribute(paged_chosen_kernel<KIND, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        TCM_CUDA(cudaFuncSetAttribute(paged_chosen_kernel<KIND, DIM>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    });
    const long long items = (long long)rows * a.v.kvheads;
    const long long steps = (most_rows + 15) / 16;
    const long long fit = kPsCtas * sm_count() / items, worth = steps / (PsGeo<KIND, DIM>::kStep / 8 * kPsWarps), need = (steps + kPdChain * kPsWarps - 1) / (kPdChain * kPsWarps);
    long long c = fit < worth ? fit : worth;
    c = c > 8 ? 8 : c;
    c = c < need ? need : c;
    c = c < 1 ? 1 : c > kPsCluster ? kPsCluster : c;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)c, a.v.kvheads, rows);
    cfg.blockDim = dim3(kPsThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream();
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)c, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    TCM_CUDA(cudaLaunchKernelEx(&cfg, paged_chosen_kernel<KIND, DIM>, a));
}

}  // namespace
}  // namespace tcm

using namespace tcm;

extern "C" {

int gpu_paged_bounds(const TcmPagedCache *cache, const TcmPagedBatch *batch, uint16_t *bounds, int *status) {
    const char *call = "gpu_paged_bounds";
    PagedView view;
    if (open_view(call, cache, batch, status, &view)) return -1;
    if (nothing(view)) return 0;
    if (!bounds || !aligned16(bounds)) return refuse(call, "bounds are 16-byte aligned device memory");
    const dim3 grid(blocks_of((long long)view.max_new + 2 * view.page - 2, view.page), view.kvheads, view.sequences);
#define CALL(K, D) launch(paged_bounds_kernel<K, D>, grid, dim3(kBoundThreads), 0, stream(), true, view, bounds, status)
    PAGED_DISPATCH(view, CALL);
#undef CALL
    return 0;
}

int gpu_paged_sparse_attention(TcmGpu *gpu, float *out, long long out_stride, const float *q, long long q_stride,
                               const TcmPagedCache *cache, const TcmPagedBatch *batch, const uint16_t *bounds, int qheads,
                               int blocks, int first, int recent, int *selected, int *status) {
    const char *call = "gpu_paged_sparse_attention";
    PagedView view;
    if (!gpu) return refuse(call, "no handle");
    if (open_view(call, cache, batch, status, &view)) return -1;
    if (qheads < 1 || qheads % view.kvheads || qheads / view.kvheads > 8) return refuse(call, "qheads is 1 to 8 times kvheads");
    if (first < 0 || recent < 1 || blocks < 1 || blocks > 8192 || (long long)first + recent > blocks)
        return refuse(call, "blocks is 1 to 8192 and holds the first and recent pages, one recent at least");
    if ((uintptr_t)selected & 3) return refuse(call, "selected is 4-byte aligned");
    if (nothing(view)) return 0;
    if (!bounds || !aligned16(bounds)) return refuse(call, "bounds are 16-byte aligned device memory");
    if (check_rows(call, q, q_stride, qheads, view.dim) || check_rows(call, out, out_stride, qheads, view.dim)) return -1;
    const int group = qheads / view.kvheads;
    // Rows in slabs whose tables stay within 64 MB.
    const long long a_row = (long long)view.kvheads * blocks + 1;
    long long slab = (64ll << 20) / 4 / a_row;
    slab = slab < 4 ? 4 : slab > 65532 ? 65532 : slab / 4 * 4;
    if (slab > view.rows) slab = view.rows;
    float *part;
    float2 *ml;
    unsigned *words;
    paged_scratch(gpu, 2, 0, 0, slab * a_row, &part, &ml, &words);
    const long long most = ((long long)view.max_length + view.page - 1) / view.page;
    const int pages = (int)(most < kChoicePages ? most : kChoicePages);
    // Rows of one sequence share the loads of its bounds, where there are rows enough and their scores leave room for two CTAs an SM.
    const bool pair = view.max_new >= 2 && (long long)view.rows * view.kvheads >= 4ll * sm_count() && choice_smem(view.dim, 2, pages) <= 100 * 1024;
    int *lengths = reinterpret_cast<int *>(words);
    PagedChoiceArgs c = {view, q, q_stride, bounds, group, blocks, first, recent, 0, 0, pages, lengths, lengths + slab, selected, status};
    PagedChosenArgs d = {view, q, out, q_stride, out_stride, group, blocks, 0, lengths, lengths + slab,
                         1.44269504088896340736f / sqrtf((float)view.dim), status};
    const long long held = (long long)blocks * view.page;
    const long long most_rows = held < view.max_length ? held : view.max_length;
    for (long long r = 0; r < view.rows; r += slab) {
        const int rows = (int)(view.rows - r < slab ? view.rows - r : slab);
        c.row0 = (int)r, c.rows = rows;
        if (view.dim == 64) pair ? choice_launch<64, 2>(c) : choice_launch<64, 1>(c);
        else pair ? choice_launch<128, 2>(c) : choice_launch<128, 1>(c);
        d.row0 = (int)r;
#define CALL(K, D) chosen_launch<K, D>(d, rows, most_rows)
        PAGED_DISPATCH(view, CALL);
#undef CALL
    }
    return 0;
}

}  // extern "C"
