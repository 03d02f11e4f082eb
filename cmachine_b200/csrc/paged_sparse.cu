// Attention over few pages of a paged K/V cache: the pages' bounds, the choice of each query's pages, and the decode
// kernel (paged_decode.cuh) over what was chosen.
//
// The choice leaves each query row a sequence of its own: one new row, a table for every KV head that names the chosen
// pages, and the length that they make. Its own page is the last of them and the only one that may be partly filled, so
// the decode kernel needs no other mask than its own.
#include "paged_host.cuh"
#include "paged_decode.cuh"
#include <float.h>
#include <math.h>

namespace tcm {
namespace {

// ---------------------------------------------------------------- bounds
// Memory bound: the page's keys are read once. A thread holds eight elements of a row, the CTA's threads DIM / 8 a row;
// what they find meets over the lanes of a warp that hold the same elements, then over the warps.
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
constexpr int kChoiceThreads = 256, kChoicePages = 16384, kChoiceBins = 512;

struct PagedChoiceArgs {
    PagedView v;
    const float *q;
    long long q_stride;
    const uint16_t *bounds;
    int group, blocks, first, recent;
    int row0;             // the slab's first row
    int *starts, *lengths, *table;  // the slab's: [rows][2], [rows], [rows][kvheads][blocks]
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

template <typename T, typename F> __device__ __forceinline__ T block_fold(T x, T *shared, F f) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
    __syncthreads();
    x = shared[0];
    for (int w = 1; w < kChoiceThreads / 32; w++) x = f(x, shared[w]);
    return x;
}

// One CTA a query row and KV head. Scores: four lanes a page, each with every fourth piece of eight elements; a bound
// is widened to 64 bits by its bits, as a number 2^-896 times as large (zero and subnormal numbers need no case of
// their own then), and the queries are 2^895 times as large. Products of a BF16 and an FP32 number are exact there.
template <int DIM> __global__ void __launch_bounds__(kChoiceThreads) paged_choice_kernel(const PagedChoiceArgs a) {
    extern __shared__ __align__(16) double score[];  // of the sequence's pages; then the queries [group][DIM]
    __shared__ double fold[kChoiceThreads / 32];
    __shared__ unsigned bins[kChoiceBins];
    __shared__ int2 sums[kChoiceThreads / 32];
    __shared__ int found, cut_bin, cut_left, cut_count;
    const PagedView &v = a.v;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = blockIdx.x, r = a.row0 + blockIdx.y;
    constexpr int T = kChoiceThreads;
    if (tid == 0) found = 0x7fffffff;
    pdl_trigger();
    pdl_wait();
    __syncthreads();
    PagedExtent e;
    for (int s = tid; s < v.sequences; s += T) {
        const int bad = choice_extent(v, s, &e);
        if (bad && !blockIdx.x && !r) paged_report(a.status, bad);
        if (r >= e.start && r < e.start + e.count) atomicMin(&found, s);
    }
    __syncthreads();
    const int s = found;
    const bool live = s < v.sequences;
    if (live) choice_extent(v, s, &e);
    const int at = live ? e.length - e.count + (r - e.start) : -1;
    const int own = at < 0 ? -1 : paged_div(&v, at), n = own + 1, count = min(n, a.blocks);
    if (h == 0 && tid == 0) {
        a.starts[2 * blockIdx.y] = live ? r : 0;
        a.starts[2 * blockIdx.y + 1] = live ? r + 1 : 0;
        a.lengths[blockIdx.y] = at < 0 ? 0 : (count - 1) * v.page + at - own * v.page + 1;
    }
    if (!live) return;
    int *table = a.table + ((int64_t)blockIdx.y * v.kvheads + h) * a.blocks;
    int *selected = a.selected ? a.selected + ((int64_t)r * v.kvheads + h) * a.blocks : nullptr;
    const int *ids = v.table + (int64_t)s * v.table_stride;
    if (selected)
        for (int i = count + tid; i < a.blocks; i += T) selected[i] = -1;
    if (n <= a.blocks) {
        for (int i = tid; i < n; i += T) {
            table[i] = ids[i];
            if (selected) selected[i] = i;
        }
        return;
    }

    // ---- scores of the pages between the first and the recent ones
    const int lo = a.first, hi = n - a.recent, want = a.blocks - a.first - a.recent;
    double cut = INFINITY;  // pages between are taken above it, and the first `ties` of those at it
    int ties = 0;
    if (want) {
        double *q = score + n;
        for (int i = tid; i < a.group * DIM; i += T)
            q[i] = (double)a.q[(long long)r * a.q_stride + (int64_t)h * a.group * DIM + i] * 0x1p895;
        __syncthreads();
        const int t = lane & 3;
        for (int p0 = lo + warp * 8; p0 < hi; p0 += T / 4) {
            const int p = p0 + (lane >> 2), id = p < hi ? ids[p] : -1;
            const bool there = id >= 0 && id < v.pages;
            const uint16_t *b = a.bounds + ((int64_t)(there ? id : 0) * v.kvheads + h) * 2 * DIM;
            double x[8];
#pragma unroll
            for (int g = 0; g < 8; g++) x[g] = 0.0;
#pragma unroll
            for (int piece = t; piece < DIM / 8; piece += 4) {
                const uint4 low4 = __ldcg(reinterpret_cast<const uint4 *>(b + piece * 8));
                const uint4 high4 = __ldcg(reinterpret_cast<const uint4 *>(b + DIM + piece * 8));
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    auto widen = [&](const uint4 &w) {
                        const uint32_t u = i % 2 ? word(w, i / 2) >> 16 : word(w, i / 2) & 0xffffu;
                        return __hiloint2double((int)(((u & 0x7fffu) << 13) | ((u & 0x8000u) << 16)), 0);
                    };
                    const double low = widen(low4), high = widen(high4);
#pragma unroll
                    for (int g = 0; g < 8; g++)
                        if (g < a.group) {
                            const double y = q[g * DIM + piece * 8 + i];
                            x[g] = fma(y, y < 0.0 ? low : high, x[g]);
                        }
                }
            }
            double best = -INFINITY;
#pragma unroll
            for (int g = 0; g < 8; g++)
                if (g < a.group) {
                    x[g] += __shfl_xor_sync(0xffffffffu, x[g], 1);
                    x[g] += __shfl_xor_sync(0xffffffffu, x[g], 2);
                    best = fmax(best, x[g]);
                }
            // Finite, so that differences are numbers.
            if (t == 0 && p < hi) score[p] = there && best >= -1e300 ? fmin(best, 1e300) : -1e300;
        }
        __syncthreads();

        // ---- the cut: bins over the range of the scores that are still open, then over the bin that it falls into
        double least = INFINITY, most = -INFINITY;
        for (int p = lo + tid; p < hi; p += T) least = fmin(least, score[p]), most = fmax(most, score[p]);
        least = block_fold(least, fold, [](double x, double y) { return fmin(x, y); });
        most = block_fold(most, fold, [](double x, double y) { return fmax(x, y); });
        int left = want;
        while (least < most) {
            const double scale = (kChoiceBins - 0.001) / (most - least);
            auto bin_of = [&](double x) {  // 0 for `least`, the last for `most`, and not falling
                return scale < 1e300 ? (int)((x - least) * scale) : x > least ? kChoiceBins - 1 : 0;
            };
            for (int i = tid; i < kChoiceBins; i += T) bins[i] = 0;
            __syncthreads();
            for (int p = lo + tid; p < hi; p += T)
                if (score[p] >= least && score[p] <= most) atomicAdd(&bins[bin_of(score[p])], 1u);
            __syncthreads();
            if (warp == 0) {  // from the top: the bin at which `left` are reached
                int above = 0;
                for (int i = kChoiceBins - 32; i >= 0; i -= 32) {
                    const int c = (int)bins[i + 31 - lane];
                    int upto = c;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int y = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += y;
                    }
                    const unsigned reached = __ballot_sync(0xffffffffu, above + upto >= left);
                    if (reached) {
                        if (lane == __ffs(reached) - 1) cut_bin = i + 31 - lane, cut_left = left - (above + upto - c), cut_count = c;
                        break;
                    }
                    above += __shfl_sync(0xffffffffu, upto, 31);
                }
            }
            __syncthreads();
            const int bin = cut_bin;
            left = cut_left;
            double down = INFINITY, up = -INFINITY;
            for (int p = lo + tid; p < hi; p += T)
                if (score[p] >= least && score[p] <= most && bin_of(score[p]) == bin)
                    down = fmin(down, score[p]), up = fmax(up, score[p]);
            down = block_fold(down, fold, [](double x, double y) { return fmin(x, y); });
            up = block_fold(up, fold, [](double x, double y) { return fmax(x, y); });
            least = down, most = up;
            if (left == cut_count) {  // all of the bin
                most = least;
                left = 0x7fffffff;
            }
            __syncthreads();
        }
        cut = least, ties = left;
    }

    // ---- the chosen pages in ascending order: each thread has a stretch of pages
    const int stretch = (n + T - 1) / T, p0 = min(n, tid * stretch), p1 = min(n, p0 + stretch);
    auto kind = [&](int p) { return p < lo || p >= hi ? 2 : score[p] > cut ? 2 : score[p] == cut ? 1 : 0; };
    int2 mine = make_int2(0, 0);  // taken, and at the cut
    for (int p = p0; p < p1; p++) {
        const int k = want || p < lo || p >= hi ? kind(p) : 0;
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
    int to = taken + min(level, ties);
    for (int p = p0; p < p1; p++) {
        const int k = want || p < lo || p >= hi ? kind(p) : 0;
        if (k == 2 || (k == 1 && level < ties)) {
            table[to] = ids[p];
            if (selected) selected[to] = p;
            to++;
        }
        level += k == 1;
    }
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
    const long long a_row = (long long)view.kvheads * blocks + 3;
    long long slab = (64ll << 20) / 4 / a_row;
    slab = slab < 1 ? 1 : slab > 65535 ? 65535 : slab;
    if (slab > kPdSequences) slab = slab / kPdSequences * kPdSequences;
    if (slab > view.rows) slab = view.rows;
    float *part;
    float2 *ml;
    unsigned *words;
    paged_scratch(gpu, 2, 0, 0, slab * a_row, &part, &ml, &words);
    const long long pages = ((long long)view.max_length + view.page - 1) / view.page;
    const size_t smem = ((size_t)(pages < kChoicePages ? pages : kChoicePages) + (size_t)group * view.dim) * sizeof(double);
    PagedChoiceArgs c = {view, q, q_stride, bounds, group, blocks, first, recent, 0, reinterpret_cast<int *>(words),
                         reinterpret_cast<int *>(words) + 2 * slab, reinterpret_cast<int *>(words) + 3 * slab, selected, status};
    // What was chosen, as a batch: one row a sequence.
    PagedDecodeArgs d = {view, out, q, out_stride, q_stride, group, 0, 0, 0, 0, 1, 1.44269504088896340736f / sqrtf((float)view.dim),
                         nullptr, nullptr, nullptr, status, 0};
    d.v.starts = c.starts, d.v.lengths = c.lengths, d.v.table = c.table;
    d.v.pairs = 1, d.v.table_head = blocks, d.v.table_stride = view.kvheads * blocks;
    d.v.max_new = 1;
    const long long held = (long long)blocks * view.page;
    d.v.max_length = held < view.max_length ? (int)held : view.max_length;
    static PerDeviceOnce once;
    once.run([] {
        const int most = (kChoicePages + 8 * 128) * (int)sizeof(double);
        TCM_CUDA(cudaFuncSetAttribute(paged_choice_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        TCM_CUDA(cudaFuncSetAttribute(paged_choice_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    });
    for (long long r = 0; r < view.rows; r += slab) {
        const int rows = (int)(view.rows - r < slab ? view.rows - r : slab);
        c.row0 = (int)r;
        const dim3 grid(view.kvheads, rows);
        if (view.dim == 64) launch(paged_choice_kernel<64>, grid, dim3(kChoiceThreads), smem, stream(), true, c);
        else launch(paged_choice_kernel<128>, grid, dim3(kChoiceThreads), smem, stream(), true, c);
        d.v.sequences = rows;
        paged_decode_rows(gpu, d);
    }
    return 0;
}

}  // extern "C"
