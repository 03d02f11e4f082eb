// Paged K/V cache: append, read back and attention of ragged batches.
//
// The reference's caches are one session's: dense FP32 slabs and the byte-codec
// ring. Here many sequences share one pool of pages (include/gpu.h); rows are
// addressed only through csrc/paged_index.h.
#include "common.cuh"
#include "paged.cuh"
#include "paged_decode.cuh"
#include "paged_chunk.cuh"
#include "paged_host.cuh"
#include "../../include/qwen_b200.h"
#include "../../include/tcm_seeded.h"
#include <math.h>

namespace tcm {
namespace {

constexpr int kRowThreads = 128;

// ---------------------------------------------------------------- append, read back
// Memory bound, and launch bound for single tokens. A warp takes kRowBatch new rows of one KV head
// (a grid row each: no division per row) at a time, K and V of each, so that its loads are in
// flight together. Measured: 42,298 rows of 128 as bytes written in 19 us (21 with one row at a
// time, 21 with four), 204,656 BF16 rows read back in 55 us (314 MB, 89 % of copy bandwidth; 65 with
// four).
constexpr int kRowBatch = 2, kReadBatch = 1;

// Byte codec: scale = max|x| / 127 (1 for a zero row) and code = clamp(roundf(x / scale), +-127),
// the divisions IEEE as in byte_cache.cu, so codes and scales are the ring's bit for bit (but for a row
// whose max|x| / 127 underflows, which the ring refuses: zeros with scale 0 here). The row's
// values are asked for before its page id, which they do not need.
template <int KIND, int DIM>
__global__ void __launch_bounds__(kRowThreads) paged_append_kernel(PagedView v, const float *k, const float *vals,
                                                                   long long stride, int *status) {
    constexpr int E = DIM / 32;
    pdl_trigger();  // the kernel that follows may be set up meanwhile; it waits before it reads anything
    const int lane = threadIdx.x & 31, h = blockIdx.y, s = blockIdx.z;
    PagedExtent e;
    int bad = paged_extent(&v, s, &e);
    const int step = gridDim.x * (kRowThreads / 32) * kRowBatch;
    for (int first = ((blockIdx.x * kRowThreads + threadIdx.x) >> 5) * kRowBatch; first < e.count; first += step) {
        float x[kRowBatch][2][E];
#pragma unroll
        for (int u = 0; u < kRowBatch; u++) {
            const long long at = (long long)(e.start + min(first + u, e.count - 1)) * stride + h * DIM + lane * E;
#pragma unroll
            for (int kind = 0; kind < 2; kind++) {
                const float *src = (kind ? vals : k) + at;
                if constexpr (E == 4) {
                    const float4 t = *reinterpret_cast<const float4 *>(src);
                    x[u][kind][0] = t.x, x[u][kind][1] = t.y, x[u][kind][2] = t.z, x[u][kind][3] = t.w;
                } else {
                    const float2 t = *reinterpret_cast<const float2 *>(src);
                    x[u][kind][0] = t.x, x[u][kind][1] = t.y;
                }
            }
        }
        int64_t row[kRowBatch];
#pragma unroll
        for (int u = 0; u < kRowBatch; u++) {
            const int j = e.length - e.count + first + u;
            row[u] = -1;
            if (first + u < e.count && j >= 0 && (row[u] = paged_slot(&v, s, j, h)) < 0) bad |= kPagedBadPage;
        }
#pragma unroll
        for (int u = 0; u < kRowBatch; u++) {
            if (row[u] < 0) continue;
#pragma unroll
            for (int kind = 0; kind < 2; kind++) {
                float(&y)[E] = x[u][kind];
                float m = 0.f, zero = 0.f;
#pragma unroll
                for (int c = 0; c < E; c++) {
                    zero = fmaf(y[c], 0.f, zero);  // NaN once a value is not finite
                    m = fmaxf(m, fabsf(y[c]));
                }
                if (!__all_sync(0xffffffffu, zero == 0.f && paged_holds<KIND>(m))) {
                    bad |= kPagedNonFinite;
                    m = 0.f;
#pragma unroll
                    for (int c = 0; c < E; c++) y[c] = 0.f;
                }
                void *dst = kind ? v.values : v.keys;
                const int64_t to = row[u] * DIM + lane * E;
                if constexpr (KIND == kPagedBytes) {
                    m = warp_max(m);
                    const float scale = m > 0.f ? __fdiv_rn(m, 127.0f) : 1.0f;
                    int8_t q[E];
                    paged_codes(y, scale, q);
                    if constexpr (E == 4)
                        *reinterpret_cast<char4 *>(static_cast<int8_t *>(dst) + to) = make_char4(q[0], q[1], q[2], q[3]);
                    else
                        *reinterpret_cast<char2 *>(static_cast<int8_t *>(dst) + to) = make_char2(q[0], q[1]);
                    if (lane == 0) v.scales[(int64_t)kind * v.pages * v.kvheads * v.page + row[u]] = scale;
                } else {
                    uint32_t w[E / 2];
#pragma unroll
                    for (int c = 0; c < E; c += 2)
                        w[c / 2] = (uint32_t)tcm_bf16_rne(y[c]) | ((uint32_t)tcm_bf16_rne(y[c + 1]) << 16);
                    uint16_t *d = static_cast<uint16_t *>(dst) + to;
                    if constexpr (E == 4) *reinterpret_cast<uint2 *>(d) = make_uint2(w[0], w[1]);
                    else *reinterpret_cast<uint32_t *>(d) = w[0];
                }
            }
        }
    }
    if (lane == 0) paged_report(status, bad);
}

// DIM / 4 lanes a row.
template <int KIND, int DIM>
__global__ void __launch_bounds__(kRowThreads) paged_read_kernel(PagedView v, float *k, float *vals, long long stride,
                                                                 int *status) {
    constexpr int L = DIM / 4, R = 32 / L;  // lanes a row, rows a warp at a time
    pdl_wait();
    const int lane = threadIdx.x & 31, h = blockIdx.y, s = blockIdx.z, c = (lane % L) * 4;
    PagedExtent e;
    int bad = paged_extent(&v, s, &e);
    const int step = gridDim.x * (kRowThreads / 32) * R * kReadBatch;
    const int64_t half = (int64_t)v.pages * v.kvheads * v.page;
    for (int first = ((blockIdx.x * kRowThreads + threadIdx.x) >> 5) * R * kReadBatch + lane / L; first < e.count; first += step) {
        float4 a[kReadBatch], b[kReadBatch];
        float sk[kReadBatch], sv[kReadBatch];
#pragma unroll
        for (int u = 0; u < kReadBatch; u++) {
            const int i = first + u * R, j = e.length - e.count + i;
            int64_t row = -1;
            if (i < e.count && j >= 0 && (row = paged_slot(&v, s, j, h)) < 0) bad |= kPagedBadPage;
            a[u] = b[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            sk[u] = sv[u] = 1.f;
            if (row >= 0) {
                a[u] = paged_load4<KIND>(v.keys, row * DIM + c);
                b[u] = paged_load4<KIND>(v.values, row * DIM + c);
                if constexpr (KIND == kPagedBytes) sk[u] = v.scales[row], sv[u] = v.scales[half + row];
            }
        }
#pragma unroll
        for (int u = 0; u < kReadBatch; u++) {
            const int i = first + u * R;
            if (i >= e.count) break;
            if constexpr (KIND == kPagedBytes) {
                a[u] = make_float4(a[u].x * sk[u], a[u].y * sk[u], a[u].z * sk[u], a[u].w * sk[u]);
                b[u] = make_float4(b[u].x * sv[u], b[u].y * sv[u], b[u].z * sv[u], b[u].w * sv[u]);
            }
            const long long at = (long long)(e.start + i) * stride + h * DIM + c;
            *reinterpret_cast<float4 *>(k + at) = a[u];
            *reinterpret_cast<float4 *>(vals + at) = b[u];
        }
    }
    paged_report(status, bad);
}

// ---------------------------------------------------------------- host
// Sequences with at most this many query rows a KV head are the decode kernel's, in row tiles of 8, 16
// or 32, those with more the chunk kernel's. Measured with 32 sequences of 4096 rows, 8 KV heads of 128
// (decode kernel, chunk kernel): 32 rows of BF16 183 and 425 us, 64 rows 353 and 428; of bytes 154 and
// 253 us, 64 rows 307 and 254.
int few_rows(int kind) { return kind == kPagedBf16 ? 64 : 32; }

// Most rows of one sequence that the queries of one tile can see.
long long visible_rows(const PagedView &v, int window, int sinks) {
    const long long most = window ? (long long)window + sinks + v.max_new + 32 : v.max_length;
    return most < v.max_length ? most : v.max_length;
}

// Most steps one KV head of one sequence of the decode kernel can have: rows below the length, for each
// of up to 8 row tiles. Below 2^30.
long long decode_steps(const PagedView &v, int few, int group) {
    const long long rows = (long long)(v.max_new < few ? v.max_new : few) * group;
    return ((long long)v.max_length / 16 + 2 + kPdSegmentCost) * ((rows + 7) / 8);
}
template <int KIND, int DIM, int R> void decode_launch_rows(TcmGpu *gpu, PagedDecodeArgs a) {
    constexpr size_t smem = kPdSmem<KIND, DIM, R>;
    static PerDeviceOnce once;
    once.run([] {
        TCM_CUDA(cudaFuncSetAttribute(paged_decode_kernel<KIND, DIM, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    });
    const int ctas = sm_count() * kPdCtas<KIND, DIM, R>;
    paged_scratch(gpu, 0, 2ll * ctas * R, DIM, ctas, &a.part, &a.ml, &a.counters);
    // As many sequences a launch as it counts, and KV heads and sequences with fewer than 2^31 steps in all.
    const PagedView all = a.v;
    const long long steps = decode_steps(all, a.few, a.group);
    const int heads = 0x7fffffff / steps < all.kvheads ? (int)(0x7fffffff / steps) : all.kvheads;
    const long long fit = 0x7fffffff / (steps * heads);
    const int most = fit < kPdSequences ? (int)fit : kPdSequences;
    for (int s = 0; s < all.sequences; s += most)
        for (a.head0 = 0; a.head0 < all.kvheads; a.head0 += heads) {
            a.heads = all.kvheads - a.head0 < heads ? all.kvheads - a.head0 : heads;
            a.v.sequences = all.sequences - s < most ? all.sequences - s : most;
            a.v.starts = all.starts + s;
            a.v.lengths = all.lengths + s;
            a.v.table = all.table + (int64_t)s * all.table_stride;
            launch(paged_decode_kernel<KIND, DIM, R>, dim3(ctas), dim3(kPdThreads), smem, stream(), true, a);
            // The next one follows this launch, whose counters and partials it uses again: it waits for them.
            a.beside = 0;
        }
}
template <int KIND, int DIM> void decode_launch(TcmGpu *gpu, PagedDecodeArgs a) {
    const int rows = (a.v.max_new < a.few ? a.v.max_new : a.few) * a.group;
    if (rows <= 8) decode_launch_rows<KIND, DIM, 8>(gpu, a);
    else if (rows <= 16) decode_launch_rows<KIND, DIM, 16>(gpu, a);
    else decode_launch_rows<KIND, DIM, 32>(gpu, a);
}

// One kernel of the chunks' tiles, then (`few`, unless null) the decode kernel beside its last
// CTAs, and if tiles are split one that joins the parts.
template <int KIND, int DIM> void chunk_launch(TcmGpu *gpu, PagedChunkArgs a, PagedDecodeArgs *few) {
    const PagedView &v = a.v;
    static PerDeviceOnce once;
    once.run([] {
        TCM_CUDA(cudaFuncSetAttribute(paged_chunk_kernel<KIND, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)PcGeo<DIM>::kSmem));
        // The warpgroups' register shares are taken from what the launch allots.
        cudaFuncAttributes attr;
        TCM_CUDA(cudaFuncGetAttributes(&attr, paged_chunk_kernel<KIND, DIM>));
        if (attr.numRegs != kPcRegs) TCM_FATAL("paged attention: built with %d registers, not %d", attr.numRegs, kPcRegs);
    });
    // CTAs for every item that there can be, and for those there probably are with their splits; the device
    // counts them and takes the splits that fit.
    const long long tiles = (visible_rows(v, a.window, a.sinks) + kPcTile - 1) / kPcTile + 1, room = 8ll * sm_count();
    const long long guess = v.kvheads * paged_tile_guess(v.sequences, v.rows, v.max_new, a.group, a.few, kPcRows);
    const long long split = guess * paged_splits(guess, (int)tiles, sm_count(), room, kPcSplitsMax);
    const long long bound = paged_tile_bound(v.sequences, v.rows, v.max_new, a.group, a.few, kPcRows);
    const long long grid = split > v.kvheads * bound ? split : v.kvheads * bound;
    a.sms = sm_count();
    a.slots = tiles < 4 ? 0 : (int)(grid < room ? grid : room);  // at most 160 MB of parts
    unsigned *count;
    paged_scratch(gpu, 1, (long long)a.slots * kPcRows, DIM, 4 * (grid / v.kvheads + 3), &a.part, &a.ml, &count);
    a.plan = reinterpret_cast<int4 *>(count) + 1;
    a.err = a.status ? reinterpret_cast<unsigned *>(a.status) : count;
    launch(paged_chunk_kernel<KIND, DIM>, dim3((unsigned)grid), dim3(kPcThreads), PcGeo<DIM>::kSmem, stream(), true, a);
    if (few) {
        few->beside = 1;
        decode_launch<KIND, DIM>(gpu, *few);
    }
    // Joins: four CTAs an SM at most (two took 2 us longer over 6144 split rows, eight 0.4 us longer where none is split).
    const long long joins = v.kvheads * bound * (kPcRows / (kPcJoinThreads / 32)), most = 4ll * sm_count();
    if (a.slots)
        launch(paged_chunk_join_kernel<DIM>, dim3((unsigned)(joins < most ? joins : most)), dim3(kPcJoinThreads), 0, stream(), true, a);
}

// gpu_paged_attention, and its self-check.
int attention(const char *name, TcmGpu *gpu, float *out, long long out_stride, const float *q, long long q_stride,
              const TcmPagedCache *cache, const TcmPagedBatch *batch, int qheads, int window, int sinks, int *status,
              int starve) {
    PagedView view;
    if (!gpu) return refuse(name, "no handle");
    if (open_view(name, cache, batch, status, &view)) return -1;
    if (qheads < 1 || qheads % view.kvheads || qheads / view.kvheads > 8)
        return refuse(name, "qheads is 1 to 8 times kvheads");
    if (window < 0 || sinks < 0) return refuse(name, "window and sinks are not negative");
    if (nothing(view)) return 0;
    if (check_rows(name, q, q_stride, qheads, view.dim) || check_rows(name, out, out_stride, qheads, view.dim)) return -1;
    const int group = qheads / view.kvheads, few = few_rows(view.kind) / group;
    if (view.max_new > few &&
        view.kvheads * paged_tile_bound(view.sequences, view.rows, view.max_new, group, 0, kPcRows) > 0x7fffffff)
        return refuse(name, "too many rows and sequences for one call");
    const float scale2 = 1.44269504088896340736f / sqrtf((float)view.dim);  // log2(e) / sqrt(dim): base-2 scores
    // A lone sequence that may have more rows than the decode kernel's is the chunk kernel's whatever it
    // has: it nearly always has them, and an empty launch of the other takes 2.6 us of the device.
    const bool lone = view.sequences == 1 && view.max_new > few;
    PagedDecodeArgs d = {view, out, q, out_stride, q_stride, group, window, sinks, 0, 0, few, scale2, nullptr, nullptr,
                         nullptr, status, 0};
    PagedChunkArgs c = {view, out, q, out_stride, q_stride, group, window, sinks, lone ? 0 : few, 0, 0, scale2, nullptr, nullptr,
                        nullptr, status, nullptr, starve};
#define CALL(K, D)                                            \
    if (view.max_new <= few) decode_launch<K, D>(gpu, d);     \
    else chunk_launch<K, D>(gpu, c, lone ? nullptr : &d)
    PAGED_DISPATCH(view, CALL);
#undef CALL
    return 0;
}

}  // namespace

void set_wait_limit_paged(unsigned long long ns) { set_module_wait_limit(ns); }

}  // namespace tcm

using namespace tcm;

extern "C" {

int gpu_paged_append(const TcmPagedCache *cache, const TcmPagedBatch *batch, const float *k, const float *v,
                     long long stride, int *status) {
    PagedView view;
    if (open_view("gpu_paged_append", cache, batch, status, &view)) return -1;
    if (nothing(view)) return 0;
    if (check_rows("gpu_paged_append", k, stride, view.kvheads, view.dim) ||
        check_rows("gpu_paged_append", v, stride, view.kvheads, view.dim))
        return -1;
    const dim3 grid(blocks_of(view.max_new, kRowThreads / 32 * kRowBatch), view.kvheads, view.sequences);
#define CALL(K, D) paged_append_kernel<K, D><<<grid, kRowThreads, 0, stream()>>>(view, k, v, stride, status)
    PAGED_DISPATCH(view, CALL);
#undef CALL
    TCM_CUDA(cudaGetLastError());
    return 0;
}

int gpu_paged_read(const TcmPagedCache *cache, const TcmPagedBatch *batch, float *k, float *v, long long stride,
                   int *status) {
    PagedView view;
    if (open_view("gpu_paged_read", cache, batch, status, &view)) return -1;
    if (nothing(view)) return 0;
    if (check_rows("gpu_paged_read", k, stride, view.kvheads, view.dim) ||
        check_rows("gpu_paged_read", v, stride, view.kvheads, view.dim))
        return -1;
    const dim3 grid(blocks_of(view.max_new, kRowThreads / 32 * (128 / view.dim) * kReadBatch), view.kvheads, view.sequences);
#define CALL(K, D) launch(paged_read_kernel<K, D>, grid, dim3(kRowThreads), 0, stream(), true, view, k, v, stride, status)
    PAGED_DISPATCH(view, CALL);
#undef CALL
    return 0;
}

int gpu_paged_attention(TcmGpu *gpu, float *out, long long out_stride, const float *q, long long q_stride,
                        const TcmPagedCache *cache, const TcmPagedBatch *batch, int qheads, int window, int sinks,
                        int *status) {
    return attention("gpu_paged_attention", gpu, out, out_stride, q, q_stride, cache, batch, qheads, window, sinks, status, 0);
}

int qwen_b200_paged_check(TcmGpu *gpu, float *out, long long out_stride, const float *q, long long q_stride,
                          const TcmPagedCache *cache, const TcmPagedBatch *batch, int qheads, int window, int sinks,
                          int *status, int starve) {
    if (starve < 0 || starve > 2) return refuse("qwen_b200_paged_check", "starve is 0, 1 or 2");
    return attention("qwen_b200_paged_check", gpu, out, out_stride, q, q_stride, cache, batch, qheads, window, sinks, status, starve);
}

}  // extern "C"
