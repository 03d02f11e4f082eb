// Paged K/V cache: append, read back and attention of ragged batches.
//
// The reference's caches are one session's: dense FP32 slabs and the byte-codec
// ring. Here many sequences share one pool of pages (include/gpu.h); rows are
// addressed only through csrc/paged_index.h.
#include "common.cuh"
#include "paged.cuh"
#include "paged_decode.cuh"
#include "paged_chunk.cuh"
#include "kernels.h"
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
                // BF16 rounds from 2^128 - 2^119 on to infinity; 127 times FP32's largest number over 127 is one too.
                if (!__all_sync(0xffffffffu, zero == 0.f && m < (KIND == kPagedBytes ? 0x1.fffffep127f : 0x1.ffp127f))) {
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
                    // A row so small that m / 127 underflows stands for zeros (scale 0, codes 0).
                    // The quotient by a reciprocal is within 5e-5 of the divided one; only where it comes near a
                    // half does the division decide (all of them by division: 26 us instead of 20 for 42,000 rows).
                    // The largest scale, 2^128 / 127, still has a reciprocal.
                    int8_t q[E];
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
int refuse(const char *call, const char *why) {
    fprintf(stderr, "%s: %s\n", call, why);
    return -1;
}
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// The call's descriptors as a view; 0, or -1 with a message.
int open_view(const char *call, const TcmPagedCache *c, const TcmPagedBatch *b, const int *status, PagedView *v) {
    if (!c || !b) return refuse(call, "no cache or no batch");
    if (c->kind != kPagedBf16 && c->kind != kPagedBytes) return refuse(call, "kind is 2 (BF16) or 3 (bytes)");
    if (c->dim != 64 && c->dim != 128) return refuse(call, "dim is 64 or 128");
    if (c->pages < 1 || c->page < 1 || c->page > 65536 || c->kvheads < 1 || c->kvheads > 1024)
        return refuse(call, "pages, page or kvheads out of range");
    if (!c->keys || !c->values || !aligned16(c->keys) || !aligned16(c->values))
        return refuse(call, "keys and values are 16-byte aligned device memory");
    if (c->kind == kPagedBytes && (!c->scales || ((uintptr_t)c->scales & 3))) return refuse(call, "a byte cache has scales");
    if (b->sequences < 0 || b->sequences > 65535 || b->rows < 0 || b->max_new < 0 || b->max_length < 0 ||
        b->max_length > 1 << 30)
        return refuse(call, "sequences, rows, max_new or max_length out of range");
    if (b->sequences && (!b->starts || !b->lengths || !b->table || b->table_stride < 1))
        return refuse(call, "a batch has starts, lengths and a table");
    if (((uintptr_t)b->starts | (uintptr_t)b->lengths | (uintptr_t)b->table) & 3)
        return refuse(call, "starts, lengths and table are 4-byte aligned");
    if ((uintptr_t)status & 3) return refuse(call, "status is 4-byte aligned");
    const int max_new = b->max_new < b->rows ? b->max_new : b->rows;
    // No sequence is longer than its table either.
    const long long held = (long long)b->table_stride * c->page;
    const int max_length = b->max_length < held ? b->max_length : (int)held;
    if ((long long)max_new * c->kvheads > 0x7fffffff / 8) return refuse(call, "too many new rows for one call");
    *v = PagedView{c->kind, c->pages, c->page, c->kvheads, c->dim, c->keys, c->values, c->scales, b->sequences, b->rows,
                   max_new, max_length, b->table_stride, b->starts, b->lengths, b->table, 0, 0};
    paged_divider(v);
    return 0;
}
int check_rows(const char *call, const void *p, long long stride, int heads, int dim) {
    if (!p || !aligned16(p)) return refuse(call, "row buffers are 16-byte aligned device memory");
    if (stride < (long long)heads * dim || stride % 4) return refuse(call, "a row stride is a multiple of 4 and holds a row");
    return 0;
}
// Nothing to do: no sequence, or none that may have a new row.
bool nothing(const PagedView &v) { return !v.sequences || !v.rows || !v.max_new; }

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

unsigned blocks_of(long long items, int a_block) {
    const long long blocks = (items + a_block - 1) / a_block;
    return (unsigned)(blocks < 4096 ? blocks : 4096);
}

#define PAGED_DISPATCH(view, call)                                      \
    do {                                                                \
        if ((view).kind == kPagedBf16) {                                \
            if ((view).dim == 64) { call(kPagedBf16, 64); }             \
            else { call(kPagedBf16, 128); }                             \
        } else {                                                        \
            if ((view).dim == 64) { call(kPagedBytes, 64); }            \
            else { call(kPagedBytes, 128); }                            \
        }                                                               \
    } while (0)

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
