// Rotated append: each head's norm and rotation of new rows, written to the paged cache in the same pass.
//
// A row of a projection holds query, key and value heads. A head of DIM elements belongs to DIM / 4 lanes, each with
// two of its rotation's pairs (d, d + R / 2), so that a head is read once, its sum of squares is a reduction over those
// lanes, and the pairs turn in registers. (Elements that do not turn, from R on, are dealt to the other lanes four at a
// time.) Of many rows a CTA has four at a time: their heads share the cosines, and their reductions the exchanges.
//
// A row is read once, queries are written once, keys and values in their stored form. Sums, angles and rotations are
// 64-bit: the choice of pages (paged_sparse.cu) and the codes of a stored row go by values next to borders.
//
// What bounds it: 21,149 rows of 12 query heads and 2 of keys and of values, byte rows, take 78 us, their bytes 48: 160
// instructions a head's row (24 of them FP64, 8 conversions), at 64 % of the issue slots. Without norm and rotation it is
// 51. With eight rows a tile and 24 warps an SM it took 92, without the prefetch 83, at 9 or 10 CTAs an SM, in fewer
// registers, 81 and 86. A single token takes 5 us, of which 3 are its sequence's extent, its page and the row one after another.
#include "paged_host.cuh"
#include "../../include/tcm_seeded.h"
#include <math.h>
#include <string.h>
#include <type_traits>

namespace tcm {
namespace {

constexpr int kTurnTile = 4, kTurnThreads = 128, kTurnCtas = 8;  // rows of a CTA at a time, where there are many; CTAs an SM
constexpr long long kTurnStride = 1 << 27;  // floats: a tile's offsets stay within 32 bits

struct PagedTurnArgs {
    PagedView v;
    const float *q, *k, *values;
    float *q_out;
    long long stride, q_out_stride;
    const float *qnorm, *knorm;
    double eps;
    int qheads, half;  // half: pairs that turn
    int *status;
    double rate[64];  // half turns a place: theta^(-2d/R) / pi
};

// x over the L lanes of a head, of R = 4 rows at once: two exchanges leave every lane with one row's, so that a quarter
// of the warp adds up, and forms the root of, a row each. turn_row says which, turn_of brings a row's value back.
template <int L> __device__ __forceinline__ double turn_sum(const double (&x)[4], int lane) {
    const bool far = lane & (L / 2), odd = lane & (L / 4);
    const double y0 = (far ? x[2] : x[0]) + __shfl_xor_sync(0xffffffffu, far ? x[0] : x[2], L / 2);
    const double y1 = (far ? x[3] : x[1]) + __shfl_xor_sync(0xffffffffu, far ? x[1] : x[3], L / 2);
    double y = (odd ? y1 : y0) + __shfl_xor_sync(0xffffffffu, odd ? y0 : y1, L / 4);
#pragma unroll
    for (int o = L / 8; o; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    return y;
}
template <int L> __device__ __forceinline__ double turn_of(double y, int row, int lane) {
    return __shfl_sync(0xffffffffu, y, (lane & ~(L - 1)) + (row >> 1) * (L / 2) + (row & 1) * (L / 4));
}
template <int L> __device__ __forceinline__ double turn_sum(const double (&x)[1], int) {
    double y = x[0];
#pragma unroll
    for (int o = L / 2; o; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    return y;
}

// Keys and values of a lane's four elements in their stored form, at row `row` of the pool; a row that it cannot hold is zeros.
template <int KIND, int DIM, int L>
__device__ __forceinline__ void turn_store(const PagedView &v, float (&y)[4], bool is_k, int64_t row, int e0, int e1, int lane, int &bad) {
    // The largest magnitude by its bits: a NaN's are above infinity's.
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < 4; c++) most = max(most, __float_as_uint(y[c]) & 0x7fffffffu);
    if constexpr (L == 32) most = __reduce_max_sync(0xffffffffu, most);
    else
#pragma unroll
        for (int o = L / 2; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    float m = __uint_as_float(most);
    if (row < 0) return;
    if (!paged_holds<KIND>(m)) {
        bad |= kPagedNonFinite;
        m = 0.f;
#pragma unroll
        for (int c = 0; c < 4; c++) y[c] = 0.f;
    }
    void *dst = is_k ? v.keys : v.values;
    const int64_t to = row * DIM;
    if constexpr (KIND == kPagedBytes) {
        const float scale = m > 0.f ? __fdiv_rn(m, 127.0f) : 1.0f;
        int8_t code[4];
        paged_codes(y, scale, code);
        *reinterpret_cast<char2 *>(static_cast<int8_t *>(dst) + to + e0) = make_char2(code[0], code[1]);
        *reinterpret_cast<char2 *>(static_cast<int8_t *>(dst) + to + e1) = make_char2(code[2], code[3]);
        if (lane % L == 0) v.scales[(is_k ? 0 : (int64_t)v.pages * v.kvheads * v.page) + row] = scale;
    } else {
        uint16_t *d = static_cast<uint16_t *>(dst) + to;
        *reinterpret_cast<uint32_t *>(d + e0) = (uint32_t)tcm_bf16_rne(y[0]) | ((uint32_t)tcm_bf16_rne(y[1]) << 16);
        *reinterpret_cast<uint32_t *>(d + e1) = (uint32_t)tcm_bf16_rne(y[2]) | ((uint32_t)tcm_bf16_rne(y[3]) << 16);
    }
}

// Single tokens, a CTA each: a warp forms the cosines that it needs while its row is on the way, and waits for no other.
template <int KIND, int DIM>
__global__ void __launch_bounds__(512) paged_turn_kernel(const __grid_constant__ PagedTurnArgs a) {
    constexpr int L = DIM / 4, H = 32 / L, W = 512 / 32;  // lanes a head, heads a warp, warps
    const PagedView &v = a.v;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane / L, pair = 2 * (lane % L), s = blockIdx.y;
    // Where the lane's two pieces of two elements lie in a head.
    const bool turns = pair < a.half;
    const int e0 = turns ? pair : 2 * pair, e1 = turns ? a.half + pair : 2 * pair + 2;
    const int heads = a.qheads + 2 * v.kvheads;
    pdl_trigger();
    pdl_wait();
    PagedExtent e;
    int bad = paged_extent(&v, s, &e);
    for (int first = blockIdx.x; first < e.count; first += gridDim.x) {
        const int place = e.length - e.count + first;
        for (int group = warp; group * H < heads; group += W) {
            const int head = group * H + sub, kv_head = head - a.qheads;
            const bool there = head < heads, is_q = kv_head < 0, is_k = !is_q && kv_head < v.kvheads;
            const bool moves = there && (is_q || is_k);
            const int h = is_k ? kv_head : kv_head - v.kvheads;  // of the pool
            const float *src = is_q ? a.q + head * DIM : (is_k ? a.k : a.values) + h * DIM;
            const float *norm = !moves ? nullptr : is_q ? a.qnorm : a.knorm;
            const bool any_moves = __any_sync(0xffffffffu, moves), any_norm = __any_sync(0xffffffffu, norm != nullptr);
            const bool any_stored = __any_sync(0xffffffffu, there && !is_q);
            float2 x0 = make_float2(0.f, 0.f), x1 = x0;
            if (there) {
                const float *x = src + (long long)(e.start + first) * a.stride;
                x0 = *reinterpret_cast<const float2 *>(x + e0);
                x1 = *reinterpret_cast<const float2 *>(x + e1);
            }
            float y[4] = {x0.x, x0.y, x1.x, x1.y};
            if (any_moves) {
                double2 t0 = make_double2(1.0, 0.0), t1 = t0;
                if (turns) {
                    sincospi((double)place * a.rate[pair], &t0.y, &t0.x);
                    sincospi((double)place * a.rate[pair + 1], &t1.y, &t1.x);
                }
                double z0 = y[0], z1 = y[1], z2 = y[2], z3 = y[3];
                if (any_norm) {
                    const double sum[1] = {z0 * z0 + z1 * z1 + (z2 * z2 + z3 * z3)};
                    const double r = rsqrt(turn_sum<L>(sum, lane) * (1.0 / DIM) + a.eps);
                    if (norm) {
                        const float2 w0 = *reinterpret_cast<const float2 *>(norm + e0), w1 = *reinterpret_cast<const float2 *>(norm + e1);
                        z0 *= r * w0.x, z1 *= r * w0.y, z2 *= r * w1.x, z3 *= r * w1.y;
                    }
                }
                if (turns) {
                    const double u0 = z0, u1 = z1;
                    z0 = u0 * t0.x - z2 * t0.y, z1 = u1 * t1.x - z3 * t1.y;
                    z2 = z2 * t0.x + u0 * t0.y, z3 = z3 * t1.x + u1 * t1.y;
                }
                if (moves) y[0] = (float)z0, y[1] = (float)z1, y[2] = (float)z2, y[3] = (float)z3;
            }
            if (there && is_q) {
                float *dst = a.q_out + (long long)(e.start + first) * a.q_out_stride + head * DIM;
                *reinterpret_cast<float2 *>(dst + e0) = make_float2(y[0], y[1]);
                *reinterpret_cast<float2 *>(dst + e1) = make_float2(y[2], y[3]);
            }
            if (!any_stored) continue;
            int64_t row = -1;
            if (there && !is_q && place >= 0 && (row = paged_slot(&v, s, place, h)) < 0) bad |= kPagedBadPage;
            turn_store<KIND, DIM, L>(v, y, is_k, row, e0, e1, lane, bad);
        }
    }
    paged_report(a.status, bad);
}

// Tiles of four rows. Their cosines, and where their rows are in the pool, are in shared memory; a warp has a group of heads
// of one sort, all four rows of it at a time. Rows behind the tile's last are copies of it that nothing stores.
enum { kTurnQ, kTurnK, kTurnV };
struct TurnTile {
    int rows;
    const float *q, *k, *values;  // the first row's
    float *q_out;
};
template <int KIND, int DIM>
__global__ void __launch_bounds__(kTurnThreads, kTurnCtas) paged_turn_tile_kernel(const __grid_constant__ PagedTurnArgs a) {
    constexpr int T = kTurnThreads, L = DIM / 4, H = 32 / L, W = T / 32;
    __shared__ __align__(16) double2 turn[kTurnTile][DIM / 2];  // cosine, sine
    __shared__ int64_t slot[kTurnTile];                         // of KV head 0; -1: nowhere
    const PagedView &v = a.v;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane / L, pair = 2 * (lane % L), s = blockIdx.y;
    const bool turns = pair < a.half;
    const int e0 = turns ? pair : 2 * pair, e1 = turns ? a.half + pair : 2 * pair + 2;
    const int q_groups = (a.qheads + H - 1) / H, kv_groups = (v.kvheads + H - 1) / H;
    const uint32_t stride = (uint32_t)a.stride, q_out_stride = (uint32_t)a.q_out_stride;  // of at most kTurnStride
    pdl_trigger();
    pdl_wait();
    PagedExtent e;
    int bad = paged_extent(&v, s, &e);
    auto run = [&](auto sort, const TurnTile &tile, int group) {
        constexpr int SORT = decltype(sort)::value;
        const int head = group * H + sub;
        const bool there = head < (SORT == kTurnQ ? a.qheads : v.kvheads);
        const float *src = (SORT == kTurnQ ? tile.q : SORT == kTurnK ? tile.k : tile.values) + (there ? head * DIM : 0);
        const float *norm = SORT == kTurnQ ? a.qnorm : a.knorm;
        double w[4];
        if (SORT != kTurnV && norm) {
            const float2 w0 = *reinterpret_cast<const float2 *>(norm + e0), w1 = *reinterpret_cast<const float2 *>(norm + e1);
            w[0] = w0.x, w[1] = w0.y, w[2] = w1.x, w[3] = w1.y;
        }
        float y[4][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float *x = src + min(i, tile.rows - 1) * stride;
            const float2 x0 = *reinterpret_cast<const float2 *>(x + e0), x1 = *reinterpret_cast<const float2 *>(x + e1);
            y[i][0] = x0.x, y[i][1] = x0.y, y[i][2] = x1.x, y[i][3] = x1.y;
        }
        if (SORT != kTurnV && (norm || a.half)) {
            double root = 1.0;
            if (norm) {
                double sum[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const double z0 = y[i][0], z1 = y[i][1], z2 = y[i][2], z3 = y[i][3];
                    sum[i] = z0 * z0 + z1 * z1 + (z2 * z2 + z3 * z3);
                }
                root = rsqrt(turn_sum<L>(sum, lane) * (1.0 / DIM) + a.eps);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                double z0 = y[i][0], z1 = y[i][1], z2 = y[i][2], z3 = y[i][3];
                if (norm) {
                    const double r = turn_of<L>(root, i, lane);
                    z0 *= r * w[0], z1 *= r * w[1], z2 *= r * w[2], z3 *= r * w[3];
                }
                if (turns) {
                    const double2 t0 = turn[i][pair], t1 = turn[i][pair + 1];
                    const double u0 = z0, u1 = z1;
                    z0 = u0 * t0.x - z2 * t0.y, z1 = u1 * t1.x - z3 * t1.y;
                    z2 = z2 * t0.x + u0 * t0.y, z3 = z3 * t1.x + u1 * t1.y;
                }
                y[i][0] = (float)z0, y[i][1] = (float)z1, y[i][2] = (float)z2, y[i][3] = (float)z3;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (SORT == kTurnQ) {
                if (there && i < tile.rows) {
                    float *dst = tile.q_out + head * DIM + i * q_out_stride;
                    *reinterpret_cast<float2 *>(dst + e0) = make_float2(y[i][0], y[i][1]);
                    *reinterpret_cast<float2 *>(dst + e1) = make_float2(y[i][2], y[i][3]);
                }
            } else {
                const int64_t at = slot[i];
                turn_store<KIND, DIM, L>(v, y[i], SORT == kTurnK, there && at >= 0 ? at + head * v.page : -1, e0, e1, lane, bad);
            }
        }
    };
    for (int first = blockIdx.x * kTurnTile; first < e.count; first += gridDim.x * kTurnTile) {
        const long long row = e.start + first;
        const TurnTile tile = {min(kTurnTile, e.count - first), a.q + row * a.stride, a.k + row * a.stride, a.values + row * a.stride,
                               a.q_out + row * a.q_out_stride};
        const int place = e.length - e.count + first;
        // The rows are on their way to L2 while the cosines are formed.
        for (int i = tid; i < tile.rows * (a.qheads + 2 * v.kvheads) * (DIM / 32); i += T) {
            const int heads = a.qheads + 2 * v.kvheads, unit = i / (DIM / 32), r = unit / heads, head = unit - r * heads, kv = head - a.qheads;
            const float *x = kv < 0 ? tile.q + head * DIM : kv < v.kvheads ? tile.k + kv * DIM : tile.values + (kv - v.kvheads) * DIM;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(x + r * stride + i % (DIM / 32) * 32));
        }
        if (tid < kTurnTile) {
            int64_t at = -1;
            if (tid < tile.rows && place + tid >= 0 && (at = paged_slot(&v, s, place + tid, 0)) < 0) bad |= kPagedBadPage;
            slot[tid] = at;
        }
        for (int i = tid; i < tile.rows * (DIM / 2); i += T) {
            const int r = i / (DIM / 2), d = i % (DIM / 2);
            if (d < a.half) {
                double sn, cs;
                sincospi((double)(place + r) * a.rate[d], &sn, &cs);
                turn[r][d] = make_double2(cs, sn);
            }
        }
        __syncthreads();
        for (int group = warp; group < q_groups + 2 * kv_groups; group += W) {
            if (group < q_groups) run(std::integral_constant<int, kTurnQ>{}, tile, group);
            else if (group < q_groups + kv_groups) run(std::integral_constant<int, kTurnK>{}, tile, group - q_groups);
            else run(std::integral_constant<int, kTurnV>{}, tile, group - q_groups - kv_groups);
        }
        __syncthreads();
    }
    paged_report(a.status, bad);
}

// The table of one rotation, kept for the thread's next call: 64 powers are 5 us.
void rates(double *out, float theta, int rotary) {
    static thread_local double table[64];
    static thread_local float key_theta = 0.f;
    static thread_local int key_rotary = 0;
    if (key_rotary != rotary || key_theta != theta) {
        for (int d = 0; d < rotary / 2; d++)
            table[d] = (double)(powl((long double)theta, -2.0L * d / rotary) / 3.14159265358979323846264338327950288L);
        key_theta = theta;
        key_rotary = rotary;
    }
    memcpy(out, table, sizeof(table));
}

}  // namespace
}  // namespace tcm

using namespace tcm;

extern "C" int gpu_paged_rotate_append(const TcmPagedCache *cache, const TcmPagedBatch *batch, const TcmHeadRotation *turn,
                                       float *q_out, long long q_out_stride, const float *q, const float *k, const float *v,
                                       long long stride, int qheads, int *status) {
    const char *call = "gpu_paged_rotate_append";
    PagedTurnArgs a;
    memset(&a, 0, sizeof(a));
    if (open_view(call, cache, batch, status, &a.v)) return -1;
    if (!turn) return refuse(call, "no rotation");
    if (qheads < 1 || qheads % a.v.kvheads || qheads / a.v.kvheads > 8) return refuse(call, "qheads is 1 to 8 times kvheads");
    if (!(turn->eps >= 0.f) || isinf(turn->eps)) return refuse(call, "eps is finite and not negative");
    if (turn->rotary < 0 || turn->rotary > a.v.dim || turn->rotary % 4) return refuse(call, "rotary is a multiple of 4, at most dim");
    if (turn->rotary && (!(turn->theta > 0.f) || isinf(turn->theta))) return refuse(call, "theta is finite and positive");
    if (((uintptr_t)turn->qnorm | (uintptr_t)turn->knorm) & 7) return refuse(call, "norms are 8-byte aligned");
    if (nothing(a.v)) return 0;
    if (check_rows(call, q, stride, qheads, a.v.dim) || check_rows(call, k, stride, a.v.kvheads, a.v.dim) ||
        check_rows(call, v, stride, a.v.kvheads, a.v.dim) || check_rows(call, q_out, q_out_stride, qheads, a.v.dim))
        return -1;
    if (q_out == q && q_out_stride != stride) return refuse(call, "q_out in the place of q has its stride");
    a.q = q, a.k = k, a.values = v, a.q_out = q_out;
    a.stride = stride, a.q_out_stride = q_out_stride;
    a.qnorm = turn->qnorm, a.knorm = turn->knorm, a.eps = turn->eps;
    a.qheads = qheads, a.half = turn->rotary / 2, a.status = status;
    rates(a.rate, turn->theta, turn->rotary);
    // Tiles of rows only where they leave no SM without work, and sequences have the rows to fill them.
    const bool tiles = a.v.max_new >= 4 && a.v.rows >= 4 * sm_count() && stride <= kTurnStride && q_out_stride <= kTurnStride;
    const dim3 grid(blocks_of(a.v.max_new, tiles ? kTurnTile : 1), a.v.sequences);
#define CALL(K, D)                                                                                        \
    if (tiles) launch(paged_turn_tile_kernel<K, D>, grid, dim3(kTurnThreads), 0, stream(), true, a);      \
    else launch(paged_turn_kernel<K, D>, grid, dim3(512), 0, stream(), true, a)
    PAGED_DISPATCH(a.v, CALL);
#undef CALL
    return 0;
}
