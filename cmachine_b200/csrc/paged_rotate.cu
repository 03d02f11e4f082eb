// Rotated append: each head's norm and rotation of new rows, written to the paged cache in the same pass.
//
// A row of a projection holds query, key and value heads. A head of DIM elements belongs to DIM / 4 lanes, each with
// two of its rotation's pairs (d, d + R / 2), so that a head is read once, its sum of squares is a reduction over those
// lanes, and the pairs turn in registers. (Elements that do not turn, from R on, are dealt to the other lanes four at a
// time.) The cosines of a row are shared by its heads: the CTA forms those of its rows first, in shared memory.
//
// Memory bound: a row is read once, queries are written once, keys and values in their stored form. Sums, angles and
// rotations are 64-bit: the choice of pages (paged_sparse.cu) and the codes of a stored row go by values next to
// borders, and the FP64 pipe is idle otherwise.
#include "paged_host.cuh"
#include "../../include/tcm_seeded.h"
#include <math.h>
#include <string.h>

namespace tcm {
namespace {

constexpr int kTurnThreads = 256, kTurnRows = 8;  // rows a CTA forms the cosines of together, at most

struct PagedTurnArgs {
    PagedView v;
    const float *q, *k, *values;
    float *q_out;
    long long stride, q_out_stride;
    const float *qnorm, *knorm;
    double eps;
    int qheads, half, tile;  // half: pairs that turn; tile: rows of a CTA at a time
    int *status;
    double rate[64];  // half turns a place: theta^(-2d/R) / pi
};

template <int KIND, int DIM>
__global__ void __launch_bounds__(kTurnThreads) paged_turn_kernel(const __grid_constant__ PagedTurnArgs a) {
    constexpr int L = DIM / 4, H = 32 / L, W = kTurnThreads / 32;  // lanes a head, heads a warp, warps
    __shared__ __align__(16) double2 turn[kTurnRows][DIM / 2];     // cosine, sine
    const PagedView &v = a.v;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane / L, pair = 2 * (lane % L), s = blockIdx.y;
    const unsigned mine = L == 32 ? 0xffffffffu : 0xffffu << (lane & 16);
    // Where the lane's two pieces of two elements lie in a head.
    const bool turns = pair < a.half;
    const int e0 = turns ? pair : 2 * pair, e1 = turns ? a.half + pair : 2 * pair + 2;
    const int heads = a.qheads + 2 * v.kvheads, groups = (heads + H - 1) / H;
    pdl_trigger();
    pdl_wait();
    PagedExtent e;
    int bad = paged_extent(&v, s, &e);
    for (int first = blockIdx.x * a.tile; first < e.count; first += gridDim.x * a.tile) {
        const int rows = min(a.tile, e.count - first), items = rows * groups, place = e.length - e.count + first;
        struct Item {
            float2 x[2];
            int64_t row;  // of the pool, for keys and values
            int head, at;
        };
        auto load = [&](int it) {
            Item r;
            r.at = it / groups;
            r.head = (it - r.at * groups) * H + sub;
            r.row = -1;
            r.x[0] = r.x[1] = make_float2(0.f, 0.f);
            if (it < items && r.head < heads) {
                const bool key = r.head < a.qheads + v.kvheads;
                const float *src = r.head < a.qheads ? a.q + r.head * DIM
                                   : key             ? a.k + (r.head - a.qheads) * DIM
                                                     : a.values + (r.head - a.qheads - v.kvheads) * DIM;
                src += (long long)(e.start + first + r.at) * a.stride;
                r.x[0] = *reinterpret_cast<const float2 *>(src + e0);
                r.x[1] = *reinterpret_cast<const float2 *>(src + e1);
                const int j = place + r.at;
                if (r.head >= a.qheads && j >= 0 &&
                    (r.row = paged_slot(&v, s, j, r.head - a.qheads - (key ? 0 : v.kvheads))) < 0)
                    bad |= kPagedBadPage;
            }
            return r;
        };
        Item next = load(warp);
        for (int i = tid; i < rows * (DIM / 2); i += kTurnThreads) {
            const int r = i / (DIM / 2), d = i % (DIM / 2);
            double sn, cs;
            if (d < a.half) {
                sincospi((double)(place + r) * a.rate[d], &sn, &cs);
                turn[r][d] = make_double2(cs, sn);
            }
        }
        __syncthreads();
        for (int it = warp; it < items; it += W) {
            const Item c = next;
            next = load(it + W);
            const bool there = c.head < heads, is_q = c.head < a.qheads, is_k = !is_q && c.head < a.qheads + v.kvheads;
            float y[4] = {c.x[0].x, c.x[0].y, c.x[1].x, c.x[1].y};
            if (__any_sync(0xffffffffu, there && (is_q || is_k))) {
                double z[4] = {y[0], y[1], y[2], y[3]};
                const float *norm = is_q ? a.qnorm : is_k ? a.knorm : nullptr;
                if (a.qnorm || a.knorm) {
                    double sum = z[0] * z[0] + z[1] * z[1] + (z[2] * z[2] + z[3] * z[3]);
#pragma unroll
                    for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (norm) {
                        const double r = rsqrt(sum * (1.0 / DIM) + a.eps);
                        const float2 w0 = *reinterpret_cast<const float2 *>(norm + e0);
                        const float2 w1 = *reinterpret_cast<const float2 *>(norm + e1);
                        z[0] *= r * w0.x, z[1] *= r * w0.y, z[2] *= r * w1.x, z[3] *= r * w1.y;
                    }
                }
                if (turns && (is_q || is_k)) {
                    const double2 t0 = turn[c.at][pair], t1 = turn[c.at][pair + 1];
                    const double a0 = z[0], a1 = z[1], b0 = z[2], b1 = z[3];
                    z[0] = a0 * t0.x - b0 * t0.y, z[1] = a1 * t1.x - b1 * t1.y;
                    z[2] = b0 * t0.x + a0 * t0.y, z[3] = b1 * t1.x + a1 * t1.y;
                }
                if (is_q || is_k)
#pragma unroll
                    for (int i = 0; i < 4; i++) y[i] = (float)z[i];
            }
            if (there && is_q) {
                float *dst = a.q_out + (long long)(e.start + first + c.at) * a.q_out_stride + c.head * DIM;
                *reinterpret_cast<float2 *>(dst + e0) = make_float2(y[0], y[1]);
                *reinterpret_cast<float2 *>(dst + e1) = make_float2(y[2], y[3]);
            }
            // ---- keys and values in their stored form
            if (!__any_sync(0xffffffffu, c.row >= 0)) continue;
            float m = 0.f, zero = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                zero = fmaf(y[i], 0.f, zero);  // NaN once a value is not finite
                m = fmaxf(m, fabsf(y[i]));
            }
            if ((__ballot_sync(0xffffffffu, zero == 0.f && paged_holds<KIND>(m)) & mine) != mine) {
                if (c.row >= 0) bad |= kPagedNonFinite;
                m = 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = 0.f;
            }
            void *dst = is_k ? v.keys : v.values;
            const int64_t to = c.row * DIM;
            if constexpr (KIND == kPagedBytes) {
#pragma unroll
                for (int o = 1; o < L; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                const float scale = m > 0.f ? __fdiv_rn(m, 127.0f) : 1.0f;
                int8_t code[4];
                paged_codes(y, scale, code);
                if (c.row >= 0) {
                    *reinterpret_cast<char2 *>(static_cast<int8_t *>(dst) + to + e0) = make_char2(code[0], code[1]);
                    *reinterpret_cast<char2 *>(static_cast<int8_t *>(dst) + to + e1) = make_char2(code[2], code[3]);
                    if (lane % L == 0) v.scales[(is_k ? 0 : (int64_t)v.pages * v.kvheads * v.page) + c.row] = scale;
                }
            } else if (c.row >= 0) {
                uint16_t *d = static_cast<uint16_t *>(dst) + to;
                *reinterpret_cast<uint32_t *>(d + e0) = (uint32_t)tcm_bf16_rne(y[0]) | ((uint32_t)tcm_bf16_rne(y[1]) << 16);
                *reinterpret_cast<uint32_t *>(d + e1) = (uint32_t)tcm_bf16_rne(y[2]) | ((uint32_t)tcm_bf16_rne(y[3]) << 16);
            }
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
    // A row a CTA while that leaves SMs free, up to eight where there are many.
    const int each = a.v.rows / (3 * sm_count());
    a.tile = each < 1 ? 1 : each > kTurnRows ? kTurnRows : each;
    const dim3 grid(blocks_of(a.v.max_new, a.tile), a.v.sequences);
#define CALL(K, D) launch(paged_turn_kernel<K, D>, grid, dim3(kTurnThreads), 0, stream(), true, a)
    PAGED_DISPATCH(a.v, CALL);
#undef CALL
    return 0;
}
