// Sampling: one token a row of logits, with temperature, top-k, top-p and min-p, by a given uniform number.
//
// A thread-block cluster has one row. Each of its CTAs has a contiguous slice of it, in shared memory where it fits (the
// row is read from HBM once then, twice otherwise). All three filters keep a prefix of the tokens in descending order of
// their logits (equal ones by id), so what is kept is described by the last token that is, the cut: a logit and an id. The
// row is never sorted:
//   1. one pass finds the largest logit and, for top-k and top-p, counts the tokens in bins of a 128th of the temperature
//      whose borders do not depend on the row: a circle of 8192 bins, of which the cluster adds up the 4096 below the
//      largest logit. Where the row's range passes the circle, or its bins hold too many, a pass over the row's own range
//      counts again;
//   2. the bin of the k-th token is known then; that of top-p's last token is estimated from the counts and the bins'
//      middles;
//   3. one pass adds up the weights above those bins, and lists the few tokens inside them;
//   4. every CTA searches the list for the cut, then finds the id at which the kept weights pass the uniform number's
//      share; the warp that holds this id writes the result.
// Where the estimate was wrong, or the bins hold more than a list (many equal logits), sample_slowly() narrows the range
// bin by bin instead.
//
// Weights exp((l - max) / T) are whole numbers, 2^44 or next to it for the largest: their sums are exact whatever the order,
// so that atomics and the CTAs' shares leave results the same from call to call, and a sum of 2^19 of them stays below 2^64.
//
// What bounds it (rows of 151,936): one row, five barriers of the cluster and the search, 1 to 3 us each (20 us; 11 with
// neither top-k nor top-p). 256 rows with top-p, 138 us, an SM's two CTAs: 40 us of the first pass and 63 of the weights',
// which take 9 FP64 instructions an element at two cycles or more of an SM's quarter, and some 25 others; the other 35 are
// steps 2 and 4. A row's slices are as long as one another, so an SM with two CTAs is waited for by those with one.
#include "common.cuh"
#include "kernels.h"
#include "sample_bins.h"
#include "../../include/gpu.h"
#include <cooperative_groups.h>
#include <float.h>
#include <math.h>
#include <type_traits>
#include <utility>

namespace cg = cooperative_groups;

namespace tcm {
namespace {

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kSampleShifts = 256, kSampleList = 2048, kSlowBins = 1024, kSubBins = 256, kFew = kSampleThreads / 4;
constexpr int kSampleVocab = 1 << 19, kSampleCluster = 16;
constexpr int kSampleOwnSm = 180 * 1024, kSampleHalfSm = 76 * 1024;  // bytes of a slice in shared memory: one CTA an SM, two
typedef unsigned long long u64;

struct SampleArgs {
    int *ids;
    float *logprobs;
    int *kept;
    const float *logits;
    long long stride;
    int vocab, slice;
    const TcmSampling *params;
    const float *uniforms;
    int *status;
};

// What a CTA of the cluster tells the others of its slice.
struct SampleSlice {
    uint32_t most, counted;  // keys of the logits above -infinity: the largest, the least that the first pass counted
    int live, bad;         // logits above -infinity; a NaN or +infinity among them
};
struct SampleSums {
    u64 all, above, kept;  // weights: of the tokens that top-p takes a share of, above its bins, and above all bins and min-p
    int kept_count, listed;
};

struct SampleShared {
    TcmSampling set;             // the row's settings, its uniform number, 1 / T
    float uniform;
    double cold;
    u64 buffer[2][kSampleList];  // own counts, then own list; the cluster's counts, then its list
    SampleSlice slices[kSampleCluster];
    SampleSums sums[kSampleCluster];
    int first[kSampleCluster];       // greedy rows: the lowest id of the largest logit
    float2 ends[kSampleCluster];     // least and largest logit above -infinity, or of the slow search's bin
    u64 part_mass[kSampleCluster];
    double shift[kSampleShifts];     // the row's: see SampleRow
    int part_count[kSampleCluster];
    u64 warp_mass[kSampleWarps], warp_more[kSampleWarps], warp_kept[kSampleWarps];
    int warp_count[kSampleWarps];
    float warp_low[kSampleWarps], warp_high[kSampleWarps];
    u64 whole, before, heavier, everything;  // of the row: see SampleSums; before: kept in CTAs before this one
    u64 list_before, list_kept, list_counted;
    int kept, listed, list_count;
    int bin, above, in_bin;  // of top-k's cut
    float mass_whole;        // what top-p takes its share of, estimated
    int mass_from, mass_to;  // top-p's bins, first and last,
    int list_from, list_to;  // and the tokens above the first, up to the last
    // The search for the cut in the list.
    u64 found, found_mass;
    uint32_t sub_least, sub_most;
    int sub_bin, sub_above, few_count;
    float border[4];
    int list_start[kSampleCluster], list_total;
    u64 slow_mass;
};

__device__ __forceinline__ u64 warp_sum64(u64 x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// p * x, for p of [0, 1), down to a whole number, or up. FP64 would round x first, and a share that falls between two of
// many equal weights be one token off.
__device__ __forceinline__ u64 sample_share(float p, u64 x, bool up) {
    const unsigned bits = __float_as_uint(p), e = bits >> 23;  // p is at least zero
    if (!bits || bits >> 31) return 0;
    const u64 m = (bits & 0x7fffffu) | (e ? 0x800000u : 0);
    const int s = 150 - (int)(e ? e : 1);  // p = m / 2^s, s from 24 to 149
    const u64 high = __umul64hi(m, x), low = m * x;
    const u64 y = s < 64 ? high << (64 - s) | low >> s : s < 128 ? high >> (s - 64) : 0;
    const u64 rest = s < 64 ? low << (64 - s) : s == 64 ? low : s < 128 ? low | high << (128 - s) : low | high;
    return y + (up && rest);
}
// Floats in ascending order as unsigned numbers, and back. Both zeros are one number.
__device__ __forceinline__ uint32_t sample_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sample_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// (2^f - 1) / f for |f| <= 1/2, interpolated at the seven Chebyshev points there: 2^f is off by 2^-33 at most.
__constant__ double kSampleSeries[7] = {0.6931471805599453,    0.24022650922288757,   0.055504108839096185,  0.009618056678524632,
                                        0.0013333502386162978, 0.00015461444698571227, 1.5297323760649362e-05};

constexpr int kSampleDown = 64;  // powers of two below the largest weight, at which nothing is left
struct SampleRow {
    double slope;                       // log2(e) / T
    float lowest;                       // a logit that is kSampleDown to 3 kSampleDown powers of two below the largest
    float unit, origin, step;           // a power of two, the largest logit times that; slope / unit
    uint32_t shift;                     // where in shared memory -top * slope - n is for the n whose bits are zero: n steps of 8 bytes
    // The product is off by 2^-44 of itself, 2^-14 at most as no slope is larger than 2^30 / |top|, at which FP32's next lower
    // number weighs nothing. All weights of the row are off by that one factor, and weight(high) by the same: the product's
    // last bits are cut off so that adding n is exact. A thread writes a number of `table`.
    __device__ SampleRow(float high, double cold, double *table) {
        const double top = high;
        slope = 1.4426950408889634074 * cold;
        if (slope * fabs(top) > 0x1p30) slope = 0x1p30 / fabs(top);
        // Differences, and what they are multiplied by, stay normal numbers of FP32.
        unit = slope > 1e30 ? 0x1p100f : slope < 1e-30 ? 0.25f : 1.f;
        origin = high * unit, step = (float)(slope / (double)unit);
        lowest = fmaxf(__double2float_rd(top - kSampleDown / slope), -FLT_MAX);  // 2^7 powers of two are a step of FP32 at most
        const double product = top * slope;
        if (threadIdx.x < kSampleShifts)
            table[kSampleShifts - 1 - threadIdx.x] = threadIdx.x - __hiloint2double(__double2hiint(product), __double2loint(product) & ~0xff);
        shift = (uint32_t)__cvta_generic_to_shared(table + kSampleShifts - 1) - (__float_as_uint(0x1.8p23f) << 3);
    }
    __device__ float logprob(float l, float high, double cold, u64 whole) const {
        return (float)(((double)l - (double)high) * cold - log((double)whole / (double)weight(high)));
    }
    __device__ u64 weight(float l) const {  // of a logit no larger than the largest
        // The power of two by FP32 arithmetic, and what is left to it, a half and little more at most, in FP64.
        l = fmaxf(l, lowest);
        const int n = __float_as_int(fmaf(fmaf(l, unit, -origin), step, 0x1.8p23f));  // its lower bits; 0 to -193
        double z, less;
        asm volatile("ld.shared.f64 %0, [%1];" : "=d"(less) : "r"(shift + ((unsigned)n << 3)));
        const double f = fma((double)l, slope, less);
        z = kSampleSeries[6];
#pragma unroll
        for (int k = 5; k >= 0; k--) z = fma(z, f, kSampleSeries[k]);
        z = fma(z, f, 1.0);
        z = __hiloint2double(__double2hiint(z) + (n << 20), __double2loint(z));
        return (u64)(__double_as_longlong(z + 0x1.8p8) - __double_as_longlong(0x1.8p8));  // in units of 2^-44
    }
};

// A CTA's slice of the row: `off` elements behind a 16-byte boundary, in shared memory with -infinity around it, or where
// it is in global memory, read again by every pass (from L2, mostly).
template <bool RESIDENT> struct SampleLogits {
    const float *x;  // of the first element's quad
    int off, n;
    __device__ float at(int i) const { return RESIDENT ? x[off + i] : __ldcg(x + off + i); }
    __device__ float4 quad(int q) const {
        if constexpr (RESIDENT) return reinterpret_cast<const float4 *>(x)[q];
        else {
            if (4 * q >= off && 4 * q + 3 < off + n) return __ldcg(reinterpret_cast<const float4 *>(x) + q);
            float l[4];
#pragma unroll
            for (int k = 0; k < 4; k++) l[k] = 4 * q + k >= off && 4 * q + k < off + n ? __ldcg(x + 4 * q + k) : -INFINITY;
            return make_float4(l[0], l[1], l[2], l[3]);
        }
    }
};

// The quads from, from + STEP, ... below `to` of a thread, out of global memory: kRing of them are on the way at a time, as
// HBM and L2 are some 2000 cycles away, into a ring of the thread's own in shared memory or (KEEP) to where the quad stays
// there. (Four ahead in registers left the weights' pass of 256 rows waiting half of its 85 us.) The copies start with
// the constructor; run() calls f(q, quad).
constexpr int kRing = 8, kRingBytes = kRing * kSampleThreads * 16;
template <int STEP, bool KEEP> struct QuadStream {
    const SampleLogits<false> x;
    float4 *const memory;
    int q, ahead, to;
    bool cut_first, cut_last;  // quads that the slice's ends cut
    uint32_t at;               // bytes from the memory's start to quad q
    __device__ QuadStream(const SampleLogits<false> &x_, float4 *memory_, int from, int to_) : x(x_), memory(memory_) {
        const int whole = (x.off + x.n) / 4;
        cut_first = from == 0 && x.off && to_ > 0;
        cut_last = to_ > whole && from <= whole && (whole - from) % STEP == 0 && !(cut_first && whole == 0);
        q = cut_first ? from + STEP : from, to = min(to_, whole), ahead = q, at = 16 * (KEEP ? q : threadIdx.x);
#pragma unroll
        for (int i = 0; i < kRing; i++) copy(KEEP ? at + i * (STEP * 16) : at + i * (kSampleThreads * 16));
    }
    __device__ __forceinline__ void copy(uint32_t to_at) {
        if (ahead < to)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(memory) + to_at),
                         "l"(reinterpret_cast<const float4 *>(x.x) + ahead) : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
        ahead += STEP;
    }
    template <typename F> __device__ __forceinline__ void run(F f) {
        auto cut = [&](int quad) {
            const float4 y = x.quad(quad);
            if (KEEP) memory[quad] = y;
            f(quad, y);
        };
        if (cut_first) cut(0);
        for (; q < to; q += STEP) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
            const float4 y = *reinterpret_cast<const float4 *>(reinterpret_cast<const char *>(memory) + at);
            copy(KEEP ? at + kRing * STEP * 16 : at);
            at = KEEP ? at + STEP * 16 : (at + kSampleThreads * 16) & (kRingBytes - 1);
            f(q, y);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (cut_last) cut((x.off + x.n) / 4);
    }
};
// The same of a slice wherever it is.
template <int STEP, bool RESIDENT, typename F>
__device__ __forceinline__ void each_quad(const SampleLogits<RESIDENT> &x, float4 *ring, int from, int to, F f) {
    if constexpr (RESIDENT)
        for (int q = from; q < to; q += STEP) f(q, x.quad(q));
    else QuadStream<STEP, false>(x, ring, from, to).run(f);
}

// The cut by repeated histograms of the cluster: counts and weights in bins of the range in which it must lie, then of the
// bin that it falls into, until that holds one value. Then who is kept, and the token. All threads of the cluster call it.
template <bool RESIDENT>
__device__ __noinline__ void sample_slowly(const SampleArgs &a, SampleShared &sh, float *slice_memory, int row, float high_all, int live, float min_logit) {
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const TcmSampling p = sh.set;
    const int base = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - base);
    const float *src = a.logits + (long long)row * a.stride + base;
    const int off = (int)((uintptr_t)src >> 2) & 3;
    const SampleLogits<RESIDENT> x = {RESIDENT ? slice_memory : src - off, off, n};
    const SampleRow r(high_all, sh.cold, sh.shift);  // `shift` as it is
    u64 *mass = sh.buffer[0], *all_mass = sh.buffer[1];
    unsigned *count = reinterpret_cast<unsigned *>(mass + kSlowBins), *all_count = reinterpret_cast<unsigned *>(all_mass + kSlowBins);
    static_assert(kSampleList * 8 >= kSlowBins * 12, "the slow search's bins fit the buffers");

    // The cut: tokens above `value` and the first `ties` at it, `tokens` in all, of weight `weight`.
    struct Cut {
        float value;
        int ties, tokens;
        u64 weight;
    };
    // The least prefix of the tokens above `floor` that holds `tokens` of them (by_mass false) or weighs `share` or more.
    // There is one.
    auto find = [&](bool by_mass, int tokens, u64 share, float floor) {
        Cut cut = {0.f, 0, 0, 0};
        float low = fmaxf(-FLT_MAX, floor), high = high_all;
        // Weights end 32 temperatures below the largest; what lies lower is one bin until the cut is known to be there.
        const float reach = (float)((double)high_all - 32.0 * (double)p.temperature);
        float from = low < reach && reach < high ? reach : low;
        // A pass narrows the range a thousandfold, and FP32's spans less than 2^280: 64 are never reached.
        for (int pass = 0;; pass++) {
            const SampleBins bins = sample_bins_over(from, high, kSlowBins);
            auto open = [&](float l) { return l <= high && l >= low && l > floor; };
            __syncthreads();
            for (int i = tid; i < kSlowBins; i += kSampleThreads) mass[i] = 0, count[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kSampleThreads)
                if (const float l = x.at(i); open(l)) {
                    const int b = sample_bin(&bins, l);
                    atomicAdd(&count[b], 1u);
                    atomicAdd(&mass[b], r.weight(l));
                }
            cluster.sync();
            // Each CTA adds up its share of the bins and tells the others.
            const int share_of = kSlowBins / C;
            for (int i = tid; i < share_of; i += kSampleThreads) {
                const int b = rank * share_of + i;
                unsigned c = 0;
                u64 m = 0;
                for (int k = 0; k < C; k++) c += cluster.map_shared_rank(count, k)[b], m += cluster.map_shared_rank(mass, k)[b];
                for (int k = 0; k < C; k++) cluster.map_shared_rank(all_count, k)[b] = c, cluster.map_shared_rank(all_mass, k)[b] = m;
            }
            cluster.sync();
            if (warp == 0) {
                int above = cut.tokens;
                u64 heavier = cut.weight;
                for (int b = 0; b < kSlowBins; b += 32) {
                    int c = (int)all_count[b + lane], upto = c;
                    u64 m = all_mass[b + lane], sum = m;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int y = __shfl_up_sync(0xffffffffu, upto, o);
                        const u64 z = __shfl_up_sync(0xffffffffu, sum, o);
                        if (lane >= o) upto += y, sum += z;
                    }
                    const bool here = by_mass ? c && heavier + sum >= share : above + upto >= tokens;
                    const unsigned reached = __ballot_sync(0xffffffffu, here);
                    if (reached) {
                        if (lane == __ffs(reached) - 1)
                            sh.bin = b + lane, sh.above = above + upto - c, sh.in_bin = c, sh.slow_mass = heavier + sum - m;
                        break;
                    }
                    above += __shfl_sync(0xffffffffu, upto, 31);
                    heavier += __shfl_sync(0xffffffffu, sum, 31);
                }
            }
            __syncthreads();
            const int bin = sh.bin, in_bin = sh.in_bin;
            cut.tokens = sh.above;
            cut.weight = sh.slow_mass;
            float down = INFINITY, up = -INFINITY;
            for (int i = tid; i < n; i += kSampleThreads)
                if (const float l = x.at(i); open(l) && sample_bin(&bins, l) == bin) down = fminf(down, l), up = fmaxf(up, l);
            down = -warp_max(-down), up = warp_max(up);
            if (lane == 0) sh.warp_low[warp] = down, sh.warp_high[warp] = up;
            __syncthreads();
            if (tid < C) {
                for (int w = 0; w < kSampleWarps; w++) down = fminf(down, sh.warp_low[w]), up = fmaxf(up, sh.warp_high[w]);
                cluster.map_shared_rank(sh.ends, tid)[rank] = make_float2(down, up);
            }
            cluster.sync();
            down = INFINITY, up = -INFINITY;
            for (int c = 0; c < C; c++) down = fminf(down, sh.ends[c].x), up = fmaxf(up, sh.ends[c].y);
            low = from = down, high = up;
            if (low == high || pass == 63) {  // one value: how many of its tokens
                const u64 w = r.weight(low);
                int t;
                if (!by_mass) t = tokens - cut.tokens;
                else {
                    const u64 need = share > cut.weight && w ? (share - cut.weight + w - 1) / w : 1;
                    t = need > (u64)in_bin ? in_bin : (int)need;
                }
                cut.value = low, cut.ties = t;
                cut.tokens += t;
                cut.weight += w * (u64)t;
                return cut;
            }
        }
    };

    // ---- top-k, then top-p of what it leaves
    Cut cut = {-INFINITY, 0, live, 0};
    if (p.top_k > 0 && p.top_k < live) cut = find(false, p.top_k, 0, -INFINITY);
    if (p.top_p < 1.f) {
        u64 whole = cut.weight;
        if (cut.value == -INFINITY) {  // of the row
            u64 m = 0;
            for (int i = tid; i < n; i += kSampleThreads) m += r.weight(x.at(i));
            m = warp_sum64(m);
            __syncthreads();
            if (lane == 0) sh.warp_mass[warp] = m;
            __syncthreads();
            if (tid < C) {
                m = 0;
                for (int w = 0; w < kSampleWarps; w++) m += sh.warp_mass[w];
                cluster.map_shared_rank(sh.part_mass, tid)[rank] = m;
            }
            cluster.sync();
            for (int c = 0; c < C; c++) whole += sh.part_mass[c];
        }
        const u64 share = sample_share(p.top_p, whole, true);
        // Inside the ties of top-k's cut, or above them.
        const u64 w = cut.value == -INFINITY ? 0 : r.weight(cut.value), above = cut.weight - w * (u64)cut.ties;
        if (cut.value != -INFINITY && above < share) {
            const u64 need = w ? (share - above + w - 1) / w : 1;
            const int t = need > (u64)cut.ties ? cut.ties : (int)need;
            cut.tokens -= cut.ties - t;
            cut.ties = t;
        } else if (cut.value != -INFINITY && cut.tokens == cut.ties) {  // nothing above them
            cut.tokens = cut.ties = 1;
        } else {
            cut = find(true, 0, share, cut.value);
        }
    }

    // ---- what is kept, by id: tokens above the cut, and the first ties at it; min-p among them
    const int per_warp = (n + kSampleWarps - 1) / kSampleWarps, w0 = min(n, warp * per_warp), w1 = min(n, w0 + per_warp);
    int ties_before = 0;
    if (cut.ties) {
        int t = 0;
        for (int i = w0 + lane; i < w1; i += 32) t += x.at(i) == cut.value;
        t = __reduce_add_sync(0xffffffffu, t);
        cluster.sync();  // the search's sums have been read
        if (lane == 0) sh.warp_count[warp] = t;
        __syncthreads();
        if (tid < C) {
            t = 0;
            for (int w = 0; w < kSampleWarps; w++) t += sh.warp_count[w];
            cluster.map_shared_rank(sh.part_count, tid)[rank] = t;
        }
        for (int w = 0; w < warp; w++) ties_before += sh.warp_count[w];
        cluster.sync();
        for (int c = 0; c < rank; c++) ties_before += sh.part_count[c];
    }
    // Calls f(i, kept, weight) in order of i, 32 lanes at a time; f says whether to stop.
    auto walk = [&](auto f) {
        int level = ties_before;
        for (int i0 = w0; i0 < w1; i0 += 32) {
            const int i = i0 + lane;
            const float l = i < w1 ? x.at(i) : -INFINITY;
            const bool tie = cut.ties && l == cut.value && i < w1;
            const unsigned tied = __ballot_sync(0xffffffffu, tie);
            const bool keep = l > cut.value || (tie && level + __popc(tied & ((1u << lane) - 1u)) < cut.ties);
            level += __popc(tied);
            const bool stays = keep && l >= min_logit;
            if (f(i, stays, stays ? r.weight(l) : 0ull)) break;
        }
    };
    u64 sum = 0;
    int tokens = 0;
    walk([&](int, bool stays, u64 w) {
        sum += w, tokens += stays;
        return false;
    });
    sum = warp_sum64(sum);
    tokens = __reduce_add_sync(0xffffffffu, tokens);
    __syncthreads();
    if (lane == 0) sh.warp_mass[warp] = sum, sh.warp_count[warp] = tokens;
    cluster.sync();
    if (tid < C) {
        u64 m = 0;
        int k = 0;
        for (int w = 0; w < kSampleWarps; w++) m += sh.warp_mass[w], k += sh.warp_count[w];
        cluster.map_shared_rank(sh.part_mass, tid)[rank] = m;
        cluster.map_shared_rank(sh.part_count, tid)[rank] = k;
    }
    cluster.sync();
    u64 whole = 0, before = 0;
    int kept = 0;
    for (int c = 0; c < C; c++) {
        if (c < rank) before += sh.part_mass[c];
        whole += sh.part_mass[c];
        kept += sh.part_count[c];
    }
    const u64 target = sample_share(sh.uniform, whole, false);
    for (int w = 0; w < warp; w++) before += sh.warp_mass[w];
    if (target < before || target >= before + sum) return;  // one warp of the cluster has the token
    walk([&](int i, bool, u64 w) {
        u64 upto = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const unsigned reached = __ballot_sync(0xffffffffu, before + upto > target);
        if (reached && lane == __ffs(reached) - 1) {
            a.ids[row] = base + i;
            if (a.logprobs) a.logprobs[row] = r.logprob(x.at(i), high_all, sh.cold, whole);
            if (a.kept) a.kept[row] = kept;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
        return reached != 0;
    });
}

// The memory of the search for the cut in the list, in the place of the cluster's counts.
struct SampleSearch {
    // A bin's count above its weight's upper bits, and the next 21 and 21 of it, so that native atomics add them up: a loop
    // for 64 bits took 31 us where 400 equal logits met in a bin.
    unsigned top[kSubBins], middle[kSubBins], low[kSubBins];
    u64 few[kFew], few_mass[kFew];
    __device__ unsigned count(int b) const { return top[b] >> 16; }
    __device__ u64 mass(int b) const { return ((u64)(top[b] & 0xffff) << 42) + ((u64)middle[b] << 21) + low[b]; }
};
static_assert(kSampleList * 8 <= 0xffff && (u64)kSampleList << 21 <= 1ull << 32, "the parts' sums fit");
static_assert(sizeof(SampleSearch) <= sizeof(SampleShared::buffer[1]), "the search's memory fits the buffer");

// A CTA's share of the cluster's list: every thread holds up to four tokens, as (descending logit, id) in one number.
constexpr int kIdBits = 19;
static_assert(kSampleVocab == 1 << kIdBits, "ids fit");
__device__ __forceinline__ float token_logit(u64 token) { return sample_value(~(uint32_t)(token >> kIdBits)); }
__device__ __forceinline__ int token_id(u64 token) { return (int)(token & (kSampleVocab - 1)); }
constexpr int kEach = kSampleList / kSampleThreads;

// How many of the few come before `mine`, and their weights, added to what is there. Four lanes a token.
__device__ __forceinline__ void rank_few(const SampleSearch &in, int few, u64 mine, int &above, u64 &heavier) {
    u64 sum = 0;
#pragma unroll 4
    for (int i = threadIdx.x % 4; i < few; i += 4)
        if (in.few[i] < mine) above++, sum += in.few_mass[i];
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o), sum += __shfl_xor_sync(0xffffffffu, sum, o);
    heavier += sum;
}

// Of the tokens marked as members, the first in order with which `tokens` of them are reached (by_mass false), or with
// which `heavier` and their weights make `share`: bins over the range of their numbers, until one holds kFew of them at
// most (there are `most_members` in all at most), which are compared with one another. All threads call it; ~0
// where there is none. Numbers are unique, so it ends.
__device__ u64 search_list(SampleShared &sh, const u64 (&token)[kEach], const u64 (&w)[kEach], const bool (&member)[kEach], int most_members,
                           bool by_mass, int tokens, u64 share, u64 heavier) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    SampleSearch &in = *reinterpret_cast<SampleSearch *>(sh.buffer[1]);
    u64 base = 0, width = ~0ull;
    __syncthreads();
    if (tid == 0) sh.few_count = 0, sh.found = ~0ull;
    if (most_members > kFew) {
        if (tid == 0) sh.sub_least = 0xffffffffu, sh.sub_most = 0;
        __syncthreads();
        uint32_t least = 0xffffffffu, most = 0;
#pragma unroll
        for (int k = 0; k < kEach; k++)
            if (member[k]) least = min(least, (uint32_t)(token[k] >> kIdBits)), most = max(most, (uint32_t)(token[k] >> kIdBits));
        least = __reduce_min_sync(0xffffffffu, least), most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0 && least <= most) atomicMin(&sh.sub_least, least), atomicMax(&sh.sub_most, most);
        __syncthreads();
        if (sh.sub_least > sh.sub_most) return ~0ull;
        base = (u64)sh.sub_least << kIdBits, width = ((u64)(sh.sub_most - sh.sub_least) << kIdBits) | (kSampleVocab - 1);
        int shift = 64 - __clzll((long long)width) - 8;
        for (;;) {
            for (int i = tid; i < kSubBins; i += kSampleThreads) in.top[i] = in.middle[i] = in.low[i] = 0;
            if (tid == 0) sh.sub_bin = -1;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kEach; k++)
                if (member[k] && token[k] - base <= width) {
                    const int b = (int)((token[k] - base) >> shift);
                    atomicAdd(&in.top[b], 0x10000u + (unsigned)(w[k] >> 42));
                    if (by_mass) atomicAdd(&in.middle[b], (unsigned)(w[k] >> 21) & 0x1fffffu), atomicAdd(&in.low[b], (unsigned)w[k] & 0x1fffffu);
                }
            __syncthreads();
            if (warp == 0) {
                constexpr int per_lane = kSubBins / 32;
                unsigned c[per_lane], upto = 0;
                u64 m[per_lane], sum = 0;
#pragma unroll
                for (int k = 0; k < per_lane; k++) {
                    c[k] = in.count(lane * per_lane + k), m[k] = in.mass(lane * per_lane + k);
                    upto += c[k], sum += m[k];
                }
                const unsigned mine = upto;
                const u64 mine_mass = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned y = __shfl_up_sync(0xffffffffu, upto, o);
                    const u64 z = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o) upto += y, sum += z;
                }
                const bool here = by_mass ? mine && heavier + sum >= share : upto >= (unsigned)tokens;
                const unsigned reached = __ballot_sync(0xffffffffu, here);
                if (reached && lane == __ffs(reached) - 1) {
                    unsigned above = upto - mine;
                    u64 mass = heavier + sum - mine_mass;
#pragma unroll
                    for (int k = 0; k < per_lane; k++) {
                        if (sh.sub_bin < 0 && c[k] && (by_mass ? mass + m[k] >= share : above + c[k] >= (unsigned)tokens))
                            sh.sub_bin = lane * per_lane + k, sh.sub_above = (int)above, sh.found_mass = mass;
                        above += c[k], mass += m[k];
                    }
                }
            }
            __syncthreads();
            const int bin = sh.sub_bin;
            if (bin < 0) return ~0ull;
            tokens -= sh.sub_above;
            if (by_mass) heavier = sh.found_mass;
            base += (u64)bin << shift;
            width = ((u64)1 << shift) - 1;
            if (in.count(bin) <= kFew) break;
            shift = shift > 8 ? shift - 8 : 0;
            __syncthreads();
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kEach; k++)
        if (member[k] && token[k] - base <= width) {
            const int i = atomicAdd(&sh.few_count, 1);
            in.few[i] = token[k], in.few_mass[i] = w[k];
        }
    __syncthreads();
    const int few = sh.few_count;
    if (warp * 8 < few) {  // four lanes a token
        const int at = min(tid / 4, few - 1);
        const u64 mine = in.few[at], mass = in.few_mass[at];
        int above = 0;
        rank_few(in, few, mine, above, heavier);
        // The first at which it is reached: the one before it does not reach it.
        if (by_mass ? heavier + mass >= share && (!above || heavier < share) : above + 1 == tokens) atomicMin(&sh.found, mine);
    }
    __syncthreads();
    return sh.found;
}

template <bool RESIDENT> __global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
    extern __shared__ __align__(16) float slice_memory[];
    __shared__ __align__(16) SampleShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    auto started = cluster.barrier_arrive();  // no CTA's shared memory is written before the CTA runs
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int base = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - base);
    for (int i = tid; i < kSampleList; i += kSampleThreads) reinterpret_cast<uint4 *>(sh.buffer[0])[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) sh.listed = sh.list_count = 0, sh.list_before = sh.list_kept = sh.list_counted = 0;
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    const float *src = a.logits + (long long)row * a.stride + base;

    // ---- what there is in the slice. In shared memory it starts as far from a 16-byte boundary as in global memory, so
    // that everything goes by whole quads.
    const int off = (int)((uintptr_t)src >> 2) & 3, quads = (off + n + 3) / 4;
    const SampleLogits<RESIDENT> x = {RESIDENT ? slice_memory : src - off, off, n};
    const SampleLogits<false> global = {src - off, off, n};
    float4 *ring = reinterpret_cast<float4 *>(slice_memory);  // where the slice is not there
    QuadStream<kSampleThreads, RESIDENT> stream(global, ring, tid, quads);
    const TcmSampling &p = sh.set;
    if (tid == 0) sh.set = a.params[row], sh.uniform = a.uniforms[row], sh.cold = 1.0 / (double)sh.set.temperature;
    __syncthreads();
    // Where cuts are asked for, tokens are counted as they come, in bins of a 128th of the temperature whose borders do not
    // depend on the row: a circle of 8192, as numbers of 16 bits where a slice has no more tokens than they count. Tokens
    // that are masked with a large number, -1e4 or -FLT_MAX, are left out (sample_slots_hold() says when they may be).
    // Where they count more, the slice is not in shared memory, and the cluster's counts go to the ring.
    const bool packed = C > 1 && a.slice <= 0xffff;
    unsigned *own = reinterpret_cast<unsigned *>(sh.buffer[0]), *counts = RESIDENT || packed ? reinterpret_cast<unsigned *>(sh.buffer[1]) : reinterpret_cast<unsigned *>(slice_memory);
    const float fixed_scale = 128.f / p.temperature;
    const bool early = (p.top_k > 0 || p.top_p < 1.f) && fixed_scale > 0.f && fixed_scale < INFINITY;
    const float fixed_floor = sample_floor(fixed_scale);
    float most = -INFINITY, least_counted = INFINITY;
    bool bad = false;
    int live = 0, most_at = 0;  // for greedy rows: the first quad that has the largest
    auto first_pass = [&](auto early, auto packed) {
        constexpr bool kEarly = decltype(early)::value, kPacked = decltype(packed)::value;
        const float floor = kEarly ? fixed_floor : -INFINITY;
        auto look = [&](int q, const float4 &y) {
            const float l[4] = {y.x, y.y, y.z, y.w};
            const float largest = fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)), smallest = fminf(fminf(y.x, y.y), fminf(y.z, y.w));
            if (!kEarly && largest > most) most_at = q;
            most = fmaxf(most, largest);
            if ((smallest > floor) & ((y.x + y.y) + (y.z + y.w) < INFINITY)) {  // four usual tokens: 20 instructions fewer
                live += 4;
                if constexpr (kEarly) {
                    least_counted = fminf(least_counted, smallest);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int b = sample_slot(l[k], fixed_scale);
                        if constexpr (kPacked) atomicAdd(&own[b >> 1], b & 1 ? 0x10000u : 1u);
                        else atomicAdd(&own[b], 1u);
                    }
                }
                return;
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                bad |= !(l[k] < INFINITY);
                live += l[k] > -INFINITY;
                if constexpr (kEarly)
                    if (l[k] > floor) {
                        const int b = sample_slot(l[k], fixed_scale);
                        least_counted = fminf(least_counted, l[k]);
                        atomicAdd(&own[kPacked ? b >> 1 : b], kPacked && b & 1 ? 0x10000u : 1u);
                    }
            }
        };
        stream.run(look);
    };
    if (!early) first_pass(std::false_type{}, std::false_type{});
    else if (packed) first_pass(std::true_type{}, std::true_type{});
    else first_pass(std::true_type{}, std::false_type{});
    const uint32_t warp_most = __reduce_max_sync(0xffffffffu, sample_key(most));
    const uint32_t warp_counted = __reduce_min_sync(0xffffffffu, sample_key(least_counted));
    bad = __any_sync(0xffffffffu, bad);
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 0) {
        sh.warp_count[warp] = live;
        reinterpret_cast<uint32_t *>(sh.warp_high)[warp] = warp_most, reinterpret_cast<uint32_t *>(sh.warp_low)[warp] = warp_counted;
        sh.warp_mass[warp] = bad;
    }
    __syncthreads();
    cluster.barrier_wait(std::move(started));
    if (warp == 0) {  // lane c tells CTA c
        const int w = lane % kSampleWarps;
        SampleSlice z;
        z.most = __reduce_max_sync(0xffffffffu, reinterpret_cast<uint32_t *>(sh.warp_high)[w]);
        z.counted = __reduce_min_sync(0xffffffffu, reinterpret_cast<uint32_t *>(sh.warp_low)[w]);
        z.live = __reduce_add_sync(0xffffffffu, lane < kSampleWarps ? sh.warp_count[w] : 0);
        z.bad = __any_sync(0xffffffffu, sh.warp_mass[w] != 0);
        if (lane < C) cluster.map_shared_rank(sh.slices, lane)[rank] = z;
    }
    cluster.sync();
    float high, low_counted;
    int all_live;
    {
        const SampleSlice z = sh.slices[lane < C ? lane : 0];
        high = sample_value(__reduce_max_sync(0xffffffffu, z.most));
        low_counted = sample_value(__reduce_min_sync(0xffffffffu, z.counted));
        all_live = __reduce_add_sync(0xffffffffu, lane < C ? z.live : 0);
        bad = __any_sync(0xffffffffu, z.bad);
    }
    const float u = sh.uniform;
    const bool wrong = !(p.temperature >= 0.f && p.temperature < INFINITY && u >= 0.f && u < 1.f && p.min_p <= 1.f) ||
                       p.top_p != p.top_p;
    if (bad || !all_live || wrong) {  // the whole cluster alike
        if (rank == 0 && tid == 0) {
            a.ids[row] = -1;
            if (a.logprobs) a.logprobs[row] = 0.f;
            if (a.kept) a.kept[row] = 0;
            if (a.status) atomicOr(a.status, (bad ? 1 : 0) | (!bad && !all_live ? 2 : 0) | (wrong ? 4 : 0));
        }
        return;
    }
    if (p.temperature == 0.f) {
        int first = 0x7fffffff;
        if (most == high) {  // both zeros are one number
            const float4 y = x.quad(most_at);
            first = base + 4 * most_at - off + (y.x == high ? 0 : y.y == high ? 1 : y.z == high ? 2 : 3);
        }
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0) sh.warp_count[warp] = first;
        __syncthreads();
        if (warp == 0) {
            first = __reduce_min_sync(0xffffffffu, sh.warp_count[lane % kSampleWarps]);
            if (lane == 0) cluster.map_shared_rank(sh.first, 0)[rank] = first;
        }
        cluster.sync();
        if (rank == 0 && tid == 0) {
            for (int c = 0; c < C; c++) first = min(first, sh.first[c]);
            a.ids[row] = first;
            if (a.logprobs) a.logprobs[row] = 0.f;
            if (a.kept) a.kept[row] = 1;
        }
        return;
    }

    const SampleRow r(high, sh.cold, sh.shift);
    __syncthreads();
    // min-p as the least logit that it keeps: next to the one that arithmetic gives, the one that satisfies the definition.
    float min_logit = -FLT_MAX;
    if (p.min_p > 0.f) {
        const double coldest = log((double)p.min_p);
        auto exponent = [&](float l) { return ((double)l - (double)high) * sh.cold; };
        float l = fmaxf((float)((double)high + coldest * (double)p.temperature), -FLT_MAX);
        if (!(exponent(l) >= coldest)) l = nextafterf(l, INFINITY);
        else if (l > -FLT_MAX && exponent(nextafterf(l, -INFINITY)) >= coldest) l = nextafterf(l, -INFINITY);
        min_logit = fminf(l, high);
    }

    // ---- the bins in which the cuts lie
    const bool by_count = p.top_k > 0 && p.top_k < all_live, by_mass = p.top_p < 1.f, cuts = by_count || by_mass;
    const float reach = (float)((double)high - 32.0 * (double)p.temperature);
    SampleBins bins = sample_bins_of(high, fixed_scale);
    bool fixed = early && sample_slots_hold(&bins, high, low_counted);
    int count_bin = kSampleBins, mass_from = kSampleBins, mass_to = -1;  // top-k's bin; top-p's, first and last
    int tokens_left = 0, in_count_bin = 0;                               // of top-k in its bin, and how many that has
    int listed = 0;
    bool all_listed = false;
    for (; cuts; fixed = false) {  // again, with bins over the row's own range, where those hold too many or not at all
        if (!fixed) {
            float low = INFINITY;
            each_quad<kSampleThreads>(x, ring, tid, quads, [&](int, const float4 &y) {
                const float l[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int k = 0; k < 4; k++) low = fminf(low, l[k] > -INFINITY ? l[k] : INFINITY);
            });
            low = -warp_max(-low);
            __syncthreads();
            if (lane == 0) sh.warp_low[warp] = low;
            __syncthreads();
            if (tid < C) {
                for (int w = 0; w < kSampleWarps; w++) low = fminf(low, sh.warp_low[w]);
                cluster.map_shared_rank(sh.ends, tid)[rank] = make_float2(low, high);
            }
            if (C > 1) cluster.sync();
            else __syncthreads();
            for (int c = 0; c < C; c++) low = fminf(low, sh.ends[c].x);
            bins = sample_bins_over(low < reach && reach < high ? reach : low, high, kSampleBins);
            for (int i = tid; i < kSampleBins / 4; i += kSampleThreads) reinterpret_cast<uint4 *>(own)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            each_quad<kSampleThreads>(x, ring, tid, quads, [&](int, const float4 &l) {
                if (l.x > -INFINITY) atomicAdd(&own[sample_bin(&bins, l.x)], 1u);
                if (l.y > -INFINITY) atomicAdd(&own[sample_bin(&bins, l.y)], 1u);
                if (l.z > -INFINITY) atomicAdd(&own[sample_bin(&bins, l.z)], 1u);
                if (l.w > -INFINITY) atomicAdd(&own[sample_bin(&bins, l.w)], 1u);
            });
            if (C > 1) cluster.sync();
            else __syncthreads();
        }
        if (tid == 0) sh.bin = kSampleBins, sh.mass_from = sh.mass_to = kSampleBins - 1;
        if (C > 1) {
            // Each CTA adds up its share of the bins and tells the others.
            const int share_of = kSampleBins / C;
            for (int i = tid; i < share_of; i += kSampleThreads) {
                const int b = rank * share_of + i, at = fixed ? (bins.top - b) & (kSampleSlots - 1) : b;
                unsigned c = 0;
#pragma unroll 8
                for (int k = 0; k < C; k++) {
                    const unsigned *theirs = cluster.map_shared_rank(own, k);
                    c += fixed && packed ? reinterpret_cast<const unsigned short *>(theirs)[at] : theirs[at];
                }
#pragma unroll 8
                for (int k = 0; k < C; k++) cluster.map_shared_rank(counts, k)[b] = c;
            }
            cluster.sync();
        } else {
            __syncthreads();
        }
        constexpr int each = kSampleBins / kSampleThreads;
        unsigned c[each], upto = 0;
        float mass[each], total = 0.f, squares = 0.f;
        // A bin's width, in powers of two of weight.
        const float step = bins.scale > 0.f ? (float)(-r.slope / ((double)bins.scale * (double)bins.unit)) : 0.f;
        static_assert(each == 8, "two quads");
        const bool circle = C == 1 && fixed;  // in which bins go down
        const unsigned *from = C > 1 ? counts + tid * each : circle ? own + ((bins.top - tid * each - (each - 1)) & (kSampleSlots - 1)) : own + tid * each;
        const uint4 some_low = reinterpret_cast<const uint4 *>(from)[0], some_high = reinterpret_cast<const uint4 *>(from)[1];
        const unsigned some[each] = {some_low.x, some_low.y, some_low.z, some_low.w, some_high.x, some_high.y, some_high.z, some_high.w};
#pragma unroll
        for (int k = 0; k < each; k++) {
            const int b = tid * each + k;
            c[k] = circle ? some[7 - k] : some[k];
            if (b == kSampleBins - 1) c[k] = 0;  // and all that lie lower: what the others leave
            const float weight = b == kSampleBins - 1 ? 0.f : exp2f((float)b * step);
            mass[k] = (float)c[k] * weight;
            upto += c[k], total += mass[k], squares += mass[k] * weight;
        }
        unsigned mine = upto;
        const float mine_mass = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, upto, o);
            const float z = __shfl_up_sync(0xffffffffu, total, o);
            if (lane >= o) upto += y, total += z;
        }
        squares = warp_sum(squares);
        if (lane == 31) sh.warp_count[warp] = (int)upto, sh.warp_high[warp] = total, sh.warp_low[warp] = squares;
        __syncthreads();
        unsigned before = upto - mine;
        float lighter = total - mine_mass, whole = 0.f;
        squares = 0.f;
#pragma unroll
        for (int w = 0; w < kSampleWarps; w++) {
            squares += sh.warp_low[w];
            if (w < warp) before += (unsigned)sh.warp_count[w], lighter += sh.warp_high[w];
            whole += sh.warp_high[w];
        }
        if (tid == kSampleThreads - 1) c[each - 1] = (unsigned)all_live - before - mine, mine += c[each - 1];
        if (by_count) {
            const unsigned k = (unsigned)p.top_k;
            if (before < k && k <= before + mine) {
                unsigned above = before;
                float heavier = lighter;
#pragma unroll
                for (int b = 0; b < each; b++) {
                    if (above < k && k <= above + c[b]) {
                        sh.bin = tid * each + b, sh.above = (int)above, sh.in_bin = (int)c[b];
                        sh.mass_whole = heavier + mass[b] * ((float)(k - above) / (float)c[b]);
                    }
                    above += c[b], heavier += mass[b];
                }
            }
            __syncthreads();
            count_bin = sh.bin, tokens_left = p.top_k - sh.above, in_count_bin = sh.in_bin;
            whole = sh.mass_whole;
        }
        all_listed = by_count && sh.above + sh.in_bin <= kSampleList;
        listed = in_count_bin;
        if (all_listed) {  // a small k: all tokens down to its bin, and no estimate
            mass_from = 0, mass_to = count_bin;
            listed += sh.above, tokens_left = p.top_k;
        } else if (by_mass) {
            // The bins at which the estimated sum passes the share, a little before and a little behind it.
            // A token's weight is estimated within half a bin's width, so a sum of independent ones within some 0.3 widths
            // of the root of their squares' sum; four times that, and what FP32 sums are off by.
            const float share = fmaxf(p.top_p, 0.f) * whole, slack = -0.8f * step * sqrtf(squares) + 2e-5f * whole;
            const int last = min(kSampleBins - 1, count_bin);
            // A thread's last sum is the next one's first, so that every value is passed by one of them.
            float behind = __shfl_down_sync(0xffffffffu, lighter, 1), sum = lighter;
            if (lane == 31) {
                behind = 0.f;
                for (int w = 0; w <= warp; w++) behind += sh.warp_high[w];
            }
#pragma unroll
            for (int k = 0; k < each; k++) {
                const int b = tid * each + k;
                const float next = k == each - 1 ? behind : sum + mass[k];
                if (sum < share - slack && next >= share - slack) atomicMin(&sh.mass_from, b);
                if (sum < share + slack && next >= share + slack) atomicMin(&sh.mass_to, b);
                sum = next;
            }
            if (tid == 0 && !(share > slack)) atomicMin(&sh.mass_from, 0);
            __syncthreads();
            mass_from = min(sh.mass_from, last), mass_to = max(min(sh.mass_to, last), mass_from);
            // How many tokens they hold: those up to the last but not above the first.
#pragma unroll
            for (int k = 0; k < each; k++) {
                const int b = tid * each + k;
                if (b == mass_from) sh.list_from = (int)before;
                before += c[k];
                if (b == mass_to) sh.list_to = (int)before;
            }
            __syncthreads();
            listed = sh.list_to - sh.list_from + (mass_to < count_bin ? in_count_bin : 0);
        }
        if (C == 1) __syncthreads();  // the counts have been read: the list takes their place
        if (listed <= kSampleList) break;
        if (!fixed) {
            sample_slowly<RESIDENT>(a, sh, slice_memory, row, high, all_live, min_logit);
            return;
        }
    }

    // ---- weights above the bins, and the list of what is in them. A warp has a contiguous stretch of ids.
    const int per_warp = (quads + kSampleWarps - 1) / kSampleWarps, w0 = min(quads, warp * per_warp), w1 = min(quads, w0 + per_warp);
    u64 *own_list = sh.buffer[0];
    u64 sum_above = 0, sum_all = 0, sum_kept = 0;
    int kept = 0;
    if (cuts) {
        // The bins' borders as logits: the least of a bin and those above it, found by trial as the arithmetic of sample_bin(&bins, )
        // has it. Tokens from `sure` on are above the bins in question and kept; from `in_from` down to `in_to` in top-p's,
        // from `count_from` down to `count_to` in top-k's.
        if (warp < 4) {  // a warp a border: 32 numbers at a time cut the range into 33
            const int b = warp == 0 ? (by_mass || all_listed ? mass_from : count_bin) - 1 : warp == 1 ? mass_to : warp == 2 ? count_bin - 1 : count_bin;
            uint32_t down = sample_key(-FLT_MAX), up = sample_key(high);  // sample_bin(&bins, up) <= b, or none is
            if (b < sample_bin(&bins, high)) down = up = sample_key(INFINITY);
            while (down < up) {
                const uint32_t step = (up - down) / 33 + 1, at = up - down > (lane + 1) * step ? up - (lane + 1) * step : down;
                const unsigned in = __ballot_sync(0xffffffffu, sample_bin(&bins, sample_value(at)) <= b);  // the first lanes
                const uint32_t most = up - down, passed = __popc(in);
                up = most > passed * step ? up - passed * step : down;
                if (passed < 32) down = most > (passed + 1) * step ? up - step + 1 : down + 1;
            }
            if (lane == 0) sh.border[warp] = sample_value(up);
        }
        __syncthreads();
        const float sure = sh.border[0], in_to = by_mass || all_listed ? sh.border[1] : INFINITY;
        // As many as the bins counted; whatever they counted, no more than there is room for.
        auto append = [&](float l, int i) {
            const int at = atomicAdd(&sh.listed, 1);
            if (at < kSampleList) own_list[at] = ((u64)~sample_key(l) << kIdBits) | (unsigned)(base + i);
        };
        // Lists those of a quad that `in` marks.
        auto append_some = [&](int q, const float (&l)[4], auto in) {
            if (in(l[0]) | in(l[1]) | in(l[2]) | in(l[3]))
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (in(l[k])) append(l[k], 4 * q + k - off);
        };
        if (all_listed) {
            each_quad<32>(x, ring, w0 + lane, w1, [&](int q, const float4 &y) {
                const float l[4] = {y.x, y.y, y.z, y.w};
                append_some(q, l, [&](float z) { return z >= in_to; });
            });
        } else if (by_count) {
            const float count_from = sh.border[2], count_to = sh.border[3];
            each_quad<32>(x, ring, w0 + lane, w1, [&](int q, const float4 &y) {
                if (!(fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)) >= count_to)) return;
                const float l[4] = {y.x, y.y, y.z, y.w};
                append_some(q, l, [&](float z) { return (!(z >= sure) & (z >= in_to)) | (!(z >= count_from) & (z >= count_to)); });
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const u64 w = r.weight(l[k]);
                    if (l[k] >= count_from) sum_all += w;
                    if (l[k] >= sure) sum_above += w;
                    if (l[k] >= sure && l[k] < min_logit) sum_kept += w, kept--;
                }
            });
        } else if (p.min_p > 0.f) {
            each_quad<32>(x, ring, w0 + lane, w1, [&](int q, const float4 &y) {
                const float l[4] = {y.x, y.y, y.z, y.w};
                append_some(q, l, [&](float z) { return !(z >= sure) & (z >= in_to); });
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const u64 w = r.weight(l[k]);
                    sum_all += w;
                    if (l[k] >= sure) sum_above += w;
                    if (l[k] >= sure && l[k] < min_logit) sum_kept += w, kept--;
                }
            });
        } else {
            each_quad<32>(x, ring, w0 + lane, w1, [&](int q, const float4 &y) {
                const float l[4] = {y.x, y.y, y.z, y.w};
                append_some(q, l, [&](float z) { return !(z >= sure) & (z >= in_to); });
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const u64 w = r.weight(l[k]);
                    sum_all += w;
                    if (l[k] >= sure) sum_above += w;
                }
            });
        }
        // How many there are above the bins is known of the whole row; sum_kept and kept are what min-p takes away of them.
        if (rank == 0 && tid == 0) kept += all_listed ? 0 : by_mass ? sh.list_from : sh.above;
        sum_kept = sum_above - sum_kept;
    } else {
        if (p.min_p > 0.f)
            each_quad<32>(x, ring, w0 + lane, w1, [&](int, const float4 &y) {
                if (!(fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)) >= min_logit)) return;
                const float l[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const u64 w = r.weight(l[k]);
                    if (l[k] >= min_logit) sum_kept += w, kept++;
                }
            });
        else {
            each_quad<32>(x, ring, w0 + lane, w1, [&](int, const float4 &y) {  // masked tokens weigh nothing
                sum_kept += (r.weight(y.x) + r.weight(y.y)) + (r.weight(y.z) + r.weight(y.w));
            });
            if (rank == 0 && tid == 0) kept = all_live;
        }
    }
    if (by_mass) sum_all = warp_sum64(sum_all), sum_above = warp_sum64(sum_above);
    sum_kept = warp_sum64(sum_kept);
    kept = __reduce_add_sync(0xffffffffu, kept);
    if (lane == 0) {
        sh.warp_mass[warp] = sum_all, sh.warp_more[warp] = sum_above, sh.warp_kept[warp] = sum_kept;
        sh.warp_count[warp] = kept;
    }
    __syncthreads();
    if (warp == 0) {  // lane c tells CTA c
        const int w = lane % kSampleWarps;
        SampleSums z = {0, 0, 0, 0, 0};
        if (lane < kSampleWarps) z.all = sh.warp_mass[w], z.above = sh.warp_more[w], z.kept = sh.warp_kept[w], z.kept_count = sh.warp_count[w];
        if (by_mass) z.all = warp_sum64(z.all), z.above = warp_sum64(z.above);
        z.kept = warp_sum64(z.kept);
        z.kept_count = __reduce_add_sync(0xffffffffu, z.kept_count);
        z.listed = min(sh.listed, kSampleList);
        if (lane < C) cluster.map_shared_rank(sh.sums, lane)[rank] = z;
    }
    cluster.sync();
    if (warp == 1) {
        SampleSums z = {0, 0, 0, 0, 0};
        if (lane < C) z = sh.sums[lane];
        const u64 before = warp_sum64(lane < rank ? z.kept : 0), whole = warp_sum64(z.kept);
        if (by_mass) z.above = warp_sum64(z.above), z.all = warp_sum64(z.all);
        z.kept_count = __reduce_add_sync(0xffffffffu, z.kept_count);
        if (lane == 0) sh.before = before, sh.whole = whole, sh.heavier = z.above, sh.everything = z.all, sh.kept = z.kept_count;
        int upto = z.listed;
#pragma unroll
        for (int o = 1; o < kSampleCluster; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        if (lane < C) sh.list_start[lane] = upto - z.listed;
        if (lane == C - 1) sh.list_total = upto;
    }
    if (lane == 0) sh.warp_more[warp] = 0;
    // ---- the cut in the cluster's list
    u64 cut = 0;
    if (cuts) {
        __syncthreads();
        const int m = min(listed, sh.list_total);  // tokens that are there, so each once: the search ends
        u64 token[kEach], w[kEach];
        bool member[kEach], counted[kEach];
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            const int i = tid + k * kSampleThreads;
            token[k] = ~0ull;
            member[k] = i < m;
            if (member[k]) {
                int c = 0;
#pragma unroll
                for (int j = 1; j < kSampleCluster; j++) c += j < C && sh.list_start[j] <= i;
                token[k] = cluster.map_shared_rank(own_list, c)[i - sh.list_start[c]];
            }
        }
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            w[k] = 0, counted[k] = false;
            if (k * kSampleThreads + warp * 32 >= m) continue;
            const float l = token_logit(token[k]);
            w[k] = member[k] ? r.weight(l) : 0;
            counted[k] = member[k] && by_count && sample_bin(&bins, l) <= count_bin && (all_listed || sample_bin(&bins, l) == count_bin);
        }
        if (C > 1) cluster.barrier_arrive();  // the others' lists have been read; a CTA leaves when its own has
        cut = ~0ull;
        // Few tokens are compared with one another once, for both cuts. (One row with top-k 40 and top-p: 20.3 us, 22.7 with two
        // searches.)
        const bool at_once = m > 0 && m <= kFew && (all_listed || !by_count);
        u64 share = 0;
        if (at_once) {
            SampleSearch &in = *reinterpret_cast<SampleSearch *>(sh.buffer[1]);
            if (tid < m) in.few[tid] = token[0], in.few_mass[tid] = w[0];
            if (tid == 0) sh.found = ~0ull;
            __syncthreads();
            const int at = min(tid / 4, m - 1);
            const u64 mine = in.few[at], mass = in.few_mass[at];
            int above = 0;
            u64 heavier = sh.heavier;
            rank_few(in, m, mine, above, heavier);
            const bool counts_in = !by_count || above < tokens_left;
            if (by_mass) {
                u64 all_of = sh.everything;
                if (by_count) {
                    const u64 sum = warp_sum64(counts_in && lane % 4 == 0 && tid / 4 < m ? mass : 0);
                    if (lane == 0 && sum) atomicAdd(&sh.list_counted, sum);
                    __syncthreads();
                    all_of += sh.list_counted;
                }
                share = sample_share(p.top_p, all_of, true);
                if (counts_in && heavier + mass >= share && (!above || heavier < share)) atomicMin(&sh.found, mine);
            } else if (above + 1 == tokens_left) {
                atomicMin(&sh.found, mine);
            }
            __syncthreads();
            cut = sh.found;
        }
        if (by_count && !at_once) cut = search_list(sh, token, w, counted, m, false, tokens_left, 0, 0);
        if (by_mass && !at_once) {
            u64 all_of = sh.everything;
            if (by_count) {
                u64 sum = 0;
#pragma unroll
                for (int k = 0; k < kEach; k++) {
                    member[k] = member[k] && token[k] <= cut;
                    if (counted[k] && member[k]) sum += w[k];
                }
                sum = warp_sum64(sum);
                if (lane == 0 && sum) atomicAdd(&sh.list_counted, sum);
                __syncthreads();
                all_of += sh.list_counted;
            }
            share = sample_share(p.top_p, all_of, true);
            cut = search_list(sh, token, w, member, m, true, 0, share, sh.heavier);
        }
        // There is one, top-p's in its bins, or the estimate or the counts were wrong.
        const bool fine = cut != ~0ull && (!by_mass || ((mass_from == 0 || sh.heavier < share) && sample_bin(&bins, token_logit(cut)) <= mass_to));
        if (!fine) {  // the whole cluster alike
            if (C > 1) cluster.barrier_wait();
            sample_slowly<RESIDENT>(a, sh, slice_memory, row, high, all_live, min_logit);
            return;
        }
        // What is kept of the list, by where it is.
        u64 sum = 0, ahead = 0;
        int count = 0;
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            if (!member[k] || token[k] > cut || token_logit(token[k]) < min_logit) continue;
            const int at = token_id(token[k]) - base;
            sum += w[k], count++;
            if (at < 0) ahead += w[k];
            else if (at < n) atomicAdd(&sh.warp_more[(at + off) / 4 / per_warp], w[k]);
        }
        sum = warp_sum64(sum), ahead = warp_sum64(ahead);
        count = __reduce_add_sync(0xffffffffu, count);
        if (lane == 0 && count) {
            atomicAdd(&sh.list_kept, sum);
            atomicAdd(&sh.list_count, count);
            if (ahead) atomicAdd(&sh.list_before, ahead);
        }
    }
    __syncthreads();
    u64 whole = sh.whole, before = sh.before;
    const float cut_value = cuts ? token_logit(cut) : -INFINITY;
    const unsigned cut_id = token_id(cut);
    if (cuts) whole += sh.list_kept, before += sh.list_before;
    const u64 target = sample_share(sh.uniform, whole, false);

    // ---- the token: the warp's stretch that holds it, in 16 parts for the warps, then the part by one warp
    auto weights = [&](int q, const float4 &y, u64 (&w)[4]) {  // what is kept of a quad
        const float l[4] = {y.x, y.y, y.z, y.w};
        u64 sum = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const unsigned id = (unsigned)(base + 4 * q + k - off);
            const bool stays = (l[k] > cut_value || (l[k] == cut_value && id <= cut_id)) && l[k] >= min_logit;
            w[k] = r.weight(l[k]);
            if (!stays) w[k] = 0;
            sum += w[k];
        }
        return sum;
    };
    // Which of 16 consecutive sums passes the target; -1: none. `before` moves to its start.
    auto holder = [&](u64 mine) {
        u64 upto = mine;
#pragma unroll
        for (int o = 1; o < kSampleWarps; o <<= 1) {
            const u64 z = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += z;
        }
        const unsigned reached = __ballot_sync(0xffffffffu, lane < kSampleWarps && target >= before + upto - mine && target < before + upto);
        const int who = __ffs(reached) - 1;
        if (who >= 0) before += __shfl_sync(0xffffffffu, upto - mine, who);
        return who;
    };
    const int who = holder(lane < kSampleWarps ? sh.warp_kept[lane] + sh.warp_more[lane] : 0);
    if (who >= 0) {  // this CTA has it
        const int s0 = min(quads, who * per_warp), s1 = min(quads, s0 + per_warp), part = (s1 - s0 + kSampleWarps - 1) / kSampleWarps;
        u64 w[4], sum = 0;
        each_quad<32>(x, ring, s0 + warp * part + lane, min(s1, s0 + (warp + 1) * part), [&](int q, const float4 &y) { sum += weights(q, y, w); });
        sum = warp_sum64(sum);
        if (lane == 0) sh.warp_mass[warp] = sum;
        __syncthreads();
        const int mine = holder(lane < kSampleWarps ? sh.warp_mass[lane] : 0);
        if (warp == mine) {
            const int q1 = min(s1, s0 + (warp + 1) * part);
            bool found = false;
            constexpr int kLoads = 4;  // at a time
            for (int q0 = s0 + warp * part; q0 < q1 && !found; q0 += 32 * kLoads) {
                float4 y[kLoads];
#pragma unroll
                for (int i = 0; i < kLoads; i++) {
                    const int q = q0 + 32 * i + lane;
                    y[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (q < q1) y[i] = x.quad(q);
                }
#pragma unroll
                for (int i = 0; i < kLoads; i++) {
                    const int q = q0 + 32 * i + lane;
                    w[0] = w[1] = w[2] = w[3] = 0;
                    u64 upto = q < q1 ? weights(q, y[i], w) : 0;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const u64 z = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += z;
                    }
                    const unsigned reached = found ? 0 : __ballot_sync(0xffffffffu, before + upto > target);
                    if (reached && lane == __ffs(reached) - 1) {
                        u64 to = before + upto;
                        int id = 0;
#pragma unroll
                        for (int k = 3; k >= 0; k--) {  // the first of the four at which the sum passes the target
                            if (to > target && w[k]) id = 4 * q + k - off;
                            to -= w[k];
                        }
                        a.ids[row] = base + id;
                        if (a.logprobs) a.logprobs[row] = r.logprob(x.at(id), high, sh.cold, whole);
                        if (a.kept) a.kept[row] = sh.kept + (cuts ? sh.list_count : 0);
                    }
                    found |= reached != 0;
                    before += __shfl_sync(0xffffffffu, upto, 31);
                }
            }
        }
    }
    if (cuts && C > 1) cluster.barrier_wait();
}

int refuse(const char *why) {
    fprintf(stderr, "gpu_sample: %s\n", why);
    return -1;
}

}  // namespace
}  // namespace tcm

using namespace tcm;

extern "C" int gpu_sample(TcmGpu *gpu, int *ids, float *logprobs, int *kept, const float *logits, long long stride, int rows,
                          int vocab, const TcmSampling *params, const float *uniforms, int *status) {
    if (!gpu) return refuse("no handle");
    if (rows < 0 || rows > 1 << 24) return refuse("rows is 0 to 2^24");
    if (vocab < 1 || vocab > kSampleVocab) return refuse("vocab is 1 to 524288");
    if (stride && stride < vocab) return refuse("a stride is 0 or holds a row");
    if (!rows) return 0;
    if (!ids || !logits || !params || !uniforms) return refuse("no ids, logits, settings or uniforms");
    if (((uintptr_t)ids | (uintptr_t)logprobs | (uintptr_t)kept | (uintptr_t)logits | (uintptr_t)params | (uintptr_t)uniforms |
         (uintptr_t)status) & 3)
        return refuse("arrays are 4-byte aligned");
    static PerDeviceOnce once;
    once.run([] {
        TCM_CUDA(cudaFuncSetAttribute(sample_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleOwnSm));
        TCM_CUDA(cudaFuncSetAttribute(sample_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes));
        TCM_CUDA(cudaFuncSetAttribute(sample_kernel<true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        TCM_CUDA(cudaFuncSetAttribute(sample_kernel<false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    });
    // As many CTAs a row as run at once for all rows, of 1024 tokens at least; 8 and 16 only where every CTA has an SM of its own.
    // Measured with rows of 151,936 and top-p, us for 1, 2, 4, 8, 16 CTAs a row: 1 row 81, 55, 35, 29, 26; 32 rows 91, 67, 36,
    // 43, 74; 64 rows 109, 80, 57, 75, 132; 128 rows 128, 84, 115, 146, 249; 256 rows 136, 163, 212, 279, 480.
    int cluster = kSampleCluster;
    while (cluster > 4 && (long long)rows * cluster > sm_count()) cluster /= 2;
    while (cluster > 1 && (vocab < cluster * 1024 || (long long)rows * cluster > 2 * sm_count())) cluster /= 2;
    const int slice = ((vocab + cluster - 1) / cluster + 3) / 4 * 4;
    // In shared memory where that takes no CTA off its SM.
    const long long smem = (slice + 8) * 4ll;
    const bool resident = smem <= ((long long)rows * cluster <= sm_count() && smem > kSampleHalfSm ? kSampleOwnSm : kSampleHalfSm);
    const SampleArgs args = {ids, logprobs, kept, logits, stride, vocab, slice, params, uniforms, status};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * cluster);
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = resident ? (size_t)smem : kRingBytes;
    cfg.stream = stream();
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)cluster, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (resident) TCM_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<true>, args));
    else TCM_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<false>, args));
    return 0;
}
