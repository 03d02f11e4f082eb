// Sampling: one token a row of logits, with temperature, top-k, top-p and min-p, by a given uniform number.
//
// A thread-block cluster has one row. Each of its CTAs brings a contiguous slice of the row into shared memory, and
// everything after that runs on chip: the row is read from HBM once. All three filters keep a prefix of the tokens in
// descending order of their logits (equal ones by id), so what is kept is described by the last token that is, the cut:
// a logit and an id. The row is never sorted:
//   1. the largest logit (a cluster barrier);
//   2. for top-k and top-p, how many tokens each of 4096 bins of the logits' range has (two barriers). The bin of the
//      k-th token is known then; that of top-p's last token is estimated from the counts and the bins' middles;
//   3. one pass adds up the weights above those bins, and lists the few tokens inside them (a barrier);
//   4. every CTA sorts the list and finds the cut in it, then the id at which the kept weights pass the uniform number's
//      share; the warp that holds this id writes the result.
// Where the estimate was wrong, or the bins hold more than a list (many equal logits), sample_slowly() narrows the range
// bin by bin instead.
//
// Weights exp((l - max) / T) are whole numbers, 2^44 for the largest: their sums are exact whatever the order, so that
// atomics and the CTAs' shares leave results the same from call to call, and a sum of 2^19 of them stays below 2^64.
// What bounds it: the weights' 13 FP64 instructions an element (26 cycles of an SM's quarter) beside HBM.
#include "common.cuh"
#include "kernels.h"
#include "../../include/gpu.h"
#include <cooperative_groups.h>
#include <float.h>
#include <math.h>
#include <utility>

namespace cg = cooperative_groups;

namespace tcm {
namespace {

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 4096, kSampleList = 2048, kSlowBins = 1024;
constexpr int kSampleVocab = 1 << 19, kSampleCluster = 16;
constexpr int kSampleSlice = kSampleVocab / kSampleCluster;  // logits a CTA holds at most
constexpr double kSampleOne = 0x1p44;
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
    uint32_t most, least;  // keys of the logits above -infinity
    int live, bad;         // logits above -infinity; a NaN or +infinity among them
};
struct SampleSums {
    u64 all, above, kept;  // weights: of the tokens that top-p takes a share of, above its bins, and above all bins and min-p
    int kept_count, listed;
};

struct SampleShared {
    u64 buffer[2][kSampleList];  // own counts, then own list; the cluster's counts, then its list
    SampleSlice slices[kSampleCluster];
    SampleSums sums[kSampleCluster];
    int first[kSampleCluster];       // greedy rows: the lowest id of the largest logit
    float2 ends[kSampleCluster];     // least and largest logit of the slow search's bin
    u64 part_mass[kSampleCluster];
    int part_count[kSampleCluster];
    u64 warp_mass[kSampleWarps], warp_more[kSampleWarps], warp_kept[kSampleWarps];
    int warp_count[kSampleWarps];
    float warp_low[kSampleWarps], warp_high[kSampleWarps];
    u64 whole, before, heavier, everything;  // of the row: see SampleSums; before: kept in CTAs before this one
    u64 list_before, list_kept, at_first, at_last;
    int kept, listed, list_count;
    int bin, above, in_bin;  // of top-k's cut
    float mass_whole;        // what top-p takes its share of, estimated
    int mass_from, mass_to;  // top-p's bins, first and last,
    int list_from, list_to;  // and the tokens above the first, up to the last
    int cut;                 // index in the list of top-p's last token
    int settled;             // whether the cut is in the list
    uint32_t cut_key;
    unsigned cut_id;
    u64 slow_mass;
};

__device__ __forceinline__ u64 warp_sum64(u64 x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
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
__device__ constexpr double kSampleSeries[7] = {0.6931471805599453,    0.24022650922288757,   0.055504108839096185,  0.009618056678524632,
                                                0.0013333502386162978, 0.00015461444698571227, 1.5297323760649362e-05};

struct SampleRow {
    double top, cold, slope;  // the largest logit, 1 / T, log2(e) / T
    __device__ double exponent(float l) const { return ((double)l - top) * cold; }
    __device__ u64 weight(float l) const {
        const double y0 = ((double)l - top) * slope;
        // At most zero; from -64 on (its upper word decides) nothing is left of it.
        const double y = __hiloint2double((int)min((unsigned)__double2hiint(y0), 0xc0500000u), __double2loint(y0));
        const double t = y + 0x1.8p52, f = y - (t - 0x1.8p52);
        double z = kSampleSeries[6];
#pragma unroll
        for (int k = 5; k >= 0; k--) z = fma(z, f, kSampleSeries[k]);
        z = fma(z, f, 1.0);
        z = __hiloint2double(__double2hiint(z) + (__double2loint(t) << 20), __double2loint(z));
        return (u64)(__double_as_longlong(z + 0x1.8p8) - __double_as_longlong(0x1.8p8));  // in units of 2^-44
    }
};

// Bins over [from, high]: 0 for `high`, and not falling as l falls; all below `from` are the last.
struct SampleBins {
    float from, high, unit, scale;
    int last;
    __device__ SampleBins(float from_, float high_, int bins) : from(from_), high(high_), last(bins - 1) {
        // Differences in a power of two at which neither they nor the scale leave FP32's range.
        const float span = high - from;
        unit = span > 1e30f ? 0.25f : span < 1e-25f ? 0x1p100f : 1.f;
        scale = span > 0.f ? (float)(bins - 2) * 0.999999f / (high * unit - from * unit) : 0.f;
        high *= unit;
    }
    __device__ int of(float l) const {
        const int b = __float_as_int(fmaf(high - l * unit, scale, 0x1p23f)) & 0x7fffff;
        return l < from ? last : b;
    }
    __device__ float width() const { return scale > 0.f ? 1.f / scale / unit : 0.f; }  // a bin's
};

// The cut by repeated histograms of the cluster: counts and weights in bins of the range in which it must lie, then of the
// bin that it falls into, until that holds one value. Then who is kept, and the token. All threads of the cluster call it.
__device__ __noinline__ void sample_slowly(const SampleArgs &a, const SampleRow &r, SampleShared &sh, const float *x, int n, int base,
                                           int row, float low_all, float high_all, int live, float min_logit) {
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const TcmSampling p = a.params[row];
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
    auto find = [&](bool by_mass, int tokens, double share, float floor) {
        Cut cut = {0.f, 0, 0, 0};
        float low = fmaxf(low_all, floor), high = high_all;
        // Weights end 32 temperatures below the largest; what lies lower is one bin until the cut is known to be there.
        const float reach = (float)(r.top - 32.0 * (double)p.temperature);
        float from = low < reach && reach < high ? reach : low;
        // A pass narrows the range a thousandfold, and FP32's spans less than 2^280: 64 are never reached.
        for (int pass = 0;; pass++) {
            const SampleBins bins(from, high, kSlowBins);
            auto open = [&](float l) { return l <= high && l >= low && l > floor; };
            __syncthreads();
            for (int i = tid; i < kSlowBins; i += kSampleThreads) mass[i] = 0, count[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kSampleThreads)
                if (open(x[i])) {
                    const int b = bins.of(x[i]);
                    atomicAdd(&count[b], 1u);
                    atomicAdd(&mass[b], r.weight(x[i]));
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
                    const bool here = by_mass ? c && (double)(heavier + sum) >= share : above + upto >= tokens;
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
                if (open(x[i]) && bins.of(x[i]) == bin) down = fminf(down, x[i]), up = fmaxf(up, x[i]);
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
                    const double need = ceil((share - (double)cut.weight) / (double)(w ? w : 1));
                    t = need < 1.0 ? 1 : need > (double)in_bin ? in_bin : (int)need;
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
    if (p.top_k > 0 && p.top_k < live) cut = find(false, p.top_k, 0.0, -INFINITY);
    if (p.top_p < 1.f) {
        u64 whole = cut.weight;
        if (cut.value == -INFINITY) {  // of the row
            u64 m = 0;
            for (int i = tid; i < n; i += kSampleThreads) m += r.weight(x[i]);
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
        const double share = fmax(0.0, (double)p.top_p) * (double)whole;
        // Inside the ties of top-k's cut, or above them.
        const u64 w = cut.value == -INFINITY ? 0 : r.weight(cut.value), above = cut.weight - w * (u64)cut.ties;
        if (cut.value != -INFINITY && (double)above < share) {
            const double need = ceil((share - (double)above) / (double)(w ? w : 1));
            const int t = need < 1.0 ? 1 : need > (double)cut.ties ? cut.ties : (int)need;
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
        for (int i = w0 + lane; i < w1; i += 32) t += x[i] == cut.value;
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
            const float l = i < w1 ? x[i] : -INFINITY;
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
    u64 target = (u64)((double)a.uniforms[row] * (double)whole);
    if (target >= whole) target = whole - 1;
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
            if (a.logprobs) a.logprobs[row] = (float)(r.exponent(x[i]) - log((double)whole / kSampleOne));
            if (a.kept) a.kept[row] = kept;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
        return reached != 0;
    });
}

// The first kResolve threads of a CTA settle the list.
constexpr int kResolve = 128;
__device__ __forceinline__ void resolve_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kResolve) : "memory"); }

__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) float slice_memory[];
    __shared__ __align__(16) SampleShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    auto started = cluster.barrier_arrive();  // no CTA's shared memory is written before the CTA runs
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int base = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - base);
    pdl_trigger();
    pdl_wait();
    const float *src = a.logits + (long long)row * a.stride + base;
    const TcmSampling p = a.params[row];
    const float u = a.uniforms[row];

    // ---- the slice, and what there is in it. It starts in shared memory as far from a 16-byte boundary as in global
    // memory, with -infinity around it, so that everything after this goes by whole quads.
    const int off = (int)((uintptr_t)src >> 2) & 3, quads = (off + n + 3) / 4;
    float *x = slice_memory + off;
    float4 *x4 = reinterpret_cast<float4 *>(slice_memory);
    float most = -INFINITY, least = INFINITY;
    bool bad = false;
    auto meet = [&](float l) {
        bad |= !(l < INFINITY);
        most = fmaxf(most, l), least = fminf(least, l);
    };
    const int q0 = off ? 1 : 0, q1 = (off + n) / 4;  // whole quads
#pragma unroll 4
    for (int q = q0 + tid; q < q1; q += kSampleThreads) {
        const float4 l = __ldcg(reinterpret_cast<const float4 *>(src - off) + q);
        x4[q] = l;
        meet(l.x), meet(l.y), meet(l.z), meet(l.w);
    }
    if (warp == 0) {  // the ends: lanes 0 .. 3 the first quad, 4 .. 7 the last
        const int i = (lane < 4 ? 0 : 4 * q1) + lane % 4 - off;  // of the slice
        if ((lane < 4 && q0) || (lane >= 4 && lane < 8 && q1 < quads && (q1 || !q0))) {
            const bool there = i >= 0 && i < n;
            const float l = there ? src[i] : -INFINITY;
            x[i] = l;
            if (there) meet(l);
        }
    }
    const uint32_t warp_most = __reduce_max_sync(0xffffffffu, sample_key(most));
    uint32_t warp_least = __reduce_min_sync(0xffffffffu, sample_key(least));
    bad = __any_sync(0xffffffffu, bad);
    int live = 0;
    const bool masked = __syncthreads_or(least == -INFINITY);
    if (masked) {  // what there is beside masked tokens
        least = INFINITY;
        for (int i = tid; i < n; i += kSampleThreads)
            if (x[i] > -INFINITY) live++, least = fminf(least, x[i]);
        warp_least = __reduce_min_sync(0xffffffffu, sample_key(least));
        live = __reduce_add_sync(0xffffffffu, live);
    }
    if (lane == 0) {
        sh.warp_count[warp] = live;
        reinterpret_cast<uint32_t *>(sh.warp_high)[warp] = warp_most, reinterpret_cast<uint32_t *>(sh.warp_low)[warp] = warp_least;
        sh.warp_mass[warp] = bad;
    }
    const bool ranked = p.top_k > 0 || p.top_p < 1.f;
    if (ranked)
        for (int i = tid; i < kSampleBins / 4; i += kSampleThreads) reinterpret_cast<uint4 *>(sh.buffer[0])[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) sh.listed = sh.list_count = 0, sh.list_before = sh.list_kept = 0;
    __syncthreads();
    cluster.barrier_wait(std::move(started));
    if (warp == 0) {  // lane c tells CTA c
        const int w = lane % kSampleWarps;
        SampleSlice z;
        z.most = __reduce_max_sync(0xffffffffu, reinterpret_cast<uint32_t *>(sh.warp_high)[w]);
        z.least = __reduce_min_sync(0xffffffffu, reinterpret_cast<uint32_t *>(sh.warp_low)[w]);
        z.live = __reduce_add_sync(0xffffffffu, lane < kSampleWarps ? sh.warp_count[w] : 0);
        z.bad = __any_sync(0xffffffffu, sh.warp_mass[w] != 0);
        if (!masked) z.live = n;
        if (lane < C) cluster.map_shared_rank(sh.slices, lane)[rank] = z;
    }
    cluster.sync();
    float high, low;
    int all_live;
    {
        const SampleSlice z = sh.slices[lane < C ? lane : 0];
        high = sample_value(__reduce_max_sync(0xffffffffu, z.most)), low = sample_value(__reduce_min_sync(0xffffffffu, z.least));
        all_live = __reduce_add_sync(0xffffffffu, lane < C ? z.live : 0);
        bad = __any_sync(0xffffffffu, z.bad);
    }
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
        for (int i = tid; i < n; i += kSampleThreads)
            if (x[i] == high) first = min(first, base + i);
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

    SampleRow r;
    r.top = high, r.cold = 1.0 / (double)p.temperature, r.slope = 1.4426950408889634074 * r.cold;
    // min-p as the least logit that it keeps: next to the one that arithmetic gives, the one that satisfies the definition.
    float min_logit = -FLT_MAX;
    if (p.min_p > 0.f) {
        const double coldest = log((double)p.min_p);
        float l = fmaxf((float)(r.top + coldest * (double)p.temperature), -FLT_MAX);
        if (!(r.exponent(l) >= coldest)) l = nextafterf(l, INFINITY);
        else if (l > -FLT_MAX && r.exponent(nextafterf(l, -INFINITY)) >= coldest) l = nextafterf(l, -INFINITY);
        min_logit = fminf(l, high);
    }

    // ---- the bins in which the cuts lie
    const bool by_count = p.top_k > 0 && p.top_k < all_live, by_mass = p.top_p < 1.f;
    const float reach = (float)(r.top - 32.0 * (double)p.temperature);
    const SampleBins bins(low < reach && reach < high ? reach : low, high, kSampleBins);
    int count_bin = kSampleBins, mass_from = kSampleBins, mass_to = -1;  // top-k's bin; top-p's, first and last
    int tokens_left = 0, in_count_bin = 0;                               // of top-k in its bin, and how many that has
    int listed = 0;
    if (by_count || by_mass) {
        unsigned *own = reinterpret_cast<unsigned *>(sh.buffer[0]), *counts = reinterpret_cast<unsigned *>(sh.buffer[1]);
        for (int q = tid; q < quads; q += kSampleThreads) {
            const float4 l = x4[q];
            if (l.x > -INFINITY) atomicAdd(&own[bins.of(l.x)], 1u);
            if (l.y > -INFINITY) atomicAdd(&own[bins.of(l.y)], 1u);
            if (l.z > -INFINITY) atomicAdd(&own[bins.of(l.z)], 1u);
            if (l.w > -INFINITY) atomicAdd(&own[bins.of(l.w)], 1u);
        }
        cluster.sync();
        // Each CTA adds up its share of the bins and tells the others.
        const int share_of = kSampleBins / C;
        for (int i = 4 * tid; i < share_of; i += 4 * kSampleThreads) {
            const int b = rank * share_of + i;
            uint4 c = make_uint4(0, 0, 0, 0);
#pragma unroll 8
            for (int k = 0; k < C; k++) {
                const uint4 y = *reinterpret_cast<const uint4 *>(cluster.map_shared_rank(own, k) + b);
                c.x += y.x, c.y += y.y, c.z += y.z, c.w += y.w;
            }
#pragma unroll 8
            for (int k = 0; k < C; k++) *reinterpret_cast<uint4 *>(cluster.map_shared_rank(counts, k) + b) = c;
        }
        if (tid == 0) sh.bin = kSampleBins, sh.mass_from = sh.mass_to = kSampleBins - 1;
        cluster.sync();
        constexpr int each = kSampleBins / kSampleThreads;
        unsigned c[each], upto = 0;
        float mass[each], total = 0.f;
        const float step = -bins.width() * (float)r.slope;
#pragma unroll
        for (int k = 0; k < each; k += 4) {
            const uint4 y = *reinterpret_cast<const uint4 *>(counts + tid * each + k);
            c[k] = y.x, c[k + 1] = y.y, c[k + 2] = y.z, c[k + 3] = y.w;
        }
#pragma unroll
        for (int k = 0; k < each; k++) {
            const int b = tid * each + k;
            mass[k] = b == kSampleBins - 1 ? 0.f : (float)c[k] * exp2f((float)b * step);
            upto += c[k], total += mass[k];
        }
        const unsigned mine = upto;
        const float mine_mass = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, upto, o);
            const float z = __shfl_up_sync(0xffffffffu, total, o);
            if (lane >= o) upto += y, total += z;
        }
        if (lane == 31) sh.warp_count[warp] = (int)upto, sh.warp_high[warp] = total;
        __syncthreads();
        unsigned before = upto - mine;
        float lighter = total - mine_mass, whole = 0.f;
#pragma unroll
        for (int w = 0; w < kSampleWarps; w++) {
            if (w < warp) before += (unsigned)sh.warp_count[w], lighter += sh.warp_high[w];
            whole += sh.warp_high[w];
        }
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
        listed = in_count_bin;
        if (by_mass) {
            // The bins at which the estimated sum passes the share, a little before and a little behind it.
            const float share = fmaxf(p.top_p, 0.f) * whole, slack = 2e-5f * whole;
            const int last = min(kSampleBins - 1, count_bin);
            float sum = lighter;
#pragma unroll
            for (int k = 0; k < each; k++) {
                const int b = tid * each + k;
                const float next = sum + mass[k];
                if (c[k]) {
                    if (sum < share - slack || before == 0) {
                        if (next >= share - slack) atomicMin(&sh.mass_from, b);
                    }
                    if ((sum < share + slack || before == 0) && next >= share + slack) atomicMin(&sh.mass_to, b);
                }
                before += c[k], sum = next;
            }
            before -= mine;
            __syncthreads();
            mass_from = min(sh.mass_from, last), mass_to = min(sh.mass_to, last);
            if (mass_to < mass_from) mass_to = mass_from;
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
        if (listed > kSampleList) {
            sample_slowly(a, r, sh, x, n, base, row, low, high, all_live, min_logit);
            return;
        }
    }

    // ---- weights above the bins, and the list of what is in them. A warp has a contiguous stretch of ids.
    const int kept_to = by_mass ? mass_from : count_bin;  // bins below this are kept whole
    const int per_warp = (quads + kSampleWarps - 1) / kSampleWarps, w0 = min(quads, warp * per_warp), w1 = min(quads, w0 + per_warp);
    u64 *own_list = sh.buffer[0], *list = sh.buffer[1];
    u64 sum_all = 0, sum_above = 0, sum_kept = 0;
    int kept = 0;
    if (by_count || by_mass) {
        const int needed = by_count ? count_bin : kSampleBins - 1;  // weights end here
        for (int q = w0 + lane; q < w1; q += 32) {
            const float4 y = x4[q];
            const float l[4] = {y.x, y.y, y.z, y.w};
            int b[4];
            bool any = false;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                b[k] = l[k] > -INFINITY ? bins.of(l[k]) : kSampleBins;
                any |= b[k] <= needed;
            }
            if (!any) continue;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if ((b[k] >= mass_from && b[k] <= mass_to) || (b[k] == count_bin && by_count))
                    own_list[atomicAdd(&sh.listed, 1)] = ((u64)~sample_key(l[k]) << 32) | (unsigned)(base + 4 * q + k - off);
            u64 w[4];
#pragma unroll
            for (int k = 0; k < 4; k++) w[k] = r.weight(l[k]);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (b[k] < count_bin) sum_all += w[k];
                if (b[k] < kept_to) {
                    sum_above += w[k];
                    if (l[k] >= min_logit) sum_kept += w[k], kept++;
                }
            }
        }
    } else {
        for (int q = w0 + lane; q < w1; q += 32) {
            const float4 y = x4[q];
            const float l[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const u64 w = r.weight(l[k]);
                if (l[k] >= min_logit) sum_kept += w, kept++;
            }
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
        z.listed = sh.listed;
        if (lane < C) cluster.map_shared_rank(sh.sums, lane)[rank] = z;
    }
    cluster.sync();
    if (warp == 1) {
        SampleSums z = {0, 0, 0, 0, 0};
        if (lane < C) z = sh.sums[lane];
        const u64 before = warp_sum64(lane < rank ? z.kept : 0), whole = warp_sum64(z.kept);
        if (by_mass) z.above = warp_sum64(z.above), z.all = warp_sum64(z.all);
        z.kept_count = __reduce_add_sync(0xffffffffu, z.kept_count);
        if (lane == 0) sh.before = before, sh.whole = whole, sh.heavier = z.above, sh.everything = z.all, sh.kept = z.kept_count, sh.cut = kSampleList;
    }
    if (lane == 0) sh.warp_more[warp] = 0;
    // ---- the list of the cluster, sorted by a few warps: logits descending, ids ascending
    if (by_count || by_mass) {
        const int m = listed;
        for (int c = 0, to = 0; c < C; c++) {
            const int k = sh.sums[c].listed;
            const u64 *from = cluster.map_shared_rank(own_list, c);
            for (int i = tid; i < k; i += kSampleThreads) list[to + i] = from[i];
            to += k;
        }
        cluster.barrier_arrive();  // the others' lists have been read; a CTA leaves when its own has
        int size = 32;
        while (size < m) size <<= 1;
        for (int i = m + tid; i < size; i += kSampleThreads) list[i] = ~0ull;
        __syncthreads();
        if (tid < kResolve) {
            for (int k = 2; k <= size; k <<= 1)
                for (int j = k >> 1; j; j >>= 1) {
                    for (int i = tid; i < size / 2; i += kResolve) {
                        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                        const u64 y = list[lo], z = list[hi];
                        if ((y > z) == ((lo & k) == 0)) list[lo] = z, list[hi] = y;
                    }
                    resolve_barrier();
                }
            auto logit_at = [&](int i) { return sample_value(~(uint32_t)(list[i] >> 32)); };
            const int each = size > kResolve ? size / kResolve : 1, i0 = min(m, tid * each), i1 = min(m, i0 + each);
            int cut = tokens_left - 1;
            bool fine = true;
            if (by_mass) {
                // Sums of weights up to each thread's places.
                u64 mine = 0;
                for (int i = i0; i < i1; i++) mine += r.weight(logit_at(i));
                u64 upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                if (lane == 31) sh.warp_mass[warp] = upto;
                resolve_barrier();
                upto -= mine;
                for (int k = 0; k < warp; k++) upto += sh.warp_mass[k];
                u64 all_of = sh.everything;
                const int first = m - in_count_bin, last = first + tokens_left - 1;  // of top-k's bin, its tokens
                if (by_count) {
                    u64 sum = upto;
                    for (int i = i0; i < i1; i++) {
                        if (i == first) sh.at_first = sum;
                        sum += r.weight(logit_at(i));
                        if (i == last) sh.at_last = sum;
                    }
                    resolve_barrier();
                    all_of += sh.at_last - sh.at_first;
                }
                const double share = fmax(0.0, (double)p.top_p) * (double)all_of;
                fine = mass_from == 0 || (double)sh.heavier < share;
                u64 sum = sh.heavier + upto;
                int i = i0;
                for (; i < i1; i++) {
                    sum += r.weight(logit_at(i));
                    if ((double)sum >= share) break;
                }
                if (i < i1 && (i == 0 || (double)(sum - r.weight(logit_at(i))) < share)) sh.cut = i;
                resolve_barrier();
                cut = sh.cut;
                // In top-p's bins, or the estimate was wrong.
                fine = fine && cut < m && (!by_count || cut <= last);
                if (fine) fine = bins.of(logit_at(cut)) <= mass_to;
            }
            if (tid == 0) {
                sh.settled = fine;
                if (fine) sh.cut_key = ~(uint32_t)(list[cut] >> 32), sh.cut_id = (unsigned)list[cut];
            }
            if (fine) {  // what is kept of the list, by where it is
                for (int i = i0; i < i1 && i <= cut; i++) {
                    const float l = logit_at(i);
                    if (l < min_logit) continue;
                    const u64 w = r.weight(l);
                    const int at = (int)(unsigned)list[i] - base;
                    atomicAdd(&sh.list_kept, w);
                    atomicAdd(&sh.list_count, 1);
                    if (at < 0) atomicAdd(&sh.list_before, w);
                    else if (at < n) atomicAdd(&sh.warp_more[(at + off) / 4 / per_warp], w);
                }
            }
        }
    }
    __syncthreads();
    float cut_value = -INFINITY;
    unsigned cut_id = 0;
    u64 whole = sh.whole, before = sh.before;
    if (by_count || by_mass) {
        if (!sh.settled) {  // the whole cluster alike
            cluster.barrier_wait();
            sample_slowly(a, r, sh, x, n, base, row, low, high, all_live, min_logit);
            return;
        }
        cut_value = sample_value(sh.cut_key), cut_id = sh.cut_id;
        whole += sh.list_kept, before += sh.list_before;
    }
    u64 target = (u64)((double)u * (double)whole);
    if (target >= whole) target = whole - 1;
    {
        const u64 w = lane < kSampleWarps ? sh.warp_kept[lane] + sh.warp_more[lane] : 0;  // of each warp's stretch
        before += warp_sum64(lane < warp ? w : 0);
        const u64 own = __shfl_sync(0xffffffffu, w, warp);
        if (target >= before && target < before + own) {  // one warp of the cluster has the token
            for (int q0 = w0; q0 < w1; q0 += 32) {
                const int q = q0 + lane;
                const float4 y = q < w1 ? x4[q] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                const float l[4] = {y.x, y.y, y.z, y.w};
                u64 w4[4], mine = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const unsigned id = (unsigned)(base + 4 * q + k - off);
                    const bool stays = (l[k] > cut_value || (l[k] == cut_value && id <= cut_id)) && l[k] >= min_logit;
                    w4[k] = r.weight(l[k]);
                    if (!stays) w4[k] = 0;
                    mine += w4[k];
                }
                u64 upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 z = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += z;
                }
                const unsigned reached = __ballot_sync(0xffffffffu, before + upto > target);
                if (reached) {
                    if (lane == __ffs(reached) - 1) {
                        u64 sum = before + upto;
                        int id = 0;
                        float logit = 0.f;
#pragma unroll
                        for (int k = 3; k >= 0; k--) {  // the first of the four at which the sum passes the target
                            if (sum > target && w4[k]) id = base + 4 * q + k - off, logit = l[k];
                            sum -= w4[k];
                        }
                        a.ids[row] = id;
                        if (a.logprobs) a.logprobs[row] = (float)(r.exponent(logit) - log((double)whole / kSampleOne));
                        if (a.kept) a.kept[row] = sh.kept + ((by_count || by_mass) ? sh.list_count : 0);
                    }
                    break;
                }
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
    }
    if (by_count || by_mass) cluster.barrier_wait();
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
        TCM_CUDA(cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kSampleSlice + 8) * 4));
        TCM_CUDA(cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    });
    // Few rows take all the SMs that help; many rows the fewest CTAs whose slices leave room for two an SM.
    int cluster = kSampleCluster;
    while (cluster > 1 && (vocab < cluster * 1024 || (rows * cluster > 2 * sm_count() && vocab <= cluster / 2 * 19456))) cluster /= 2;
    const int slice = ((vocab + cluster - 1) / cluster + 3) / 4 * 4;
    const SampleArgs args = {ids, logprobs, kept, logits, stride, vocab, slice, params, uniforms, status};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * cluster);
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = (size_t)(slice + 8) * 4;
    cfg.stream = stream();
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)cluster, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    TCM_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel, args));
    return 0;
}
