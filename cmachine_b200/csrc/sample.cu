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
// What bounds it: the weights' 15 FP64 instructions an element (28 cycles of an SM's quarter) beside HBM.
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
    float most, least;  // of the logits above -infinity
    int live, bad;      // logits above -infinity; a NaN or +infinity among them
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
    u64 list_before, list_kept, at_first, at_last;
    int listed, list_count;
    int bin, above, in_bin;  // of top-k's cut
    int mass_bin;            // of top-p's, estimated
    int cut;                 // index in the list
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

// 2^f = sum of (f ln 2)^k / k!: for |f| <= 1/2 the terms from the tenth on are below 2^-37 together.
struct SampleSeries {
    double c[10];
    constexpr SampleSeries() : c() {
        c[0] = 1.0;
        for (int k = 1; k < 10; k++) c[k] = c[k - 1] * 0.69314718055994530942 / k;
    }
};
__device__ constexpr SampleSeries kSampleSeries{};

struct SampleRow {
    double top, cold, slope;  // the largest logit, 1 / T, log2(e) / T
    __device__ double exponent(float l) const { return ((double)l - top) * cold; }
    __device__ u64 weight(float l) const {
        const double y0 = ((double)l - top) * slope;
        // At most zero; from -64 on (its upper word decides) nothing is left of it.
        const double y = __hiloint2double((int)min((unsigned)__double2hiint(y0), 0xc0500000u), __double2loint(y0));
        const double t = y + 0x1.8p52, f = y - (t - 0x1.8p52);
        double z = kSampleSeries.c[9];
#pragma unroll
        for (int k = 8; k >= 0; k--) z = fma(z, f, kSampleSeries.c[k]);
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
    __device__ double middle(int b) const { return scale > 0.f ? (double)b / ((double)scale * (double)unit) : 0.0; }  // below high
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

    // ---- the slice, and what there is in it. It starts in shared memory as far from a 16-byte boundary as in global memory.
    const int off = (int)((uintptr_t)src >> 2) & 3;
    float *x = slice_memory + off;
    float most = -INFINITY, least = INFINITY;
    bool bad = false;
    auto meet = [&](float l) {
        bad |= !(l < INFINITY);
        most = fmaxf(most, l), least = fminf(least, l);
    };
    const int head = min(n, (4 - off) & 3), quads = (n - head) / 4;
    if (tid < head) {
        const float l = src[tid];
        x[tid] = l;
        meet(l);
    }
#pragma unroll 4
    for (int i = tid; i < quads; i += kSampleThreads) {
        const float4 l = __ldcg(reinterpret_cast<const float4 *>(src + head) + i);
        reinterpret_cast<float4 *>(x + head)[i] = l;
        meet(l.x), meet(l.y), meet(l.z), meet(l.w);
    }
    if (tid < (n - head) % 4) {
        const int i = head + 4 * quads + tid;
        const float l = src[i];
        x[i] = l;
        meet(l);
    }
    most = warp_max(most);
    least = -warp_max(-least);
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) sh.warp_high[warp] = most, sh.warp_low[warp] = least, sh.warp_count[warp] = bad;
    __syncthreads();
    int live = n;
    {
        float low = INFINITY;
        for (int w = 0; w < kSampleWarps; w++) low = fminf(low, sh.warp_low[w]);
        if (low == -INFINITY) {  // masked tokens: what else there is
            int count = 0;
            least = INFINITY;
            for (int i = tid; i < n; i += kSampleThreads)
                if (x[i] > -INFINITY) count++, least = fminf(least, x[i]);
            least = -warp_max(-least);
            count = __reduce_add_sync(0xffffffffu, count);
            __syncthreads();
            if (lane == 0) sh.warp_low[warp] = least, sh.warp_mass[warp] = count;
            __syncthreads();
            live = 0;
            for (int w = 0; w < kSampleWarps; w++) live += (int)sh.warp_mass[w];
        }
    }
    cluster.barrier_wait(std::move(started));
    if (tid < C) {  // thread c tells CTA c
        SampleSlice z = {-INFINITY, INFINITY, live, 0};
        for (int w = 0; w < kSampleWarps; w++) {
            z.most = fmaxf(z.most, sh.warp_high[w]), z.least = fminf(z.least, sh.warp_low[w]);
            z.bad |= sh.warp_count[w];
        }
        cluster.map_shared_rank(sh.slices, tid)[rank] = z;
    }
    for (int i = tid; i < kSampleBins / 2; i += kSampleThreads) sh.buffer[0][i] = 0;
    if (tid == 0) sh.listed = sh.list_count = 0, sh.list_before = sh.list_kept = 0;
    cluster.sync();
    SampleSlice all = sh.slices[0];
    for (int c = 1; c < C; c++) {
        const SampleSlice &z = sh.slices[c];
        all.most = fmaxf(all.most, z.most), all.least = fminf(all.least, z.least);
        all.live += z.live;
        all.bad |= z.bad;
    }
    const bool wrong = !(p.temperature >= 0.f && p.temperature < INFINITY && u >= 0.f && u < 1.f && p.min_p <= 1.f) ||
                       p.top_p != p.top_p;
    if (all.bad || !all.live || wrong) {  // the whole cluster alike
        if (rank == 0 && tid == 0) {
            a.ids[row] = -1;
            if (a.logprobs) a.logprobs[row] = 0.f;
            if (a.kept) a.kept[row] = 0;
            if (a.status) atomicOr(a.status, (all.bad ? 1 : 0) | (!all.bad && !all.live ? 2 : 0) | (wrong ? 4 : 0));
        }
        return;
    }
    if (p.temperature == 0.f) {
        int first = 0x7fffffff;
        for (int i = tid; i < n; i += kSampleThreads)
            if (x[i] == all.most) first = min(first, base + i);
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0) sh.warp_count[warp] = first;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < kSampleWarps; w++) first = min(first, sh.warp_count[w]);
            cluster.map_shared_rank(sh.first, 0)[rank] = first;
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
    r.top = all.most, r.cold = 1.0 / (double)p.temperature, r.slope = 1.4426950408889634074 * r.cold;
    // min-p as the least logit that it keeps: next to the one that arithmetic gives, the one that satisfies the definition.
    float min_logit = -FLT_MAX;
    if (p.min_p > 0.f) {
        const double coldest = log((double)p.min_p);
        float l = fmaxf((float)(r.top + coldest * (double)p.temperature), -FLT_MAX);
        if (!(r.exponent(l) >= coldest)) l = nextafterf(l, INFINITY);
        else if (l > -FLT_MAX && r.exponent(nextafterf(l, -INFINITY)) >= coldest) l = nextafterf(l, -INFINITY);
        min_logit = fminf(l, all.most);
    }

    // ---- the bins in which the cuts lie
    const bool by_count = p.top_k > 0 && p.top_k < all.live, by_mass = p.top_p < 1.f;
    const float reach = (float)(r.top - 32.0 * (double)p.temperature);
    const SampleBins bins(all.least < reach && reach < all.most ? reach : all.least, all.most, kSampleBins);
    int count_bin = kSampleBins, mass_from = kSampleBins, mass_to = -1;  // top-k's bin; top-p's, first and last
    int tokens_left = 0, in_count_bin = 0;                               // of top-k in its bin, and how many that has
    int listed_all = 0;
    if (by_count || by_mass) {
        unsigned *own = reinterpret_cast<unsigned *>(sh.buffer[0]), *counts = reinterpret_cast<unsigned *>(sh.buffer[1]);
        for (int i = tid; i < n; i += kSampleThreads)
            if (x[i] > -INFINITY) atomicAdd(&own[bins.of(x[i])], 1u);
        cluster.sync();
        // Each CTA adds up its share of the bins and tells the others.
        const int share_of = kSampleBins / C;
        for (int i = tid; i < share_of; i += kSampleThreads) {
            const int b = rank * share_of + i;
            unsigned c = 0;
#pragma unroll 8
            for (int k = 0; k < C; k++) c += cluster.map_shared_rank(own, k)[b];
#pragma unroll 8
            for (int k = 0; k < C; k++) cluster.map_shared_rank(counts, k)[b] = c;
        }
        cluster.sync();
        constexpr int each = kSampleBins / kSampleThreads;
        unsigned c[each], upto = 0;
        float mass[each], total = 0.f;
#pragma unroll
        for (int k = 0; k < each; k++) {
            const int b = tid * each + k;
            c[k] = counts[b];
            mass[k] = b == bins.last ? 0.f : (float)c[k] * exp2f((float)(-bins.middle(b) * r.slope));
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
        if (tid == 0) sh.mass_bin = bins.last, sh.bin = kSampleBins;
        __syncthreads();
        unsigned before = upto - mine;
        float lighter = total - mine_mass, whole = 0.f;
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
                        sh.ends[0].x = heavier + mass[b] * ((float)(k - above) / (float)c[b]);
                    }
                    above += c[b], heavier += mass[b];
                }
            }
            __syncthreads();
            count_bin = sh.bin, tokens_left = p.top_k - sh.above, in_count_bin = sh.in_bin;
            whole = sh.ends[0].x;
        }
        if (by_mass) {
            const float share = fmaxf(p.top_p, 0.f) * whole;
            int here = kSampleBins;
#pragma unroll
            for (int b = each - 1; b >= 0; b--) {
                float sum = lighter;
#pragma unroll
                for (int m = 0; m <= b; m++) sum += mass[m];
                if (c[b] && sum >= share) here = tid * each + b;
            }
            if (here < kSampleBins && (lighter < share || !(share > 0.f))) atomicMin(&sh.mass_bin, here);
            __syncthreads();
            const int bin = min(sh.mass_bin, count_bin < kSampleBins ? count_bin : bins.last);
            mass_from = max(bin - 1, 0), mass_to = min(bin + 1, count_bin < kSampleBins ? count_bin : bins.last);
        }
        // How many tokens these bins hold: within a list, or the slow way. The estimate's neighbours only where they fit.
        for (int tries = 0; tries < 2; tries++) {
            int listed = 0;
#pragma unroll
            for (int k = 0; k < each; k++) {
                const int b = tid * each + k;
                if ((b >= mass_from && b <= mass_to) || b == count_bin) listed += (int)c[k];
            }
            listed = __reduce_add_sync(0xffffffffu, listed);
            __syncthreads();
            if (lane == 0) sh.warp_count[warp] = listed;
            __syncthreads();
            listed_all = 0;
            for (int w = 0; w < kSampleWarps; w++) listed_all += sh.warp_count[w];
            if (listed_all <= kSampleList || !by_mass || tries) break;
            mass_from = mass_to = min(sh.mass_bin, count_bin < kSampleBins ? count_bin : bins.last);
        }
        if (listed_all > kSampleList) {
            sample_slowly(a, r, sh, x, n, base, row, all.least, all.most, all.live, min_logit);
            return;
        }
    }

    // ---- weights above the bins, and the list of what is in them. A warp has a contiguous stretch of ids.
    const int kept_to = by_mass ? mass_from : count_bin;  // bins below this are kept whole
    const int per_warp = (n + kSampleWarps - 1) / kSampleWarps, w0 = min(n, warp * per_warp), w1 = min(n, w0 + per_warp);
    u64 *own_list = sh.buffer[0], *list = sh.buffer[1];
    SampleSums sums = {0, 0, 0, 0, 0};
    if (by_count || by_mass) {
        const int needed = max(by_mass ? mass_to : 0, by_count ? count_bin : by_mass ? bins.last : 0);  // weights end here
        for (int i = w0 + lane; i < w1; i += 32) {
            const float l = x[i];
            const int b = l > -INFINITY ? bins.of(l) : kSampleBins;
            if (b > needed) continue;
            if ((b >= mass_from && b <= mass_to) || b == count_bin)
                own_list[atomicAdd(&sh.listed, 1)] = ((u64)~sample_key(l) << 32) | (unsigned)(base + i);
            const bool below = b < kept_to;
            if (!by_mass && !below) continue;
            const u64 w = r.weight(l);
            if (b < count_bin) sums.all += w;
            if (below) {
                sums.above += w;
                if (l >= min_logit) sums.kept += w, sums.kept_count++;
            }
        }
    } else {
        for (int i = w0 + lane; i < w1; i += 32) {
            const float l = x[i];
            if (l >= min_logit) sums.kept += r.weight(l), sums.kept_count++;
        }
    }
    sums.all = warp_sum64(sums.all), sums.above = warp_sum64(sums.above), sums.kept = warp_sum64(sums.kept);
    sums.kept_count = __reduce_add_sync(0xffffffffu, sums.kept_count);
    const u64 warp_kept = sums.kept;
    if (lane == 0) {
        sh.warp_mass[warp] = sums.all, sh.warp_more[warp] = sums.above, sh.warp_kept[warp] = sums.kept;
        sh.warp_count[warp] = sums.kept_count;
    }
    __syncthreads();
    if (tid < C) {
        SampleSums z = {0, 0, 0, 0, sh.listed};
        for (int w = 0; w < kSampleWarps; w++) {
            z.all += sh.warp_mass[w], z.above += sh.warp_more[w], z.kept += sh.warp_kept[w];
            z.kept_count += sh.warp_count[w];
        }
        cluster.map_shared_rank(sh.sums, tid)[rank] = z;
    }
    cluster.sync();
    u64 whole = 0, before = 0, heavier = 0, everything = 0;
    int kept = 0;
    for (int c = 0; c < C; c++) {
        const SampleSums &z = sh.sums[c];
        if (c < rank) before += z.kept;
        whole += z.kept, heavier += z.above, everything += z.all;
        kept += z.kept_count;
    }
    for (int w = 0; w < warp; w++) before += sh.warp_kept[w];
    float cut_value = -INFINITY;
    unsigned cut_id = 0;
    u64 warp_listed = 0;  // kept weights of the list in this warp's stretch
    bool gathered = false;
    if (by_count || by_mass) {
        // ---- the list of the cluster, sorted: logits descending, ids ascending
        const int m = listed_all;
        for (int c = 0, to = 0; c < C; c++) {
            const int k = sh.sums[c].listed;
            const u64 *from = cluster.map_shared_rank(own_list, c);
            for (int i = tid; i < k; i += kSampleThreads) list[to + i] = from[i];
            to += k;
        }
        cluster.barrier_arrive();  // the others' lists have been read; a CTA leaves when its own has
        gathered = true;
        int size = 32;
        while (size < m) size <<= 1;
        for (int i = m + tid; i < size; i += kSampleThreads) list[i] = ~0ull;
        for (int k = 2; k <= size; k <<= 1)
            for (int j = k >> 1; j; j >>= 1) {
                __syncthreads();
                for (int i = tid; i < size / 2; i += kSampleThreads) {
                    const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                    const u64 y = list[lo], z = list[hi];
                    if ((y > z) == ((lo & k) == 0)) list[lo] = z, list[hi] = y;
                }
            }
        __syncthreads();
        // Sums of weights up to each place of the list, four places a thread.
        constexpr int each = kSampleList / kSampleThreads;
        u64 w[each], upto = 0;
#pragma unroll
        for (int k = 0; k < each; k++) {
            const int i = tid * each + k;
            w[k] = i < m && (by_mass || by_count) ? r.weight(sample_value(~(uint32_t)(list[min(i, kSampleList - 1)] >> 32))) : 0;
            upto += w[k];
        }
        const u64 mine = upto;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        if (lane == 31) sh.warp_mass[warp] = upto;
        if (tid == 0) sh.cut = kSampleList, sh.at_first = 0;
        __syncthreads();
        upto -= mine;
        for (int k = 0; k < warp; k++) upto += sh.warp_mass[k];
        int cut = kSampleList;
        bool fine = true;
        const int first_counted = m - in_count_bin, last_counted = first_counted + tokens_left - 1;  // of top-k's bin
        if (by_count) cut = last_counted;
        if (by_mass) {
            u64 all_of = everything;
            if (by_count) {
                u64 sum = upto;
#pragma unroll
                for (int k = 0; k < each; k++) {
                    if (tid * each + k == first_counted) sh.at_first = sum;
                    sum += w[k];
                    if (tid * each + k == last_counted) sh.at_last = sum;
                }
                __syncthreads();
                all_of += sh.at_last - sh.at_first;
            }
            const double share = fmax(0.0, (double)p.top_p) * (double)all_of;
            fine = mass_from == 0 || (double)heavier < share;
            u64 sum = heavier + upto;
            int here = kSampleList;
#pragma unroll
            for (int k = 0; k < each; k++) {
                sum += w[k];
                if (here == kSampleList && tid * each + k < m && (double)sum >= share) here = tid * each + k;
            }
            if (here < kSampleList) atomicMin(&sh.cut, here);
            __syncthreads();
            cut = sh.cut;
            // In top-p's bins, or the estimate was wrong.
            fine = fine && cut < m && (!by_count || cut <= last_counted);
            if (fine) fine = bins.of(sample_value(~(uint32_t)(list[cut] >> 32))) <= mass_to;
        }
        if (!fine) {  // the whole cluster alike
            cluster.barrier_wait();
            sample_slowly(a, r, sh, x, n, base, row, all.least, all.most, all.live, min_logit);
            return;
        }
        const u64 last = list[cut];
        cut_value = sample_value(~(uint32_t)(last >> 32)), cut_id = (unsigned)last;
        // What is kept of the list, by where it is.
        if (lane == 0) sh.warp_more[warp] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < each; k++) {
            const int i = tid * each + k;
            if (i > cut || i >= m) continue;
            const u64 y = list[i];
            if (sample_value(~(uint32_t)(y >> 32)) < min_logit) continue;
            const int at = (int)(unsigned)y - base;
            atomicAdd(&sh.list_kept, w[k]);
            atomicAdd(&sh.list_count, 1);
            if (at < 0) atomicAdd(&sh.list_before, w[k]);
            else if (at < n) atomicAdd(&sh.warp_more[at / per_warp], w[k]);
        }
        __syncthreads();
        whole += sh.list_kept, kept += sh.list_count, before += sh.list_before;
        for (int k = 0; k < warp; k++) before += sh.warp_more[k];
        warp_listed = sh.warp_more[warp];
    }
    u64 target = (u64)((double)u * (double)whole);
    if (target >= whole) target = whole - 1;
    if (target >= before && target < before + warp_kept + warp_listed) {  // one warp of the cluster has the token
        for (int i0 = w0; i0 < w1; i0 += 32) {
            const int i = i0 + lane;
            const float l = i < w1 ? x[i] : -INFINITY;
            const bool stays = (l > cut_value || (l == cut_value && (unsigned)(base + i) <= cut_id)) && l >= min_logit;
            u64 upto = stays ? r.weight(l) : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            const unsigned reached = __ballot_sync(0xffffffffu, before + upto > target);
            if (reached) {
                if (lane == __ffs(reached) - 1) {
                    a.ids[row] = base + i;
                    if (a.logprobs) a.logprobs[row] = (float)(r.exponent(l) - log((double)whole / kSampleOne));
                    if (a.kept) a.kept[row] = kept;
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    if (gathered) cluster.barrier_wait();
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
        TCM_CUDA(cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kSampleSlice + 4) * 4));
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
    cfg.dynamicSmemBytes = (size_t)(slice + 4) * 4;
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
