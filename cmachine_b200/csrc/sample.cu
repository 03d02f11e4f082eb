// Sampling: one token a row of logits, with temperature, top-k, top-p and min-p, by a given uniform number.
//
// A thread-block cluster has one row. Each of its CTAs brings a contiguous slice of the row into shared memory, and
// everything after that runs on chip: the row is read from HBM once. All three filters keep a prefix of the tokens in
// descending order of their logits, so what is kept is described by a cut: a logit, and how many of the tokens at it (by
// id) still belong. The cut is found by histograms of counts and weights over the range of logits in which it must lie,
// then over the bin that it falls into, until that holds one value; the whole row is never sorted.
//
// Weights exp((l - max) / T) are whole numbers, 2^44 for the largest: their sums are exact whatever the order, so
// atomics keep results the same from call to call, and a sum of 2^19 of them stays below 2^64.
#include "common.cuh"
#include "kernels.h"
#include "../../include/gpu.h"
#include <cooperative_groups.h>
#include <math.h>
#include <utility>

namespace cg = cooperative_groups;

namespace tcm {
namespace {

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32, kSampleBins = 1024;
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

// What a CTA of the cluster knows of its slice.
struct SampleSlice {
    float most, least;  // of the logits above -infinity
    int first;          // the lowest id at `most`
    int live, bad;      // logits above -infinity; a NaN or +infinity among them
};

struct SampleShared {
    SampleSlice slices[kSampleCluster];
    u64 mass[kSampleBins];
    unsigned count[kSampleBins];
    u64 all_mass[kSampleBins];      // of the cluster
    unsigned all_count[kSampleBins];
    float2 ends[kSampleCluster];    // least and largest logit of the cut's bin
    u64 part_mass[kSampleCluster];
    int part_count[kSampleCluster];
    u64 warp_mass[kSampleWarps];
    int warp_count[kSampleWarps];
    float warp_low[kSampleWarps], warp_high[kSampleWarps];
    u64 cut_mass;  // above the cut's bin
    int cut_bin, cut_above, cut_count;
};

__device__ __forceinline__ u64 warp_sum64(u64 x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// The cut: tokens above `value` and the first `ties` at it. Among them `count` tokens of weight `mass`.
struct SampleCut {
    float value;
    int ties;
    int count;
    u64 mass;
};

__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) float x[];  // the slice
    __shared__ SampleShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    auto started = cluster.barrier_arrive();  // no CTA's shared memory is written before the CTA runs
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int base = rank * a.slice, n = max(0, min(a.slice, a.vocab - base));
    pdl_trigger();
    pdl_wait();
    const float *src = a.logits + (long long)row * a.stride + base;

    // ---- the slice, and what there is in it
    float most = -INFINITY, least = INFINITY;
    int first = 0x7fffffff, live = 0, bad = 0;
#pragma unroll 8
    for (int i = tid; i < n; i += kSampleThreads) {
        const float l = src[i];
        x[i] = l;
        bad |= !(l < INFINITY);
        if (l > -INFINITY) {
            live++;
            least = fminf(least, l);
            if (l > most) most = l, first = base + i;
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float m = __shfl_xor_sync(0xffffffffu, most, o);
        const int f = __shfl_xor_sync(0xffffffffu, first, o);
        if (m > most || (m == most && f < first)) most = m, first = f;
    }
    least = -warp_max(-least);
    live = __reduce_add_sync(0xffffffffu, live);
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
        sh.warp_high[warp] = most, sh.warp_low[warp] = least;
        sh.warp_count[warp] = live, sh.warp_mass[warp] = ((u64)(unsigned)first << 1) | bad;
    }
    __syncthreads();
    cluster.barrier_wait(std::move(started));
    if (tid < C) {  // thread c tells CTA c
        SampleSlice z = {-INFINITY, INFINITY, 0x7fffffff, 0, 0};
        for (int w = 0; w < kSampleWarps; w++) {
            const int f = (int)(sh.warp_mass[w] >> 1);
            if (sh.warp_high[w] > z.most || (sh.warp_high[w] == z.most && f < z.first)) z.most = sh.warp_high[w], z.first = f;
            z.least = fminf(z.least, sh.warp_low[w]);
            z.live += sh.warp_count[w];
            z.bad |= (int)(sh.warp_mass[w] & 1);
        }
        cluster.map_shared_rank(&sh, tid)->slices[rank] = z;
    }
    cluster.sync();
    SampleSlice all = sh.slices[0];
    for (int c = 1; c < C; c++) {
        const SampleSlice &z = sh.slices[c];
        if (z.most > all.most) all.most = z.most, all.first = z.first;
        all.least = fminf(all.least, z.least);
        all.live += z.live;
        all.bad |= z.bad;
    }
    const TcmSampling p = a.params[row];
    const float u = a.uniforms[row];
    const bool wrong = !(p.temperature >= 0.f && p.temperature < INFINITY && u >= 0.f && u < 1.f && p.min_p <= 1.f) ||
                       p.top_p != p.top_p;
    if (all.bad || !all.live || wrong || p.temperature == 0.f) {  // the whole cluster alike
        if (rank == 0 && tid == 0) {
            const bool none = all.bad || !all.live || wrong;
            a.ids[row] = none ? -1 : all.first;
            if (a.logprobs) a.logprobs[row] = 0.f;
            if (a.kept) a.kept[row] = none ? 0 : 1;
            if (none && a.status) atomicOr(a.status, (all.bad ? 1 : 0) | (!all.bad && !all.live ? 2 : 0) | (wrong ? 4 : 0));
        }
        return;
    }

    const double top = all.most, cold = 1.0 / (double)p.temperature;
    auto exponent = [&](float l) { return ((double)l - top) * cold; };
    auto weight = [&](float l) { return __double2ull_rn(exp(exponent(l)) * kSampleOne); };

    // The least prefix of the tokens above `floor` that holds `tokens` of them (by_mass false) or weighs `share` or more.
    // There is one. All threads of the cluster call it.
    auto find = [&](bool by_mass, int tokens, double share, float floor) {
        SampleCut cut = {0.f, 0, 0, 0};
        float low = fmaxf(all.least, floor), high = all.most;
        // Weights end 32 temperatures below the largest; what lies lower is one bin until the cut is known to be there.
        const float reach = (float)(top - 32.0 * (double)p.temperature);
        float from = low < reach && reach < high ? reach : low;
        // A pass narrows the range a thousandfold, and FP32's spans less than 2^280: 64 are never reached.
        for (int pass = 0;; pass++) {
            // Differences in a power of two at which neither they nor the scale leave FP32's range.
            const float span = high - from, unit = span > 1e30f ? 0.25f : span < 1e-25f ? 0x1p100f : 1.f;
            const float scale = (kSampleBins - 1) * 0.9999f / (high * unit - from * unit);
            auto bin_of = [&](float l) {  // 0 for `high`, the last but one for `from`, and not falling as l falls
                return l < from ? kSampleBins - 1 : (int)((high * unit - l * unit) * scale);
            };
            auto open = [&](float l) { return l <= high && l >= low && l > floor; };
            for (int i = tid; i < kSampleBins; i += kSampleThreads) sh.mass[i] = 0, sh.count[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kSampleThreads)
                if (open(x[i])) {
                    const int b = bin_of(x[i]);
                    atomicAdd(&sh.count[b], 1u);
                    atomicAdd(&sh.mass[b], weight(x[i]));
                }
            cluster.sync();
            // Each CTA adds up its share of the bins and tells the others.
            const int share_of = kSampleBins / C;
            for (int i = tid; i < share_of; i += kSampleThreads) {
                const int b = rank * share_of + i;
                unsigned c = 0;
                u64 m = 0;
#pragma unroll 4
                for (int k = 0; k < C; k++) {
                    const SampleShared *o = cluster.map_shared_rank(&sh, k);
                    c += o->count[b], m += o->mass[b];
                }
                for (int k = 0; k < C; k++) {
                    SampleShared *o = cluster.map_shared_rank(&sh, k);
                    o->all_count[b] = c, o->all_mass[b] = m;
                }
            }
            cluster.sync();
            if (warp == 0) {
                int above = cut.count;
                u64 heavier = cut.mass;
                for (int b = 0; b < kSampleBins; b += 32) {
                    int c = (int)sh.all_count[b + lane], upto = c;
                    u64 m = sh.all_mass[b + lane], sum = m;
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
                            sh.cut_bin = b + lane, sh.cut_above = above + upto - c, sh.cut_count = c, sh.cut_mass = heavier + sum - m;
                        break;
                    }
                    above += __shfl_sync(0xffffffffu, upto, 31);
                    heavier += __shfl_sync(0xffffffffu, sum, 31);
                }
            }
            __syncthreads();
            const int bin = sh.cut_bin;
            cut.count = sh.cut_above;
            cut.mass = sh.cut_mass;
            float down = INFINITY, up = -INFINITY;
            for (int i = tid; i < n; i += kSampleThreads)
                if (open(x[i]) && bin_of(x[i]) == bin) down = fminf(down, x[i]), up = fmaxf(up, x[i]);
            down = -warp_max(-down), up = warp_max(up);
            if (lane == 0) sh.warp_low[warp] = down, sh.warp_high[warp] = up;
            __syncthreads();
            if (tid < C) {
                for (int w = 0; w < kSampleWarps; w++) down = fminf(down, sh.warp_low[w]), up = fmaxf(up, sh.warp_high[w]);
                cluster.map_shared_rank(&sh, tid)->ends[rank] = make_float2(down, up);
            }
            const int in_bin = sh.cut_count;
            cluster.sync();
            down = INFINITY, up = -INFINITY;
            for (int c = 0; c < C; c++) down = fminf(down, sh.ends[c].x), up = fmaxf(up, sh.ends[c].y);
            low = from = down, high = up;
            if (low == high || pass == 63) {  // one value: how many of its tokens
                const u64 w = weight(low);
                int t;
                if (!by_mass) t = tokens - cut.count;
                else {
                    const double need = ceil((share - (double)cut.mass) / (double)(w ? w : 1));
                    t = need < 1.0 ? 1 : need > (double)in_bin ? in_bin : (int)need;
                }
                cut.value = low, cut.ties = t;
                cut.count += t;
                cut.mass += w * (u64)t;
                return cut;
            }
        }
    };

    // ---- top-k, then top-p of what it leaves
    SampleCut cut = {-INFINITY, 0, all.live, 0};
    if (p.top_k > 0 && p.top_k < all.live) cut = find(false, p.top_k, 0.0, -INFINITY);
    if (p.top_p < 1.f) {
        u64 whole = cut.mass;
        if (cut.value == -INFINITY) {  // of the row
            u64 m = 0;
            for (int i = tid; i < n; i += kSampleThreads)
                if (x[i] > -INFINITY) m += weight(x[i]);
            m = warp_sum64(m);
            if (lane == 0) sh.warp_mass[warp] = m;
            __syncthreads();
            if (tid < C) {
                m = 0;
                for (int w = 0; w < kSampleWarps; w++) m += sh.warp_mass[w];
                cluster.map_shared_rank(&sh, tid)->part_mass[rank] = m;
            }
            cluster.sync();
            for (int c = 0; c < C; c++) whole += sh.part_mass[c];
        }
        const double share = fmax(0.0, (double)p.top_p) * (double)whole;
        // Inside the ties of top-k's cut, or above them.
        const u64 w = cut.value == -INFINITY ? 0 : weight(cut.value), above = cut.mass - w * (u64)cut.ties;
        if (cut.value != -INFINITY && (double)above < share) {
            const double need = ceil((share - (double)above) / (double)(w ? w : 1));
            const int t = need < 1.0 ? 1 : need > (double)cut.ties ? cut.ties : (int)need;
            cut.count -= cut.ties - t;
            cut.ties = t;
        } else if (cut.value != -INFINITY && cut.count == cut.ties) {  // nothing above them
            cut.count = cut.ties = 1;
        } else {
            cut = find(true, 0, share, cut.value);
        }
    }

    // ---- what is kept, by id: tokens above the cut, and the first ties at it; min-p among them
    const double coldest = p.min_p > 0.f ? log((double)p.min_p) : -INFINITY;
    const int per_warp = (n + kSampleWarps - 1) / kSampleWarps, w0 = min(n, warp * per_warp), w1 = min(n, w0 + per_warp);
    int ties_before = 0;
    if (cut.ties) {
        int t = 0;
        for (int i = w0 + lane; i < w1; i += 32) t += x[i] == cut.value;
        t = __reduce_add_sync(0xffffffffu, t);
        cluster.sync();  // the bins and ends of the search have been read
        if (lane == 0) sh.warp_count[warp] = t;
        __syncthreads();
        if (tid < C) {
            t = 0;
            for (int w = 0; w < kSampleWarps; w++) t += sh.warp_count[w];
            cluster.map_shared_rank(&sh, tid)->part_count[rank] = t;
        }
        for (int w = 0; w < warp; w++) ties_before += sh.warp_count[w];
        cluster.sync();
        for (int c = 0; c < rank; c++) ties_before += sh.part_count[c];
    }
    // Calls f(i, weight) in order of i, 32 lanes at a time, weight 0 for tokens that are not kept; f says whether to stop.
    auto walk = [&](auto f) {
        int level = ties_before;
        for (int i0 = w0; i0 < w1; i0 += 32) {
            const int i = i0 + lane;
            const float l = i < w1 ? x[i] : -INFINITY;
            const bool tie = cut.ties && l == cut.value && i < w1;
            const unsigned tied = __ballot_sync(0xffffffffu, tie);
            const bool keep = l > cut.value || (tie && level + __popc(tied & ((1u << lane) - 1u)) < cut.ties);
            level += __popc(tied);
            const bool stays = keep && exponent(l) >= coldest;
            if (f(i, stays, stays ? weight(l) : 0ull)) break;
        }
    };
    u64 mass = 0;
    int count = 0;
    walk([&](int, bool stays, u64 w) {
        mass += w, count += stays;
        return false;
    });
    mass = warp_sum64(mass);
    count = __reduce_add_sync(0xffffffffu, count);
    __syncthreads();
    if (lane == 0) sh.warp_mass[warp] = mass, sh.warp_count[warp] = count;
    cluster.sync();
    if (tid < C) {
        u64 m = 0;
        int k = 0;
        for (int w = 0; w < kSampleWarps; w++) m += sh.warp_mass[w], k += sh.warp_count[w];
        SampleShared *o = cluster.map_shared_rank(&sh, tid);
        o->part_mass[rank] = m, o->part_count[rank] = k;
    }
    cluster.sync();
    u64 whole = 0, before = 0;
    int kept = 0;
    for (int c = 0; c < C; c++) {
        if (c < rank) before += sh.part_mass[c];
        whole += sh.part_mass[c];
        kept += sh.part_count[c];
    }
    u64 target = (u64)((double)u * (double)whole);
    if (target >= whole) target = whole - 1;
    for (int w = 0; w < warp; w++) before += sh.warp_mass[w];
    if (target < before || target >= before + mass) return;  // one warp of the cluster has the token
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
            if (a.logprobs) a.logprobs[row] = (float)(exponent(x[i]) - log((double)whole / kSampleOne));
            if (a.kept) a.kept[row] = kept;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
        return reached != 0;
    });
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
        TCM_CUDA(cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleSlice * 4));
        TCM_CUDA(cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    });
    int cluster = kSampleCluster;
    while (cluster > 1 && (vocab < cluster * 1024 || (rows * cluster > 2 * sm_count() && vocab <= cluster / 2 * 20480))) cluster /= 2;
    const int slice = ((vocab + cluster - 1) / cluster + 3) / 4 * 4;
    const SampleArgs args = {ids, logprobs, kept, logits, stride, vocab, slice, params, uniforms, status};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * cluster);
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = (size_t)slice * 4;
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
