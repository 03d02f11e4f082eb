/* The bins in which gpu_sample counts a row's logits (csrc/sample.cu).
 *
 * Plain C, shared by the kernel and a CPU build of the same arithmetic
 * (oracle/sample_cpu.c): the list of tokens that decides a row has room for as
 * many as the bins counted, so the tests count rows here before a kernel does.
 */
#ifndef TCM_SAMPLE_BINS_H
#define TCM_SAMPLE_BINS_H
#include <math.h>
#include <stdint.h>
#include <string.h>
#ifdef __CUDACC__
#define TCM_SAMPLE static __host__ __device__ __forceinline__
#else
#define TCM_SAMPLE static inline
#endif

enum { kSampleBins = 4096, kSampleSlots = 8192 };
/* FP32 sums with kSampleRound are whole numbers, one to one with their bits; they go to the nearest, and to even ones
 * from between, so that bins are not off to one side of logits of 16 bits. */
#define kSampleRound 12582912.f /* 1.5 * 2^23 */
#define kSampleReach 524288.f   /* 2^19 */

TCM_SAMPLE int sample_bits(float x) {
#ifdef __CUDA_ARCH__
    return __float_as_int(x);
#else
    int32_t u;
    memcpy(&u, &x, 4);
    return u;
#endif
}
TCM_SAMPLE float sample_float(int u) {
#ifdef __CUDA_ARCH__
    return __int_as_float(u);
#else
    float x;
    memcpy(&x, &u, 4);
    return x;
#endif
}

/* Bins of the logits: one of the first eight for the largest, and not falling as l falls; `last` for all that lie so many
 * bins lower, or lower. */
typedef struct {
    float unit, origin, scale, least;
    int top, last;
} SampleBins;
TCM_SAMPLE int sample_bin(const SampleBins *b, float l) {
    return b->top - sample_bits(fmaxf(fmaf(fmaf(l, b->unit, -b->origin), b->scale, kSampleRound), b->least));
}
/* Of equal width over [from, high]; what lies below `from` is the last but one at most. */
TCM_SAMPLE SampleBins sample_bins_over(float from, float high, int bins) {
    SampleBins b;
    /* Differences in a power of two at which neither they nor the scale leave FP32's range. */
    const float span = high - from;
    b.unit = span > 1e30f ? 0.25f : span > 0.f && span < 1e-25f ? 0x1p100f : 1.f;
    b.origin = high * b.unit;
    b.scale = span > 0.f ? (float)(bins - 2) * 0.999999f / (b.origin - from * b.unit) : 0.f;
    b.last = bins - 1;
    b.top = sample_bits(kSampleRound);
    b.least = kSampleRound - (float)b.last;
    return b;
}
/* Of a width given beforehand, 1 / scale, with borders that do not move with the row: sample_slot tells one of
 * kSampleSlots in a circle without knowing `high`. |high * scale| is below kSampleReach. */
TCM_SAMPLE int sample_slot(float l, float scale) { return sample_bits(fmaf(l, scale, kSampleRound)) & (kSampleSlots - 1); }
TCM_SAMPLE SampleBins sample_bins_of(float high, float scale) {
    SampleBins b;
    b.unit = 1.f;
    b.origin = 0.f;
    b.scale = scale;
    b.last = kSampleBins - 1;
    b.top = sample_bits(fmaf(high, scale, kSampleRound)) | 7; /* so that a thread's eight slots are two aligned quads */
    b.least = sample_float(b.top - b.last);
    return b;
}
/* Logits at this one and below are not counted in slots. */
TCM_SAMPLE float sample_floor(float scale) { return -kSampleReach / scale; }
/* Do the counts of a row's slots hold for its bins? `counted` is the least logit that was counted. No slot may have two
 * bins, and the logits at the floor and below, which have no slot, must all be of the last bin, which gets what the others
 * leave: the floor is kSampleReach steps of 1 / scale below zero, so the largest must lie kSampleBins steps above it. One
 * more covers the roundings of `at` and of the floor, 2^-5 steps each. */
TCM_SAMPLE int sample_slots_hold(const SampleBins *b, float high, float counted) {
    const float at = high * b->scale;
    return at >= (float)kSampleBins + 1.f - kSampleReach && at < kSampleReach &&
           b->top - sample_bits(fmaf(counted, b->scale, kSampleRound)) < kSampleSlots;
}
#endif
