/* The sampling's bins (csrc/sample_bins.h) as host functions, for the CPU tests. */
#include "../cmachine_b200/csrc/sample_bins.h"

/* A row of n logits counted as the kernel's first pass does, in slots. Where those counts hold: 1, `counts` of the
 * bins as the kernel takes them from the slots, and `direct` by each token's own bin; else 0. */
int sample_cpu_slots(const float *l, int n, float temperature, int *counts, int *direct) {
    static int slots[kSampleSlots];
    const float scale = 128.f / temperature;
    if (!(scale > 0.f && scale < INFINITY)) return 0;
    const float floor = sample_floor(scale);
    float high = -INFINITY, counted = INFINITY;
    int live = 0, taken = 0;
    memset(slots, 0, sizeof(slots));
    for (int i = 0; i < n; i++) {
        live += l[i] > -INFINITY;
        high = fmaxf(high, l[i]);
        if (l[i] > floor) {
            slots[sample_slot(l[i], scale)]++;
            counted = fminf(counted, l[i]);
        }
    }
    const SampleBins bins = sample_bins_of(high, scale);
    if (!live || !sample_slots_hold(&bins, high, counted)) return 0;
    memset(direct, 0, kSampleBins * sizeof(int));
    for (int b = 0; b < kSampleBins - 1; b++) taken += counts[b] = slots[(bins.top - b) & (kSampleSlots - 1)];
    counts[kSampleBins - 1] = live - taken;
    for (int i = 0; i < n; i++)
        if (l[i] > -INFINITY) {
            const int b = sample_bin(&bins, l[i]);
            if (b < 0 || b >= kSampleBins) return -1;
            direct[b]++;
        }
    return 1;
}
/* The bins of n logits over the range [from, high]. */
void sample_cpu_bins(const float *l, int n, float from, float high, int bins, int *out) {
    const SampleBins b = sample_bins_over(from, high, bins);
    for (int i = 0; i < n; i++) out[i] = sample_bin(&b, l[i]);
}
