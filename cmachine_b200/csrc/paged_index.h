/* Where the rows of a paged K/V cache lie, and which of them a query sees.
 *
 * Plain C, shared by the kernels (csrc/paged*.cu*) and a CPU build of the same
 * arithmetic (oracle/paged_cpu.c), which the tests run over sizes and tables
 * that a kernel must never be tried on. Everything a kernel reads or writes in
 * the pool or in the callers' row buffers is addressed through
 * paged_extent + paged_slot, which turn every bad extent or page id into "no
 * row" plus a status bit.
 */
#ifndef TCM_PAGED_INDEX_H
#define TCM_PAGED_INDEX_H
#include <stdint.h>
#include "../../include/gpu.h"
#ifdef __CUDACC__
#define TCM_HD static __host__ __device__ __forceinline__
#else
#define TCM_HD static inline
#endif

enum { kPagedNonFinite = 1, kPagedBadPage = 2, kPagedBadExtent = 4 }; /* status bits (include/gpu.h) */

/* The two descriptors of a call, with the division by the page size prepared. */
typedef struct {
    int kind, pages, page, kvheads, dim;
    void *keys, *values;
    float *scales;
    int sequences, rows, max_new, max_length, table_stride;
    const int *starts, *lengths, *table;
    uint32_t page_mul;
    int page_shift;
} PagedView;

/* x / page as (hi32(mul * x) + x) >> shift for 0 <= x < 2^31: with l = ceil(log2 page),
 * mul = floor(2^32 (2^l - page) / page) + 1, the multiplier 2^32 + mul exceeds
 * 2^(32+l) / page by less than 2^l / page, too little to reach the next quotient
 * (division by invariant integers, Granlund and Montgomery 1994). The sum stays
 * below 2^32 because hi32(mul * x) <= x < 2^31. */
TCM_HD void paged_divider(PagedView *v) {
    int l = 0;
    while ((1u << l) < (uint32_t)v->page) l++;
    v->page_shift = l;
    v->page_mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - (uint64_t)v->page)) / (uint64_t)v->page + 1);
}
TCM_HD int paged_div(const PagedView *v, int x) {
#ifdef __CUDA_ARCH__
    const uint32_t hi = __umulhi(v->page_mul, (uint32_t)x);
#else
    const uint32_t hi = (uint32_t)(((uint64_t)v->page_mul * (uint32_t)x) >> 32);
#endif
    return (int)((hi + (uint32_t)x) >> v->page_shift);
}

/* Sequence s of the batch: its first row in the callers' buffers, its new rows
 * and its length. Returns 0, or kPagedBadExtent with no rows where the extents
 * do not fit the buffers, the declared maxima or the table. */
typedef struct {
    int start, count, length;
} PagedExtent;
TCM_HD int paged_extent_of(const PagedView *v, int start, int end, int length, PagedExtent *e) {
    e->start = start;
    e->count = end - start;
    e->length = length;
    if (start < 0 || end < start || end > v->rows || e->count > v->max_new || length < 0 || length > v->max_length ||
        (int64_t)length > (int64_t)v->table_stride * v->page) {
        e->start = e->count = e->length = 0;
        return kPagedBadExtent;
    }
    return 0;
}
TCM_HD int paged_extent(const PagedView *v, int s, PagedExtent *e) {
    return paged_extent_of(v, v->starts[s], v->starts[s + 1], v->lengths[s], e);
}

/* Row j >= 0 of KV head h under page id `id`, in rows of the [pages][kvheads][page]
 * order that keys, values and scales share; -1 when the pool has no such page. */
TCM_HD int64_t paged_row(const PagedView *v, int id, int j, int j_page, int h) {
    if (id < 0 || id >= v->pages) return -1;
    return ((int64_t)id * v->kvheads + h) * v->page + (j - j_page * v->page);
}
/* The same through the table, for 0 <= j < a sequence's length. */
TCM_HD int64_t paged_slot(const PagedView *v, int s, int j, int h) {
    const int p = paged_div(v, j);
    return paged_row(v, v->table[(int64_t)s * v->table_stride + p], j, p, h);
}

/* Does the query at place `at` see row j of its sequence? */
TCM_HD int paged_sees(int at, int j, int window, int sinks) {
    return j <= at && (window == 0 || j < sinks || (int64_t)j > (int64_t)at - window);
}
/* The tiles of `tile` rows (a power of two, 2^shift) that the queries at places
 * first..last see any row of: tiles [0, a) and [b, e), numbered 0 .. a + e - b - 1. */
typedef struct {
    int a, b, count;
} PagedTiles;
TCM_HD PagedTiles paged_tiles(int first, int last, int window, int sinks, int shift) {
    PagedTiles t = {0, 0, 0};
    if (last < 0) return t;
    if (first < 0) first = 0;
    const int e = (last >> shift) + 1;
    if (window) {
        const int64_t low64 = (int64_t)first - window + 1;
        const int low = low64 > 0 ? (int)low64 : 0;
        const int top = sinks < low ? sinks : low; /* first rows below every window */
        t.b = low >> shift;
        t.a = (int)(((int64_t)top + ((int64_t)1 << shift) - 1) >> shift);
        if (t.a > t.b) t.a = t.b;
    }
    t.count = t.a + e - t.b;
    return t;
}
TCM_HD int paged_tile(PagedTiles t, int k) { return k < t.a ? k : t.b + (k - t.a); }

/* How chunks are shared out. A row tile is `tile` query rows of one KV head; an item is a row tile of one KV head,
 * and may be split over the rows that it sees. The device counts the row tiles of a batch; the host, which knows
 * only sums and maxima, launches for a bound of them and for a guess.
 *
 * The most row tiles that sequences of more than `few` rows can have: each has at most max_new rows, and
 * ceil(n / tile) adds up to less than the sum over tile and one for each, of rows / (few + 1) sequences at most. */
TCM_HD int64_t paged_tile_bound(int sequences, int rows, int max_new, int group, int few, int tile) {
    const int64_t each = ((int64_t)max_new * group + tile - 1) / tile, live = rows / (few + 1);
    const int64_t all = (int64_t)rows * group / tile + (live < sequences ? live : sequences);
    return all < each * sequences ? all : each * sequences;
}
/* Their number when some sequences have max_new rows and the others one, as many as the rows are enough for. */
TCM_HD int64_t paged_tile_guess(int sequences, int rows, int max_new, int group, int few, int tile) {
    const int64_t bound = paged_tile_bound(sequences, rows, max_new, group, few, tile);
    int64_t full = max_new > 1 ? ((int64_t)rows - sequences + max_new - 2) / (max_new - 1) : sequences;
    if (full < 1) full = 1;
    full *= ((int64_t)max_new * group + tile - 1) / tile;
    return full < bound ? full : bound;
}
/* The time of `items` items of `mean` cached-row tiles and `longest` at most, each of them split in k: rounds of the
 * SMs, or the longest split, whose start and end count as three tiles; joining the parts counts as two. The k taken
 * is the least within 3 % of the best. (items * k is below 2^32: it passes paged_may_split, or k is 1.) */
TCM_HD float paged_split_cost(int64_t items, int k, int mean, int longest, int sms) {
    const float rounds = (float)(((uint32_t)items * (uint32_t)k + (uint32_t)sms - 1) / (uint32_t)sms);
    const float all = rounds * ((float)mean / (float)k + 3.f), one = (float)longest / (float)k + 3.f;
    return (all > one ? all : one) + (k > 1 ? 2.f : 0.f);
}
TCM_HD int paged_may_split(int64_t items, int k, int tiles, int64_t room) { return k == 1 || (2 * k <= tiles && items * k <= room); }
static inline int paged_splits(int64_t items, int tiles, int sms, int64_t room, int most) {
    float least = paged_split_cost(items, 1, tiles, tiles, sms);
    for (int k = 2; k <= most; k++)
        if (paged_may_split(items, k, tiles, room) && paged_split_cost(items, k, tiles, tiles, sms) < least)
            least = paged_split_cost(items, k, tiles, tiles, sms);
    for (int k = 1;; k++)
        if (k == most || (paged_may_split(items, k, tiles, room) && paged_split_cost(items, k, tiles, tiles, sms) <= 1.03f * least))
            return k;
}

#endif
