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

#endif
