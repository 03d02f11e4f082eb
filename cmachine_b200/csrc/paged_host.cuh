// Host side shared by the entry points over the paged K/V cache: checks of their arguments, and dispatch.
#pragma once
#include "paged.cuh"
#include "kernels.h"
#include "../../include/gpu.h"

namespace tcm {

inline int refuse(const char *call, const char *why) {
    fprintf(stderr, "%s: %s\n", call, why);
    return -1;
}
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// The call's descriptors as a view; 0, or -1 with a message.
inline int open_view(const char *call, const TcmPagedCache *c, const TcmPagedBatch *b, const int *status, PagedView *v) {
    if (!c || !b) return refuse(call, "no cache or no batch");
    if (c->kind != kPagedBf16 && c->kind != kPagedBytes) return refuse(call, "kind is 2 (BF16) or 3 (bytes)");
    if (c->dim != 64 && c->dim != 128) return refuse(call, "dim is 64 or 128");
    if (c->pages < 1 || c->page < 1 || c->page > 65536 || c->kvheads < 1 || c->kvheads > 1024)
        return refuse(call, "pages, page or kvheads out of range");
    if (!c->keys || !c->values || !aligned16(c->keys) || !aligned16(c->values))
        return refuse(call, "keys and values are 16-byte aligned device memory");
    if (c->kind == kPagedBytes && (!c->scales || ((uintptr_t)c->scales & 3))) return refuse(call, "a byte cache has scales");
    if (b->sequences < 0 || b->sequences > 65535 || b->rows < 0 || b->max_new < 0 || b->max_length < 0 ||
        b->max_length > 1 << 30)
        return refuse(call, "sequences, rows, max_new or max_length out of range");
    if (b->sequences && (!b->starts || !b->lengths || !b->table || b->table_stride < 1))
        return refuse(call, "a batch has starts, lengths and a table");
    if (((uintptr_t)b->starts | (uintptr_t)b->lengths | (uintptr_t)b->table) & 3)
        return refuse(call, "starts, lengths and table are 4-byte aligned");
    if ((uintptr_t)status & 3) return refuse(call, "status is 4-byte aligned");
    const int max_new = b->max_new < b->rows ? b->max_new : b->rows;
    // No sequence is longer than its table either.
    const long long held = (long long)b->table_stride * c->page;
    const int max_length = b->max_length < held ? b->max_length : (int)held;
    if ((long long)max_new * c->kvheads > 0x7fffffff / 8) return refuse(call, "too many new rows for one call");
    *v = PagedView{c->kind, c->pages, c->page, c->kvheads, c->dim, c->keys, c->values, c->scales, b->sequences, b->rows,
                   max_new, max_length, b->table_stride, b->starts, b->lengths, b->table, 0, 0};
    paged_divider(v);
    return 0;
}
inline int check_rows(const char *call, const void *p, long long stride, int heads, int dim) {
    if (!p || !aligned16(p)) return refuse(call, "row buffers are 16-byte aligned device memory");
    if (stride < (long long)heads * dim || stride % 4) return refuse(call, "a row stride is a multiple of 4 and holds a row");
    return 0;
}
// Nothing to do: no sequence, or none that may have a new row.
inline bool nothing(const PagedView &v) { return !v.sequences || !v.rows || !v.max_new; }

inline unsigned blocks_of(long long items, int a_block) {
    const long long blocks = (items + a_block - 1) / a_block;
    return (unsigned)(blocks < 4096 ? blocks : 4096);
}

#define PAGED_DISPATCH(view, call)                                      \
    do {                                                                \
        if ((view).kind == kPagedBf16) {                                \
            if ((view).dim == 64) { call(kPagedBf16, 64); }             \
            else { call(kPagedBf16, 128); }                             \
        } else {                                                        \
            if ((view).dim == 64) { call(kPagedBytes, 64); }            \
            else { call(kPagedBytes, 128); }                            \
        }                                                               \
    } while (0)

}  // namespace tcm
