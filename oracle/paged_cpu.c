/* The paged cache's index arithmetic (csrc/paged_index.h) as host functions, for
 * the CPU tests. */
#include "../cmachine_b200/csrc/paged_index.h"

int paged_cpu_div(int page, int x) {
    PagedView v = {0};
    v.page = page;
    paged_divider(&v);
    return paged_div(&v, x);
}
int paged_cpu_extent(int rows, int max_new, int max_length, int table_stride, int page, int start, int end, int length,
                     int *out) {
    PagedView v = {0};
    v.rows = rows;
    v.max_new = max_new;
    v.max_length = max_length;
    v.table_stride = table_stride;
    v.page = page;
    PagedExtent e;
    const int bad = paged_extent_of(&v, start, end, length, &e);
    out[0] = e.start;
    out[1] = e.count;
    out[2] = e.length;
    return bad;
}
int64_t paged_cpu_slot(int pages, int page, int kvheads, const int *table, int table_stride, int s, int j, int h) {
    PagedView v = {0};
    v.pages = pages;
    v.page = page;
    v.kvheads = kvheads;
    v.table = table;
    v.table_stride = table_stride;
    paged_divider(&v);
    return paged_slot(&v, s, j, h);
}
int paged_cpu_sees(int at, int j, int window, int sinks) { return paged_sees(at, j, window, sinks); }
int paged_cpu_tiles(int first, int last, int window, int sinks, int shift, int *out, int most) {
    const PagedTiles t = paged_tiles(first, last, window, sinks, shift);
    for (int k = 0; k < t.count && k < most; k++) out[k] = paged_tile(t, k);
    return t.count;
}
int64_t paged_cpu_tile_bound(int sequences, int rows, int max_new, int group, int few, int tile) {
    return paged_tile_bound(sequences, rows, max_new, group, few, tile);
}
int64_t paged_cpu_tile_guess(int sequences, int rows, int max_new, int group, int few, int tile) {
    return paged_tile_guess(sequences, rows, max_new, group, few, tile);
}
int paged_cpu_splits(int64_t items, int tiles, int sms, int64_t room, int most) {
    return paged_splits(items, tiles, sms, room, most);
}
