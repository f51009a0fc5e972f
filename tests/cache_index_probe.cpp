// The cache's index arithmetic (csrc/cache_index.h) as a small C library for
// the CPU tests.
#include "../mxfp8-quantizer_b200/csrc/cache_index.h"

using namespace mxfp8;

extern "C" {
int64_t probe_row(int64_t pages, int heads, int shift, int64_t page, int head, int offset) {
    return cache_row(CacheShape{pages, heads, shift, 128}, page, head, offset);
}
int64_t probe_table(const int32_t* table, int64_t stride, int64_t max_pages, int64_t b, int64_t at, int shift) {
    return table_page(table, stride, max_pages, b, at, shift);
}
int64_t probe_sequence(const int32_t* starts, int64_t batch, int64_t first_row, int64_t row) {
    int64_t from = -1;  // as the kernel counts
    for (int64_t b = 0; b <= batch; ++b) from += starts[b] <= first_row;
    return sequence_from(starts, batch, from, row);
}
int64_t probe_begin(int64_t i, int64_t n, int64_t total) { return split_begin(make_split(n, total), i); }
int64_t probe_part(int64_t x, int64_t n, int64_t total) { return split_part(make_split(n, total), x); }
int64_t probe_visible(int64_t length, int64_t max_pages, int shift) { return visible_length(length, max_pages, shift); }
}
