// cache_index.h -- index arithmetic of the paged cache: which row a position
// lives in, which sequence an output row belongs to, and how the attention's
// tiles are split over warps.  Plain C++, so that the CPU tests compile it too.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define MXFP8_HD __host__ __device__ __forceinline__
#else
#define MXFP8_HD inline
#endif

namespace mxfp8 {

// Geometry of a cache; page_size = 1 << page_shift.
struct CacheShape {
    int64_t num_pages;
    int heads;
    int page_shift;
    int dim;
};

constexpr int64_t kNoRow = -1;

// Row (of dim bytes, of dim / 32 scale bytes) of a page's position for head
// h, or kNoRow for a page outside the cache.
MXFP8_HD int64_t cache_row(const CacheShape& c, int64_t page, int head, int offset) {
    if (page < 0 || page >= c.num_pages) return kNoRow;
    return ((page * c.heads + head) << c.page_shift) + offset;
}

// Page of position `at` of sequence b, or -1 if it lies past the table's row.
MXFP8_HD int64_t table_page(const int32_t* table, int64_t stride, int64_t max_pages, int64_t b, int64_t at,
                            int page_shift) {
    const int64_t i = at >> page_shift;
    return at < 0 || i >= max_pages ? -1 : table[b * stride + i];
}

// The sequence that covers output row `row`: the last b with starts[b] <=
// row; batch if the row lies past the last sequence, -1 before the first.
// `from` is a number of that kind for a row at or before this one: the count of
// starts that are <= that row, less one.
MXFP8_HD int64_t sequence_from(const int32_t* starts, int64_t batch, int64_t from, int64_t row) {
    int64_t b = from;
    while (b < batch && starts[b + 1] <= row) ++b;
    return b;
}

// `total` units over n parts, the first total % n parts one unit longer: part i
// takes [begin(i), begin(i + 1)).
struct Split {
    int64_t each, longer;
};
// a / b, both at least 0: in 32 bits where they allow it, the common case.
MXFP8_HD int64_t quotient(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
MXFP8_HD Split make_split(int64_t n, int64_t total) {
    const int64_t each = quotient(total, n);
    return Split{each, total - each * n};
}
MXFP8_HD int64_t split_begin(const Split& s, int64_t i) { return i * s.each + (i < s.longer ? i : s.longer); }
// The part that holds unit x < total.
MXFP8_HD int64_t split_part(const Split& s, int64_t x) {
    const int64_t edge = s.longer * (s.each + 1);  // end of the longer parts
    return x < edge ? quotient(x, s.each + 1) : s.longer + quotient(x - edge, s.each);
}

// Positions of a sequence that the attention visits.
MXFP8_HD int64_t visible_length(int64_t length, int64_t max_pages, int page_shift) {
    const int64_t room = max_pages << page_shift;
    return length < 0 ? 0 : length < room ? length : room;
}

}  // namespace mxfp8
