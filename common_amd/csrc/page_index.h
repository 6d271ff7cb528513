// Where rows of a paged cache lie: the index arithmetic that its kernels share, on whatever the device arrays hold.
// Every function returns an index inside its array, or -1, for any contents (negative, descending, past the end).
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#define AR_HD __host__ __device__ inline
#else
#define AR_HD inline
#endif

// Page of row `row` of sequence `seq`, or -1: no such sequence, column or page.
AR_HD int page_of_row(const int32_t* table, int seqs, int max_pages, int pages, int page_shift, int seq, int row) {
    if (seq < 0 || seq >= seqs || row < 0) return -1;
    const int col = row >> page_shift;
    if (col >= max_pages) return -1;
    const int page = table[(int64_t)seq * max_pages + col];
    return page >= 0 && page < pages ? page : -1;
}

// Cache row of row j of a chunk that begins at cache row `at`, or -1 (not in the cache, or past 2^31 - 1).
AR_HD int cache_row(int at, int j) {
    if (at < 0 || j < 0 || at > 0x7fffffff - j) return -1;
    return at + j;
}

// Chunks are cut into tiles of `span` units, `per_row` of them in a row (the query heads that share a KV head).  Tile
// slots run over all chunks: chunk i has the slots from chunk_slot(i) to chunk_slot(i + 1) - 1, which are enough for its
// tiles (c units from unit s on cross at most floor((s + c) / span) - floor(s / span) + 1 >= ceil(c / span) of them) and
// can be found without a prefix sum; a slot past the chunk's last tile is empty.  All of them: at most
// rows * per_row / span + n.
AR_HD int64_t chunk_slot(int32_t start, int i, int per_row, int span) {
    // (floor also for negative starts: the slots of ascending starts ascend)
    const int64_t s = (int64_t)start * per_row;
    return (s >= 0 ? s / span : -((-s + span - 1) / span)) + i;
}

// Rows of chunk i as (first, count) within 0 .. rows; count 0 where start descends or leaves the range.
AR_HD void chunk_rows(const int32_t* start, int i, int rows, int* first, int* count) {
    if (!start) {
        *first = i;
        *count = i < rows ? 1 : 0;
        return;
    }
    const int a = start[i], b = start[i + 1];
    *first = a;
    *count = a >= 0 && b > a && b <= rows ? b - a : 0;
}

// The chunk that holds slot `slot`: the last i with chunk_slot(start[i], i) <= slot.  For starts that ascend; for others
// some i in 0 .. n-1.  Each round asks `ways` chunks at once: `below(i, k, len)` tells how
// many of the chunks i, i + k, i + 2k, ... below i + len satisfy the condition before the first that does not.
template <typename F>
AR_HD int chunk_search(int n, int ways, F below) {
    int lo = 0, len = n;
    while (len > 1) {
        const int step = (len + ways - 1) / ways;
        int c = below(lo, step, len);
        if (c < 1) c = 1;
        lo += (c - 1) * step;
        len -= (c - 1) * step;
        if (len > step) len = step;
    }
    return lo;
}

// Units of a split: the fewest in lo .. hi whose tasks `fits` accepts, or hi, where none below it is accepted.  `fits` is
// monotone (more units in a split, fewer tasks).  At most log2(hi - lo) + 1 questions, whatever the answers are.
template <typename F>
AR_HD int fewest_units(int lo, int hi, F fits) {
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (fits(mid)) hi = mid;
        else lo = mid + 1;
    }
    return hi;
}

// The chunk that holds row `row`, or -1.
AR_HD int chunk_of_row(const int32_t* start, int n, int rows, int row) {
    if (row < 0 || row >= rows) return -1;
    if (!start) return row < n ? row : -1;
    int lo = 0, hi = n - 1;  // the last i with start[i] <= row
    while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (start[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    int first, count;
    chunk_rows(start, lo, rows, &first, &count);
    return row >= first && (int64_t)row - first < count ? lo : -1;
}
