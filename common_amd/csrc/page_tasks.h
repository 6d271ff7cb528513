// How a paged attention call is cut into tasks: the arithmetic that its kernels and its host side share.
//
// Tasks are the tiles of ROWS packed rows of every chunk (a chunk's row t * group + g: token t, head g of the query heads
// that share a KV head).  Where there are enough of them to fill the GPU, a tile is a task (target 0) and has a slot
// (chunk_slot).  Otherwise every block adds up what all chunks' tiles see, so that splits of `per` units of
// kUnit<ROWS> keys make about `target` tasks of equal length whatever the lengths of the sequences are, and finds its task
// in their order.  In a chunk of several tiles, tile j's tasks begin at floor(S(j) / L) + j, with L keys in a split and
// S(j) the keys that the tiles before j see, from above and in closed form: at least as many as its splits, and found
// without a sum over tiles; those past its splits are empty.
//
// P, in what follows: a call's sizes, with the members n, rows, group, seqs, max_pages, shift and few_rows.
#pragma once

#include <cmath>

#include "page_index.h"

template <int ROWS>
constexpr int kUnit = ROWS == 16 ? 128 : 64;  // a round of the few-row kernel's wavefronts; the tile kernel's largest key tile

// Units of a split, at least.  (One token over 4,096 rows in splits of one unit: 17.0 us, of two 14.1; tiles over few keys
// want all the blocks they can get: 509 tokens over 609 rows 33.5 us, with two units 36.7.)
template <int ROWS>
constexpr float kLeast = ROWS == 16 ? 2.f : 1.f;

constexpr int kMostUnits = 1 << 24;  // of 64 keys: a table's 2^30 rows

struct Task {
    int seq, first, count;  // chunk
    int at;                 // cache row of its first token
    int r0, rows;           // packed rows: first, and how many there are
    int units;              // key units its chunk's last row sees
    int per, splits, split; // units of a split, splits, and which
    int base;               // the tile's first task
};

AR_HD int lesser(int a, int b) { return a < b ? a : b; }
AR_HD int greater(int a, int b) { return a > b ? a : b; }

// Of a chunk that has rows a .. b - 1 of the call (b - a <= 0: none), at cache row `at` of sequence `seq`: its fields of
// *t, and the number of its tiles; 0: it is not this kernel's.
template <int ROWS, typename P>
AR_HD int tiles_of_chunk(const P& p, int a, int b, int at, int seq, Task* t) {
    t->first = a;
    t->count = a >= 0 && b > a && b <= p.rows ? b - a : 0;
    t->seq = seq;
    t->at = at;
    const int cap = p.max_pages << p.shift;  // (at most 2^30)
    const int end = at < 0 || seq < 0 || seq >= p.seqs ? 0 : at >= cap ? cap : lesser(at + t->count, cap);
    t->units = (end + kUnit<ROWS> - 1) / kUnit<ROWS>;
    const int packed = t->count * p.group;  // (at most 2^30)
    if (t->count == 0 || (ROWS == 16 ? packed > p.few_rows : packed <= p.few_rows)) return 0;
    return (packed + ROWS - 1) / ROWS;
}

// Keys that tile j of the chunk sees; S(j) above; first task of tile j.
template <int ROWS, typename P>
AR_HD int tile_end(const P& p, const Task& c, int j) {
    const int cap = p.max_pages << p.shift, packed = c.count * p.group;
    return c.units == 0 ? 0 : c.at >= cap ? cap : lesser(c.at + (lesser((j + 1) * ROWS, packed) - 1) / p.group + 1, cap);
}
template <int ROWS, typename P>
AR_HD double keys_before(const P& p, const Task& c, int j) {
    const double at = lesser(c.at, p.max_pages << p.shift) + 1;
    return c.units == 0 ? 0. : j * at + 0.5 * ROWS * j * (j + 1.) / p.group;
}
template <int ROWS, typename P>
AR_HD int first_task(const P& p, const Task& c, int j, double inv) {
    return (int)(keys_before<ROWS>(p, c, j) * inv) + j;
}

// Keys of a chunk of n tiles, for the sum over all chunks.
template <int ROWS, typename P>
AR_HD float keys_of_chunk(const P& p, const Task& c, int n) {
    return n == 1 ? (float)c.units * kUnit<ROWS> : (float)keys_before<ROWS>(p, c, n);
}

// Units of a split for `target` tasks of equal length (and one more a tile) out of `keys` in all: a little more than the
// even share, for the sum's roundings.
template <int ROWS>
AR_HD float even_share(float keys, int target) {
    return fmaxf(kLeast<ROWS>, ceilf(keys * 1.0001f / ((float)target * kUnit<ROWS>)));
}
// The same by the fewest units whose tasks are at most `most`, for chunks of one tile: from where fewest_units begins.
template <int ROWS>
AR_HD int least_share(float keys, int most, int per) {
    return (int)fminf(fmaxf(kLeast<ROWS>, ceilf(keys / ((float)most * kUnit<ROWS>)) - 1.f), (float)per);
}

// Splits of `units` units; tasks of a chunk of n tiles.
AR_HD int splits_of(int units, int per) { return greater(1, (units + per - 1) / per); }
template <int ROWS, typename P>
AR_HD int tasks_of_chunk(const P& p, const Task& c, int n, int per, double inv) {
    return n == 0 ? 0 : n == 1 ? splits_of(c.units, per) : first_task<ROWS>(p, c, n, inv);
}

// Tile of a chunk of n tiles that has the chunk's task q: the last whose tasks begin at q or before.
template <int ROWS, typename P>
AR_HD int tile_of_task(const P& p, const Task& c, int n, int q, double inv) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (first_task<ROWS>(p, c, mid, inv) <= q) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// A tile's first task within its chunk, and its splits.
template <int ROWS, typename P>
AR_HD int tile_begin(const P& p, const Task& c, int n, int tile, double inv) {
    return n == 1 ? 0 : first_task<ROWS>(p, c, tile, inv);
}
template <int ROWS, typename P>
AR_HD int tile_splits(const P& p, const Task& c, int tile, int per) {
    return splits_of((tile_end<ROWS>(p, c, tile) + kUnit<ROWS> - 1) / kUnit<ROWS>, per);
}

// ---- host side ----------------------------------------------------------------------------------------------

// A kernel's share of a call: its tiles at most, and how many tasks to cut their keys into (0: none; one more per tile
// for its last split, and one for what rounding makes of where its tasks begin).
struct Part {
    int tiles = 0, target = 0, blocks = 0;  // (blocks: resident at once)
    int tasks() const { return !target ? tiles : target + tiles + 1 > blocks ? target + tiles + 1 : blocks; }
};

// The launches of a call.  The host knows the numbers of rows and of chunks, not which chunk has how many.  Up to 32
// packed rows a chunk on average, all chunks go to the few-row kernel (16 sequences, 8 tokens, 4 heads a KV head, 22 rows
// on average: 36 us, tiles 46; 16 tokens, 45 rows: 49 us, tiles 39).  One chunk of more rows goes to the tile kernel.
// Otherwise one launch holds both kernels' blocks, and chunks of up to kFewRows rows are the few-row kernel's (decode
// steps and a prompt together, fp16 and fp32: 143 and 290 us, all as tiles 162 and 338; kFewRows 64 instead of 16: 16
// chunks of 16 tokens 53 us instead of 39 in bf16, 63 instead of 44 in fp32).  The average also sends one longer chunk
// among many single tokens to the few-row kernel: 127 tokens over 1,500 rows and 512 over 1,512, 32 / 8 heads of 128, 194
// us in bf16, the two apart 151 and 46.
struct Plan {
    int few_rows = 0;  // packed rows up to which a chunk is the few-row kernel's
    Part few, tile;
};

constexpr int kFewRows = 16, kMaxSplitChunks = 1024;

// Tasks to cut the keys for, of n chunks over tables of `cap` rows: `blocks`, the number that is resident at once, unless
// the tiles alone are as many (1,024 tokens of three sequences, 537 tiles for 512 blocks: whole tiles 609 us, cut ones
// 632).  Each tile takes one of them, so that a long context among nearly as many short ones is hardly cut: 31,999 rows
// beside 62 (63) of 1,000 in fp16, 8 KV heads: 217 us (372), 79 by their bytes; beside 30: 52, its floor.
inline void cut_keys(long long blocks, long long cap, long long tiles, int n, int unit, Part* out) {
    if (tiles >= blocks || n > kMaxSplitChunks) return;
    if (cap <= unit) return;  // (one split of any sequence)
    // (a tile's last split is a task of its own, so that there may be `tiles` more; and no more than units)
    const long long most = (tiles > n ? tiles : n) * ((cap + unit - 1) / unit), want = blocks - tiles < most ? blocks - tiles : most;
    out->target = want > 1 ? (int)want : 1;
    out->blocks = (int)blocks;
}

// Of n chunks (`starts`: of any lengths, not one row each; the rows behind those are no work) with `rows` rows in all and
// `group` query heads a KV head, over tables of `cap` rows of `kv_heads` KV heads, fp32 or not, on a GPU of `cus` CUs.
inline Plan plan_tasks(int cus, int kv_heads, bool fp32, long long cap, bool starts, int n, int rows, int group) {
    Plan a;
    const long long packed = (starts ? rows : n) * (long long)group;
    // (Few rows over fp32, which keep twice the bytes in flight: one block a CU, 46 us for 8 sequences of 4,000 rows, two
    // 52; 16-bit caches: two, 82 us for 16 of 8,192, one 88.  Tiles: two, 46 us for the fp32 chunk, one 52.)
    const long long few = (fp32 ? 1LL : 2LL) * cus / kv_heads, tile = 2LL * cus / kv_heads;
    if (!starts || packed <= 32LL * n) {
        a.few_rows = 0x7fffffff;
        a.few.tiles = (int)(starts ? packed / 16 + n : n * ((group + 15LL) / 16));
        cut_keys(few, cap, packed / 16 > n ? packed / 16 : n, n, kUnit<16>, &a.few);
    } else {
        a.tile.tiles = (int)(packed / 128 + n);
        cut_keys(tile, cap, packed / 128, n, kUnit<128>, &a.tile);
        if (n > 1) {
            a.few_rows = kFewRows;
            cut_keys(few, cap, 0, n, kUnit<16>, &a.few);
            const long long any = packed / 16 + n, cut = kFewRows / 16LL * n;
            a.few.tiles = (int)(a.few.target && cut < any ? cut : any);
        }
    }
    return a;
}
