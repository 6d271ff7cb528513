// How the paged attention's keys are cut into tasks (common_amd/csrc/page_tasks.h), against plain loops and at the
// largest sizes that its calls accept; built with the address and undefined-behaviour sanitizers.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../common_amd/csrc/page_tasks.h"

static std::mt19937 rng(11);
static int pick(int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); }
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); exit(1); } } while (0)

// Units of a split for one-tile chunks of `units` units each, and how often the number of tasks was asked for.
struct Fit {
    int units, asked;
};
static long long tasks_of(const std::vector<int>& units, int per) {
    long long sum = 0;
    for (int u : units) sum += u == 0 ? 1 : (u + per - 1) / per;
    return sum;
}
static Fit fit(const std::vector<int>& units, int lo, int hi, int most) {
    Fit f{0, 0};
    f.units = fewest_units(lo, hi, [&](int per) {
        f.asked++;
        return tasks_of(units, per) <= most;
    });
    return f;
}

static void fewest_units_of_a_split() {
    for (int t = 0; t < 20000; t++) {
        std::vector<int> units(pick(1, 64));
        for (int& u : units) u = pick(0, 1 << pick(1, 10));
        const int lo = pick(1, 40), hi = lo + pick(0, 300), most = pick(1, 256);
        int want = lo;  // step by step
        while (want < hi && tasks_of(units, want) > most) want++;
        const Fit f = fit(units, lo, hi, most);
        CHECK(f.units == want && f.asked <= 10);
    }
    // tables of 2^30 rows: 2^23 units a chunk, splits of up to 2^24 (from which on a float counts no further)
    const int top = 1 << 24;
    for (int most : {1, 16, 63, 64, 65, 512, 1 << 30}) {
        const std::vector<int> units(64, 1 << 23);
        const Fit f = fit(units, 1, top, most);
        CHECK(f.asked <= 25);
        CHECK(f.units == (most < 64 ? top : (int)(((1LL << 23) + most / 64 - 1) / (most / 64))));
        CHECK(fit(units, top, top, most).units == top && fit(units, top - 1, top, most).asked <= 1);
    }
}

// A call: its sizes as the kernels have them, and its chunks.
struct Call {
    int n, rows, group, seqs, max_pages, shift, few_rows;
    std::vector<int> start, at, seq;
};

// The tasks of one kernel's part, found the way its blocks do: every split of every tile has a task of its own, and all of
// them lie below tasks().  Returns how many packed rows the part takes.
template <int ROWS>
static long long check_part(const Call& c, const Part& part) {
    std::vector<Task> chunk(c.n);
    std::vector<int> tiles(c.n);
    long long rows = 0, all_tiles = 0;
    for (int i = 0; i < c.n; i++) {
        tiles[i] = tiles_of_chunk<ROWS>(c, c.start[i], c.start[i + 1], c.at[i], c.seq[i], &chunk[i]);
        all_tiles += tiles[i];
        if (tiles[i]) rows += (long long)chunk[i].count * c.group;
        CHECK(tiles[i] == 0 || ((tiles[i] - 1LL) * ROWS < (long long)chunk[i].count * c.group));
        CHECK((long long)tiles[i] * ROWS >= (tiles[i] ? (long long)chunk[i].count * c.group : 0));
    }
    CHECK(all_tiles <= part.tiles);
    if (part.target == 0) {
        CHECK(chunk_slot(c.start[c.n], c.n, c.group, ROWS) - chunk_slot(c.start[0], 0, c.group, ROWS) <= part.tiles);
        return rows;
    }
    // the sum over all keys, added up by 64 lanes and then by halves
    float lanes[64] = {};
    bool single = c.n <= 64;
    for (int i = 0; i < c.n; i++) {
        lanes[i & 63] += keys_of_chunk<ROWS>(c, chunk[i], tiles[i]);
        single &= tiles[i] <= 1;
    }
    for (int d = 32; d; d /= 2)
        for (int i = 0; i < d; i++) lanes[i] += lanes[i + d];
    const float share = even_share<ROWS>(lanes[0], part.target);
    const double inv = 1. / ((double)share * kUnit<ROWS>);
    int per = (int)fminf(share, kMostUnits);
    if (ROWS == 16 && single) {
        const int most = part.blocks < part.tasks() ? part.blocks : part.tasks();
        per = fewest_units(least_share<ROWS>(lanes[0], most, per), per, [&](int units) {
            long long sum = 0;
            for (int i = 0; i < c.n; i++) sum += tiles[i] ? splits_of(chunk[i].units, units) : 0;
            return sum <= most;
        });
    }
    CHECK(per >= 1 && per <= kMostUnits);
    long long tasks = 0;
    for (int i = 0; i < c.n; i++) {
        const int mine = tasks_of_chunk<ROWS>(c, chunk[i], tiles[i], per, inv);
        int end = 0;
        for (int j = 0; j < tiles[i]; j++) {
            const int begin = tile_begin<ROWS>(c, chunk[i], tiles[i], j, inv), splits = tile_splits<ROWS>(c, chunk[i], j, per);
            CHECK(begin >= end && splits >= 1);
            end = begin + splits;
            CHECK(end <= mine);
            CHECK(tile_of_task<ROWS>(c, chunk[i], tiles[i], begin, inv) == j);
            CHECK(tile_of_task<ROWS>(c, chunk[i], tiles[i], end - 1, inv) == j);
        }
        tasks += mine;
    }
    CHECK(tasks <= part.tasks());
    return rows;
}

static void every_split_has_a_task() {
    int cut[2] = {}, whole = 0;
    for (int t = 0; t < 60000; t++) {
        Call c;
        c.n = pick(0, 9) ? pick(1, 70) : pick(1, 1100);
        c.group = pick(0, 2) ? 1 << pick(0, 5) : pick(1, 40);
        c.shift = pick(4, 8);
        c.seqs = pick(1, 5);
        const int wide = pick(0, 3) == 0, longest = 1 << (wide ? pick(0, 30 - c.shift) : pick(0, 12));
        c.max_pages = pick(0, 1) ? longest : pick(1, longest);
        const int cap = c.max_pages << c.shift, most = 1 << pick(0, c.n > 100 ? 4 : 11), long_one = pick(0, c.n - 1);
        c.start.push_back(0);
        for (int i = 0; i < c.n; i++) {
            const int kind = pick(0, 19);
            const int count = i == long_one ? pick(0, 4 * most) : kind < 2 ? 0 : kind < 12 ? 1 : pick(1, most);
            c.start.push_back(c.start.back() + count);
            const int near = cap - pick(0, cap < 300 ? cap : 300);
            c.at.push_back(kind == 0 ? -1 : kind == 1 ? INT_MAX - pick(0, 5) : kind < 6 ? near : pick(0, pick(0, 1) ? cap : cap / 2 + 1));
            c.seq.push_back(pick(0, 30) ? pick(0, c.seqs - 1) : pick(-1, c.seqs));
        }
        c.rows = c.start.back() + pick(0, 3);
        const int kv_heads = pick(0, 5) ? 1 << pick(0, 5) : pick(1, 700);
        if (((long long)c.rows * c.group / 16 + c.n) * kv_heads >= 1 << 23) continue;  // (refused)
        const Plan plan = plan_tasks(pick(0, 3) ? 256 : pick(1, 304), kv_heads, pick(0, 1), cap, true, c.n, c.rows, c.group);
        c.few_rows = plan.few_rows;
        // (whoever has no tasks is not launched)
        long long rows = 0;
        if (plan.few.tasks()) rows += check_part<16>(c, plan.few);
        if (plan.tile.tasks()) rows += check_part<128>(c, plan.tile);
        CHECK(rows == (long long)c.start.back() * c.group);
        cut[0] += plan.few.target > 0;
        cut[1] += plan.tile.target > 0;
        whole += plan.few.target == 0 && plan.tile.target == 0;
    }
    CHECK(cut[0] > 5000 && cut[1] > 5000 && whole > 5000);
}

// Chunks of one row each in row arrays of a fixed size: the rows behind them change nothing.
static void rows_behind_single_tokens() {
    for (int t = 0; t < 2000; t++) {
        const int cus = pick(1, 304), kv_heads = pick(1, 40), n = pick(1, 1100), group = pick(1, 40);
        const long long cap = 1LL << pick(4, 30);
        const bool fp32 = pick(0, 1);
        const Plan a = plan_tasks(cus, kv_heads, fp32, cap, false, n, n, group);
        const Plan b = plan_tasks(cus, kv_heads, fp32, cap, false, n, n + pick(1, 1 << 22), group);
        CHECK(a.few_rows == b.few_rows && a.few.tiles == b.few.tiles && a.few.target == b.few.target && a.few.blocks == b.few.blocks);
        CHECK(a.tile.tasks() == 0 && b.tile.tasks() == 0);
    }
}

int main() {
    rows_behind_single_tokens();
    every_split_has_a_task();
    fewest_units_of_a_split();
    printf("ok\n");
    return 0;
}
