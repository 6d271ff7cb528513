// How the paged attention's keys are cut into tasks (common_amd/csrc/page_index.h), against plain loops and at the
// largest sizes that its calls accept; built with the address and undefined-behaviour sanitizers.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../common_amd/csrc/page_index.h"

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

int main() {
    fewest_units_of_a_split();
    printf("ok\n");
    return 0;
}
