// The index arithmetic of the paged cache (common_amd/csrc/page_index.h) against plain loops, on well-formed arrays
// and on arrays full of anything; built with the address and undefined-behaviour sanitizers, so that an index outside
// its array ends the program.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../common_amd/csrc/page_index.h"

static std::mt19937 rng(7);
static int pick(int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); }
static int any() {
    static const int odd[] = {INT_MIN, INT_MIN + 1, -1000000, -1, 0, 1, 2, 63, 64, 1000000, INT_MAX - 1, INT_MAX};
    return pick(0, 1) ? odd[pick(0, 11)] : pick(-5, 200);
}
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); exit(1); } } while (0)

int main() {
    for (int t = 0; t < 20000; t++) {
        const int n = pick(1, 40), span = 1 << pick(0, 7);
        std::vector<int> start(n + 1, 0);
        for (int i = 0; i < n; i++) start[i + 1] = start[i] + (pick(0, 3) ? pick(0, 3 * span) : 0);
        const int rows = start[n] + pick(0, 9);
        // every row of a chunk is found, and no other
        std::vector<int> owner(rows + 1, -1);
        for (int i = 0; i < n; i++)
            for (int r = start[i]; r < start[i + 1]; r++) owner[r] = i;
        for (int k = 0; k < 20; k++) {
            const int r = pick(-2, rows + 1);
            CHECK(chunk_of_row(start.data(), n, rows, r) == (r < 0 || r >= rows ? -1 : owner[r]));
        }
        // the slots: every tile of every chunk has one, in order, and their number is bounded
        const int per = pick(1, 9);
        auto of_slot = [&](int64_t slot) {
            return chunk_search(n, 4, [&](int i, int k, int len) {
                int c = 0;
                for (int j = 0; j < 4 && j * k < len && chunk_slot(start[i + j * k], i + j * k, per, span) <= slot; j++) c++;
                return c;
            });
        };
        int64_t before = 0;
        for (int i = 0; i < n; i++) {
            const int64_t a = chunk_slot(start[i], i, per, span), b = chunk_slot(start[i + 1], i + 1, per, span);
            CHECK(a == before && b - a >= (per * (start[i + 1] - start[i]) + span - 1) / span);
            for (int64_t s = a; s < b; s++) CHECK(of_slot(s) == i);
            before = b;
        }
        CHECK(before <= (int64_t)rows * per / span + n);
        // one row each
        CHECK(chunk_of_row(nullptr, n, n + 3, n - 1) == n - 1 && chunk_of_row(nullptr, n, n + 3, n) == -1);
        // anything: indexes stay inside, counts stay inside the rows
        for (auto& s : start) s = any();
        for (int k = 0; k < 20; k++) {
            const int c = chunk_of_row(start.data(), n, rows, any()), d = of_slot(any());
            CHECK(c >= -1 && c < n && d >= 0 && d < n);
        }
        for (int i = 0; i < n; i++) {
            int first, count;
            chunk_rows(start.data(), i, rows, &first, &count);
            CHECK(count >= 0 && (count == 0 || (first >= 0 && (int64_t)first + count <= rows)));
        }
        // pages
        const int seqs = pick(1, 5), cols = pick(1, 6), pages = pick(1, 50), shift = pick(4, 8);
        std::vector<int> table(seqs * cols);
        for (auto& x : table) x = pick(0, 2) ? pick(0, pages - 1) : any();
        for (int k = 0; k < 40; k++) {
            const int s = pick(0, 2) ? pick(0, seqs - 1) : any(), r = pick(0, 2) ? pick(0, (cols << shift) + 5) : any();
            int want = -1;
            if (s >= 0 && s < seqs && r >= 0 && (int64_t)r < ((int64_t)cols << shift)) {
                want = table[s * cols + r / (1 << shift)];
                if (want < 0 || want >= pages) want = -1;
            }
            CHECK(page_of_row(table.data(), seqs, cols, pages, shift, s, r) == want);
        }
        const int a = any(), j = any();
        const int64_t sum = (int64_t)a + j;
        CHECK(cache_row(a, j) == (a < 0 || j < 0 || sum > INT_MAX ? -1 : (int)sum));
    }
    printf("ok\n");
    return 0;
}
