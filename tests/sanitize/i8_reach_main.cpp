// The rule for products of rows in 8 bits (common_amd/csrc/i8_plan.h) on a card of 256 CUs.  Without arguments: every kind of
// launch that it comes to over a wide sweep of sizes.  With arguments "m,n,k,gated": the launch of each.  A line is
//   gated kind parts rounds   (parts: of k; rounds of blocks on the CUs, 2 standing for all above one)
#include <cstdio>
#include <set>
#include <tuple>

#include "../../common_amd/csrc/i8_plan.h"

static std::tuple<int, int, int, int> launch(int m, int n, int k, int gated) {
    const int cus = 256;
    const I8Plan p = i8_plan(m, n, (k + 15) / 16 * 16, gated, cus);
    if (p.kind == kRows) return {gated, p.kind, 1, 1};
    const auto& t = kTileSize[p.kind];
    const long long bn = gated ? t.gated_bn : t.bn, wide = gated ? 2LL * n : n;
    const long long tasks = ((long long)m + t.bm - 1) / t.bm * ((wide + bn - 1) / bn) * p.splits;
    return {gated, p.kind, p.splits, tasks > cus * t.per_cu ? 2 : 1};
}

static void print(const std::tuple<int, int, int, int>& l) {
    std::printf("%d %d %d %d\n", std::get<0>(l), std::get<1>(l), std::get<2>(l), std::get<3>(l));
}

int main(int argc, char** argv) {
    for (int i = 1; i < argc; i++) {
        int m, n, k, gated;
        if (std::sscanf(argv[i], "%d,%d,%d,%d", &m, &n, &k, &gated) != 4) return 1;
        print(launch(m, n, k, gated));
    }
    if (argc > 1) return 0;
    std::set<std::tuple<int, int, int, int>> seen;
    for (int gated = 0; gated < 2; gated++)
        for (double m = 1; m < 20000; m *= 1.07)
            for (double n = 16; n < 200000; n *= 1.1)
                for (double k = 64; k < 20000; k *= 1.15) seen.insert(launch((int)m, (int)n, (int)k, gated));
    for (const auto& l : seen) print(l);
}
