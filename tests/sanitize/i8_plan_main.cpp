// How products of rows in 8 bits are cut (common_amd/csrc/i8_plan.h), at every kind of size: a kernel that there is, parts of
// at least four steps of k, and work space for all of them.  (Which kernels sizes come to: i8_reach_main.cpp.)
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "../../common_amd/csrc/i8_plan.h"

static void fail(const char* what, int m, int n, int k, int gated) {
    std::printf("%s at %d x %d over %d, gated %d\n", what, m, n, k, gated);
    std::exit(1);
}

int main() {
    const int sizes[] = {1, 2, 15, 16, 17, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500, 768, 1000, 2048, 2560, 5000,
                         8192, 9728, 20000, 151936, 1 << 20, 1 << 24};
    const int ks[] = {16, 112, 128, 144, 512, 1024, 2048, 2064, 4096, 9728, 16384, 131072};
    int seen[kTiles + 1] = {}, split = 0;
    for (int cus : {256, 304, 64, 8})
        for (int gated = 0; gated < 2; gated++)
            for (int m : sizes)
                for (int n : sizes)
                    for (int k : ks) {
                        const I8Plan p = i8_plan(m, n, k, gated, cus);
                        const size_t work = i8_work_bytes(m, n, k, gated, cus);
                        if (p.kind < 0 || p.kind > kTiles) fail("no such kind", m, n, k, gated);
                        seen[p.kind]++;
                        if (p.kind == kRows) {
                            if (p.splits != 1 || work) fail("rows in parts", m, n, k, gated);
                            continue;
                        }
                        const auto& t = kTileSize[p.kind];
                        const int bn = gated ? t.gated_bn : t.bn;
                        if (bn == 0) fail("no such kernel", m, n, k, gated);
                        if (p.splits < 1 || (p.splits > 1 && (!t.split || k / 128 < 4 * p.splits))) fail("parts", m, n, k, gated);
                        const unsigned long long mt = (m + t.bm - 1) / t.bm, nt = ((gated ? 2ull : 1ull) * n + bn - 1) / bn;
                        if ((work > 0) != (p.splits > 1)) fail("work space", m, n, k, gated);
                        if (p.splits > 1) {
                            split++;
                            if (work != mt * nt * p.splits * t.bm * bn * 4) fail("work space", m, n, k, gated);
                            if (mt * nt >= (unsigned)cus) fail("parts of enough tiles", m, n, k, gated);
                        }
                    }
    for (int s : seen)
        if (!s) fail("a kind that no size takes", 0, 0, 0, 0);
    if (!split) fail("nothing in parts", 0, 0, 0, 0);
    std::puts("ok");
}
