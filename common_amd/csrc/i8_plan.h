// How a product of rows in 8 bits is cut: which kernel, which tiles, k in how many parts.  No HIP in here: the host's tests
// compile it, too.
#pragma once

#include <cstddef>

// The kernels that products go to: a tile's tokens and weight rows (gated: half of them gate rows), the LDS buffers of 128
// bytes of k that it goes through, blocks on a CU at a time, and whether it takes parts of k.
enum Kind { kTile32, kTile64, kTile64x128, kTile128, kTile128x256, kTile256x192, kTile256, kTiles, kRows = kTiles };
constexpr struct TileSize {
    int bm, bn, buffers, gated_bn, gated_buffers, per_cu;
    bool split;
} kTileSize[kTiles] = {{32, 128, 4, 128, 4, 2, true},   {64, 64, 4, 128, 3, 2, true},   {64, 128, 5, 0, 0, 1, true},
                       {128, 128, 4, 128, 4, 1, true},  {128, 256, 3, 256, 3, 1, false}, {256, 192, 2, 0, 0, 1, false},
                       {256, 256, 2, 256, 2, 1, false}};
struct I8Plan {
    Kind kind;
    int splits;
};

// What a product takes by each kind of tile, in us, up to what they have in common: tiles go in rounds of per_cu blocks a CU;
// in a round a CU copies 70 KB a us, 128 bytes of k take 0.85 / (buffers - 1) us at least, the way from memory, and outputs
// are finished one after the other.  Parts of k cost a launch and their sums' way through memory.  Fitted to 520 sizes by every
// kind and number of parts (17 to 10,000 tokens, 768 to 20,000 outputs over 768 to 14,336; several sets of weights in turn, which
// the last-level cache still holds for 200 of the sizes), of which the choice is 0.7% behind the fastest on average, more than
// 4.4% in one of 20 and 15% at worst (68 x 4,096 over 14,336; MI355X; profiles/int8_tile_times.txt).  It does not know whether
// weights come from memory: 509 x 2,560 over 9,728 by 64 x 128 tiles 24.6 us from the last-level cache and 36 from memory, by
// 128 x 128 in three parts 27 to 28 and 30.5.  Both sides of it, us, from the cache: 509 x 2,560 over 9,728 by 64 x 128 tiles
// 24.6, 128 x 128 32.2, 64 x 64 30.8; 448 x 2,048 over 6,144 by 64 x 64 17.2, 64 x 128 23.8; 1,024 x
// 6,144 over 2,560 by 128 x 256 25.4, 128 x 128 33, 256 x 256 36.5; 2,048 x 6,144 over 2,560 by 256 x 192 43.2, 256 x 256 46.5,
// 128 x 256 52.8; 64 x 2,560 over 9,728 by 64 x 64 18.4, in 4 parts 13.5; 100 x 768 over 768 by 64 x 64 4.8, 256 x 256 14.9.
inline I8Plan i8_plan(int M, int N, int K, bool gated, int cus) {
    // One tile of tokens over few outputs: 16 of them a block of 8 wavefronts, without LDS on the way (8 tokens x 2,560 over
    // 4,096 5.7 us, by 32 x 128 tiles 10.3; 16 x 2,560 over 9,728 11.2 and 12.2; but 8 x 9,728 gated over 2,560 14.9 and 13.6,
    // 16 x 151,936 over 2,048 83 and 52, where part of the weights comes from the last-level cache; all from memory 60).
    if (M <= 16 && (N + 15) / 16 * (gated ? 2 : 1) <= 2 * cus) return I8Plan{kRows, 1};
    I8Plan best{kTile256, 1};
    double least = 1e30;
    for (int kind = 0; kind < kTiles; kind++) {
        const auto& t = kTileSize[kind];
        const int bn = gated ? t.gated_bn : t.bn;
        if (bn == 0) continue;
        const double buffers = gated ? t.gated_buffers : t.buffers;
        const double tiles = (double)((M + t.bm - 1) / t.bm) * ((N * (gated ? 2LL : 1LL) + bn - 1) / bn);
        const double most = t.split && tiles < cus ? (K / 512 < 8 ? K / 512 : 8) : 1;  // (four steps a part or more)
        for (int splits = 1; splits == 1 || splits <= most; splits++) {
            const double blocks = tiles * splits, rounds = (double)(long long)(blocks / (cus * t.per_cu));
            const double rest = blocks - rounds * (cus * t.per_cu);
            const auto round = [&](int on_a_cu) {
                const double copies = (t.bm + bn) * on_a_cu / 70e3, latency = 0.85 / (128 * (buffers - 1));
                const double finish = splits > 1 ? 0 : t.bm * bn * on_a_cu * (gated ? 1.7e-4 : 1.1e-4);
                return (copies > latency ? copies : latency) * K / splits + finish;
            };
            const double sums = splits > 1 ? 8.5 + 8.0 * M * N * (gated ? 2 : 1) * splits / 4e6 : 0;
            const double us = rounds * round(t.per_cu) + (rest > cus ? round(2) : rest > 0 ? round(1) : 0) + sums;
            if (us < least) {
                least = us;
                best = I8Plan{(Kind)kind, splits};
            }
        }
    }
    return best;
}

// Bytes that the parts' sums take.
inline size_t i8_work_bytes(int M, int N, int K, bool gated, int cus) {
    const I8Plan plan = i8_plan(M, N, K, gated, cus);
    if (plan.splits == 1) return 0;
    const auto& t = kTileSize[plan.kind];
    const int bn = gated ? t.gated_bn : t.bn;
    const size_t tiles = (size_t)((M + t.bm - 1) / t.bm) * ((N * (gated ? 2LL : 1LL) + bn - 1) / bn);
    return tiles * plan.splits * t.bm * bn * 4;
}
