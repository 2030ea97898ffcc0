// w4_rules.hpp -- which kernel a product with 4-bit weights takes: host functions of
// the sizes alone.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace bk {
namespace w4 {

// ---- tiles -----------------------------------------------------------------------
// Shapes of w4_tiles.hip: TM rows of x by TN rows of the weights; of two of the same
// size the DEEP one has a CU to itself and cuts K over groups of waves.
enum TileShape {
    T_32x64, T_32x128, T_32x128_DEEP, T_64x128_DEEP, T_64x256, T_128x128_DEEP, T_128x256_DEEP, T_128x256, T_192x256, T_256x256,
    T_COUNT
};
struct TileCost {
    int tm, tn;
    int share;      // tiles that share a CU
    float fixed;    // us of a round: launch, first loads, end
    float step;     // us per 64 values of K, a tile alone on its CU and few of them
    float load;     // ... how much more of that where every CU has one
    float shared;   // us per 64 values of as many tiles as share a CU
};
// Fitted to every shape's times (us) over 102 sizes of 32 to 4097 rows, N = 1000 to 60000,
// K = 512 to 14336, and 70 mixtures, bf16, weights from HBM: the picks lie 0.7% above the
// best of the ten on the average, 15% at most (of mixtures, whose counts the host does
// not know, 1.4%).  200 x 11008 x 4096: 128x128 29, 64x256 35, 128x256 44; 777 x 11007 x
// 4096: 192x256 73, 256x256 82, 128x256 85; 64 x 14336 x 4096: 32x128 deep 15.6, 32x64 18;
// 64 x 60000 x 1024: 64x256 14, 32x128 19, 128x256 18.
constexpr TileCost kTileCost[T_COUNT] = {
    {32, 64, 2, 5.6f, 0.082f, 0.36f, 0.158f},  {32, 128, 3, 6.0f, 0.138f, 0.49f, 0.377f}, {32, 128, 1, 6.0f, 0.132f, 0.0f, 0.0f},
    {64, 128, 1, 7.0f, 0.176f, 0.27f, 0.0f},   {64, 256, 2, 6.7f, 0.376f, 0.27f, 0.812f}, {128, 128, 1, 6.7f, 0.304f, 0.28f, 0.0f},
    {128, 256, 1, 9.2f, 0.468f, 0.50f, 0.0f},  {128, 256, 2, 7.9f, 0.449f, 0.78f, 1.362f}, {192, 256, 1, 8.2f, 0.862f, 0.19f, 0.0f},
    {256, 256, 1, 8.5f, 1.035f, 0.29f, 0.0f},
};
constexpr int64_t kMaxTiles = 1 << 21;      // workgroups of a launch, of up to 1024 threads

// n tiles a CU, of a launch that fills `full` of the 256 CUs' first tiles.
inline float cu_us(const TileCost &c, float n, float full, int k) {
    const float kt = (float)((k + 63) / 64), one = c.fixed + kt * c.step * (1.0f + c.load * std::min(1.0f, full));
    if (c.share == 1) return n * one;
    const float all = c.fixed + kt * c.shared, share = (float)c.share;
    if (n <= 1.0f) return one;
    return n <= share ? one + std::max(0.0f, all - one) * (n - 1.0f) / (share - 1.0f) : n / share * all;
}

// Of one matrix's rows: up to three rounds of tiles over the CUs are whole ones, later
// ones overlap.
inline float tile_us(const TileCost &c, int64_t tiles, int k) {
    const float full = (float)tiles / 256.0f;
    const int64_t rounds = (tiles + 255) / 256;
    return cu_us(c, rounds <= 3 * c.share ? (float)rounds : full + 0.5f, full, k);
}

// By expert, where the GPU alone knows the counts: the experts that can have rows are
// taken to have them with an exponential spread, tiles of rows in whole numbers.  Tiles
// that share CUs overlap their rounds, and half of one more is taken as begun.
inline float moe_tile_us(const TileCost &c, int64_t pairs, int experts, int n, int k) {
    const float active = (float)std::min<int64_t>(experts, pairs), mean = (float)pairs / active;
    const float rows = std::max(1.0f, std::round(active / (1.0f - std::exp(-0.85f * (float)c.tm / mean))));
    const float full = rows * (float)((n + c.tn - 1) / c.tn) / 256.0f;
    const float rounds = c.share == 1 && full <= 2.5f ? std::ceil(full) : full + 0.5f;
    return cu_us(c, std::max(1.0f, rounds), full, k);
}

// Tiles of rows that there can be at most.  experts: 0 where the rows are one matrix's.
inline int64_t most_tile_rows(int64_t rows, int experts, int tm) {
    return (rows + tm - 1) / tm + std::min<int64_t>(experts, rows);
}

inline TileShape tile_shape(int64_t rows, int experts, int n, int k) {
    int best = T_256x256;
    float us = 0.0f;
    for (int i = T_256x256; i >= 0; --i) {
        const TileCost &c = kTileCost[i];
        const int64_t tn = (n + c.tn - 1) / c.tn;
        if (i != T_256x256 && most_tile_rows(rows, experts, c.tm) * tn > kMaxTiles) continue;
        const float t = experts ? moe_tile_us(c, rows, experts, n, k) : tile_us(c, (rows + c.tm - 1) / c.tm * tn, k);
        if (i == T_256x256 || t < us) best = i, us = t;
    }
    return (TileShape)best;
}

// ---- few rows ---------------------------------------------------------------------
// Where w4_rows.hip takes the product: 16 rows a workgroup, so that more rows read the
// weights again (from L2), but K is cut over its waves.  Up to 16 rows always (16 x
// 28672 x 4096 17.1 us, the best tile 17.2), and more of them on grids of up to 320
// workgroups of 64 weight rows: 64 x 4096 x 4096 8.1 / 10.9, 48 x 4096 x 14336 18.6 / 27.8,
// 128 x 1024 x 4096 5.7 / 10.3, 64 x 5120 x 2880 8.5 / 9.7; past it 128 x 4096 x 4096 12.1 /
// 11.5, 32 x 14336 x 4096 14.7 / 13.2, 48 x 8192 x 8192 20.1 / 19.2.
inline bool rows_pay(int64_t rows, int n) {
    return rows <= 16 || (int64_t)((n + 63) / 64) * ((rows + 15) / 16) <= 320;
}

// By expert, with the average of rows of the experts that can have any: few rows an
// expert, or few workgroups.  us, rows / best tile: 16 tokens, 2 of 8 experts 28672 x 4096
// (average 4) 94 / 98, 32 tokens, 6 of 64 2816 x 2048 (3) 35 / 38, 64 tokens (6) 47 / 40, 8 of 128
// 1536 x 2048 (4) 44 / 40, 4 experts 8640 x 544 (4) 11 / 13, 4 experts 384 x 9216 (18) 12 / 22,
// 16 experts 816 x 3200 (13) 17 / 15.
inline bool moe_rows_pay(int64_t pairs, int experts, int n) {
    const int64_t active = std::min<int64_t>(experts, pairs), groups = (int64_t)((n + 63) / 64) * (pairs / 16 + active / 2);
    return pairs <= 3 * active || groups <= 224 || (pairs <= 6 * active && groups <= 512);
}

// Rows of x that a workgroup holds: 2, 4, 8 or 16.
inline int rows_held(int64_t rows) { return rows <= 2 ? 2 : rows <= 4 ? 4 : rows <= 8 ? 8 : 16; }

// By expert no more than 8 where most experts have fewer: 20 tokens, 2 of 16 experts 1000 x
// 512 5.7 us, 16 held 7.2; 32 tokens, 6 of 64 2816 x 2048 (average 3) 37.6, 35.3.
inline int moe_rows_held(int64_t pairs, int experts) {
    const int most = rows_held(pairs);
    return 4 * pairs < 11 * std::min<int64_t>(experts, pairs) ? std::min(most, 8) : most;
}

// ... and how many workgroups over the rows are likely.
inline int64_t moe_rows_likely(int64_t pairs, int experts, int held) {
    return std::max<int64_t>(1, pairs / held + std::min<int64_t>(experts, pairs) / 2);
}

// ---- few pairs of a mixture --------------------------------------------------------
// Up to this many sorted pairs a workgroup finds its expert's rows from the ids, 64
// positions (a chunk) at a time: bit l of head[i] is set where position 64 i + l has
// another id than the one before it, as the first position past the pairs has.
constexpr int kFewPairs = 256, kFewChunks = kFewPairs / 64;

// Where the run of equal ids began that holds position 64 i + l; `from`: the run that
// reaches into chunk i.
constexpr int run_began(uint64_t head, int i, int l, int from) {
    const uint64_t upto = head & (~0ull >> (63 - l));
    return upto ? 64 * i + 63 - __builtin_clzll(upto) : from;
}

// Positions of that run from 64 i + l on; where there are TB of them or more, TB or more.
// TB rows from any lane touch REACH chunks behind their own at most.
template <int TB>
constexpr int run_left(const uint64_t (&head)[kFewChunks], int i, int l) {
    constexpr int REACH = (TB + 62) / 64;
    const uint64_t later = l < 63 ? head[i] >> (l + 1) : 0;
    if (later) return __builtin_ctzll(later) + 1;
    int left = 64 - l;
#if defined(__clang__)
#pragma unroll
#endif
    for (int j = 1; j <= REACH; ++j) {
        if (i + j >= kFewChunks) break;
        if (head[i + j]) return left + __builtin_ctzll(head[i + j]);
        left += 64;
    }
    return left;
}

struct RowsShape {
    int blocks, waves;      // of 16 weight rows a workgroup; that divide K
};
// `slots`: workgroups over the rows.  A wider workgroup reads x fewer times, a narrower
// one fills the card with fewer weight rows; us by 1 / 2 / 4 blocks, the better of the
// waves: 1 x 28672 x 4096 13.8 / 14.5 / 15.0, 4 x 14336 x 4096 9.1 / 8.7 / 9.2, 16 x 4096 x
// 4096 5.8 / 6.3 / 8.0, 32 x 4096 x 4096 8.0 / 6.4 / 8.1, 64 x 4096 x 4096 11.9 / 8.7 / 8.1,
// 8 x 14336 x 4096 10.8 / 9.3 / 9.5, 16 x 14336 x 4096 13.8 / 10.9 / 10.3.
// Waves: eight, sixteen for a deep K on a small grid (1 x 4096 x 14336 8.2, with eight
// 10.5), four on a large grid of wide workgroups (16 x 28672 x 4096 17.1, 18.5) and for up
// to four words of K (1 x 60000 x 1024 8.4, 10.7), two of both (16 x 60000 x 1024 10.6, with
// four 12.1).  Gated, sixteen waves spill 20 to 24 registers at the end and pay on the
// smallest grids alone: 1 x 1024 x 14336 10.4, with eight 12.3, 1 x 2048 x 8192 7.9 / 8.2, but
// 1 x 4096 x 8192 9.0 / 8.9, 1 x 7168 x 8192 10.9 / 10.4, 8 x 7168 x 8192 11.7 / 11.0.
inline RowsShape rows_shape(int held, int64_t slots, int n, int k, bool gated) {
    const int64_t g = (int64_t)((n + 15) / 16) * slots;
    const int words = (k + 255) / 256;
    RowsShape s;
    if (held <= 2) s.blocks = 1;
    else if (held <= 4) s.blocks = g > 512 ? 2 : 1;
    else s.blocks = g <= 256 ? 1 : g <= 512 || (held <= 8 && g <= 1024) ? 2 : 4;
    if (gated) s.blocks = std::max(s.blocks, 2);          // gate and up
    const int64_t groups = g / s.blocks;
    s.waves = words <= 4 ? 4 : 8;
    if (s.blocks == 4 && groups >= 320) s.waves = 4;
    if (words <= 4 && s.blocks > 1 && groups >= 512) s.waves = 2;
    if (words >= 32 && s.blocks < 4 && groups <= 256) s.waves = 16;
    return s;
}

// Whether rows_shape gives this form for any sizes, so that no other is compiled: one or
// two blocks for up to 2 rows held, no four for up to 4; two waves for two blocks or more
// on 512 workgroups, which 16 rows held by two blocks never have; sixteen for fewer blocks
// than four.
constexpr bool rows_form(int held, int blocks, int waves, bool gated) {
    if (blocks == 1 ? gated : blocks == 2 ? held == 2 && !gated : held <= 4) return false;
    if (waves == 2) return blocks == 4 || (blocks == 2 && held < 16);
    return waves == 16 ? blocks < 4 : waves == 4 || waves == 8;
}


}  // namespace w4
}  // namespace bk
