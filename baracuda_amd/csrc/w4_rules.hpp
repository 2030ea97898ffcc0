// w4_rules.hpp -- which kernel a product with 4-bit weights takes: host functions of
// the sizes alone.
#pragma once

#include <algorithm>
#include <cstdint>

namespace bk {
namespace w4 {

// ---- tiles -----------------------------------------------------------------------
// Shapes of w4_tiles.hip: TM rows of x by TN rows of the weights.
enum TileShape { T_32x64, T_32x128, T_32x128_DEEP, T_64x128, T_64x256, T_128x128, T_128x256, T_192x256, T_256x256, T_COUNT };
struct TileCost {
    int tm, tn;
    float fixed;    // us of a round: launch, first loads, end
    float step;     // us per 64 values of K, a tile alone on its CU and few of them
    float load;     // ... how much more of that where every CU has one
    float paired;   // us per 64 values of two tiles that share a CU (0: LDS holds one)
};
// Fitted to every shape's times (us) over 32 to 4097 rows, N = 1024 to 60000, K = 512 to
// 14336, bf16, weights from HBM: the picks lie 0.4% above the best of the nine on the
// average of 86 sizes, 8% at most.  200 x 11008 x 4096: 128x128 28.7, 64x256 30.9, 64x128
// 37.4, 128x256 44.3; 777 x 11008 x 4096: 192x256 74.7, 256x256 82.7, 128x128 88.4; 64 x
// 14336 x 4096: 32x128 deep 15.9, 32x64 18.3, 64x128 20.1; 32 x 60000 x 1024: 32x128 13.2,
// 64x256 15.1, 32x64 16.9.
constexpr TileCost kTileCost[T_COUNT] = {
    {32, 64, 4.8f, 0.097f, 0.21f, 0.167f},  {32, 128, 4.9f, 0.181f, 0.19f, 0.288f}, {32, 128, 5.4f, 0.132f, 0.07f, 0.0f},
    {64, 128, 6.2f, 0.187f, 0.26f, 0.0f},   {64, 256, 7.0f, 0.305f, 0.45f, 0.0f},   {128, 128, 5.7f, 0.324f, 0.26f, 0.0f},
    {128, 256, 7.2f, 0.482f, 0.56f, 0.0f},  {192, 256, 6.2f, 0.882f, 0.25f, 0.0f},  {256, 256, 6.5f, 0.986f, 0.41f, 0.0f},
};
constexpr int64_t kMaxTiles = 1 << 22;      // workgroups of a launch

// Of one matrix's rows: up to three rounds of tiles over the 256 CUs are whole ones,
// later ones overlap.
inline float tile_us(const TileCost &c, int64_t tiles, int k) {
    const float kt = (float)((k + 63) / 64), full = (float)tiles / 256.0f;
    const int64_t rounds = (tiles + 255) / 256;
    const float one = c.fixed + kt * c.step * (1.0f + c.load * std::min(1.0f, full));
    if (c.paired == 0.0f) return rounds <= 3 ? (float)rounds * one : (full + 0.5f) * one;
    const float two = c.fixed + kt * c.paired;
    return rounds <= 3 ? (float)(rounds / 2) * two + (float)(rounds % 2) * one : (full + 0.5f) / 2.0f * two;
}

// By expert, where the GPU alone knows the counts: an expert's last tile is taken as
// filled by a third, and a round that may just be passed as half begun.  The picks lie
// 1.6% above the best shape on the average of 75 mixtures of 2 to 128 experts with uneven
// shares (with the last tile half full and whole rounds 3.3%).
inline float moe_tile_us(const TileCost &c, int64_t pairs, int experts, int n, int k) {
    const float rows = std::max(1.0f, (float)pairs / (float)c.tm + 0.7f * (float)std::min<int64_t>(experts, pairs));
    const float kt = (float)((k + 63) / 64), full = rows * (float)((n + c.tn - 1) / c.tn) / 256.0f;
    const float one = c.fixed + kt * c.step * (1.0f + c.load * std::min(1.0f, full)), rounds = std::max(1.0f, full + 0.5f);
    if (c.paired == 0.0f) return rounds * one;
    return rounds <= 1.0f ? one : std::max(one, rounds / 2.0f * (c.fixed + kt * c.paired));
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
// four 12.1).
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

}  // namespace w4
}  // namespace bk
