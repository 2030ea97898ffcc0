// kv4_rules.hpp -- which kernel attention over 4-bit pages takes, and how the work is
// cut: host functions of the sizes alone.
#pragma once

#include <cstddef>
#include <cstdint>

namespace bk {
namespace kv4 {

// Waves of a large block's workgroup, 32 rows each.  Heads of 256 values: the queries and O of
// 32 rows fill most of 512 registers, so a SIMD has one wave.
constexpr int prompt_waves(int D) { return D == 256 ? 4 : 8; }

// How a problem is cut, the same for the workspace's size and the launch.
struct Cut {
    int rows, row_blocks, slots, min_tiles;
    bool wide;                // one workgroup of many waves has a whole sequence
    int64_t items, grid;
    size_t part, bytes;
};

// Workgroups that the parts are made for: two a CU; heads of 256 values move
// enough bytes with fewer (40 sequences of up to 6000 tokens: 384 25.5 us, 512 29.4).
constexpr int slots_of(int D) { return D == 256 ? 384 : 512; }
constexpr int kMinTiles = 16;

// Tokens up to which one workgroup of eight waves takes a sequence whole: parts
// and their join cost a second launch.  One row, 8 kv heads, whole against cut,
// us: heads of 128, 1100 tokens 10.0 and 12.0, 2000 14.9 and 12.1; of 64, 2000 12.5
// and 12.3; of 256, 1100 12.8 and 12.6.  (Blocks of 32 rows see more.)
constexpr int whole_tokens(int D) { return D == 256 ? 1024 : D == 128 ? 1280 : 1792; }

// Blocks of 32 rows convert a token once for twice the rows of a block of 16, and
// have fewer waves for it: they pay where the blocks fill the card and their
// tokens are many.  16 rows against 32, us, heads of 64, 128, 256: 48 blocks of 32, 900
// tokens 9.5, 11.0, 15.6 and 14.4, 17.6, 46.7; 1700 tokens 12.8, 14.3, 17.6 and 13.0,
// 15.3, 26.6.  192 blocks, 6000 tokens 15.1, 23.4, 36.4 and 18.5, 23.3, 36.1.  320
// blocks, 900 tokens 11.5, 13.8, 25.1 and 15.2, 18.5, 49.0; 1500 tokens 14.2, 21.6,
// 29.9 and 14.2, 16.2, 27.0.
constexpr int64_t kManyBlocks = 256, kManySeen = 1024;

// Blocks of 16 or 32 rows, whose waves share out the tokens, or of 256 (128 for heads of
// 256 values), whose waves share the converted tokens?  The large blocks have a
// longer way in and pay where there is work for all CUs: the measure is blocks of
// 32 rows times tokens.  Large against small, us: heads of 128, 0.1 M 23 and 13, 0.6 M
// 36 and 43 (one kv head), 0.8 M 34.5 and 35.4, 1.5 M 38 and 44, 4.2 M 60 and 111, 24 M
// 187 and 278.  Heads of 64, 0.8 M 27 and 22, 1.2 M 32 and 28, 1.5 M 31 and 30, 4.2 M 45
// and 80.  Heads of 256: 0.3 M 40 and 29, 0.6 M 47 and 64, 4.2 M 131 and 233.  Up to
// kManySeen tokens against blocks of 16: heads of 128, 0.8 M 39 and 25, 2 M 36 and 36
// (of 500 tokens 35 and 44); of 256, 0.8 M 50 and 42, 2 M 59 and 71.
inline bool large_blocks(int64_t blocks, int64_t seen, int D) {
    if (seen <= kManySeen) return blocks * seen >= (D == 256 ? 1200000 : 1500000);
    return blocks * seen >= (D == 64 ? 1500000 : D == 128 ? 550000 : 500000);
}

// A launch has less than 2^32 threads, 512 of a workgroup at most.
constexpr int64_t kMaxGrid = 0x7fffff;

// Whether blocks of 256 rows, the largest there are, are too many already: past this
// the cut counts in 32 bits.
inline bool past_a_launch(int num_seqs, int max_q, int ratio, int hk) {
    return num_seqs && ((int64_t)max_q * ratio + 255) / 256 > kMaxGrid / ((int64_t)num_seqs * hk);
}

inline Cut cut_of(int num_seqs, int max_q, int64_t max_kv, int ratio, int hk, int D, int window) {
    Cut c{};
    const int64_t rows = (int64_t)max_q * ratio;
    const int64_t seen = window && window + (int64_t)max_q < max_kv ? window + (int64_t)max_q : max_kv;
    const int64_t blocks = (rows + 31) / 32 * num_seqs * hk;
    const bool large = rows > 32 && large_blocks(blocks, seen, D);
    c.rows = large ? 32 * prompt_waves(D) : rows > 16 && blocks >= kManyBlocks && seen > kManySeen ? 32 : 16;
    c.row_blocks = (int)((rows + c.rows - 1) / c.rows);
    c.items = (int64_t)num_seqs * c.row_blocks;
    if (large) {
        c.slots = seen <= 512 || c.items * hk >= 256 ? 0 : 256;
        c.min_tiles = 2 * kMinTiles;
    } else {
        c.slots = (c.rows == 16 && seen <= whole_tokens(D)) || c.items * hk >= 4096 ? 0 : slots_of(D);
        c.min_tiles = kMinTiles;
    }
    c.wide = !c.slots && c.rows == 16 && seen > 256 && c.items * hk <= 256;
    c.grid = c.items * hk + c.slots;
    if (c.slots) {
        c.grid = (c.grid + hk - 1) / hk * hk;
        c.part = ((size_t)c.items * 8 + 255) / 256 * 256;
        c.bytes = c.part + (size_t)c.grid * c.rows * (D + 2) * 4;
    }
    return c;
}

}  // namespace kv4
}  // namespace bk
