// kv4_attention.hpp -- what the attention kernels over 4-bit pages share: the
// arguments, which tokens a block of rows sees, and how the work is cut.
//
//   o = softmax(scale q k^T + mask) v
//
// A sequence's new tokens are its last ones: token i of n stands at position
// len - n + i.  `causal` hides the positions after a row's own (a row is a token
// and a head), a window w those that lie w or more before it, each by itself: a
// row with both sees the last w positions up to its own, one with a window alone
// those and all later ones.  A row that sees nothing gives zeros.  Rows of one kv head are taken
// together: row r is token r / ratio and head r % ratio of the group.
#pragma once

#include "kv4.hpp"

namespace bk {
namespace kv4 {

struct AttnArgs {
    const void *q;
    void *out;
    const uint8_t *cache;
    const int32_t *tables, *lens, *cu_q;
    int64_t q_token, q_head, out_token, out_head, table_stride, num_pages;
    int64_t part;              // bytes from `split` to the partial results
    char *split;               // workspace: int2 per item, then m and l, then O of each part
    uint32_t ratio_magic;      // ceil(2^32 / ratio) where that divides every row number exactly, else 0
    int num_seqs, total_q, hq, hk, ratio, max_pages, ps, ps_shift, causal, window;
    int row_blocks;            // blocks of rows of a sequence
    int items;                 // num_seqs * row_blocks
    int paired;                // large blocks take half their rows from a sequence's end
    int slots;                 // workgroups that the parts are made for; 0: nothing is split
    int min_tiles;             // tiles of 16 tokens that a part has at least
    float scale;               // times log2(e)
};

// A block of rows and the tokens [lo, hi) that any of them sees.
struct Item {
    int seq, q0, n, first, rows, base, len, lo, hi;
};

__device__ __forceinline__ int token_of(const AttnArgs &a, int row) {
    if (a.ratio == 1) return row;
    return a.ratio_magic ? (int)__umulhi((uint32_t)row, a.ratio_magic) : row / a.ratio;
}

// The first position that the window of a row at `pos` holds.  A row before the cache's
// start (more new tokens than it holds) has a negative one: no difference of the
// two, which may pass 32 bits.
__device__ __forceinline__ int first_seen(const AttnArgs &a, int pos) {
    return a.window && pos >= a.window ? pos - a.window + 1 : 0;
}

__device__ __forceinline__ Item item_of(const AttnArgs &a, int item, int block) {
    Item s;
    s.seq = a.row_blocks == 1 ? item : item / a.row_blocks;
    int q0 = s.seq, n = 1;
    if (a.cu_q) {
        q0 = a.cu_q[s.seq];
        n = a.cu_q[s.seq + 1] - q0;
    }
    if (q0 < 0 || n < 0 || n > a.total_q - q0) n = 0;
    const int len = a.lens[s.seq];
    const int64_t room = (int64_t)a.max_pages << a.ps_shift;
    s.q0 = q0;
    s.n = n;
    s.base = len - n;
    s.len = (int)(len < room ? len : room);
    s.first = (item - s.seq * a.row_blocks) * block;
    s.rows = min(block, n * a.ratio - s.first);
    s.lo = s.hi = 0;
    if (s.rows > 0) {
        const int i0 = token_of(a, s.first), i1 = token_of(a, s.first + s.rows - 1);
        s.hi = max(0, a.causal ? min(s.len, s.base + i1 + 1) : s.len);
        s.lo = first_seen(a, s.base + i0);
    }
    return s;
}

__device__ __forceinline__ int tiles_of(const Item &s) { return s.hi > s.lo ? (s.hi + 15) / 16 - s.lo / 16 : 0; }

// The tokens that a row sees: [lo, hi).
__device__ __forceinline__ void row_span(const AttnArgs &a, const Item &s, int r, int &lo, int &hi) {
    const int pos = s.base + token_of(a, s.first + r);
    const bool in = r < s.rows;
    hi = in ? (a.causal ? min(s.len, pos + 1) : s.len) : 0;
    lo = in ? first_seen(a, pos) : 0;
}

__device__ __forceinline__ float as_float(uint32_t x) { return __uint_as_float(x); }

// Lanes that differ in bit 4, and in bit 5: the four groups of 16 that hold
// the same row (v_permlane*_swap: no trip through LDS).
__device__ __forceinline__ float max_over_groups(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(as_float(a[0]), as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(as_float(b[0]), as_float(b[1]));
}
__device__ __forceinline__ float sum_over_groups(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = as_float(a[0]) + as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return as_float(b[0]) + as_float(b[1]);
}

// Inclusive sums over the wave's lanes (DPP row shifts and broadcasts).
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);    // within rows of 16: 1, 2, 4, 8 lanes up
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row 0's sum to row 1, row 2's to row 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // the first half's to the second
    return x;
}
// A part of an item: tiles [t0, t1) of 16 tokens.  `parts` parts have the item,
// the first of them is part `begin` of all.
struct Part {
    int item, t0, t1, parts, begin;
};

// Part `index` of all, and its item, worked out from the lengths by one wave: all
// items together are cut into about slots / hk parts of one size, so that the
// longest sequence does not hold up the launch.  Up to 64 items cost one pass
// over the lengths and are put in line by size, in powers of two: a CU is given
// parts that lie apart in line, and would with bad luck have several long ones
// (48 sequences of up to 8192 tokens: 17.2 us in line, 18.6 in their order).
// part.item < 0: there is no such part.
__device__ __forceinline__ void find_part(const AttnArgs &a, int block, int index, Part &part, Item &item) {
    const int lane = threadIdx.x & 63;
    Item s;
    // all tiles together may pass 32 bits: summed in two pieces
    int high = 0, low = 0;
    for (int i0 = 0; i0 < a.items; i0 += 64) {
        s.rows = s.lo = s.hi = 0;
        if (i0 + lane < a.items) s = item_of(a, i0 + lane, block);
        high += tiles_of(s) >> 12, low += tiles_of(s) & 4095;
    }
    const int64_t total = ((int64_t)__builtin_amdgcn_readlane(wave_scan(high), 63) << 12) +
                          __builtin_amdgcn_readlane(wave_scan(low), 63);
    const int per = max(a.min_tiles, (int)((total * a.hk + a.slots - 1) / a.slots));
    int begin = 0;
    for (int i0 = 0; i0 < a.items; i0 += 64) {
        if (a.items > 64) {
            s.rows = s.lo = s.hi = 0;
            if (i0 + lane < a.items) s = item_of(a, i0 + lane, block);
        }
        const int tiles = tiles_of(s);
        const int n = s.rows > 0 ? max(1, (tiles + per - 1) / per) : 0;
        int mine, all;
        if (a.items <= 64) {
            const int many = n > 1 ? n : 0;
            mine = wave_scan(many);
            all = __builtin_amdgcn_readlane(mine, 63);
            mine -= many;
            const int size = n > 1 ? 0 : tiles * 2 > per ? 1 : tiles * 4 > per ? 2 : tiles * 8 > per ? 3 : 4;
#pragma unroll
            for (int c = 1; c < 5; ++c) {
                const uint64_t of = __ballot(n == 1 && size == c);
                if (size == c)
                    mine = all + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(of >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)of, 0));
                all += __popcll(of);
            }
        } else {
            all = wave_scan(n);
            mine = begin + all - n;
            all = __builtin_amdgcn_readlane(all, 63);
        }
        const bool hit = index >= mine && index < mine + n;
        if (hit) {
            // equal parts of the item
            const int each = (tiles + n - 1) / n, k = index - mine, t0 = s.lo / 16;
            part = Part{i0 + lane, t0 + min(tiles, k * each), t0 + min(tiles, (k + 1) * each), n, mine};
            item = s;
        }
        if (__any(hit)) return;
        begin += all;
    }
    if (lane == 0) part.item = -1;
}

// The same in scalar registers: all lanes hold the same.
__device__ __forceinline__ Item uniform(const Item &s) {
    const auto f = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    return Item{f(s.seq), f(s.q0), f(s.n), f(s.first), f(s.rows), f(s.base), f(s.len), f(s.lo), f(s.hi)};
}
__device__ __forceinline__ Part uniform(const Part &p) {
    const auto f = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    return Part{f(p.item), f(p.t0), f(p.t1), f(p.parts), f(p.begin)};
}

template <typename T>
__device__ __forceinline__ v4f mfma_pv(const v4i &a, const v4i &b, const v4f &c);
template <>
__device__ __forceinline__ v4f mfma_pv<Bf16>(const v4i &a, const v4i &b, const v4f &c) {
    return mfma16x16x32_h<true>(a, b, c);
}
template <>
__device__ __forceinline__ v4f mfma_pv<F16>(const v4i &a, const v4i &b, const v4f &c) {
    return mfma16x16x32_h<false>(a, b, c);
}

// Byte `sel` of w, two codes, as a pair of elements under `scale` (exact for
// every scale that kv4_append writes; f16 rounds scales below 2^-23).
template <typename T>
__device__ __forceinline__ uint32_t pair_of(uint32_t w, float scale, int sel) {
    if constexpr (__is_same(T, Bf16)) {
        switch (sel) {
            case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
            case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
            case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
            default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
        }
    } else {
        switch (sel) {
            case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0));
            case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1));
            case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2));
            default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
        }
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (__is_same(T, Bf16)) {
        return f32x2_to_bf16x2(lo, hi);
    } else {
        return f32x2_to_f16x2(lo, hi);
    }
}

// The scale of a conversion: the instruction reads the exponent alone, and 255
// there makes its results NaN, so the bits around the byte may be anything.
__device__ __forceinline__ float scale_bits(uint32_t x) { return __uint_as_float(x); }

// l + the two weights of a packed pair, as they are after the rounding.
template <typename T>
__device__ __forceinline__ float add_pair(uint32_t pair, float l) {
    if constexpr (__is_same(T, Bf16)) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, pair), __builtin_bit_cast(b2, 0x3f803f80u), l, false);
    } else {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, pair), __builtin_bit_cast(f16x2_t, 0x3c003c00u), l, false);
    }
}

// How far (in powers of two) a row's maximum may pass the one that its weights
// are relative to before they are scaled anew, in large blocks of rows: weights
// grow by 2^8 at most, and most steps need no pass over O (65.7 M vector
// instructions, 57.4 with the slack, for 2047 tokens of 32 heads after 4000).  With
// few rows maxima seldom grow, and there is no slack.
constexpr float kSlack = 8.0f;

// Weights are taken relative to a row's maximum plus this (in powers of two), so that the
// sum of all of them stays at 1 at most: bf16's values reach 2^127.6, and a sum of them
// that is divided at the end must not pass 32 bits' range before.  An addend of the
// maximum, it costs nothing.  f16's values are far from there, and its weights
// have no exponents to spare.
template <typename T>
__device__ __forceinline__ float headroom(int tokens, float slack) {
    return __is_same(T, Bf16) ? (float)(32 - __builtin_clz((uint32_t)tokens | 1u)) + slack : 0.0f;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace kv4
}  // namespace bk
