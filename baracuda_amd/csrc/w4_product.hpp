// w4_product.hpp -- what the kernels of the products with 4-bit weights share:
// arguments, rows of an expert, the end of a product.
#pragma once

#include "w4.hpp"

namespace bk {
namespace w4 {

struct ProductArgs {
    const uint16_t *x;           // rows of K elements, ldx apart
    const uint8_t *w;            // packed matrices
    const float *bias;           // [matrices, N], or null
    uint16_t *out;               // rows of N (gated: N / 2) elements, ldo apart
    int64_t ldx, ldo;
    int64_t matrix;              // bytes of a packed matrix
    int M, N, K, tiles, words;
    // by expert: position p of the pairs sorted by expert has pair order[p]
    const int32_t *order, *offsets;
    const float *topk_weights;   // [size_m] by pair, or null
    int E, size_m, in_div;       // input row of a pair: pair / in_div
};

// Rows of one workgroup: its rows of the list (a matrix's own rows, or positions
// of an expert's pairs).
struct Rows {
    int e, first, rows;
};

// Tile `slot` of TB rows in the list of all experts' tiles, found by a wave from
// the offsets: 64 experts at a time, one a lane, a prefix sum of their tiles.
// False past the list.
template <int TB>
__device__ __forceinline__ bool expert_rows(const ProductArgs &a, int slot, Rows &r) {
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
        const int x = e0 + lane;
        const int o0 = x < a.E ? min(max(a.offsets[x], 0), a.size_m) : 0;
        const int n = x < a.E ? max(min(a.offsets[x + 1], a.size_m) - o0, 0) : 0;
        const int own = (n + TB - 1) / TB;
        int incl = own;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(incl, off, 64);
            if (lane >= off) incl += v;
        }
        const uint64_t past = __ballot(incl > slot);
        if (past) {
            const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)past) - 1);
            const int tile = slot - (__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(own, l));
            r.e = e0 + l;
            r.first = __builtin_amdgcn_readlane(o0, l) + tile * TB;
            r.rows = min(TB, __builtin_amdgcn_readlane(n, l) - tile * TB);
            return true;
        }
        slot -= __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}

// Input and output row of row r of a workgroup's; negative where there is none.
template <bool MOE>
__device__ __forceinline__ void row_of(const ProductArgs &a, const Rows &w, int r, int &in, int &out) {
    in = out = -1;
    if (r >= w.rows) return;
    if constexpr (MOE) {
        const int pair = a.order[w.first + r];
        if ((unsigned)pair < (unsigned)a.size_m) out = pair, in = pair / a.in_div;
    } else {
        in = out = w.first + r;
    }
}

// silu(gate) * up in 32 bits.  exp(-gate) overflows to infinity where the gate is
// below -88, and the quotient is then -0, as it should be.
__device__ __forceinline__ float gated(float gate, float up) { return gate / (1.0f + __expf(-gate)) * up; }

// The end of a product: four consecutive columns from n of an output row, bias and
// gate added in 32 bits and rounded once.  ncols: columns of the output.
template <bool BF16>
__device__ __forceinline__ void store4(const ProductArgs &a, int row, int n, int ncols, const v4f &y) {
    uint16_t *p = a.out + row * a.ldo + n;
    uint32_t lo, hi;
    if constexpr (BF16) lo = f32x2_to_bf16x2(y[0], y[1]), hi = f32x2_to_bf16x2(y[2], y[3]);
    else lo = kv4::f32x2_to_f16x2(y[0], y[1]), hi = kv4::f32x2_to_f16x2(y[2], y[3]);
    if (n + 4 <= ncols && ((uintptr_t)p & 7) == 0) {
        *(v2i *)p = v2i{(int)lo, (int)hi};
        return;
    }
    const uint16_t h[4] = {(uint16_t)lo, (uint16_t)(lo >> 16), (uint16_t)hi, (uint16_t)(hi >> 16)};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < ncols) p[i] = h[i];
}

// Four biases from row n of matrix e (zeros past N).
__device__ __forceinline__ v4f bias4(const ProductArgs &a, int e, int n) {
    v4f b = {0.0f, 0.0f, 0.0f, 0.0f};
    if (a.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.N) b[i] = a.bias[(int64_t)e * a.N + n + i];
    }
    return b;
}

}  // namespace w4
}  // namespace bk
