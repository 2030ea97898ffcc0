// w4_product.hpp -- what the kernels of the products with 4-bit weights share:
// arguments, rows of an expert, the end of a product.
#pragma once

#include "w4.hpp"
#include "w4_rules.hpp"

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
    const int32_t *order, *offsets, *expert_ids;     // offsets null: few pairs, from the ids
    int32_t *counts_out, *offsets_out;
    const float *topk_weights;   // [size_m] by pair, or null
    int E, size_m, in_div;       // size_m: pairs, or M; input row of a pair: pair / in_div
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

// Tiles of TB rows in all.
template <int TB>
__device__ __forceinline__ int expert_tiles(const ProductArgs &a) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int x = lane; x < a.E; x += 64) {
        const int o0 = min(max(a.offsets[x], 0), a.size_m);
        n += (max(min(a.offsets[x + 1], a.size_m) - o0, 0) + TB - 1) / TB;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) n += __shfl_xor(n, off, 64);
    return __builtin_amdgcn_readfirstlane(n);
}

// expert_rows for at most kFewPairs pairs, from the ids themselves: that saves the
// launch in front that counts them (about 3 us of a step of 30).  Past the list `slot`
// is left smaller by the list's length.
template <int TB>
__device__ __forceinline__ bool expert_rows_few(const ProductArgs &a, int &slot, Rows &r) {
    const int lane = threadIdx.x & 63;
    int id[kFewChunks];
    uint64_t head[kFewChunks];             // positions whose expert is not the one before
#pragma unroll
    for (int i = 0; i < kFewChunks; ++i) id[i] = 64 * i + lane < a.size_m ? a.expert_ids[64 * i + lane] : -1;
#pragma unroll
    for (int i = 0; i < kFewChunks; ++i) {
        const int before = i ? __builtin_amdgcn_readlane(id[i ? i - 1 : 0], 63) : -2, up = __shfl_up(id[i], 1, 64);
        head[i] = __ballot(id[i] != (lane ? up : before));
    }
    int from = 0;                          // where the run that reaches into this chunk began
#pragma unroll
    for (int i = 0; i < kFewChunks; ++i) {
        const uint64_t starts = __ballot((unsigned)id[i] < (unsigned)a.E && (64 * i + lane - run_began(head[i], i, lane, from)) % TB == 0);
        const int n = __popcll(starts);
        if (slot < n) {
            const bool me = (starts >> lane & 1) && __popcll(starts & ((1ull << lane) - 1)) == slot;
            const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(me)) - 1);
            r.e = __builtin_amdgcn_readlane(id[i], l);
            r.first = 64 * i + l;
            r.rows = min(min(TB, run_left<TB>(head, i, l)), a.size_m - r.first);
            return true;
        }
        slot -= n;
        from = run_began(head[i], i, 63, from);
    }
    return false;
}

template <int TB>
__device__ __forceinline__ int expert_tiles_few(const ProductArgs &a) {
    int left = INT32_MAX;
    Rows none;
    expert_rows_few<TB>(a, left, none);
    return INT32_MAX - left;
}

// expert_counts and expert_offsets of few pairs, by one whole workgroup, through
// kFewPairs words of LDS.
__device__ __forceinline__ void count_experts(const ProductArgs &a, uint32_t *ids) {
    __syncthreads();
    for (int i = threadIdx.x; i < a.size_m; i += blockDim.x) ids[i] = (uint32_t)a.expert_ids[i];
    __syncthreads();
    const auto before = [&](uint32_t e) {      // positions of experts below e
        int lo = 0, n = a.size_m;
        while (n > 0) {
            const int half = n / 2;
            const bool below = ids[lo + half] < e;
            lo = below ? lo + half + 1 : lo;
            n = below ? n - half - 1 : half;
        }
        return lo;
    };
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
        const int first = before(e), last = before(e + 1);
        a.counts_out[e] = last - first;
        a.offsets_out[e] = first;
        if (e == a.E - 1) a.offsets_out[a.E] = last;
    }
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

struct __attribute__((packed, aligned(2))) Unaligned8 {
    v2i v;
};

// The end of a product: four consecutive columns from n of an output row, bias and
// gate added in 32 bits and rounded once.  ncols: columns of the output.
template <bool BF16>
__device__ __forceinline__ void store4(const ProductArgs &a, int row, int n, int ncols, const v4f &y) {
    uint16_t *p = a.out + row * a.ldo + n;
    uint32_t lo, hi;
    if constexpr (BF16) lo = f32x2_to_bf16x2(y[0], y[1]), hi = f32x2_to_bf16x2(y[2], y[3]);
    else lo = kv4::f32x2_to_f16x2(y[0], y[1]), hi = kv4::f32x2_to_f16x2(y[2], y[3]);
    if (n + 4 <= ncols) {
        ((Unaligned8 *)p)->v = v2i{(int)lo, (int)hi};
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

int32_t launch_rows(const ProductArgs &a, bool bf16, bool moe, bool gated, hipStream_t stream);
int32_t launch_tiles(const ProductArgs &a, bool bf16, bool moe, bool gated, hipStream_t stream);

}  // namespace w4
}  // namespace bk
