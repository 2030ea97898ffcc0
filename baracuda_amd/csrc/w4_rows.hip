// w4_rows.hip -- products with 4-bit weights for few rows.
#include "gemm_mfma2.hpp"
#include "w4_product.hpp"

namespace bk {
namespace w4 {
namespace {

// Few rows: the waves of a workgroup divide K among them, so that all of it is asked
// for at once, and add their sums through LDS in the waves' order.
//
// 16 rows of x against CB blocks of 16 weight rows by the 16x16x32 product.  Lane l
// supplies weight row l % 16 and group l / 16 of four (128 values of K, from two
// tiles), and the same values of x's row l % 16.  Gated: odd blocks are rows of the
// second half of the matrix, whose products meet those of the first half in the same
// lanes.  A wave takes a word (256 values of K, four tiles) at a time: codes and
// scales into registers, the next word's asked for before this one is multiplied; x by
// LDS DMA into 512 bytes a row of its own, 16-byte unit u of row r at u ^ (r & 15).
// (Straight from L2 into registers a row's 64 bytes at a time x bounded it: 16 x 4096 x
// 4096 7.5 us, now 5.8; 16 x 28672 x 4096 20 and 17.  A second buffer of x costs more in
// workgroups that fit a CU than it hides: 16 x 14336 x 4096 11.0 and 10.5.  x and the weights are
// waited for together, so that a wave has one word of them in flight; an earlier form with
// x in registers took 12.5 us for one row of 28672 x 4096 gated, this one 13.9.)
//
// The weights' bytes bound it, behind a launch and one round trip of 2.4 us: one row of
// 131072 x 16384 moves them at 6.0 TB/s, 28672 x 4096 in 13.8 us (4.5), 4096 x 4096 in
// 3.5 to 4.4.
template <bool BF16, bool MOE, bool GATED, int HELD, int CB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void rows_kernel(const ProductArgs a) {
    extern __shared__ __attribute__((aligned(1024))) int8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Rows w;
    if constexpr (MOE) {
        int slot = blockIdx.y;
        if (!(a.offsets ? expert_rows<HELD>(a, slot, w) : expert_rows_few<HELD>(a, slot, w))) {     // the whole workgroup
            if (!a.offsets && blockIdx.x == 0 && blockIdx.y == 0) count_experts(a, (uint32_t *)lds);
            return;
        }
    } else {
        w = Rows{0, (int)blockIdx.y * HELD, min(HELD, a.M - (int)blockIdx.y * HELD)};
    }
    const int col = lane & 15, kq = lane >> 4;
    // blocks of 16 weight rows, held in pairs
    const uint8_t *matrix = a.w + w.e * a.matrix;
    const int64_t blocks = row_blocks(a.N);
    int row16[CB];
    const uint8_t *codes[CB], *scales[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) {
        row16[c] = GATED ? (int)blockIdx.x * (CB / 2) + c / 2 + (c & 1) * (a.N / 32) : (int)blockIdx.x * CB + c;
        const int b = min(row16[c] / 2, (int)blocks - 1), at = (row16[c] & 1) * 16 + col + 32 * (kq & 1);
        codes[c] = matrix + ((int64_t)b * a.tiles + (kq >> 1)) * 1024 + 16 * at;
        scales[c] = matrix + blocks * a.tiles * 1024 + (int64_t)b * a.words * 256 + 4 * at;
    }
    const int words = a.words, halves = a.tiles / 2;             // of 256 and of 128 values
    struct Weights {
        v4i code[CB][2];
        uint32_t scale[CB];
    };
    const auto weights = [&](int s, Weights &r) {
        // a word's second half may lie past the last: the first again, for zeros of x
        const int64_t at = (int64_t)4 * s * 1024, second = 2 * s + 1 < halves ? 2048 : 0;
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            r.code[c][0] = *(const v4i *)(codes[c] + at);
            r.code[c][1] = *(const v4i *)(codes[c] + at + second);
            r.scale[c] = *(const uint32_t *)(scales[c] + (int64_t)s * 256);
        }
    };
    // x: up to HELD rows, two a DMA; rows that there are not and values past K lie past the
    // extent and land as zeros
    int8_t *own = lds + wave * (HELD * 512);
    const v4i rsrc = MOE ? mfma2::make_rsrc(a.x, (uint32_t)((int64_t)((a.size_m + a.in_div - 1) / a.in_div) * a.K * 2))
                         : mfma2::make_rsrc(a.x + w.first * a.ldx, (uint32_t)(((w.rows - 1) * a.ldx + a.K) * 2));
    int off[HELD / 2];
#pragma unroll
    for (int j = 0; j < HELD / 2; ++j) {
        const int r = 2 * j + (lane >> 5);
        int in, out;
        row_of<MOE>(a, w, r, in, out);
        off[j] = in < 0 ? mfma2::kPastExtent : (int)((MOE ? in * a.ldx : r * a.ldx) * 2) + (((lane & 31) ^ (r & 15)) << 4);
    }
    const auto inputs = [&](int s) {
#pragma unroll
        for (int j = 0; j < HELD / 2; ++j) {
            if (2 * j >= w.rows) break;
            const int unit = (lane & 31) ^ ((2 * j + (lane >> 5)) & 15);
            mfma2::dma16(rsrc, 256 * s + 8 * unit < a.K ? off[j] : mfma2::kPastExtent, __builtin_amdgcn_readfirstlane(s * 512),
                         own + j * 1024);
        }
    };
    v4f acc[CB][2];
#pragma unroll
    for (int c = 0; c < CB; ++c) acc[c][0] = acc[c][1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // columns of x past the last row repeat it: nothing of them is stored
    const int8_t *mine = own + min(col, w.rows - 1) * 512;
    const int turn = min(col, w.rows - 1);
    const auto multiply = [&](const Weights &r) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v4i xf = *(const v4i *)(mine + (((16 * h + 4 * kq + i) ^ turn) << 4));
#pragma unroll
                for (int c = 0; c < CB; ++c) {
                    const v4i wf = elements8<BF16>((uint32_t)r.code[c][h][i], scale_of(r.scale[c] >> (8 * (kq >> 1)), 2 * h));
                    acc[c][h] = mfma16x16x32_h<BF16>(wf, xf, acc[c][h]);
                }
            }
    };
    Weights now, next;
    if (wave < words) {
        weights(wave, now);
        inputs(wave);
    }
    for (int s = wave; s < words; s += WAVES) {
        const bool more = s + WAVES < words;
        mfma2::wait_dma();
        if (more) weights(s + WAVES, next);
        multiply(now);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // x has been read
        if (more) inputs(s + WAVES);
        now = next;
    }
    __syncthreads();
    v4f *part = (v4f *)lds;                                      // [waves][CB][64]
#pragma unroll
    for (int c = 0; c < CB; ++c) part[(wave * CB + c) * 64 + lane] = acc[c][0] + acc[c][1];
    __syncthreads();
    const int ncols = GATED ? a.N / 2 : a.N;
    constexpr int OUT = GATED ? CB / 2 : CB;
    for (int o = wave; o < OUT; o += WAVES) {
        const int c = o * (GATED ? 2 : 1);
        v4f y = part[c * 64 + lane];
#pragma unroll
        for (int v = 1; v < WAVES; ++v) y += part[(v * CB + c) * 64 + lane];
        int in, out;
        row_of<MOE>(a, w, col, in, out);
        int n = 0;
#pragma unroll
        for (int q = 0; q < CB; ++q) n = q == c ? 16 * row16[q] + 4 * kq : n;
        if (out < 0 || n >= ncols) continue;
        y += bias4(a, w.e, n);
        if constexpr (GATED) {
            v4f u = part[(c + 1) * 64 + lane];
#pragma unroll
            for (int v = 1; v < WAVES; ++v) u += part[(v * CB + c + 1) * 64 + lane];
            u += bias4(a, w.e, n + a.N / 2);
#pragma unroll
            for (int q = 0; q < 4; ++q) y[q] = gated(y[q], u[q]);
        }
        if constexpr (MOE) {
            if (a.topk_weights) y *= a.topk_weights[out];
        }
        store4<BF16>(a, out, n, ncols, y);
    }
    if constexpr (MOE) {
        if (!a.offsets && blockIdx.x == 0 && blockIdx.y == 0) count_experts(a, (uint32_t *)lds);
    }
}

template <bool BF16, bool MOE, bool GATED, int HELD, int CB, int WAVES>
int32_t launch_held(const ProductArgs &a, int64_t slots, hipStream_t stream) {
    constexpr int per = GATED ? CB / 2 : CB;
    constexpr int bytes = std::max(std::max(WAVES * HELD * 512, WAVES * CB * 1024), 4 * kFewPairs);
    const int blocks = ((GATED ? a.N / 2 : a.N) + 16 * per - 1) / (16 * per);
    hipLaunchKernelGGL((rows_kernel<BF16, MOE, GATED, HELD, CB, WAVES>), dim3((unsigned)blocks, (unsigned)slots),
                       dim3(64 * WAVES), bytes, stream, a);
    return launch_status();
}

template <bool BF16, bool MOE, bool GATED, int HELD, int CB>
int32_t launch_blocks(const ProductArgs &a, int waves, int64_t slots, hipStream_t stream) {
#define BK_W4_WAVES(WAVES)                          \
    if constexpr (rows_form(HELD, CB, WAVES, GATED)) \
        if (waves == WAVES) return launch_held<BF16, MOE, GATED, HELD, CB, WAVES>(a, slots, stream);
    BK_W4_WAVES(2)
    BK_W4_WAVES(4)
    BK_W4_WAVES(8)
    BK_W4_WAVES(16)
#undef BK_W4_WAVES
    return kUnsupported;
}

template <bool BF16, bool MOE, bool GATED, int HELD>
int32_t launch_shape(const ProductArgs &a, const RowsShape &s, int64_t slots, hipStream_t stream) {
    switch (s.blocks) {
        case 1: return launch_blocks<BF16, MOE, GATED, HELD, 1>(a, s.waves, slots, stream);
        case 2: return launch_blocks<BF16, MOE, GATED, HELD, 2>(a, s.waves, slots, stream);
        default: return launch_blocks<BF16, MOE, GATED, HELD, 4>(a, s.waves, slots, stream);
    }
}

template <bool BF16, bool MOE, bool GATED>
int32_t launch_all(const ProductArgs &a, hipStream_t stream) {
    const int held = MOE ? moe_rows_held(a.size_m, a.E) : rows_held(a.M);
    const int64_t slots = MOE ? std::min<int64_t>(most_tile_rows(a.size_m, a.E, held), a.size_m) : (a.M + held - 1) / held;
    const RowsShape s = rows_shape(held, MOE ? moe_rows_likely(a.size_m, a.E, held) : slots, a.N, a.K, GATED);
    switch (held) {
        case 2: return launch_shape<BF16, MOE, GATED, 2>(a, s, slots, stream);
        case 4: return launch_shape<BF16, MOE, GATED, 4>(a, s, slots, stream);
        case 8: return launch_shape<BF16, MOE, GATED, 8>(a, s, slots, stream);
        default: return launch_shape<BF16, MOE, GATED, 16>(a, s, slots, stream);
    }
}

}  // namespace

int32_t launch_rows(const ProductArgs &a, bool bf16, bool moe, bool gated, hipStream_t stream) {
    if (bf16) {
        if (moe) return gated ? launch_all<true, true, true>(a, stream) : launch_all<true, true, false>(a, stream);
        return gated ? launch_all<true, false, true>(a, stream) : launch_all<true, false, false>(a, stream);
    }
    if (moe) return gated ? launch_all<false, true, true>(a, stream) : launch_all<false, true, false>(a, stream);
    return gated ? launch_all<false, false, true>(a, stream) : launch_all<false, false, false>(a, stream);
}

}  // namespace w4
}  // namespace bk
