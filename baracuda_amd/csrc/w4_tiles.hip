// w4_tiles.hip -- products with 4-bit weights for many rows: tiles of TM rows of x
// by TN rows of the weights, on the 32x32x16 matrix product.
//
// Weights become elements in registers, each wave's own 64 rows of them (the
// conversion takes the group's scale with it), so LDS holds x as elements but the
// weights as codes: a stage of 64 values of K is TM x 128 bytes of x and TN / 32
// blocks of 1 KiB of codes and 256 bytes of scales (a word of four tiles' scales,
// fetched with each of the four).  All of it comes by LDS DMA into a ring of DEPTH
// stages, DEPTH - 1 in flight, one barrier a stage, the next stage's DMA spread
// between the matrix products.  Lane l of a weights' operand is row l % 32 and
// group l / 32 of its tile, word i of its 16 bytes the eight values of product i;
// x's operand takes the same eight values, 16-byte unit 4 (l / 32) + i of its row.
//
// Large tiles are bound by the board's power: 4097 x 28672 x 4096 gated, by tiles of
// 128x256, two a CU, 1210 to 1310 TFLOP/s at 1.68 GHz with 73% of the matrix unit's clocks
// busy (without the gate 1.6 and 76%).  Tiles of few rows are bound by the DMA of x, 26
// clocks a kilobyte of a CU, and by a tile's first loads and end, 5 to 8 us, which tiles
// that share a CU hide from one another.
#include "gemm_mfma2.hpp"
#include "w4_product.hpp"

namespace bk {
namespace w4 {
namespace {

using mfma2::v16f;

// One LDS DMA of four bytes a lane, as mfma2::dma16.
__device__ __forceinline__ void dma4(const v4i &rsrc, int voff, int soff, const int8_t *lds_dst) {
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>(lds_dst));
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
                 : "memory", "m0");
}

template <bool BF16>
__device__ __forceinline__ v16f mfma32x32x16(const v4i &a, const v4i &b, const v16f &c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// TM x TN tiles; a group of WM x TN / 64 waves takes TM / WM x 64 each.  KG groups
// take 64 values of K each of a stage of 64 KG, and add their sums at the end.
template <int TM_, int TN_, int WM_, int KG_, int DEPTH_>
struct Tile {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, KG = KG_, DEPTH = DEPTH_;
    static constexpr int WN = TN / 64, GROUP = WM * WN, WAVES = KG * GROUP;
    static constexpr int TI = TM / 32 / WM;             // 32-row blocks of x a wave
    static constexpr int NB = TN / 32;                  // blocks of weight rows
    // DMAs a wave and stage: of x (8 rows by 64 values), codes (a tile) and scales (a
    // block's words, of up to four tiles each; with more waves than blocks some are
    // fetched again: every wave does the same, and none is waited for at the barrier)
    static constexpr int NX = TM / 8 / GROUP, NC = NB / GROUP, NS = (NB + WAVES - 1) / WAVES, NI = NX + NC + NS;
    static constexpr int SUB = TM * 128 + NB * 1024, SCALES = KG * SUB, STAGE = SCALES + NB * 256;
    static constexpr int LDS = DEPTH * STAGE + TM * 4;  // and the output rows
    static constexpr int SCRATCH = DEPTH * STAGE / GROUP / 1024 * 1024;      // a wave's of the first group, at the end
    static_assert(NX * GROUP * 8 == TM && NC * GROUP == NB && WAVES <= 16 && KG <= 4, "tile");
    static_assert(LDS <= 160 * 1024 && SCRATCH >= 4096 && (KG - 1) * GROUP * TI * 8192 <= DEPTH * STAGE, "tile");
};

// What a wave moves of each stage.
template <class T>
struct Source {
    v4i x, codes[T::NC], scales;             // buffer resources
    int row[T::NX];                          // byte offsets of this lane's pieces of x
    int word[T::NS];                         // byte offsets of the blocks' scales
    int8_t *lds;

    __device__ __forceinline__ void piece(int i, int stage_at, int stage) const {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
        int8_t *s = lds + stage_at;
        if (i < T::NX) {
            const int q = wave * T::NX + i, kg = q / (T::TM / 8), r = q % (T::TM / 8);
            mfma2::dma16(x, row[i], __builtin_amdgcn_readfirstlane((stage * T::KG + kg) * 128), s + kg * T::SUB + r * 1024);
        } else if (i < T::NX + T::NC) {
            const int q = wave * T::NC + i - T::NX, kg = q / T::NB, b = q % T::NB;
            mfma2::dma16(codes[i - T::NX], lane * 16, __builtin_amdgcn_readfirstlane((stage * T::KG + kg) * 1024),
                         s + kg * T::SUB + T::TM * 128 + b * 1024);
        } else {
            const int j = i - T::NX - T::NC, b = (wave * T::NS + j) % T::NB;
            dma4(scales, lane * 4, __builtin_amdgcn_readfirstlane((stage * T::KG >> 2) * 256 + word[j]),
                 s + T::SCALES + b * 256);
        }
    }

    // Units of x past K lie past its extent from here on and land as zeros (codes past
    // the last tile do of themselves).
    __device__ __forceinline__ void prepare(int stage, int K) {
        if ((stage + 1) * (T::KG * 64) <= K) return;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < T::NX; ++i) {
            const int q = wave * T::NX + i, kg = q / (T::TM / 8), r = q % (T::TM / 8) * 8 + (lane >> 3);
            if ((stage * T::KG + kg) * 64 + ((lane & 7) ^ mfma2::swz(r)) * 8 >= K) row[i] = mfma2::kPastExtent;
        }
    }
};

template <bool BF16, class T>
__device__ __forceinline__ void multiply(Source<T> &src, int K, v16f (&acc)[T::TI][2]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kg = wave / T::GROUP, wm = wave % T::GROUP / T::WN, wn = wave % T::WN;
#pragma unroll
    for (int i = 0; i < T::TI; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = v16f{0};
    const int stages = (K + T::KG * 64 - 1) / (T::KG * 64);
    for (int s = 0; s < T::DEPTH - 1; ++s) {
        src.prepare(s, K);
#pragma unroll
        for (int i = 0; i < T::NI; ++i) src.piece(i, s * T::STAGE, s);
    }
    int cur = 0, nxt = (T::DEPTH - 1) * T::STAGE;
    for (int s = 0; s < stages; ++s) {
        src.prepare(s + T::DEPTH - 1, K);
        mfma2::wait_vmcnt<(T::DEPTH - 2) * T::NI>();
        __syncthreads();
        const int8_t *st = src.lds + cur + kg * T::SUB, *sc = src.lds + cur + T::SCALES;
        v4i code[2];
        float scale[2];
        v4i xf[4][T::TI];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            code[j] = *(const v4i *)(st + T::TM * 128 + (2 * wn + j) * 1024 + lane * 16);
            scale[j] = scale_of(*(const uint32_t *)(sc + (2 * wn + j) * 256 + lane * 4), (s * T::KG + kg) & 3);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int i = 0; i < T::TI; ++i)
                xf[h][i] = *(const v4i *)(st + mfma2::lds_off((wm * T::TI + i) * 32 + (lane & 31), 4 * (lane >> 5) + h));
        constexpr int TOT = 8 * T::TI, EVERY = TOT / T::NI;
        static_assert(EVERY >= 1, "a product for each DMA");
#pragma unroll
        for (int h = 0; h < 4; ++h) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const v4i wf = elements8<BF16>((uint32_t)code[j][h], scale[j]);
#pragma unroll
                for (int i = 0; i < T::TI; ++i) {
                    acc[i][j] = mfma32x32x16<BF16>(wf, xf[h][i], acc[i][j]);
                    const int t = (h * 2 + j) * T::TI + i;
                    if (t % EVERY == 0 && t / EVERY < T::NI) {
                        // (pinned for small tiles: 128 x 4096 x 4096 11.3 us, else 11.9; large
                        // ones are better off with the compiler's order: 777 x 11008 x 4096
                        // 74.6, pinned 76.8)
                        if constexpr (T::TI == 1) __builtin_amdgcn_sched_barrier(0);
                        src.piece(t / EVERY, nxt, s + T::DEPTH - 1);
                        if constexpr (T::TI == 1) __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
        nxt = cur;
        cur = cur + T::STAGE == T::DEPTH * T::STAGE ? 0 : cur + T::STAGE;
    }
    mfma2::wait_dma();
    __syncthreads();
    if constexpr (T::KG > 1) {       // the other groups' sums, in their order
        v4f *part = (v4f *)src.lds + (wave % T::GROUP) * (T::TI * 512) + lane;      // [KG - 1][GROUP][TI][2][4][64]
        if (kg) {
            part += (kg - 1) * T::GROUP * T::TI * 512;
#pragma unroll
            for (int i = 0; i < T::TI; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        part[((i * 2 + j) * 4 + g) * 64] =
                            v4f{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        }
        __syncthreads();
        if (!kg) {
#pragma unroll
            for (int o = 0; o < T::KG - 1; ++o)
#pragma unroll
                for (int i = 0; i < T::TI; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const v4f v = part[o * T::GROUP * T::TI * 512 + ((i * 2 + j) * 4 + g) * 64];
#pragma unroll
                            for (int q = 0; q < 4; ++q) acc[i][j][4 * g + q] += v[q];
                        }
        }
        __syncthreads();
    }
}

struct __attribute__((packed, aligned(2))) Unaligned16 {
    v4i v;
};

// A wave's tile: bias, gate and router weight in 32 bits, rounded, 32 rows at a time
// through 4 KiB of LDS, so that rows are written 128 (gated: 64) bytes at once.
template <bool BF16, bool MOE, bool GATED, class T>
__device__ __forceinline__ void store_tile(const ProductArgs &a, const v16f (&acc)[T::TI][2], int8_t *scratch, const int *s_out,
                                           int e, int col0, int ncols) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / T::WN;
    constexpr int COLS = GATED ? 32 : 64, UNITS = COLS / 8;
    v4f b[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            b[j][g] = bias4(a, e, col0 + (GATED ? j * (a.N / 2) : j * 32) + 8 * g + 4 * (lane >> 5));
#pragma unroll
    for (int i = 0; i < T::TI; ++i) {
        const int *rows = s_out + (wm * T::TI + i) * 32;
        float mix = 1.0f;
        if constexpr (MOE) {
            const int row = rows[lane & 31];
            if (a.topk_weights && row >= 0) mix = a.topk_weights[row];
        }
#pragma unroll
        for (int j = 0; j < (GATED ? 1 : 2); ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float y[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if constexpr (GATED) y[q] = gated(acc[i][0][4 * g + q] + b[0][g][q], acc[i][1][4 * g + q] + b[1][g][q]);
                    else y[q] = acc[i][j][4 * g + q] + b[j][g][q];
                    if constexpr (MOE) y[q] *= mix;
                }
                v2i w;
                if constexpr (BF16) w = v2i{(int)f32x2_to_bf16x2(y[0], y[1]), (int)f32x2_to_bf16x2(y[2], y[3])};
                else w = v2i{(int)kv4::f32x2_to_f16x2(y[0], y[1]), (int)kv4::f32x2_to_f16x2(y[2], y[3])};
                const int r = lane & 31, u = j * 4 + g;
                *(v2i *)(scratch + r * 128 + ((u ^ (r & 7)) << 4) + 8 * (lane >> 5)) = w;
            }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
        const int u = lane % UNITS, n = col0 + 8 * u;
#pragma unroll
        for (int p = 0; p < 32 * UNITS / 64; ++p) {
            const int r = p * (64 / UNITS) + lane / UNITS, row = rows[r];
            if (row < 0 || n >= ncols) continue;
            const v4i v = *(const v4i *)(scratch + r * 128 + ((u ^ (r & 7)) << 4));
            uint16_t *out = a.out + row * a.ldo + n;
            if (n + 8 <= ncols) {
                ((Unaligned16 *)out)->v = v;
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (n + q < ncols) out[q] = (uint16_t)((uint32_t)v[q / 2] >> (16 * (q & 1)));
            }
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
    }
}

// Workgroup to tile.  Consecutive workgroups go to the 8 XCDs in turn, so each XCD
// gets a contiguous range of the list, in which four tiles of rows share the
// weights that its L2 holds.
__device__ __forceinline__ bool tile_of(int tiles_m, int tiles_n, int &tm, int &tn) {
    const int total = tiles_m * tiles_n, xcd = blockIdx.x % 8, q = total / 8, r = total % 8;
    if ((int)blockIdx.x / 8 >= q + (xcd < r ? 1 : 0)) return false;
    const int i = xcd * q + min(xcd, r) + blockIdx.x / 8, group = i / (4 * tiles_n), width = min(4, tiles_m - 4 * group);
    const int j = i - group * 4 * tiles_n;
    tm = 4 * group + j % width;
    tn = j / width;
    return true;
}

template <bool BF16, bool MOE, bool GATED, class T>
__global__ __launch_bounds__(64 * T::WAVES) void tiles_kernel(const ProductArgs a, int tiles_n) {
    extern __shared__ __attribute__((aligned(1024))) int8_t lds[];
    int *s_out = (int *)(lds + T::DEPTH * T::STAGE);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn;
    Rows w;
    if constexpr (MOE) {
        if (!a.offsets && blockIdx.x == 0) {
            count_experts(a, (uint32_t *)lds);
            __syncthreads();
        }
        if (!tile_of(a.offsets ? expert_tiles<T::TM>(a) : expert_tiles_few<T::TM>(a), tiles_n, tm, tn)) return;
        int slot = tm;
        if (!(a.offsets ? expert_rows<T::TM>(a, slot, w) : expert_rows_few<T::TM>(a, slot, w))) return;
    } else {
        if (!tile_of((a.M + T::TM - 1) / T::TM, tiles_n, tm, tn)) return;
        w = Rows{0, tm * T::TM, min(T::TM, a.M - tm * T::TM)};
    }
    Source<T> src;
    src.lds = lds;
    const uint8_t *matrix = a.w + w.e * a.matrix;
    const int blocks = (int)row_blocks(a.N);
    // block b of the tile's weight rows: gated, one of the first half of the matrix and
    // the same of the second in turn
    const auto block_of = [&](int b) {       // past the last one: as many as there are
        const int slot = tn * T::NB + b;
        if constexpr (GATED) return slot / 2 < a.N / 64 ? slot / 2 + (slot & 1) * (a.N / 64) : blocks;
        else return min(slot, blocks);
    };
#pragma unroll
    for (int j = 0; j < T::NC; ++j) {
        const int block = __builtin_amdgcn_readfirstlane(block_of((wave * T::NC + j) % T::NB));
        src.codes[j] = mfma2::make_rsrc(matrix + (int64_t)block * a.tiles * 1024, block < blocks ? a.tiles * 1024 : 0);
    }
    // The scales from the tile's first block on: a matrix may have more than 2^31 bytes of
    // them, of which the blocks of one tile span half and a little at most (gated).  (A block
    // past the last takes whatever follows, for columns that are not stored.)
    const int first = __builtin_amdgcn_readfirstlane(block_of(0)), block_scales = a.words * 256;
    src.scales = mfma2::make_rsrc(matrix + (int64_t)blocks * a.tiles * 1024 + (int64_t)first * block_scales,
                                  (uint32_t)(blocks - first) * (uint32_t)block_scales);
#pragma unroll
    for (int j = 0; j < T::NS; ++j)
        src.word[j] = (__builtin_amdgcn_readfirstlane(block_of((wave * T::NS + j) % T::NB)) - first) * block_scales;
    if constexpr (MOE) {
        const int x_rows = (a.size_m + a.in_div - 1) / a.in_div;
        src.x = mfma2::make_rsrc(a.x, (uint32_t)((int64_t)x_rows * a.K * 2));
    } else {
        src.x = mfma2::make_rsrc(a.x + w.first * a.ldx, (uint32_t)(((w.rows - 1) * a.ldx + a.K) * 2));
    }
#pragma unroll
    for (int i = 0; i < T::NX; ++i) {
        const int q = wave * T::NX + i, r = q % (T::TM / 8) * 8 + (lane >> 3), u = (lane & 7) ^ mfma2::swz(r);
        int in, out;
        row_of<MOE>(a, w, r, in, out);
        if (q < T::TM / 8 && (lane & 7) == 0) s_out[r] = out;
        // rows that there are not lie past the extent and land as zeros
        src.row[i] = in < 0 ? mfma2::kPastExtent : (int)((MOE ? in * a.ldx : r * a.ldx) * 2) + u * 16;
    }
    v16f acc[T::TI][2];
    multiply<BF16, T>(src, a.K, acc);
    if (wave >= T::GROUP) return;
    const int ncols = GATED ? a.N / 2 : a.N;
    const int col0 = (tn * T::WN + wave % T::WN) * (GATED ? 32 : 64);
    if (col0 >= ncols) return;
    store_tile<BF16, MOE, GATED, T>(a, acc, lds + wave * T::SCRATCH, s_out, w.e, col0, ncols);
}

template <bool BF16, bool MOE, bool GATED, class T>
int32_t launch_tile(const ProductArgs &a, hipStream_t stream) {
    const int64_t tiles_n = (a.N + T::TN - 1) / T::TN;
    const int64_t tiles_m = MOE ? most_tile_rows(a.size_m, a.E, T::TM) : (a.M + T::TM - 1) / T::TM;
    const int64_t grid = (tiles_m * tiles_n + 7) / 8 * 8;
    hipLaunchKernelGGL((tiles_kernel<BF16, MOE, GATED, T>), dim3((unsigned)grid), dim3(64 * T::WAVES), T::LDS, stream, a,
                       (int)tiles_n);
    return launch_status();
}

template <bool BF16, bool MOE, bool GATED>
int32_t launch_all(const ProductArgs &a, hipStream_t stream) {
    switch (tile_shape(a.size_m, MOE ? a.E : 0, a.N, a.K)) {
        case T_32x64: return launch_tile<BF16, MOE, GATED, Tile<32, 64, 1, 4, 3>>(a, stream);
        case T_32x128: return launch_tile<BF16, MOE, GATED, Tile<32, 128, 1, 2, 3>>(a, stream);
        case T_32x128_DEEP: return launch_tile<BF16, MOE, GATED, Tile<32, 128, 1, 4, 4>>(a, stream);
        case T_64x128_DEEP: return launch_tile<BF16, MOE, GATED, Tile<64, 128, 2, 4, 3>>(a, stream);
        case T_64x256: return launch_tile<BF16, MOE, GATED, Tile<64, 256, 2, 1, 3>>(a, stream);
        case T_128x128_DEEP: return launch_tile<BF16, MOE, GATED, Tile<128, 128, 2, 2, 3>>(a, stream);
        case T_128x256_DEEP: return launch_tile<BF16, MOE, GATED, Tile<128, 256, 2, 2, 3>>(a, stream);
        case T_128x256: return launch_tile<BF16, MOE, GATED, Tile<128, 256, 2, 1, 3>>(a, stream);
        case T_192x256: return launch_tile<BF16, MOE, GATED, Tile<192, 256, 2, 1, 4>>(a, stream);
        default: return launch_tile<BF16, MOE, GATED, Tile<256, 256, 2, 1, 3>>(a, stream);
    }
}

}  // namespace

int32_t launch_tiles(const ProductArgs &a, bool bf16, bool moe, bool gated, hipStream_t stream) {
    if (bf16) {
        if (moe) return gated ? launch_all<true, true, true>(a, stream) : launch_all<true, true, false>(a, stream);
        return gated ? launch_all<true, false, true>(a, stream) : launch_all<true, false, false>(a, stream);
    }
    if (moe) return gated ? launch_all<false, true, true>(a, stream) : launch_all<false, true, false>(a, stream);
    return gated ? launch_all<false, false, true>(a, stream) : launch_all<false, false, false>(a, stream);
}

}  // namespace w4
}  // namespace bk
