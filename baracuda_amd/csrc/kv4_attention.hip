// kv4_attention.hip -- attention over a key-value cache held in 4 bits.
//
// Few rows (decode, drafts): bound by HBM, the pages' bytes.  A wave keeps the
// rows' queries in registers as the right operand and streams tokens, 16 a
// tile: S^T = K Q^T, so that a lane holds four tokens' scores of one row, which
// are in place as the right operand of O^T = V^T P^T without any exchange.
// Codes become elements in registers (v_cvt_scalef32_pk_*_fp4, the scale with
// it).  The waves of a workgroup take steps of a part in turn, each with its
// own running maximum and sum, and are joined through LDS at the end; parts of
// a sequence that was cut are joined by a second kernel.
//
// Scores, maximum, sum and O are held in 32 bits.  P is rounded to the element's
// type for the matrix product, at most half a step of a weight, and the sum is that
// of the rounded weights: what is divided by is what was multiplied with.
#include "kv4_attention.hpp"
#include "kv4_rules.hpp"

namespace bk {
namespace {

using namespace kv4;

// What a lane holds of a tile of 16 tokens: of K the values [g D / 4, (g + 1) D / 4)
// of token lane % 16, of V run lane % 16 of tokens 4 g .. 4 g + 3 (g = lane / 16).
template <int D>
struct Tile {
    uint32_t k[D / 32], v[D / 32], ks, vs;
};

template <int W>
__device__ __forceinline__ void load_words(uint32_t (&w)[W], const uint8_t *p) {
    if constexpr (W == 2) {
        const v2i x = *(const v2i *)p;
        w[0] = x[0], w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const v4i x = *(const v4i *)(p + 4 * i);
            w[i] = x[0], w[i + 1] = x[1], w[i + 2] = x[2], w[i + 3] = x[3];
        }
    }
}

// page: uniform, off: the tile's first token in it.
template <int D>
__device__ __forceinline__ void load_tile(Tile<D> &t, const AttnArgs &a, int page, int head, int off, int lane) {
    const int r = lane & 15, g = lane >> 4;
    const uint8_t *base = a.cache + ((int64_t)page * a.hk + head) * head_bytes(a.ps, D);
    load_words(t.k, base + off * (D / 2) + r * (D / 2) + g * (D / 8));
    load_words(t.v, base + v_codes(a.ps, D) + off * (D / 2) + lane * (D / 8));
    const uint8_t *ks = base + k_scales(a.ps, D) + (off + r) * (D / 32) + g * D / 128;
    t.ks = D == 256 ? *(const uint16_t *)ks : *ks;
    t.vs = *(const uint32_t *)(base + v_scales(a.ps, D) + (((off >> 2) + g) * (D / 32) + r * D / 512) * 4);
}

// A page in the table's row, -1 where there is none.
__device__ __forceinline__ int page_of(const AttnArgs &a, const int32_t *row, int tile, int last) {
    if (tile >= last) return -1;
    const int p = row[tile >> (a.ps_shift - 4)];
    return p >= 0 && p < a.num_pages ? p : -1;
}

// MT tiles of 16 rows; NT tiles of 16 tokens a step; NW waves; AHEAD: the next
// step's loads go out before this one's products.
//
// Two tiles of tokens a step and three waves a SIMD: four tiles need a register
// file that two waves fill (48 sequences 23.1 against 19.6 us, 200001 tokens of 8
// heads 47.4 against 46.2), and four waves spill (70).  Two sequences of 200001 and
// 15 tokens: 218 MB in 45.3 us (4.8 TB/s), 40.6 with the loads alone in the same
// launch.  48 sequences of up to 8192: 47 MB in 16.8 us, of them 10 the loads' way
// in and out.  One sequence of 777: 9.2 us, of them 8 a chain of loads (lengths,
// table, page) on a cold cache.
template <typename T, int D, int MT, int NT, int NW, int OCC, bool AHEAD = true>
__global__ __launch_bounds__(64 * NW, OCC) void decode_kernel(const AttnArgs a) {
    constexpr int RB = 16 * MT, KW = D / 32, OC = D / 16;
    constexpr int LD = D + 4;
    __shared__ float lds_m[NW][RB], lds_l[NW][RB];
    __shared__ __align__(16) float lds_o[NW][RB * LD];
    __shared__ Part lds_part;
    __shared__ Item lds_item;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % a.hk, index = blockIdx.x / a.hk;

    Part part;
    Item s;
    if (a.slots) {
        if (wave == 0) find_part(a, RB, index, lds_part, lds_item);
        __syncthreads();
        part = lds_part;
        if (__builtin_amdgcn_readfirstlane(part.item) < 0) return;
        s = lds_item;
    } else {
        s = item_of(a, index, RB);
        if (s.rows <= 0) return;
        part = Part{index, s.lo / 16, s.lo / 16 + tiles_of(s), 1, index};
    }
    s = uniform(s);
    part = uniform(part);
    const int t0 = part.t0, t1 = part.t1;

    // queries: the right operand, values [g D / 4, (g + 1) D / 4) of row lane % 16
    v4i q[MT][KW];
    int lo[MT], hi[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int row = 16 * mt + r;
        row_span(a, s, row, lo[mt], hi[mt]);
#pragma unroll
        for (int kk = 0; kk < KW; ++kk) q[mt][kk] = v4i{0, 0, 0, 0};
        if (row < s.rows) {
            const int x = s.first + row;
            const char *p = (const char *)a.q +
                            2 * ((s.q0 + token_of(a, x)) * a.q_token + (head * a.ratio + x - token_of(a, x) * a.ratio) * a.q_head + g * (D / 4));
#pragma unroll
            for (int kk = 0; kk < KW; ++kk) {
                const auto m = *(const typename Raw<T>::Mem *)(p + 16 * kk);
                q[mt][kk] = v4i{(int)m.w[0], (int)m.w[1], (int)m.w[2], (int)m.w[3]};
            }
        }
    }
    // every row sees all of [all_lo, all_hi)
    int all_lo, all_hi, x_lo, x_hi;
    row_span(a, s, s.rows - 1, all_lo, x_hi);
    row_span(a, s, 0, x_lo, all_hi);

    const int32_t *table = a.tables + s.seq * a.table_stride;
    v4f o[MT][OC];
    float m[MT], l[MT];
    const float room = headroom<T>(s.len, 0.0f);
    uint32_t poison[MT];           // of a row, the lane's runs that a NaN has reached
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt] = -INFINITY, l[mt] = 0.0f, poison[mt] = 0;
#pragma unroll
        for (int c = 0; c < OC; ++c) o[mt][c] = v4f{0, 0, 0, 0};
    }

    // the pages of this wave's next 64 / NT steps, a tile a lane
    constexpr int kAhead = 64 / NT;
    const auto pages_from = [&](int step) {
        const int t = t0 + (step + lane / NT) * (NW * NT) + wave * NT + lane % NT;
        return page_of(a, table, t, t1);
    };
    const int steps = max(0, (t1 - t0 - wave * NT + NW * NT - 1) / (NW * NT));
    int pages = pages_from(0);
    const auto load_step = [&](Tile<D> (&tile)[NT], int step) {
        const int t = t0 + step * (NW * NT) + wave * NT;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int page = __builtin_amdgcn_readlane(pages, step % kAhead * NT + n);
            load_tile<D>(tile[n], a, page < 0 ? 0 : page, head, (t + n) * 16 & (a.ps - 1), lane);
        }
    };
    const auto do_step = [&](Tile<D> (&tile)[NT], int t, uint64_t held) {
        bool whole = 16 * t >= all_lo && 16 * (t + NT) <= all_hi && t + NT <= t1;
        bool there[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            there[n] = held >> n & 1;
            whole = whole && there[n];
        }
        uint64_t nan[NT][4];   // in a step with masks: the groups of NaN, a run and four tokens a lane
        bool any_nan = false;
        if (!whole) {
            // A weight of 0 keeps neither what lies behind the sequence's end nor a NaN
            // of a token that only later rows see out of a sum: the one becomes zeros,
            // the other as well and is given to the rows that see it below.
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int tok = 16 * (t + n) + 4 * g + j;
                    const uint32_t byte = 0xffu << (8 * j);
                    const bool seen = there[n] && tok >= s.lo && tok < s.hi;
                    const bool odd = (tile[n].vs & byte) == byte;
                    nan[n][j] = __ballot(seen && odd);
                    any_nan = any_nan || nan[n][j] != 0;
                    if (!seen || odd) {
                        constexpr int B = D / 32;   // bytes of a token
                        if constexpr (B == 2) tile[n].v[j / 2] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                        else
#pragma unroll
                            for (int w = 0; w < B / 4; ++w) tile[n].v[j * (B / 4) + w] = 0;
                        tile[n].vs &= ~byte;
                    }
                }
            }
        }
        // scores
        v4f sc[MT][NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) sc[mt][n] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int kk = 0; kk < KW; ++kk) {
                const float ks = scale_bits(D == 256 && kk < 4 ? tile[n].ks << 23 : D == 256 ? tile[n].ks << 15 : tile[n].ks << 23);
                v4i f;
#pragma unroll
                for (int b = 0; b < 4; ++b) f[b] = (int)pair_of<T>(tile[n].k[kk], ks, b);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) sc[mt][n] = mfma_pv<T>(f, q[mt][kk], sc[mt][n]);
            }
        }
        // softmax; m in units of the exponent
        v4i p[MT][NT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!whole) {
                        const int tok = 16 * (t + n) + 4 * g + j;
                        if (!there[n] || tok < lo[mt] || tok >= hi[mt]) sc[mt][n][j] = -INFINITY;
                    }
                    top = fmaxf(top, sc[mt][n][j]);
                }
            }
            top = fmaxf(__builtin_fmaf(max_over_groups(top), a.scale, room), m[mt]);
            if (__any(top > m[mt])) {
                const float f = top > m[mt] ? exp2_fast(m[mt] - top) : 1.0f;
                l[mt] *= f;
#pragma unroll
                for (int c = 0; c < OC; ++c) o[mt][c] *= f;
                m[mt] = top;
            }
            const float ref = m[mt] == -INFINITY ? 0.0f : -m[mt];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float e[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    e[j] = exp2_fast(__builtin_fmaf(sc[mt][n][j], a.scale, ref));
                    p[mt][n][0][j] = (int)pack2<T>(e[j], 0.0f);
                    p[mt][n][1][j] = (int)pack2<T>(0.0f, e[j]);
                    l[mt] = add_pair<T>((uint32_t)p[mt][n][0][j], l[mt]);
                }
            }
        }
        // O^T += V^T P^T.  A converted pair holds two values of one token, so the
        // product runs over (token, value of the pair) with the weights of one of
        // the two at a time: twice the matrix instructions, which have room, and
        // none to bring tokens side by side.  The zeros meet values of the weighed
        // ones' own group: where those are NaN, so are these.
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float vs[4] = {scale_bits(tile[n].vs << 23), scale_bits(tile[n].vs << 15), scale_bits(tile[n].vs << 7),
                                 scale_bits(tile[n].vs >> 1)};
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                v4i f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int b = j * (D / 32) + c;
                    f[j] = (int)pair_of<T>(tile[n].v[b / 4], vs[j], b % 4);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    o[mt][2 * c] = mfma_pv<T>(f, p[mt][n][0], o[mt][2 * c]);
                    o[mt][2 * c + 1] = mfma_pv<T>(f, p[mt][n][1], o[mt][2 * c + 1]);
                }
            }
        }
        if (!whole && any_nan) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int tok = 16 * (t + n) + 4 * k + j;
                        const uint32_t runs = (uint32_t)(nan[n][j] >> (16 * k + 4 * g)) & 15u;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) poison[mt] |= tok >= lo[mt] && tok < hi[mt] ? runs : 0u;
                    }
        }
    };
    const auto held_of = [&](int step) { return __ballot(pages >= 0) >> (step % kAhead * NT) & ((1u << NT) - 1); };
    if constexpr (!AHEAD) {
        for (int i = 0; i < steps; ++i) {
            if (i && i % kAhead == 0) pages = pages_from(i);
            Tile<D> tile[NT];
            load_step(tile, i);
            do_step(tile, t0 + i * (NW * NT) + wave * NT, held_of(i));
        }
    } else if (steps) {
        Tile<D> even[NT], odd[NT];
        load_step(even, 0);
        uint64_t held = held_of(0);
        for (int i = 0; i < steps; i += 2) {
            uint64_t next = 0;
            if (i + 1 < steps) {
                load_step(odd, i + 1);
                next = held_of(i + 1);
            }
            do_step(even, t0 + i * (NW * NT) + wave * NT, held);
            if (i + 1 >= steps) break;
            if (i + 2 < steps) {
                if ((i + 2) % kAhead == 0) pages = pages_from(i + 2);
                load_step(even, i + 2);
                held = held_of(i + 2);
            }
            do_step(odd, t0 + (i + 1) * (NW * NT) + wave * NT, next);
        }
    }

    // join the waves: O relative to the workgroup's maximum of each row
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        l[mt] = sum_over_groups(l[mt]);
        if (g == 0) lds_m[wave][16 * mt + r] = m[mt], lds_l[wave][16 * mt + r] = l[mt];
    }
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, lds_m[w][16 * mt + r]);
        const float f = m[mt] == -INFINITY ? (l[mt] == l[mt] ? 0.0f : l[mt]) : exp2_fast(m[mt] - top);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float *dst = &lds_o[wave][(16 * mt + r) * LD + (4 * g + e) * OC];
            const float w = poison[mt] >> e & 1 ? NAN : f;
#pragma unroll
            for (int c = 0; c < OC; c += 4)
                *(v4f *)(dst + c) = v4f{o[mt][c][e] * w, o[mt][c + 1][e] * w, o[mt][c + 2][e] * w, o[mt][c + 3][e] * w};
        }
    }
    __syncthreads();
    if (a.slots && blockIdx.x == part.begin * a.hk && threadIdx.x == 0)
        ((int2 *)a.split)[part.item] = make_int2(part.begin, part.parts);
    float *ml = (float *)(a.split + a.part);
    const int64_t all = (int64_t)gridDim.x * RB;
    for (int u = threadIdx.x; u < s.rows * (D / 4); u += 64 * NW) {
        const int row = u / (D / 4), d = u % (D / 4) * 4;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, lds_m[w][row]);
        v4f acc = v4f{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float mw = lds_m[w][row], lw = lds_l[w][row];
            sum += mw == -INFINITY ? (lw == lw ? 0.0f : lw) : lw * exp2_fast(mw - top);
            acc += *(const v4f *)&lds_o[w][row * LD + d];
        }
        if (part.parts == 1) {
            const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
            const int x = s.first + row;
            char *dst = (char *)a.out + 2 * ((s.q0 + token_of(a, x)) * a.out_token + (head * a.ratio + x - token_of(a, x) * a.ratio) * a.out_head + d);
            const uint32_t w0 = pack2<T>(acc[0] * inv, acc[1] * inv), w1 = pack2<T>(acc[2] * inv, acc[3] * inv);
            typedef struct __attribute__((packed, aligned(2))) { uint32_t w[2]; } Out;
            *(Out *)dst = Out{{w0, w1}};
        } else {
            const int64_t at = (int64_t)blockIdx.x * RB + row;
            if (d == 0) ml[2 * at] = top, ml[2 * at + 1] = sum;
            *(v4f *)(ml + 2 * all + at * D + d) = acc;
        }
    }
}

// ---- many rows ---------------------------------------------------------------
typedef float v16f __attribute__((ext_vector_type(16)));

template <typename T>
__device__ __forceinline__ v16f mfma32(const v4i &a, const v4i &b, const v16f &c) {
    if constexpr (__is_same(T, Bf16))
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0,
                                                      0);
}

// The 16-byte unit of a row of V^T that holds unit u: rows that are read
// together and rows that are written together lie in different banks.
template <int TT>
__device__ __forceinline__ int v_unit(int d, int u) { return u ^ ((d ^ (d >> 3)) & (TT / 8 - 1)); }
template <int D>
__device__ __forceinline__ int k_unit(int tok, int u) { return u ^ (tok & (D == 64 ? 7 : 15)); }

// The item that is `index`-th in line: longest sequence first, its last rows,
// which see the most tokens, first (more than 64 sequences: in their order).
__device__ __forceinline__ int item_in_line(const AttnArgs &a, int index) {
    int seq = index / a.row_blocks;
    const int block = a.row_blocks - 1 - index % a.row_blocks;
    if (a.num_seqs > 1 && a.num_seqs <= 64) {
        const int lane = threadIdx.x & 63;
        const int len = lane < a.num_seqs ? a.lens[lane] : 0;
        int rank = 0;
        for (int j = 0; j < a.num_seqs; ++j) {
            const int other = __builtin_amdgcn_readlane(len, j);
            rank += other > len || (other == len && j < lane);
        }
        seq = __builtin_ctzll(__ballot(lane < a.num_seqs && rank == seq));
    }
    return seq * a.row_blocks + block;
}

// Blocks of many rows: bound by issue, matrix and vector instructions in turn.
//
// S^T = K Q^T and O^T = V^T P^T as above, in 32x32x16 products, 32 rows a wave.
// The waves convert a step's tokens together, each 16 of them, into LDS: K token
// after token, V transposed, both in the order of the products' operands, so that
// a row's weights stay where the scores were.  A conversion serves 256 rows (128
// for heads of 256 values), where every wave of the small blocks converts for its
// own 32: 38 M vector instructions against 66 M.  One buffer: a second one cost
// as much in addresses as it saved (235 us each).  In the loop an
// instruction of the matrix unit lies between some of the vector unit's; apart,
// eight products and then 130 vector instructions, the two units took turns (252
// against 235 us).  2047 tokens after 3953, with two shorter prompts, 32 heads of
// 128 over 8: 169 GFLOP in 187 us, 902 TFLOP/s, a library's large product 1151; 2047
// tokens alone, a triangle, 60 us (79 with blocks of neighbouring rows).
template <typename T, int D>
__global__ __launch_bounds__(64 * prompt_waves(D), D == 256 ? 1 : 2) void prompt_kernel(const AttnArgs a) {
    constexpr int KS = D / 16, DB = D / 32, W = D / 32, NW = prompt_waves(D), TT = 16 * NW, ROWS = 32 * NW;
    __shared__ __align__(16) uint16_t lds_k[TT * D], lds_v[TT * D];
    __shared__ uint64_t lds_nan[NW][4];
    __shared__ __align__(8) uint8_t lds_any[NW];   // a wave's tile has such groups
    __shared__ Part lds_part;
    __shared__ Item lds_item;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int head = blockIdx.x % a.hk, index = blockIdx.x / a.hk;

    Part part;
    Item s;
    int row0 = 32 * wave;          // the wave's first row, counted from s.first
    if (a.slots) {
        if (wave == 0) find_part(a, ROWS, index, lds_part, lds_item);
        __syncthreads();
        part = lds_part;
        if (__builtin_amdgcn_readfirstlane(part.item) < 0) return;
        s = lds_item;
    } else {
        const int item = item_in_line(a, index);
        s = item_of(a, item, ROWS);
        if (s.rows <= 0) return;
        if (a.paired) {
            // half a block from the start and one from the end of the rows: every
            // workgroup, and every SIMD (waves w and w + 4), has as much to do.  The rows
            // end with the launch's blocks, also of a sequence that has more of them.
            constexpr int HALF = ROWS / 2;
            const int all = min(s.n * a.ratio, a.row_blocks * ROWS);
            const int blocks = (all + ROWS - 1) / ROWS, block = s.first / ROWS;
            const int low = block * HALF, high = (2 * blocks - 1 - block) * HALF;
            const int last = min(all, (high < all ? high : low) + HALF) - 1;
            row0 = wave < NW / 2 ? low + 32 * wave : high + 32 * (wave - NW / 2);
            s.first = 0, s.rows = all;
            s.hi = max(0, min(s.len, s.base + token_of(a, last) + 1));
        }
        part = Part{item, s.lo / 16, s.lo / 16 + tiles_of(s), 1, index};
    }
    s = uniform(s);
    part = uniform(part);
    const int t0 = part.t0, t1 = part.t1;
    const int row = row0 + n;
    int lo, hi;
    row_span(a, s, row, lo, hi);
    // what all of the wave's rows see, and what any of them does
    const int wave_rows = min(32, s.rows - row0);
    int all_lo = 0, all_hi = 0, any_lo = 0, any_hi = 0;
    if (wave_rows > 0) {
        row_span(a, s, row0 + wave_rows - 1, all_lo, any_hi);
        row_span(a, s, row0, any_lo, all_hi);
    }
    v4i q[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) q[k] = v4i{0, 0, 0, 0};
    const int x = s.first + row;
    const int64_t x_token = s.q0 + token_of(a, x), x_head = head * a.ratio + x - token_of(a, x) * a.ratio;
    if (row < s.rows) {
        const char *p = (const char *)a.q + 2 * (x_token * a.q_token + x_head * a.q_head + 8 * h);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const auto m = *(const typename Raw<T>::Mem *)(p + 32 * k);
            q[k] = v4i{(int)m.w[0], (int)m.w[1], (int)m.w[2], (int)m.w[3]};
        }
    }

    // A wave loads and converts 16 of the step's tokens: of K values
    // [(lane % 4) D / 4, ...) of token lane / 4, of V run lane % 16 of tokens
    // 4 (lane / 16) ...
    const int32_t *table = a.tables + s.seq * a.table_stride;
    // the step that is loaded, and which of its tiles are there
    uint32_t kw[W], vw[W], ks, vs, next_held = 0;
    // the pages of 64 / NW steps, a tile a lane
    int pages = page_of(a, table, t0 + lane, t1), page;
    const auto load = [&](int t) {
        if ((t - t0) % 64 == 0 && t > t0) pages = page_of(a, table, t + lane, t1);
        page = __builtin_amdgcn_readlane(pages, (t - t0) % 64 + wave);
        next_held = (uint32_t)(__ballot(pages >= 0) >> ((t - t0) % 64)) & ((1u << NW) - 1);
        const int off = (t + wave) * 16 & (a.ps - 1);
        const uint8_t *base = a.cache + ((int64_t)(page < 0 ? 0 : page) * a.hk + head) * head_bytes(a.ps, D);
        load_words(kw, base + off * (D / 2) + lane * (D / 8));
        load_words(vw, base + v_codes(a.ps, D) + off * (D / 2) + lane * (D / 8));
        const uint8_t *p = base + k_scales(a.ps, D) + off * (D / 32) + lane * D / 128;
        ks = D == 256 ? *(const uint16_t *)p : *p;
        vs = *(const uint32_t *)(base + v_scales(a.ps, D) + (((off >> 2) + (lane >> 4)) * (D / 32) + (lane & 15) * D / 512) * 4);
    };
    const auto convert = [&](int t) {
        uint16_t *lk = lds_k, *lv = lds_v;
        const int tok = 16 * wave + lane / 4;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float sc = scale_bits(D == 256 && w >= 4 ? ks << 15 : ks << 23);
            v4i f;
#pragma unroll
            for (int b = 0; b < 4; ++b) f[b] = (int)pair_of<T>(kw[w], sc, b);
            *(v4i *)(lk + tok * D + k_unit<D>(tok, lane % 4 * W + w) * 8) = f;
        }
        // Tokens that no row sees may hold anything, and a weight of 0 would not
        // keep a NaN from the other rows either: what is unseen becomes zeros,
        // groups of NaN are noted and become zeros as well.
        const int pos = 16 * (t + wave);
        const bool inside = page >= 0 && pos >= s.lo && pos + 16 <= s.hi;
        const uint32_t low7 = ~vs & 0x7f7f7f7fu;
        const bool odd = (((low7 + 0x7f7f7f7fu) | ~vs) & 0x80808080u) != 0x80808080u;   // a byte of 255
        int any = 0;
        if (!inside || __any(odd)) {
            uint64_t nan[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = pos + 4 * (lane >> 4) + j;
                const uint32_t byte = 0xffu << (8 * j);
                const bool seen = page >= 0 && at >= s.lo && at < s.hi;
                nan[j] = __ballot(seen && (vs & byte) == byte);
                if (!seen || (vs & byte) == byte) {
                    constexpr int B = D / 32;
                    if constexpr (B == 2) vw[j / 2] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                    else
#pragma unroll
                        for (int w = 0; w < B / 4; ++w) vw[j * (B / 4) + w] = 0;
                    vs &= ~byte;
                }
            }
            any = (nan[0] | nan[1] | nan[2] | nan[3]) != 0;
            if (any && lane == 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) lds_nan[wave][j] = nan[j];
            }
        }
        if (lane == 0) lds_any[wave] = (uint8_t)any;
        const float sc[4] = {scale_bits(vs << 23), scale_bits(vs << 15), scale_bits(vs << 7), scale_bits(vs >> 1)};
        // four tokens are 8 bytes of a row of V^T, in the order of the scores' lanes
        const int g = lane >> 4, unit = 2 * wave + (g & 1), place = 4 * (g >> 1);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = j * (D / 32) + c;
                w[j] = pair_of<T>(vw[b / 4], sc[j], b % 4);
            }
            const int d = (lane & 15) * (D / 16) + 2 * c;
            *(v2i *)(lv + d * TT + v_unit<TT>(d, unit) * 8 + place) =
                v2i{(int)__builtin_amdgcn_perm(w[1], w[0], 0x05040100u), (int)__builtin_amdgcn_perm(w[3], w[2], 0x05040100u)};
            *(v2i *)(lv + (d + 1) * TT + v_unit<TT>(d + 1, unit) * 8 + place) =
                v2i{(int)__builtin_amdgcn_perm(w[1], w[0], 0x07060302u), (int)__builtin_amdgcn_perm(w[3], w[2], 0x07060302u)};
        }
    };

    // where this lane's operands lie: of K unit 2 k + h of token n (32 b + n: an
    // offset), of V unit 2 k + h of value n, with the block b and d exchanged
    // by their exclusive or (value 32 d + n, unit 4 b + 2 k + h)
    int at_k[KS], at_v[2][NW / 2];
#pragma unroll
    for (int k = 0; k < KS; ++k) at_k[k] = n * D + k_unit<D>(n, 2 * k + h) * 8;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < NW / 2; ++e) at_v[k][e] = n * TT + v_unit<TT>(n, 4 * e + 2 * k + h) * 8;

    v16f o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    const float room = headroom<T>(s.len, kSlack);
    uint32_t poison = 0;           // blocks of 32 values that a NaN has reached

    const auto products = [&](int t, uint32_t there) {
        if (16 * t >= any_hi || 16 * (t + NW) <= any_lo) return;
        const uint16_t *lk = lds_k, *lv = lds_v;
        const bool whole = 16 * t >= all_lo && 16 * (t + NW) <= all_hi && there == (1u << NW) - 1;
        const auto read_k = [&](int b, int k) { return *(const v4i *)(lk + at_k[k] + 32 * b * D); };
        const auto read_v = [&](int b, int u) {
            return *(const v4i *)(lv + at_v[u / DB][(b ^ (u % DB)) & (NW / 2 - 1)] + 32 * (u % DB) * TT);
        };
        const auto mask = [&](v16f &sc, int b) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int tok = 16 * t + 32 * b + 8 * (i / 4) + 4 * h + i % 4;
                if (!(there >> (2 * b + i / 8) & 1) || tok < lo || tok >= hi) sc[i] = -INFINITY;
                top = fmaxf(top, sc[i]);
            }
            return top;
        };
        // While the matrix unit has the next block's scores, the vector unit has this
        // one's weights: an instruction of the one between some of the other, and
        // operands read two products ahead.
        constexpr int PV = 2 * DB;
        v16f sc;
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) sc = mfma32<T>(read_k(0, k), q[k], sc);
        float top = sc[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, sc[i]);
        if (!whole) top = mask(sc, 0);
#pragma unroll
        for (int b = 0; b < NW / 2; ++b) {
            const bool last = b + 1 == NW / 2;
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__builtin_fmaf(fmaxf(as_float(both[0]), as_float(both[1])), a.scale, room), m);
            if (__any(top > m + kSlack)) {
                const float f = top > m ? exp2_fast(m - top) : 1.0f;
                l *= f;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] *= f;
                m = top;
            }
            const float ref = m == -INFINITY ? 0.0f : -m;
            v16f next;
#pragma unroll
            for (int i = 0; i < 16; ++i) next[i] = 0.0f;
            v4i p[2], f[KS], g[PV];
            if (!last) f[0] = read_k(b + 1, 0), f[1] = read_k(b + 1, 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                if (!last && k + 2 < KS) f[k + 2] = read_k(b + 1, k + 2);
                if (k + 2 >= KS) g[k + 2 - KS] = read_v(b, k + 2 - KS);
#pragma unroll
                for (int x = 8 * k / KS; x < 8 * (k + 1) / KS; ++x) {
                    const float e0 = exp2_fast(__builtin_fmaf(sc[2 * x], a.scale, ref));
                    const float e1 = exp2_fast(__builtin_fmaf(sc[2 * x + 1], a.scale, ref));
                    const uint32_t pair = pack2<T>(e0, e1);
                    l = add_pair<T>(pair, l);
                    p[x / 4][x % 4] = (int)pair;
                }
                if (!last) next = mfma32<T>(f[k], q[k], next);
                __builtin_amdgcn_sched_barrier(0);
            }
            top = -INFINITY;
#pragma unroll
            for (int u = 0; u < PV; ++u) {
                if (u + 2 < PV) g[u + 2] = read_v(b, u + 2);
                o[u % DB] = mfma32<T>(g[u], p[u / DB], o[u % DB]);
                if (!last) {
#pragma unroll
                    for (int i = 16 * u / PV; i < 16 * (u + 1) / PV; ++i) top = fmaxf(top, next[i]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            sc = next;
            if (!last && !whole) top = mask(sc, b + 1);
        }
        // groups of NaN, to the rows that see their token
        uint32_t any = 0;
#pragma unroll
        for (int w = 0; w < NW; w += 4) any |= *(const uint32_t *)(lds_any + w);
        if (__builtin_amdgcn_readfirstlane(any) == 0) return;
        for (int w = 0; w < NW; ++w) {
            if (!lds_any[w]) continue;
            for (int j = 0; j < 4; ++j) {
                const uint64_t bits = lds_nan[w][j];
                for (int g = 0; g < 4; ++g) {
                    const int tok = 16 * (t + w) + 4 * g + j;
                    const bool seen = tok >= lo && tok < hi;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
                        poison |= seen && (bits >> (16 * g + d * 512 / D) & 1) ? 1u << d : 0u;
                }
            }
        }
    };

    if (t0 < t1) {
        load(t0);
        uint32_t held = next_held;
        convert(t0);
        if (t0 + NW < t1) load(t0 + NW);
        __syncthreads();
        for (int t = t0; t < t1; t += NW) {
            products(t, held);
            __syncthreads();
            if (t + NW < t1) {
                held = next_held;
                convert(t + NW);
                if (t + 2 * NW < t1) load(t + 2 * NW);
            }
            __syncthreads();
        }
    }
    {
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = as_float(both[0]) + as_float(both[1]);
    }
    if (a.slots && blockIdx.x == part.begin * a.hk && threadIdx.x == 0)
        ((int2 *)a.split)[part.item] = make_int2(part.begin, part.parts);
    if (row >= s.rows) return;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] += poison >> d & 1 ? NAN : 0.0f;
    if (part.parts == 1) {
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        char *dst = (char *)a.out + 2 * (x_token * a.out_token + x_head * a.out_head + 4 * h);
        typedef struct __attribute__((packed, aligned(2))) { uint32_t w[2]; } Out;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(Out *)(dst + 2 * (32 * d + 2 * i)) =
                    Out{{pack2<T>(o[d][i] * inv, o[d][i + 1] * inv), pack2<T>(o[d][i + 2] * inv, o[d][i + 3] * inv)}};
    } else {
        float *ml = (float *)(a.split + a.part);
        const int64_t at = (int64_t)blockIdx.x * ROWS + row;
        if (h == 0) ml[2 * at] = m, ml[2 * at + 1] = l;
        float *dst = ml + 2 * (int64_t)gridDim.x * ROWS + at * D + 4 * h;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) *(v4f *)(dst + 32 * d + 2 * i) = v4f{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
    }
}

// Joins the parts of the rows of items that were cut: W waves a row take the
// parts in turn, eight parts' values in flight in each.  With few rows there are
// waves to spare: two sequences of 64 heads and 32 parts take 4.7 us with four
// waves a row and 8.0 with one, 24 sequences of 200 rows 6.7 and 4.0.
template <typename T, int D, int RB, int W>
__global__ __launch_bounds__(256) void join_kernel(const AttnArgs a, int64_t all) {
    constexpr int V = D / 64, U = 8;
    typedef float vec __attribute__((ext_vector_type(V)));
    __shared__ float lds_m[W], lds_l[W];
    __shared__ vec lds_o[W][64];
    const int lane = threadIdx.x & 63, id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = W == 1 ? 0 : id;
    const int item = blockIdx.x / a.hk, head = blockIdx.x % a.hk, row = W == 1 ? blockIdx.y * 4 + id : blockIdx.y;
    const int2 cut = ((const int2 *)a.split)[item];
    const Item s = item_of(a, item, RB);
    if (row >= s.rows || cut.y < 2) return;
    const float *ml = (const float *)(a.split + a.part);
    const float *o = ml + 2 * all + lane * V;
    const auto place = [&](int k) { return ((int64_t)(cut.x + k) * a.hk + head) * RB + row; };
    float top = -INFINITY, sum = 0.0f;
    vec acc = 0.0f;
    for (int k0 = wave; k0 < cut.y; k0 += W * U) {
        float m[U], l[U];
        vec x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = place(min(k0 + W * u, cut.y - 1));
            m[u] = ml[2 * at], l[u] = ml[2 * at + 1];
            x[u] = *(const vec *)(o + at * D);
        }
        float high = top;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 + W * u >= cut.y) m[u] = -INFINITY, l[u] = 0.0f, x[u] = 0.0f;
            high = fmaxf(high, m[u]);
        }
        const float f = top == -INFINITY ? 0.0f : exp2_fast(top - high);
        sum *= f;
        acc *= f;
        top = high;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float e = m[u] == -INFINITY ? (l[u] == l[u] ? 0.0f : l[u]) : exp2_fast(m[u] - top);
            sum += l[u] * e;
            acc += x[u] * e;
        }
    }
    if constexpr (W > 1) {
        lds_o[wave][lane] = acc;
        if (lane == 0) lds_m[wave] = top, lds_l[wave] = sum;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, lds_m[w]);
        sum = 0.0f;
        acc = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float mw = lds_m[w], lw = lds_l[w];
            const float e = mw == -INFINITY ? (lw == lw ? 0.0f : lw) : exp2_fast(mw - top);
            sum += lw * e;
            acc += lds_o[w][lane] * e;
        }
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    const int x = s.first + row;
    uint16_t *dst = (uint16_t *)a.out + (s.q0 + token_of(a, x)) * a.out_token + (head * a.ratio + x - token_of(a, x) * a.ratio) * a.out_head + lane * V;
    if constexpr (V == 1) {
        dst[0] = (uint16_t)pack2<T>(acc[0] * inv, 0.0f);
    } else {
        typedef struct __attribute__((packed, aligned(2))) { uint32_t w[V / 2]; } Out;
        Out out;
#pragma unroll
        for (int v = 0; v < V; v += 2) out.w[v / 2] = pack2<T>(acc[v] * inv, acc[v + 1] * inv);
        *(Out *)dst = out;
    }
}

constexpr int kJoinWide = 2048;   // rows up to which four waves join one

template <typename T, int D, int RB>
void launch_join(const AttnArgs &a, const Cut &c, hipStream_t stream) {
    const unsigned items = (unsigned)(c.items * a.hk);
    if (items * RB <= kJoinWide)
        hipLaunchKernelGGL((join_kernel<T, D, RB, 4>), dim3(items, RB), dim3(256), 0, stream, a, c.grid * RB);
    else
        hipLaunchKernelGGL((join_kernel<T, D, RB, 1>), dim3(items, RB / 4), dim3(256), 0, stream, a, c.grid * RB);
}

template <typename T, int D>
int32_t launch_attention(AttnArgs a, const Cut &c, hipStream_t stream) {
    constexpr int TWO = D == 256 ? 2 : 4;
    const dim3 grid((unsigned)c.grid);
    if (c.rows > 32)
        hipLaunchKernelGGL((prompt_kernel<T, D>), grid, dim3(64 * prompt_waves(D)), 0, stream, a);
    else if (c.rows == 32)
        hipLaunchKernelGGL((decode_kernel<T, D, 2, 2, TWO, 2>), grid, dim3(64 * TWO), 0, stream, a);
    else if (c.wide)
        hipLaunchKernelGGL((decode_kernel<T, D, 1, 2, 8, 2, D != 256>), grid, dim3(512), 0, stream, a);
    else
        hipLaunchKernelGGL((decode_kernel<T, D, 1, 2, 4, D == 256 ? 2 : 3>), grid, dim3(256), 0, stream, a);
    const int32_t st = launch_status();
    if (st != kOk || !c.slots) return st;
    if (c.rows == 16) launch_join<T, D, 16>(a, c, stream);
    else if (c.rows == 32) launch_join<T, D, 32>(a, c, stream);
    else launch_join<T, D, 32 * prompt_waves(D)>(a, c, stream);
    return launch_status();
}

int32_t sizes_ok(int num_seqs, int total_q, int max_q, int64_t max_kv, int hq, int hk, int D, int ps, int64_t num_pages,
                 int max_pages, int element, int window, float scale) {
    if (num_seqs < 0 || total_q < 0 || max_q < 0 || max_kv < 0 || hk < 1 || hq < hk || D < 1 || ps < 1 || num_pages < 1 ||
        max_pages < 1 || window < 0 || element < kF32 || element > kBf16 || !(scale > 0.0f) || scale > 1e30f)
        return kInvalid;
    if (hq % hk) return kInvalid;
    if (!head_dim_ok(D) || !page_size_ok(ps) || element == kF32) return kUnsupported;
    if (num_pages > 0x7fffffff || max_kv > 0x7fffff00 || hq > 32768) return kUnsupported;
    // rows are counted in 32 bits, also those of a sequence that is longer than max_q
    if ((int64_t)total_q * (hq / hk) > 0x7ffffc00) return kUnsupported;
    if (past_a_launch(num_seqs, max_q, hq / hk, hk)) return kUnsupported;
    return cut_of(num_seqs, max_q, max_kv, hq / hk, hk, D, window).grid > kMaxGrid ? kUnsupported : kOk;
}

}  // namespace
}  // namespace bk

using namespace bk;

extern "C" int32_t baracuda_kernels_kv4_attention_gfx950_can_implement(
    int32_t num_seqs, int32_t total_q, int32_t max_q, int64_t max_kv, int32_t num_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t page_size, int64_t num_pages, int32_t max_pages, int32_t element, int32_t causal,
    int32_t window, float scale) {
    (void)causal;
    return sizes_ok(num_seqs, total_q, max_q, max_kv, num_heads, num_kv_heads, head_dim, page_size, num_pages, max_pages,
                    element, window, scale);
}

extern "C" size_t baracuda_kernels_kv4_attention_gfx950_workspace_size(int32_t num_seqs, int32_t max_q, int64_t max_kv,
                                                                       int32_t num_heads, int32_t num_kv_heads,
                                                                       int32_t head_dim, int32_t window) {
    if (num_seqs < 1 || max_q < 1 || max_kv < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || head_dim < 1 || window < 0)
        return 0;
    if (past_a_launch(num_seqs, max_q, num_heads / num_kv_heads, num_kv_heads)) return 0;
    return cut_of(num_seqs, max_q, max_kv, num_heads / num_kv_heads, num_kv_heads, head_dim, window).bytes;
}

extern "C" int32_t baracuda_kernels_kv4_attention_gfx950_run(
    int32_t num_seqs, int32_t total_q, int32_t max_q, int64_t max_kv, int32_t num_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t page_size, int64_t num_pages, int32_t max_pages, int32_t element, int32_t causal,
    int32_t window, float scale, const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *cache,
    const int32_t *tables, int64_t table_stride, const int32_t *kv_lens, const int32_t *cu_q, void *out,
    int64_t out_token_stride, int64_t out_head_stride, void *workspace, size_t workspace_bytes, void *stream) {
    const int32_t st = sizes_ok(num_seqs, total_q, max_q, max_kv, num_heads, num_kv_heads, head_dim, page_size, num_pages,
                                max_pages, element, window, scale);
    if (st != kOk) return st;
    if (num_seqs == 0 || total_q == 0 || max_q == 0) return kOk;
    if (!q || !cache || !tables || !kv_lens || !out) return kInvalid;
    if (!cu_q && (max_q != 1 || total_q != num_seqs)) return kInvalid;
    if (((uintptr_t)q & 1u) || ((uintptr_t)out & 1u) || ((uintptr_t)cache & 15u)) return kMisaligned;
    const Cut c = cut_of(num_seqs, max_q, max_kv, num_heads / num_kv_heads, num_kv_heads, head_dim, window);
    if (c.bytes) {
        if (!workspace || workspace_bytes < c.bytes) return kWorkspace;
        if ((uintptr_t)workspace & 15u) return kMisaligned;
    }
    AttnArgs a{};
    a.q = q, a.out = out, a.cache = (const uint8_t *)cache;
    a.tables = tables, a.lens = kv_lens, a.cu_q = cu_q;
    a.q_token = q_token_stride, a.q_head = q_head_stride;
    a.out_token = out_token_stride, a.out_head = out_head_stride;
    a.table_stride = table_stride, a.num_pages = num_pages;
    a.split = (char *)workspace, a.part = (int64_t)c.part;
    a.num_seqs = num_seqs, a.total_q = total_q;
    a.hq = num_heads, a.hk = num_kv_heads, a.ratio = num_heads / num_kv_heads;
    // x magic / 2^32 falls short of the next whole number by less than x ratio / 2^32
    // (of any row there is, should a sequence have more tokens than max_q)
    const uint64_t rows = (uint64_t)total_q * (uint64_t)a.ratio + 512;
    a.ratio_magic = a.ratio > 1 && rows * (uint64_t)a.ratio < (1ull << 32) ? (uint32_t)(((1ull << 32) + a.ratio - 1) / a.ratio) : 0;
    a.max_pages = max_pages, a.ps = page_size, a.ps_shift = log2i(page_size);
    a.causal = causal != 0, a.window = window;
    a.paired = causal && !window && !c.slots && head_dim != 256;
    a.row_blocks = c.row_blocks, a.items = (int)c.items, a.slots = c.slots, a.min_tiles = c.min_tiles;
    a.scale = scale * 1.44269504088896340736f;
    const hipStream_t s = (hipStream_t)stream;
    const bool half = element == kF16;
    if (head_dim == 64) return half ? launch_attention<F16, 64>(a, c, s) : launch_attention<Bf16, 64>(a, c, s);
    if (head_dim == 128) return half ? launch_attention<F16, 128>(a, c, s) : launch_attention<Bf16, 128>(a, c, s);
    return half ? launch_attention<F16, 256>(a, c, s) : launch_attention<Bf16, 256>(a, c, s);
}
