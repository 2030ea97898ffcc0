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
// Scores, maximum, sum and O are held in 32 bits.  P is rounded to the
// element's type for the matrix product, at most half a step of a weight; the
// sum is that of the weights before the rounding, whose mean error is none.
#include "kv4_attention.hpp"

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

// MT tiles of 16 rows; NT tiles of 16 tokens a step; NW waves.
template <typename T, int D, int MT, int NT, int NW, int OCC>
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
    const int t0 = __builtin_amdgcn_readfirstlane(part.t0), t1 = __builtin_amdgcn_readfirstlane(part.t1);

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
                            2 * ((s.q0 + x / a.ratio) * a.q_token + (head * a.ratio + x % a.ratio) * a.q_head + g * (D / 4));
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
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt] = -INFINITY, l[mt] = 0.0f;
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
        if (!whole) {
            // V of tokens that no row sees may be anything, also a NaN, and 0 times it would be one
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int tok = 16 * (t + n) + 4 * g + j;
                    if (!there[n] || tok < s.lo || tok >= s.hi) {
                        constexpr int B = D / 32;   // bytes of a token
                        if constexpr (B == 2) tile[n].v[j / 2] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                        else
#pragma unroll
                            for (int w = 0; w < B / 4; ++w) tile[n].v[j * (B / 4) + w] = 0;
                        tile[n].vs &= ~(0xffu << (8 * j));
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
            top = fmaxf(max_over_groups(top) * a.scale, m[mt]);
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
                }
                l[mt] += (e[0] + e[1]) + (e[2] + e[3]);
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
    };
    const auto held_of = [&](int step) { return __ballot(pages >= 0) >> (step % kAhead * NT) & ((1u << NT) - 1); };
    if constexpr (NW >= 8) {
        for (int i = 0; i < steps; ++i) {
            if (i && i % kAhead == 0) pages = pages_from(i);
            Tile<D> tile[NT];
            load_step(tile, i);
            do_step(tile, t0 + i * (NW * NT) + wave * NT, held_of(i));
        }
    } else if (steps) {
        // the next step's loads go out before this one's products
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
#pragma unroll
            for (int c = 0; c < OC; c += 4)
                *(v4f *)(dst + c) = v4f{o[mt][c][e] * f, o[mt][c + 1][e] * f, o[mt][c + 2][e] * f, o[mt][c + 3][e] * f};
        }
    }
    __syncthreads();
    if (a.slots && part.parts > 1 && blockIdx.x == part.begin * a.hk && threadIdx.x == 0)
        ((int2 *)a.split)[part.item] = make_int2(part.begin, part.parts);
    if (a.slots && part.parts == 1 && head == 0 && threadIdx.x == 0) ((int2 *)a.split)[part.item] = make_int2(part.begin, 1);
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
            char *dst = (char *)a.out + 2 * ((s.q0 + x / a.ratio) * a.out_token + (head * a.ratio + x % a.ratio) * a.out_head + d);
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
    uint16_t *dst = (uint16_t *)a.out + (s.q0 + x / a.ratio) * a.out_token + (head * a.ratio + x % a.ratio) * a.out_head + lane * V;
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

// How a problem is cut, the same for the workspace's size and the launch.
struct Cut {
    int mt, rows, row_blocks, slots, min_tiles;
    bool wide;                // one workgroup of many waves has a whole sequence
    int64_t items, grid;
    size_t part, bytes;
};

constexpr int kSlots = 512;
constexpr int kMinTiles = 16;
constexpr int kJoinWide = 2048;   // rows up to which four waves join one
constexpr int kWhole = 1024;      // tokens up to which nothing is cut

Cut cut_of(int num_seqs, int max_q, int64_t max_kv, int ratio, int hk, int D, int window) {
    Cut c{};
    c.mt = (int64_t)max_q * ratio <= 16 ? 1 : 2;
    c.rows = 16 * c.mt;
    c.row_blocks = (int)(((int64_t)max_q * ratio + c.rows - 1) / c.rows);
    c.items = (int64_t)num_seqs * c.row_blocks;
    const int64_t seen = window && window + (int64_t)max_q < max_kv ? window + (int64_t)max_q : max_kv;
    c.slots = seen <= kWhole || c.items * hk >= 8 * kSlots ? 0 : kSlots;
    c.min_tiles = kMinTiles;
    c.wide = !c.slots && c.mt == 1 && seen > 256 && c.items * hk <= 256;
    c.grid = c.items * hk + c.slots;
    if (c.slots) {
        c.grid = (c.grid + hk - 1) / hk * hk;
        c.part = ((size_t)c.items * 8 + 255) / 256 * 256;
        c.bytes = c.part + (size_t)c.grid * c.rows * (D + 2) * 4;
    }
    return c;
}

template <typename T, int D>
int32_t launch_attention(AttnArgs a, const Cut &c, hipStream_t stream) {
    constexpr int WIDE = D == 256 ? 8 : 16, TWO = D == 256 ? 2 : 4;
    const dim3 grid((unsigned)c.grid);
    if (c.mt == 2)
        hipLaunchKernelGGL((decode_kernel<T, D, 2, 2, TWO, 2>), grid, dim3(64 * TWO), 0, stream, a);
    else if (c.wide)
        hipLaunchKernelGGL((decode_kernel<T, D, 1, 2, WIDE, WIDE / 4>), grid, dim3(64 * WIDE), 0, stream, a);
    else
        hipLaunchKernelGGL((decode_kernel<T, D, 1, 2, 4, D == 256 ? 2 : 3>), grid, dim3(256), 0, stream, a);
    const int32_t st = launch_status();
    if (st != kOk || !c.slots) return st;
    const int items = (int)c.items * a.hk;
    if (items * c.rows <= kJoinWide) {
        const dim3 grid((unsigned)items, (unsigned)c.rows);
        if (c.mt == 1) hipLaunchKernelGGL((join_kernel<T, D, 16, 4>), grid, dim3(256), 0, stream, a, c.grid * 16);
        else hipLaunchKernelGGL((join_kernel<T, D, 32, 4>), grid, dim3(256), 0, stream, a, c.grid * 32);
    } else {
        const dim3 grid((unsigned)items, (unsigned)((c.rows + 3) / 4));
        if (c.mt == 1) hipLaunchKernelGGL((join_kernel<T, D, 16, 1>), grid, dim3(256), 0, stream, a, c.grid * 16);
        else hipLaunchKernelGGL((join_kernel<T, D, 32, 1>), grid, dim3(256), 0, stream, a, c.grid * 32);
    }
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
    const Cut c = cut_of(num_seqs, max_q, max_kv, hq / hk, hk, D, window);
    if (c.grid > 0x7fffffff || c.items > 0x3fffffff || c.items * hk > 0x7fffffff) return kUnsupported;
    return kOk;
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
    a.max_pages = max_pages, a.ps = page_size, a.ps_shift = log2i(page_size);
    a.causal = causal != 0, a.window = window;
    a.row_blocks = c.row_blocks, a.items = (int)c.items, a.slots = c.slots, a.min_tiles = c.min_tiles;
    a.scale = scale * 1.44269504088896340736f;
    const hipStream_t s = (hipStream_t)stream;
    const bool half = element == kF16;
    if (head_dim == 64) return half ? launch_attention<F16, 64>(a, c, s) : launch_attention<Bf16, 64>(a, c, s);
    if (head_dim == 128) return half ? launch_attention<F16, 128>(a, c, s) : launch_attention<Bf16, 128>(a, c, s);
    return half ? launch_attention<F16, 256>(a, c, s) : launch_attention<Bf16, 256>(a, c, s);
}
