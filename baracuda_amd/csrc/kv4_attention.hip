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
template <typename T, int D, int MT, int NT, int NW>
__global__ __launch_bounds__(64 * NW) void decode_kernel(const AttnArgs a) {
    constexpr int RB = 16 * MT, KW = D / 32, OC = D / 16;
    constexpr int LD = D + 4;
    __shared__ float lds_m[NW][RB], lds_l[NW][RB];
    __shared__ __align__(16) float lds_o[NW][RB * LD];
    __shared__ Part lds_part;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % a.hk, index = blockIdx.x / a.hk;

    Part part;
    Item s;
    if (a.slots) {
        if (wave == 0) {
            part = find_part(a, RB, index);
            if (lane == 0) lds_part = part;
        }
        __syncthreads();
        part = lds_part;
        part.item = __builtin_amdgcn_readfirstlane(part.item);
        if (part.item < 0) return;
        s = item_of(a, part.item, RB);
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

    for (int t = t0 + wave * NT; t < t1; t += NW * NT) {
        Tile<D> tile[NT];
        bool whole = 16 * t >= all_lo && 16 * (t + NT) <= all_hi && t + NT <= t1;
        bool there[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int page = page_of(a, table, t + n, t1);
            there[n] = page >= 0;
            whole = whole && there[n];
            load_tile<D>(tile[n], a, page < 0 ? 0 : page, head, (t + n) * 16 & (a.ps - 1), lane);
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
                const float ks = scale_value(D == 256 ? (tile[n].ks >> (kk >= 4 ? 8 : 0)) & 0xffu : tile[n].ks);
                v4i f;
#pragma unroll
                for (int b = 0; b < 4; ++b) f[b] = (int)pair_of<T>(tile[n].k[kk], ks, b);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) sc[mt][n] = mfma_pv<T>(f, q[mt][kk], sc[mt][n]);
            }
        }
        // softmax
        v4i p[MT][(NT + 1) / 2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float top = m[mt];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float v = sc[mt][n][j] * a.scale;
                    if (!whole) {
                        const int tok = 16 * (t + n) + 4 * g + j;
                        if (!there[n] || tok < lo[mt] || tok >= hi[mt]) v = -INFINITY;
                    }
                    sc[mt][n][j] = v;
                    top = fmaxf(top, v);
                }
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__any(top > m[mt])) {
                const float f = top > m[mt] ? exp2_fast(m[mt] - top) : 1.0f;
                l[mt] *= f;
#pragma unroll
                for (int c = 0; c < OC; ++c) o[mt][c] *= f;
                m[mt] = top;
            }
            const float ref = m[mt] == -INFINITY ? 0.0f : m[mt];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float e[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) e[j] = exp2_fast(sc[mt][n][j] - ref);
                l[mt] += (e[0] + e[1]) + (e[2] + e[3]);
                p[mt][n / 2][(n & 1) * 2] = (int)pack2<T>(e[0], e[1]);
                p[mt][n / 2][(n & 1) * 2 + 1] = (int)pack2<T>(e[2], e[3]);
            }
        }
        // O^T += V^T P^T, two tiles of tokens a product
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            float vs[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) vs[h][j] = scale_value((tile[n + h].vs >> (8 * j)) & 0xffu);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                v4i even, odd;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        const int b0 = j * (D / 32) + c, b1 = (j + 1) * (D / 32) + c;
                        const uint32_t x = pair_of<T>(tile[n + h].v[b0 / 4], vs[h][j], b0 % 4);
                        const uint32_t y = pair_of<T>(tile[n + h].v[b1 / 4], vs[h][j + 1], b1 % 4);
                        even[2 * h + j / 2] = (int)__builtin_amdgcn_perm(y, x, 0x05040100u);
                        odd[2 * h + j / 2] = (int)__builtin_amdgcn_perm(y, x, 0x07060302u);
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    o[mt][2 * c] = mfma_pv<T>(even, p[mt][n / 2], o[mt][2 * c]);
                    o[mt][2 * c + 1] = mfma_pv<T>(odd, p[mt][n / 2], o[mt][2 * c + 1]);
                }
            }
        }
    }

    // join the waves: O relative to the workgroup's maximum of each row
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        l[mt] += __shfl_xor(l[mt], 16, 64);
        l[mt] += __shfl_xor(l[mt], 32, 64);
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

// Joins the parts of the rows of items that were cut.  A wave a row.
template <typename T, int D, int RB>
__global__ __launch_bounds__(256) void join_kernel(const AttnArgs a, int64_t all) {
    constexpr int V = D / 64;
    const int lane = threadIdx.x & 63;
    const int item = blockIdx.x / a.hk, head = blockIdx.x % a.hk;
    const int row = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
    const Item s = item_of(a, item, RB);
    if (row >= s.rows) return;
    const int2 cut = ((const int2 *)a.split)[item];
    if (cut.y < 2) return;
    const float *ml = (const float *)(a.split + a.part);
    const float *o = ml + 2 * all + lane * V;
    float top = -INFINITY;
    for (int k = lane; k < cut.y; k += 64) top = fmaxf(top, ml[2 * (((int64_t)(cut.x + k) * a.hk + head) * RB + row)]);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x, 64));
    float sum = 0.0f, acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.0f;
    for (int k = 0; k < cut.y; ++k) {
        const int64_t at = ((int64_t)(cut.x + k) * a.hk + head) * RB + row;
        const float mk = ml[2 * at], lk = ml[2 * at + 1];
        const float f = mk == -INFINITY ? 0.0f : exp2_fast(mk - top);
        sum += lk == lk ? lk * f : lk;
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] += o[at * D + v] * f;
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    const int x = s.first + row;
    uint16_t *dst = (uint16_t *)a.out + (s.q0 + x / a.ratio) * a.out_token + (head * a.ratio + x % a.ratio) * a.out_head + lane * V;
#pragma unroll
    for (int v = 0; v < V; ++v) dst[v] = (uint16_t)pack2<T>(acc[v] * inv, 0.0f);
}

// How a problem is cut, the same for the workspace's size and the launch.
struct Cut {
    int mt, rows, row_blocks, slots, min_tiles;
    int64_t items, grid;
    size_t part, bytes;
};

constexpr int kSlots = 512;
constexpr int kMinTiles = 16;
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
    constexpr int NT = D == 256 ? 2 : 4;
    const dim3 grid((unsigned)c.grid);
    if (c.mt == 1) hipLaunchKernelGGL((decode_kernel<T, D, 1, NT, 4>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((decode_kernel<T, D, 2, NT, D == 256 ? 2 : 4>), grid, dim3(D == 256 ? 128 : 256), 0, stream, a);
    const int32_t st = launch_status();
    if (st != kOk || !c.slots) return st;
    const dim3 rows((unsigned)(c.items * a.hk), (unsigned)((c.rows + 3) / 4));
    if (c.mt == 1) hipLaunchKernelGGL((join_kernel<T, D, 16>), rows, dim3(256), 0, stream, a, c.grid * 16);
    else hipLaunchKernelGGL((join_kernel<T, D, 32>), rows, dim3(256), 0, stream, a, c.grid * 32);
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
