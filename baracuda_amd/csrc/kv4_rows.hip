// kv4_rows.hip -- what lies between the QKV projection and attention:
//
//   qk_norm_rope   RMS norm of each head of Q and K and the position rotation
//   kv4_append     the same, then K and V into the pages of a 4-bit cache
//   kv4_read       the values that slots of such a cache stand for
//
// A head x of D values becomes y = x w / sqrt(mean(x^2) + eps); then each pair
// (a, b) of its first rope_dim values becomes (a cos - b sin, b cos + a sin),
// with the cosine and sine of the pair's column in the table's row of the
// token's position on the pair's axis.  Pairs are (i, i + rope_dim / 2), or
// (2i, 2i + 1) when interleaved.
//
// A lane holds eight values, a head D / 8 lanes; a workgroup has one token, so
// a lane reads its cosines and sines once for all the heads that it sees.
// Bound by HBM: one read of the projection's rows, one write of the results.
//
// Q, and K without a cache, are computed in 32 bits and rounded once.  K that
// is quantized is computed in 64 bits: it is rounded to the element's type
// first and then to 4 bits, and a value next to a border between two codes has
// to fall on the side of the exact one, or equal prefixes would give unequal
// pages.
#include "kv4.hpp"

namespace bk {
namespace {

using namespace kv4;

constexpr int kWaves = 4;

struct RowArgs {
    const void *src[3];        // Q, K, V
    int64_t src_token[3], src_head[3];
    void *dst[2];              // Q, K (K unused with a cache)
    int64_t dst_token[2], dst_head[2];
    const void *weight[2];
    const int32_t *positions;  // [axes, tokens]
    const float *cosine, *sine;   // [table_rows, rope / 2]
    const int32_t *pair_axis;  // [rope / 2]
    int64_t tokens, table_rows;
    uint8_t *cache;
    const int64_t *slots;
    int64_t num_slots;
    double eps;
    int hq, hk, D, rope, axes, ps, ps_shift, most;
};

template <typename A>
__device__ __forceinline__ A inv_root(A x);
template <>
__device__ __forceinline__ float inv_root<float>(float x) { return 1.0f / __builtin_sqrtf(x); }
template <>
__device__ __forceinline__ double inv_root<double>(double x) { return 1.0 / __builtin_sqrt(x); }

// Lane exchanges within the G lanes of a head, for a sum: after step k all
// lanes of 2^(k+1) hold the same, so a mirrored lane serves as well as the one
// across.  DPP and v_permlane16_swap: no trip through LDS.
template <int M>
__device__ __forceinline__ uint32_t across(uint32_t x) {
    constexpr int ctrl = M == 1 ? 0xB1 : M == 2 ? 0x4E : M == 4 ? 0x141 : 0x140;
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, true);
}
template <int M>
__device__ __forceinline__ float add_across(float x) {
    if constexpr (M == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    } else {
        return x + __uint_as_float(across<M>(__float_as_uint(x)));
    }
}
template <int M>
__device__ __forceinline__ double add_across(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    if constexpr (M == 16) {
        const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
        return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) +
               __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
    } else {
        const uint64_t o = (uint64_t)across<M>((uint32_t)(b >> 32)) << 32 | across<M>((uint32_t)b);
        return x + __builtin_bit_cast(double, o);
    }
}
template <typename A, int G>
__device__ __forceinline__ A head_sum(A x) {
    x = add_across<1>(x);
    x = add_across<2>(x);
    x = add_across<4>(x);
    if constexpr (G >= 16) x = add_across<8>(x);
    if constexpr (G >= 32) x = add_across<16>(x);
    return x;
}

// The norm and the rotation of one head in type A: eight values a lane (x), the
// other sides of their pairs (z) and both sides' weights.
template <typename A, int G>
__device__ __forceinline__ void norm_rope(const float (&x)[8], const float (&z)[8], float (&y)[8], const float (&w)[8],
                                          const float (&wz)[8], bool norm, double eps, int D, bool turn, const float (&c)[8],
                                          const float (&s)[8]) {
    A r = 1;
    if (norm) {
        A sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_elementwise_fma((A)x[i], (A)x[i], sum);
        r = inv_root<A>(head_sum<A, G>(sum) / (A)D + (A)eps);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        A v = (A)x[i], o = (A)z[i];
        if (norm) v = v * r * (A)w[i], o = o * r * (A)wz[i];
        const A t = __builtin_elementwise_fma(v, (A)c[i], o * (A)s[i]);
        y[i] = (float)(turn ? t : v);
    }
}

// G lanes a head, ITERS heads a lane, `share` of the workgroup's waves a token.
// T: the element; KV4: K and V go into the cache.
template <typename T, int G, int ITERS, bool KV4>
__global__ __launch_bounds__(64 * kWaves) void rows_kernel(const RowArgs a, int share, bool inter) {
    typedef typename Raw<T>::Mem Mem;
    constexpr int HPW = 64 / G, W = sizeof(Mem) / 4;
    __shared__ __align__(16) float lds_c[kWaves][128], lds_s[kWaves][128];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t token = (int64_t)blockIdx.x * (kWaves / share) + wave / share;
    const int l = lane % G, at = 8 * l;
    const int heads = a.hq + a.hk * (KV4 ? 2 : 1);
    const int first = (blockIdx.y * share + wave % share) * HPW * ITERS + lane / G;
    const bool here = token < a.tokens, mine = here && at < a.D;

    Mem raw[ITERS];
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        const int h = first + it * HPW;
        const int kind = h < a.hq ? 0 : h < a.hq + a.hk ? 1 : 2;
        const int hh = h - (kind == 0 ? 0 : kind == 1 ? a.hq : a.hq + a.hk);
        raw[it] = Mem{};
        if (mine && h < heads) {
            const int64_t off = token * a.src_token[kind] + hh * a.src_head[kind] + at;
            raw[it] = *(const Mem *)((const char *)a.src[kind] + off * (int64_t)(sizeof(Mem) / 8));
        }
    }

    // the token's cosines and sines, once for all its heads, through LDS
    const int half = a.rope / 2;
    float *lc = lds_c[wave / share], *ls = lds_s[wave / share];
    if (here) {
        for (int p = wave % share * 64 + lane; p < half; p += 64 * share) {
            const int axis = a.pair_axis ? a.pair_axis[p] : 0;
            int64_t row = -1;
            if ((unsigned)axis < (unsigned)a.axes) row = a.positions[(int64_t)axis * a.tokens + token];
            const bool ok = row >= 0 && row < a.table_rows;
            lc[p] = ok ? a.cosine[row * half + p] : __uint_as_float(0x7fc00000u);
            ls[p] = ok ? a.sine[row * half + p] : 0.0f;
        }
    }

    // this lane's, the sine with the sign of its side, and the lane that holds
    // the other side of its pairs (its own when interleaved)
    const bool turn = at < a.rope, low = at < half;
    const int other = inter || !turn ? l : low ? l + half / 8 : l - half / 8;
    const bool norm = a.weight[0] != nullptr;
    float w[2][8], wz[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        Mem m{}, z{};
        if (norm && at < a.D) {
            m = *(const Mem *)((const char *)a.weight[k] + (int64_t)at * (sizeof(Mem) / 8));
            z = *(const Mem *)((const char *)a.weight[k] + (int64_t)(8 * other) * (sizeof(Mem) / 8));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) w[k][i] = Raw<T>::get(m, i), wz[k][i] = Raw<T>::get(z, inter ? i ^ 1 : i);
    }
    int64_t slot = 0;
    if constexpr (KV4) slot = here ? a.slots[token] : -1;
    __syncthreads();
    if (!here) return;
    float c[8], s[8];
    if (turn) {
        const int p0 = inter ? at / 2 : low ? at : at - half;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = p0 + (inter ? i / 2 : i);
            c[i] = lc[p];
            s[i] = (inter ? (i & 1) == 0 : low) ? -ls[p] : ls[p];
        }
    }

#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        const int h = first + it * HPW;
        if (h - lane / G >= heads) break;
        const int kind = h < a.hq ? 0 : h < a.hq + a.hk ? 1 : 2;
        const int hh = h - (kind == 0 ? 0 : kind == 1 ? a.hq : a.hq + a.hk);
        float x[8], z[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = Raw<T>::get(raw[it], i);
        if (inter) {
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = x[i ^ 1];
        } else {
            Mem m;
#pragma unroll
            for (int i = 0; i < W; ++i) m.w[i] = (uint32_t)__shfl((int)raw[it].w[i], other, G);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = Raw<T>::get(m, i);
        }
        if (!KV4 || kind == 0) {
            float wh[8], wo[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) wh[i] = w[KV4 ? 0 : kind == 1][i], wo[i] = wz[KV4 ? 0 : kind == 1][i];
            norm_rope<float, G>(x, z, y, wh, wo, norm, a.eps, a.D, turn, c, s);
            if (mine && h < heads) {
                Mem out;
                Raw<T>::put(out, y);
                const int64_t off = token * a.dst_token[kind] + hh * a.dst_head[kind] + at;
                *(Mem *)((char *)a.dst[kind] + off * (int64_t)(sizeof(Mem) / 8)) = out;
            }
        } else if constexpr (KV4) {
            if (kind == 1) {
                norm_rope<double, G>(x, z, y, w[1], wz[1], norm, a.eps, a.D, turn, c, s);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = Raw<T>::round(y[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i];
            }
            // four lanes share a scale
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
            top = max(top, across<1>(top));
            top = max(top, across<2>(top));
            const bool good = top < 0x7f800000u;
            const int byte = good ? scale_byte(top, a.most) : 255;
            const uint32_t code = good ? encode8(y, byte) : 0u;
            if (mine && h < heads && slot >= 0 && slot < a.num_slots) {
                const int off = (int)(slot & (a.ps - 1)), few = a.D / 32;
                uint8_t *base = a.cache + ((slot >> a.ps_shift) * a.hk + hh) * head_bytes(a.ps, a.D);
                if (kind == 1) {
                    *(uint32_t *)(base + off * (a.D / 2) + 4 * l) = code;
                    if (l % 4 == 0) base[k_scales(a.ps, a.D) + off * few + l / 4] = (uint8_t)byte;
                } else {
                    uint8_t *p = base + v_codes(a.ps, a.D) + (off >> 2) * 64 * few + (off & 3) * few;
                    if (few == 2) {          // a lane holds two runs
                        *(uint16_t *)(p + (2 * l) * 8) = (uint16_t)code;
                        *(uint16_t *)(p + (2 * l + 1) * 8) = (uint16_t)(code >> 16);
                    } else if (few == 4) {   // one
                        *(uint32_t *)(p + l * 16) = code;
                    } else {                 // or half of one
                        *(uint32_t *)(p + (l / 2) * 32 + (l & 1) * 4) = code;
                    }
                    if (l % 4 == 0) base[v_scales(a.ps, a.D) + ((off >> 2) * few + l / 4) * 4 + (off & 3)] = (uint8_t)byte;
                }
            }
        }
    }
}

// A lane reads eight values of K or V of one token; slots out of range read as zeros.
template <typename T>
__global__ __launch_bounds__(256) void read_kernel(const uint8_t *__restrict__ cache, const int64_t *__restrict__ slots,
                                                   int64_t num_slots, void *k_out, int64_t k_token, int64_t k_head,
                                                   void *v_out, int64_t v_token, int64_t v_head, int hk, int D, int ps,
                                                   int ps_shift) {
    typedef typename Raw<T>::Mem Mem;
    const int64_t token = blockIdx.x;
    const int lanes = D / 8, few = D / 32;
    const int64_t slot = slots[token];
    const bool in = slot >= 0 && slot < num_slots;
    const int off = (int)(slot & (ps - 1));
    for (int u = blockIdx.y * blockDim.x + threadIdx.x; u < 2 * hk * lanes; u += gridDim.y * blockDim.x) {
        const int l = u % lanes, row = u / lanes;
        const bool is_v = row >= hk;
        const int h = is_v ? row - hk : row;
        uint32_t code = 0, byte = 0;
        if (in) {
            const uint8_t *base = cache + ((slot >> ps_shift) * hk + h) * head_bytes(ps, D);
            if (!is_v) {
                code = *(const uint32_t *)(base + off * (D / 2) + 4 * l);
                byte = base[k_scales(ps, D) + off * few + l / 4];
            } else {
                const uint8_t *p = base + v_codes(ps, D) + (off >> 2) * 64 * few + (off & 3) * few;
                if (few == 2)
                    code = *(const uint16_t *)(p + (2 * l) * 8) | (uint32_t) * (const uint16_t *)(p + (2 * l + 1) * 8) << 16;
                else if (few == 4)
                    code = *(const uint32_t *)(p + l * 16);
                else
                    code = *(const uint32_t *)(p + (l / 2) * 32 + (l & 1) * 4);
                byte = base[v_scales(ps, D) + ((off >> 2) * few + l / 4) * 4 + (off & 3)];
            }
        }
        float x[8];
        decode8(code, byte, x);
        Mem out;
        Raw<T>::put(out, x);
        char *dst = (char *)(is_v ? v_out : k_out);
        const int64_t at = token * (is_v ? v_token : k_token) + h * (is_v ? v_head : k_head) + 8 * l;
        *(Mem *)(dst + at * (int64_t)(sizeof(Mem) / 8)) = out;
    }
}

template <typename T, int G, bool KV4>
void launch_lanes(const RowArgs &a, bool inter, hipStream_t stream) {
    const int heads = a.hq + a.hk * (KV4 ? 2 : 1), rounds = (heads + 64 / G - 1) / (64 / G);
    // a wave has up to three rounds of heads of a token where there are tokens
    // enough to fill the card without cutting them finer
    const int iters = rounds > 2 * kWaves && a.tokens >= 512 ? 3 : 1;
    const int waves = (rounds + iters - 1) / iters;
    const int share = waves >= 3 ? 4 : waves;
    const dim3 grid((unsigned)((a.tokens + kWaves / share - 1) / (kWaves / share)), (unsigned)((waves + share - 1) / share));
    if (iters == 3) hipLaunchKernelGGL((rows_kernel<T, G, 3, KV4>), grid, dim3(64 * kWaves), 0, stream, a, share, inter);
    else hipLaunchKernelGGL((rows_kernel<T, G, 1, KV4>), grid, dim3(64 * kWaves), 0, stream, a, share, inter);
}

template <typename T, bool KV4>
int32_t launch_style(const RowArgs &a, bool inter, hipStream_t stream) {
    if (a.D <= 64) launch_lanes<T, 8, KV4>(a, inter, stream);
    else if (a.D <= 128) launch_lanes<T, 16, KV4>(a, inter, stream);
    else launch_lanes<T, 32, KV4>(a, inter, stream);
    return launch_status();
}

int32_t sizes_ok(int64_t tokens, int hq, int hk, int D, int rope, int axes, int element) {
    if (tokens < 0 || hq < 0 || hk < 1 || D < 1 || rope < 0 || rope > D || axes < 1) return kInvalid;
    if (element < kF32 || element > kBf16) return kInvalid;
    if (D % 16 || D > 256 || rope % 16 || axes > 16) return kUnsupported;
    if (tokens > 0x7fffffff || hq > 32768 || hk > 32768) return kUnsupported;
    return kOk;
}

int32_t cache_ok(int D, int ps, int64_t num_pages, int element) {
    if (num_pages < 1) return kInvalid;
    if (!head_dim_ok(D) || !page_size_ok(ps) || element == kF32) return kUnsupported;
    return kOk;
}

bool aligned(const void *p, int element) { return ((uintptr_t)p & (element == kF32 ? 3u : 1u)) == 0; }

}  // namespace
}  // namespace bk

using namespace bk;

extern "C" int32_t baracuda_kernels_qk_norm_rope_gfx950_can_implement(
    int64_t tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t rope_dim, int32_t axes,
    int32_t element) {
    return sizes_ok(tokens, num_heads, num_kv_heads, head_dim, rope_dim, axes, element);
}

extern "C" int32_t baracuda_kernels_qk_norm_rope_gfx950_run(
    int64_t tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t rope_dim, int32_t axes,
    int32_t interleaved, int32_t element, double eps, const void *q, int64_t q_token_stride, int64_t q_head_stride,
    const void *k, int64_t k_token_stride, int64_t k_head_stride, void *q_out, int64_t q_out_token_stride,
    int64_t q_out_head_stride, void *k_out, int64_t k_out_token_stride, int64_t k_out_head_stride, const void *q_weight,
    const void *k_weight, const int32_t *positions, const float *cosine, const float *sine, int64_t table_rows,
    const int32_t *pair_axis, void *stream) {
    const int32_t st = sizes_ok(tokens, num_heads, num_kv_heads, head_dim, rope_dim, axes, element);
    if (st != kOk) return st;
    if (tokens == 0) return kOk;
    if ((num_heads && (!q || !q_out)) || !k || !k_out || !q_weight != !k_weight) return kInvalid;
    if (rope_dim && (!positions || !cosine || !sine || table_rows < 1 || (axes > 1 && !pair_axis))) return kInvalid;
    if (!(eps >= 0.0)) return kInvalid;
    for (const void *p : {q, k, (const void *)q_out, (const void *)k_out, q_weight, k_weight})
        if (!aligned(p, element)) return kMisaligned;
    RowArgs a{};
    a.src[0] = q, a.src[1] = k;
    a.src_token[0] = q_token_stride, a.src_token[1] = k_token_stride;
    a.src_head[0] = q_head_stride, a.src_head[1] = k_head_stride;
    a.dst[0] = q_out, a.dst[1] = k_out;
    a.dst_token[0] = q_out_token_stride, a.dst_token[1] = k_out_token_stride;
    a.dst_head[0] = q_out_head_stride, a.dst_head[1] = k_out_head_stride;
    a.weight[0] = q_weight, a.weight[1] = k_weight;
    a.positions = positions, a.cosine = cosine, a.sine = sine;
    a.pair_axis = axes > 1 ? pair_axis : nullptr;
    a.tokens = tokens, a.table_rows = table_rows, a.eps = eps;
    a.hq = num_heads, a.hk = num_kv_heads, a.D = head_dim, a.rope = rope_dim, a.axes = axes;
    const hipStream_t s = (hipStream_t)stream;
    if (element == kF32) return launch_style<float, false>(a, interleaved != 0, s);
    if (element == kF16) return launch_style<F16, false>(a, interleaved != 0, s);
    return launch_style<Bf16, false>(a, interleaved != 0, s);
}

extern "C" int32_t baracuda_kernels_kv4_append_gfx950_can_implement(
    int64_t tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t rope_dim, int32_t axes,
    int32_t element, int32_t page_size, int64_t num_pages) {
    const int32_t st = sizes_ok(tokens, num_heads, num_kv_heads, head_dim, rope_dim, axes, element);
    return st != kOk ? st : cache_ok(head_dim, page_size, num_pages, element);
}

extern "C" int32_t baracuda_kernels_kv4_append_gfx950_run(
    int64_t tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t rope_dim, int32_t axes,
    int32_t interleaved, int32_t element, double eps, int32_t page_size, int64_t num_pages, const void *q,
    int64_t q_token_stride, int64_t q_head_stride, const void *k, int64_t k_token_stride, int64_t k_head_stride,
    const void *v, int64_t v_token_stride, int64_t v_head_stride, void *q_out, int64_t q_out_token_stride,
    int64_t q_out_head_stride, void *cache, const int64_t *slots, const void *q_weight, const void *k_weight,
    const int32_t *positions, const float *cosine, const float *sine, int64_t table_rows, const int32_t *pair_axis,
    void *stream) {
    int32_t st = sizes_ok(tokens, num_heads, num_kv_heads, head_dim, rope_dim, axes, element);
    if (st == kOk) st = cache_ok(head_dim, page_size, num_pages, element);
    if (st != kOk) return st;
    if (tokens == 0) return kOk;
    if ((num_heads && (!q || !q_out)) || !k || !v || !cache || !slots || !q_weight != !k_weight) return kInvalid;
    if (rope_dim && (!positions || !cosine || !sine || table_rows < 1 || (axes > 1 && !pair_axis))) return kInvalid;
    if (!(eps >= 0.0)) return kInvalid;
    for (const void *p : {q, k, v, (const void *)q_out, q_weight, k_weight})
        if (!aligned(p, element)) return kMisaligned;
    if ((uintptr_t)cache & 15u) return kMisaligned;
    RowArgs a{};
    a.src[0] = q, a.src[1] = k, a.src[2] = v;
    a.src_token[0] = q_token_stride, a.src_token[1] = k_token_stride, a.src_token[2] = v_token_stride;
    a.src_head[0] = q_head_stride, a.src_head[1] = k_head_stride, a.src_head[2] = v_head_stride;
    a.dst[0] = q_out;
    a.dst_token[0] = q_out_token_stride, a.dst_head[0] = q_out_head_stride;
    a.weight[0] = q_weight, a.weight[1] = k_weight;
    a.positions = positions, a.cosine = cosine, a.sine = sine;
    a.pair_axis = axes > 1 ? pair_axis : nullptr;
    a.tokens = tokens, a.table_rows = table_rows, a.eps = eps;
    a.hq = num_heads, a.hk = num_kv_heads, a.D = head_dim, a.rope = rope_dim, a.axes = axes;
    a.cache = (uint8_t *)cache, a.slots = slots, a.num_slots = num_pages * page_size;
    a.ps = page_size, a.ps_shift = log2i(page_size), a.most = element == kF16 ? 13 : 125;
    const hipStream_t s = (hipStream_t)stream;
    if (element == kF16) return launch_style<F16, true>(a, interleaved != 0, s);
    return launch_style<Bf16, true>(a, interleaved != 0, s);
}

extern "C" int32_t baracuda_kernels_kv4_read_gfx950_can_implement(int64_t tokens, int32_t num_kv_heads,
                                                                  int32_t head_dim, int32_t element, int32_t page_size,
                                                                  int64_t num_pages) {
    const int32_t st = sizes_ok(tokens, 0, num_kv_heads, head_dim, 0, 1, element);
    if (st != kOk) return st;
    // reading back into 32 bits needs no rounding, so it is offered as well
    return cache_ok(head_dim, page_size, num_pages, element == kF32 ? kBf16 : element);
}

extern "C" int32_t baracuda_kernels_kv4_read_gfx950_run(
    int64_t tokens, int32_t num_kv_heads, int32_t head_dim, int32_t element, int32_t page_size, int64_t num_pages,
    const void *cache, const int64_t *slots, void *k_out, int64_t k_token_stride, int64_t k_head_stride, void *v_out,
    int64_t v_token_stride, int64_t v_head_stride, void *stream) {
    const int32_t st = baracuda_kernels_kv4_read_gfx950_can_implement(tokens, num_kv_heads, head_dim, element, page_size,
                                                                      num_pages);
    if (st != kOk) return st;
    if (tokens == 0) return kOk;
    if (!cache || !slots || !k_out || !v_out) return kInvalid;
    if (!aligned(k_out, element) || !aligned(v_out, element) || ((uintptr_t)cache & 15u)) return kMisaligned;
    const int units = 2 * num_kv_heads * (head_dim / 8);
    const dim3 grid((unsigned)tokens, (unsigned)((units + 255) / 256 < 4 ? (units + 255) / 256 : 4));
    const hipStream_t s = (hipStream_t)stream;
    const uint8_t *c = (const uint8_t *)cache;
    const int64_t n = num_pages * page_size;
    const int sh = log2i(page_size);
    if (element == kF32)
        hipLaunchKernelGGL((read_kernel<float>), grid, dim3(256), 0, s, c, slots, n, k_out, k_token_stride,
                           k_head_stride, v_out, v_token_stride, v_head_stride, num_kv_heads, head_dim, page_size, sh);
    else if (element == kF16)
        hipLaunchKernelGGL((read_kernel<F16>), grid, dim3(256), 0, s, c, slots, n, k_out, k_token_stride,
                           k_head_stride, v_out, v_token_stride, v_head_stride, num_kv_heads, head_dim, page_size, sh);
    else
        hipLaunchKernelGGL((read_kernel<Bf16>), grid, dim3(256), 0, s, c, slots, n, k_out, k_token_stride,
                           k_head_stride, v_out, v_token_stride, v_head_stride, num_kv_heads, head_dim, page_size, sh);
    return launch_status();
}
