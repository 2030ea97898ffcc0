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
// A lane holds eight values, a head D / 8 lanes.  A token's cosines and sines
// come through LDS once, and a wave has up to six rounds of heads of one token, all
// loaded before the first is used.  Bound by HBM, with the vector unit close behind:
// 6145 tokens of 40 heads of 128, three position axes, 129 MB in 36 us (3.5 TB/s;
// a large copy 4.8), 22 us of them vector instructions' issue.  What it took: heads
// of all kinds in one wave and the table read by every lane 132 us; the table
// through LDS, three rounds a wave 53; rounds of one kind, norm's and rotation's
// factors multiplied once 36; six rounds 33.5 (twelve 33.8); a look at whether 32
// bits held what came out, 1.9 more.  8191 tokens of 16 + 4 heads of 256 into the cache:
// 157 MB in 47 us, of which a wave waits 60%: its workgroup loads two tokens, meets a
// barrier, stores and ends.
//
// Q, and K without a cache, are computed in 32 bits and rounded once; heads that
// leave their range, in 64.  K that is quantized is computed in 64 bits: it is
// rounded to the element's type first and then to 4 bits, and a value next to a
// border between two codes has to fall on the side of the exact one, or equal
// prefixes would give unequal pages.
#include "kv4.hpp"

namespace bk {
namespace {

using namespace kv4;

constexpr int kWaves = 4;
constexpr int kIters = 6;          // rounds of heads of a wave where there are many tokens
constexpr int64_t kManyTokens = 512;  // below, a round a wave: the card is not full

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
    float inv_D;
    int hq, hk, D, rope, axes, ps, ps_shift, most;
};

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

// G lanes a head, ITERS rounds of 64 / G heads a wave, `share` of the workgroup's
// waves a token.  A round has heads of one kind (Q, K or V), so what differs
// between them is scalar.  T: the element; KV4: K and V go into the cache.
template <typename T, int G, int ITERS, bool KV4>
__global__ __launch_bounds__(64 * kWaves) void rows_kernel(const RowArgs a, int share, bool inter) {
    typedef typename Raw<T>::Mem Mem;
    constexpr int HPW = 64 / G, W = sizeof(Mem) / 4, SIZE = sizeof(Mem) / 8;
    __shared__ __align__(16) float lds_c[kWaves][128], lds_s[kWaves][128];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t token = (int64_t)blockIdx.x * (kWaves / share) + wave / share;
    const int l = lane % G, at = 8 * l, sub = lane / G;
    const int rq = (a.hq + HPW - 1) / HPW, rk = (a.hk + HPW - 1) / HPW, rounds = rq + rk * (KV4 ? 2 : 1);
    const int first = (blockIdx.y * share + wave % share) * ITERS;
    const bool here = token < a.tokens;
    const auto kind_of = [&](int r) { return r < rq ? 0 : r < rq + rk ? 1 : 2; };
    const auto head_of = [&](int r, int kind) { return (r - (kind == 0 ? 0 : kind == 1 ? rq : rq + rk)) * HPW + sub; };

    Mem raw[ITERS];
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        raw[it] = Mem{};
        const int r = first + it, kind = kind_of(r), head = head_of(r, kind);
        if (here && r < rounds && at < a.D && head < (kind ? a.hk : a.hq))
            raw[it] = *(const Mem *)((const char *)a.src[kind] +
                                     (token * a.src_token[kind] + head * a.src_head[kind] + at) * SIZE);
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
    int64_t slot = 0;
    if constexpr (KV4) slot = here ? a.slots[token] : -1;
    __syncthreads();
    if (!here) return;

    // this lane's, the sine with the sign of its side, and the lane that holds
    // the other side of its pairs (its own when interleaved)
    const bool turn = at < a.rope, low = at < half;
    const int other = inter || !turn ? l : low ? l + half / 8 : l - half / 8;
    const bool norm = a.weight[0] != nullptr;
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 1.0f, s[i] = 0.0f;
    if (turn) {
        const int p0 = inter ? at / 2 : low ? at : at - half;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = p0 + (inter ? i / 2 : i);
            c[i] = lc[p];
            s[i] = (inter ? (i & 1) == 0 : low) ? -ls[p] : ls[p];
        }
    }
    // the weights of both sides, and their products with cosine and sine
    Mem mw{}, mz{};
    float cw[8], sw[8];
    int held = -1;
    uint32_t redo = 0;             // rounds that 32 bits do not hold

    const auto top_of = [](const float (&y)[8]) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
        return top;
    };
    // K's or V's codes, and the scale that four lanes share; top: the lane's own top_of
    const auto store_codes = [&](int kind, int head, const float (&y)[8], uint32_t top) {
        top = max(top, across<1>(top));
        top = max(top, across<2>(top));
        const bool good = top < 0x7f800000u;
        const int byte = good ? scale_byte(top, a.most) : 255;
        const uint32_t code = good ? encode8(y, byte) : 0u;
        if (at >= a.D || head >= a.hk || slot < 0 || slot >= a.num_slots) return;
        const int off = (int)(slot & (a.ps - 1)), few = a.D / 32;
        uint8_t *base = a.cache + ((slot >> a.ps_shift) * a.hk + head) * head_bytes(a.ps, a.D);
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
    };
    const auto store_row = [&](int kind, int head, const float (&y)[8]) {
        if (at >= a.D || head >= (kind ? a.hk : a.hq)) return;
        Mem out;
        Raw<T>::put(out, y);
        *(Mem *)((char *)a.dst[kind] + (token * a.dst_token[kind] + head * a.dst_head[kind] + at) * SIZE) = out;
    };

#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        const int r = first + it;
        if (r >= rounds) break;
        const int kind = kind_of(r), head = head_of(r, kind);
        if (norm && kind < 2 && kind != held) {
            held = kind;
            if (at < a.D) {
                mw = *(const Mem *)((const char *)a.weight[kind] + at * SIZE);
                mz = *(const Mem *)((const char *)a.weight[kind] + 8 * other * SIZE);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                cw[i] = c[i] * Raw<T>::get(mw, i);
                sw[i] = s[i] * Raw<T>::get(mz, inter ? i ^ 1 : i);
            }
        }
        float x[8], z[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = Raw<T>::get(raw[it], i);
        if (kind < 2) {
            if (inter) {
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = turn ? x[i ^ 1] : 0.0f;
            } else {
                Mem m;
#pragma unroll
                for (int i = 0; i < W; ++i) m.w[i] = (uint32_t)__shfl((int)raw[it].w[i], other, G);
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = Raw<T>::get(m, i);
            }
        }
        if (!KV4 || kind == 0) {
            if (norm) {
                float sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(x[i], x[i], sum);
                const float mean = __builtin_fmaf(head_sum<float, G>(sum), a.inv_D, (float)a.eps);
                const float root = __builtin_amdgcn_rsqf(mean);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = root * __builtin_fmaf(z[i], sw[i], x[i] * cw[i]);
                if constexpr (!__is_same(T, F16)) {
                    // of a pair's two products that leave the range, one sum at least is infinite
                    float high = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) high = fmaxf(high, __builtin_fabsf(y[i]));
                    if (__any(!(mean > 0x1p-40f && mean < 0x1p100f && high < INFINITY))) {
                        redo |= 1u << it;
                        continue;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = turn ? __builtin_fmaf(z[i], s[i], x[i] * c[i]) : x[i];
            }
            store_row(kind, head, y);
        } else if constexpr (KV4) {
            uint32_t top;
            if (kind == 1) {
                double root = 1, sum = 0;
                if (norm) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum = __builtin_fma((double)x[i], (double)x[i], sum);
                    sum = head_sum<double, G>(sum);
                    root = 1.0 / __builtin_sqrt(sum / (double)a.D + a.eps);
                }
                float least = INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float v = x[i], o = z[i];
                    // 22 bits at most: exact while it is in range
                    if (norm) v *= Raw<T>::get(mw, i), o *= Raw<T>::get(mz, inter ? i ^ 1 : i);
                    const double t = turn ? __builtin_fma((double)v, (double)c[i], (double)o * (double)s[i]) : (double)v;
                    y[i] = Raw<T>::round((float)(t * root));
                    least = fminf(least, __builtin_fabsf(y[i]));
                }
                top = top_of(y);
                if constexpr (!__is_same(T, F16)) {
                    // a product past the range, or bits of one below it
                    if (norm && __any(sum != 0 && !(least >= 0x1p-60f && top < 0x7f800000u && root < 0x1p30))) {
                        redo |= 1u << it;
                        continue;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i];
                top = top_of(y);
            }
            store_codes(kind, head, y, top);
        }
    }

    // Heads whose squares or products with the weights leave 32 bits (f16's cannot): from
    // the inputs on in 64, a round at a time
    if constexpr (!__is_same(T, F16)) {
        for (; redo; redo &= redo - 1) {
            // a copy of its own: addresses kept from above cost the loop above a register (97,
            // a wave a SIMD less)
            int place = at;
            asm volatile("" : "+v"(place));
            const int r = first + __builtin_ctz(redo), kind = kind_of(r), head = head_of(r, kind);
            Mem m{}, w{}, u{}, far;
            if (at < a.D) {
                if (head < (kind ? a.hk : a.hq))
                    m = *(const Mem *)((const char *)a.src[kind] + (token * a.src_token[kind] + head * a.src_head[kind] + at) * SIZE);
                w = *(const Mem *)((const char *)a.weight[kind] + at * SIZE);
                u = *(const Mem *)((const char *)a.weight[kind] + 8 * other * SIZE);
            }
#pragma unroll
            for (int i = 0; i < W; ++i) far.w[i] = (uint32_t)__shfl((int)m.w[i], other, G);
            double sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = __builtin_fma((double)Raw<T>::get(m, i), (double)Raw<T>::get(m, i), sum);
            const double root = 1.0 / __builtin_sqrt(head_sum<double, G>(sum) / (double)a.D + a.eps);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double v = (double)Raw<T>::get(m, i) * (double)Raw<T>::get(w, i);
                const double o = (double)Raw<T>::get(far, inter ? i ^ 1 : i) * (double)Raw<T>::get(u, inter ? i ^ 1 : i);
                double t = v;
                if (turn) {
                    const int p = inter ? place / 2 + i / 2 : (low ? place : place - half) + i;
                    const double cosine = lc[p], sine = (inter ? (i & 1) == 0 : low) ? -ls[p] : ls[p];
                    t = __builtin_fma(v, cosine, o * sine);
                }
                y[i] = Raw<T>::round((float)(t * root));
            }
            if (KV4 && kind) store_codes(kind, head, y, top_of(y));
            else store_row(kind, head, y);
        }
    }
}

// A lane reads eight values of K or V of one token; slots out of range read as
// zeros.  A workgroup has `several` tokens, or part of one.  Bound by its chain of loads,
// slot, then code and scale, before the one store of a lane: 8191 tokens of 2 heads of
// 256, 21 MB in 7.2 us (2.9 TB/s), half of a wave's time waited.
template <typename T>
__global__ __launch_bounds__(256) void read_kernel(const uint8_t *__restrict__ cache, const int64_t *__restrict__ slots,
                                                   int64_t tokens, int64_t num_slots, void *k_out, int64_t k_token,
                                                   int64_t k_head, void *v_out, int64_t v_token, int64_t v_head, int hk,
                                                   int lane_shift, int ps, int ps_shift, int several) {
    typedef typename Raw<T>::Mem Mem;
    const int lanes = 1 << lane_shift, D = 8 * lanes, few = D / 32, units = 2 * hk * lanes;
    int64_t token = blockIdx.x;
    int first = blockIdx.y * blockDim.x + threadIdx.x;
    if (several > 1) {
        const int mine = first / units;
        token = token * several + mine;
        first -= mine * units;
        if (mine >= several || token >= tokens) return;
    }
    const int64_t slot = slots[token];
    const bool in = slot >= 0 && slot < num_slots;
    const int off = (int)(slot & (ps - 1));
    for (int u = first; u < units; u += gridDim.y * blockDim.x) {
        const int l = u & (lanes - 1), row = u >> lane_shift;
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
    constexpr int HPW = 64 / G;
    const int rounds = (a.hq + HPW - 1) / HPW + (a.hk + HPW - 1) / HPW * (KV4 ? 2 : 1);
    const int iters = a.tokens >= kManyTokens ? kIters : 1;
    const int waves = (rounds + iters - 1) / iters;
    const int share = waves >= 3 ? 4 : waves;
    const dim3 grid((unsigned)((a.tokens + kWaves / share - 1) / (kWaves / share)), (unsigned)((waves + share - 1) / share));
    if (iters > 1) hipLaunchKernelGGL((rows_kernel<T, G, kIters, KV4>), grid, dim3(64 * kWaves), 0, stream, a, share, inter);
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
    // a launch has less than 2^32 threads
    if (tokens > 0x7fffff || hq > 32768 || hk > 32768) return kUnsupported;
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
    a.tokens = tokens, a.table_rows = table_rows, a.eps = eps, a.inv_D = 1.0f / (float)head_dim;
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
    a.tokens = tokens, a.table_rows = table_rows, a.eps = eps, a.inv_D = 1.0f / (float)head_dim;
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
    const int units = 2 * num_kv_heads * (head_dim / 8), several = units < 256 ? 256 / units : 1;
    const dim3 grid((unsigned)((tokens + several - 1) / several), (unsigned)((units + 255) / 256 < 4 ? (units + 255) / 256 : 4));
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t *)cache, slots, tokens,
                           num_pages * page_size, k_out, k_token_stride, k_head_stride, v_out, v_token_stride, v_head_stride,
                           num_kv_heads, log2i(head_dim / 8), page_size, log2i(page_size), several);
    };
    if (element == kF32) launch(read_kernel<float>);
    else if (element == kF16) launch(read_kernel<F16>);
    else launch(read_kernel<Bf16>);
    return launch_status();
}
