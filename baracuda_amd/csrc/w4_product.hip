// w4_product.hip -- products with 4-bit weights: x W^T for the rows of a matrix,
// and by expert for the pairs of a mixture.
#include "moe_offsets.hpp"
#include "w4_product.hpp"

namespace bk {
namespace w4 {
namespace {

// Few rows: eight waves divide K among them, so that every workgroup asks for its
// weights at once, and add their sums through LDS in the waves' order.
//
// MF x 16 rows of x against CB blocks of 16 weight rows by the 16x16x32 product.
// Lane l supplies weight row l % 16 and group l / 16 of four (128 values of K,
// two tiles), and the same values of x's row l % 16.  Gated: odd blocks are rows
// of the second half of the matrix, whose products meet those of the first half
// in the same lanes.
constexpr int kWaves = 8;

template <bool BF16, bool MOE, bool GATED, int MF, int CB>
__global__ __launch_bounds__(64 * kWaves) void rows_kernel(const ProductArgs a) {
    extern __shared__ __attribute__((aligned(16))) int8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Rows w;
    if constexpr (MOE) {
        if (!expert_rows<16 * MF>(a, blockIdx.y, w)) return;     // the whole workgroup
    } else {
        w = Rows{0, (int)blockIdx.y * 16 * MF, min(16 * MF, a.M - (int)blockIdx.y * 16 * MF)};
    }
    const int col = lane & 15, kq = lane >> 4;
    const uint16_t *xp[MF];
    bool here[MF];
#pragma unroll
    for (int f = 0; f < MF; ++f) {
        int in, out;
        row_of<MOE>(a, w, 16 * f + col, in, out);
        here[f] = in >= 0;
        xp[f] = a.x + (here[f] ? in * a.ldx : 0) + 32 * kq;
    }
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
    v4f acc[CB][MF];
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int f = 0; f < MF; ++f) acc[c][f] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    for (int s = wave; s < a.words; s += kWaves) {               // 256 values of K
        uint32_t sc[CB];
#pragma unroll
        for (int c = 0; c < CB; ++c) sc[c] = *(const uint32_t *)(scales[c] + (int64_t)s * 256);
#pragma unroll
        for (int h = 0; h < 2; ++h) {                            // 128 of them
            const int k = 256 * s + 128 * h;
            if (k >= a.K) break;
            const bool inside = k + 32 * kq < a.K;
            v4i cw[CB], xf[MF][4];
#pragma unroll
            for (int c = 0; c < CB; ++c) cw[c] = *(const v4i *)(codes[c] + (int64_t)(4 * s + 2 * h) * 1024);
#pragma unroll
            for (int f = 0; f < MF; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    xf[f][i] = v4i{0, 0, 0, 0};
                    if (here[f] && inside) xf[f][i] = *(const v4i *)(xp[f] + k + 8 * i);
                }
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                const float scale = scale_of(sc[c] >> (8 * (kq >> 1)), 2 * h);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const v4i wf = elements8<BF16>((uint32_t)cw[c][i], scale);
#pragma unroll
                    for (int f = 0; f < MF; ++f) acc[c][f] = mfma16x16x32_h<BF16>(wf, xf[f][i], acc[c][f]);
                }
            }
        }
    }
    v4f *part = (v4f *)lds;                                      // [waves][CB][MF][64]
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int f = 0; f < MF; ++f) part[((wave * CB + c) * MF + f) * 64 + lane] = acc[c][f];
    __syncthreads();
    const int ncols = GATED ? a.N / 2 : a.N;
    constexpr int OUT = GATED ? CB / 2 : CB;
    for (int o = wave; o < OUT * MF; o += kWaves) {
        const int c = o / MF * (GATED ? 2 : 1), f = o % MF;
        v4f y = part[(c * MF + f) * 64 + lane], u;
#pragma unroll
        for (int v = 1; v < kWaves; ++v) y += part[((v * CB + c) * MF + f) * 64 + lane];
        int in, out;
        row_of<MOE>(a, w, 16 * f + col, in, out);
        int n = 0;
#pragma unroll
        for (int q = 0; q < CB; ++q) n = q == c ? 16 * row16[q] + 4 * kq : n;
        if (out < 0 || n >= ncols) continue;
        y += bias4(a, w.e, n);
        if constexpr (GATED) {
            u = part[((c + 1) * MF + f) * 64 + lane];
#pragma unroll
            for (int v = 1; v < kWaves; ++v) u += part[((v * CB + c + 1) * MF + f) * 64 + lane];
            u += bias4(a, w.e, n + a.N / 2);
#pragma unroll
            for (int q = 0; q < 4; ++q) y[q] = gated(y[q], u[q]);
        }
        if constexpr (MOE) {
            if (a.topk_weights) y *= a.topk_weights[out];
        }
        store4<BF16>(a, out, n, ncols, y);
    }
}

template <bool BF16, bool MOE, bool GATED>
int32_t launch_rows(const ProductArgs &a, hipStream_t stream) {
    constexpr int CB = 2;
    const int per = GATED ? CB / 2 : CB;
    const int blocks = ((GATED ? a.N / 2 : a.N) + 16 * per - 1) / (16 * per);
#define BK_W4_ROWS(MF)                                                                                               \
    {                                                                                                                \
        const int64_t slots = MOE ? (a.size_m + 16 * MF - 1) / (16 * MF) + std::min(a.E, a.size_m)                   \
                                  : (a.M + 16 * MF - 1) / (16 * MF);                                                 \
        hipLaunchKernelGGL((rows_kernel<BF16, MOE, GATED, MF, CB>), dim3((unsigned)blocks, (unsigned)slots),          \
                           dim3(64 * kWaves), (size_t)kWaves * CB * MF * 1024, stream, a);                           \
    }
    const int rows = MOE ? a.size_m / a.E : a.M;
    if (rows <= 16) BK_W4_ROWS(1) else BK_W4_ROWS(4)
#undef BK_W4_ROWS
    return launch_status();
}

template <bool MOE>
int32_t launch(const ProductArgs &a, int element, bool gated, hipStream_t stream) {
    if (element == kv4::kBf16) return gated ? launch_rows<true, MOE, true>(a, stream) : launch_rows<true, MOE, false>(a, stream);
    return gated ? launch_rows<false, MOE, true>(a, stream) : launch_rows<false, MOE, false>(a, stream);
}

int32_t product_ok(int32_t n, int32_t k, int32_t element, int32_t gated) {
    if (n < 1 || k < 1) return kInvalid;
    if ((element != kv4::kF16 && element != kv4::kBf16) || k % kGroup || (gated && n % 64)) return kUnsupported;
    if (n > (1 << 24) || k > (1 << 22)) return kUnsupported;
    return kOk;
}

void sizes(ProductArgs &a, int32_t n, int32_t k) {
    a.N = n, a.K = k, a.tiles = tiles(k), a.words = scale_words(k), a.matrix = matrix_bytes(n, k);
}

}  // namespace
}  // namespace w4
}  // namespace bk

using namespace bk;
using namespace bk::w4;

extern "C" {

int32_t baracuda_kernels_w4_linear_gfx950_can_implement(int32_t m, int32_t n, int32_t k, int32_t element, int32_t gated) {
    if (m < 0) return kInvalid;
    if (m > (1 << 20)) return kUnsupported;
    return product_ok(n, k, element, gated);
}

size_t baracuda_kernels_w4_linear_gfx950_workspace_size(int32_t m, int32_t n, int32_t k, int32_t element, int32_t gated) {
    (void)m; (void)n; (void)k; (void)element; (void)gated;
    return 0;
}

int32_t baracuda_kernels_w4_linear_gfx950_run(int32_t m, int32_t n, int32_t k, int32_t element, int32_t gated, const void *x,
                                              int64_t ldx, const void *packed, const float *bias, void *out, int64_t ldo,
                                              void *workspace, size_t workspace_bytes, void *stream) {
    (void)workspace; (void)workspace_bytes;
    const int32_t st = baracuda_kernels_w4_linear_gfx950_can_implement(m, n, k, element, gated);
    if (st != kOk || m == 0) return st;
    if (!x || !packed || !out || (m > 1 && (ldx < 0 || ldo < (gated ? n / 2 : n)))) return kInvalid;
    if ((uintptr_t)x % 16 || (uintptr_t)packed % 16 || (m > 1 && ldx % 8) || (uintptr_t)out % 2 || (uintptr_t)bias % 4)
        return kMisaligned;
    ProductArgs a{};
    a.x = (const uint16_t *)x, a.w = (const uint8_t *)packed, a.bias = bias, a.out = (uint16_t *)out;
    a.ldx = m > 1 ? ldx : 0, a.ldo = m > 1 ? ldo : 0, a.M = m;
    sizes(a, n, k);
    return launch<false>(a, element, gated != 0, (hipStream_t)stream);
}

int32_t baracuda_kernels_moe_w4_grouped_gfx950_can_implement(int32_t num_experts, int32_t topk, int32_t size_m, int32_t n,
                                                             int32_t k, int32_t element, int32_t gated) {
    if (num_experts < 1 || topk < 1 || size_m < 0 || topk > num_experts) return kInvalid;
    if (num_experts > kMaxExperts || size_m > (1 << 20)) return kUnsupported;
    return product_ok(n, k, element, gated);
}

size_t baracuda_kernels_moe_w4_grouped_gfx950_workspace_size(int32_t num_experts, int32_t topk, int32_t size_m, int32_t n,
                                                             int32_t k, int32_t element, int32_t gated) {
    (void)num_experts; (void)topk; (void)size_m; (void)n; (void)k; (void)element; (void)gated;
    return 0;
}

int32_t baracuda_kernels_moe_w4_grouped_gfx950_run(
    int32_t num_experts, int32_t topk, int32_t size_m, int32_t n, int32_t k, int32_t element, int32_t gated, const void *x,
    const void *packed, const int32_t *sorted_token_ids, const int32_t *expert_ids, const float *topk_weights,
    const float *bias, void *out, int32_t *expert_counts, int32_t *expert_offsets, void *workspace, size_t workspace_bytes,
    void *stream) {
    (void)workspace; (void)workspace_bytes;
    const int32_t st = baracuda_kernels_moe_w4_grouped_gfx950_can_implement(num_experts, topk, size_m, n, k, element, gated);
    if (st != kOk || size_m == 0) return st;
    if (!x || !packed || !sorted_token_ids || !expert_ids || !out || !expert_counts || !expert_offsets) return kInvalid;
    if ((uintptr_t)x % 16 || (uintptr_t)packed % 16 || (uintptr_t)out % 2) return kMisaligned;
    ProductArgs a{};
    a.x = (const uint16_t *)x, a.w = (const uint8_t *)packed, a.bias = bias, a.out = (uint16_t *)out;
    a.ldx = k, a.ldo = gated ? n / 2 : n;
    a.order = sorted_token_ids, a.offsets = expert_offsets, a.topk_weights = topk_weights;
    a.E = num_experts, a.size_m = size_m, a.in_div = topk_weights ? 1 : topk;
    sizes(a, n, k);
    hipLaunchKernelGGL(moe_offsets_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, expert_ids, size_m, num_experts,
                       expert_counts, expert_offsets);
    if (hipPeekAtLastError() != hipSuccess) return kLaunch;
    return launch<true>(a, element, gated != 0, (hipStream_t)stream);
}

}  // extern "C"
