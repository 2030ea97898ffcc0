// w4_product.hip -- the entry points of the products with 4-bit weights.
#include "gemm_mfma2.hpp"
#include "moe_offsets.hpp"
#include "w4_product.hpp"

namespace bk {
namespace w4 {
namespace {

int32_t product_ok(int32_t n, int32_t k, int32_t element, int32_t gated) {
    if (n < 1 || k < 1) return kInvalid;
    if ((element != kv4::kF16 && element != kv4::kBf16) || k % kGroup || (gated && n % 64)) return kUnsupported;
    if (n > (1 << 24) || k > (1 << 22) || (int64_t)n * k > (1ll << 36)) return kUnsupported;
    return kOk;
}

// A launch's workgroups of the largest tiles.
bool too_many(int64_t rows, int32_t experts, int32_t n) {
    return most_tile_rows(rows, experts, 256) * ((n + 255) / 256) > kMaxTiles;
}

// Byte offsets of x within a tile, or of all rows that pairs name, fit 31 bits.
bool extent_ok(int64_t rows, int64_t ld, int32_t k) { return ((rows - 1) * ld + k) * 2 < mfma2::kPastExtent; }

// Rows of x that pairs name, in_div pairs a row.
int64_t x_rows(int32_t size_m, int32_t in_div) { return ((int64_t)size_m + in_div - 1) / in_div; }

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
    const int32_t st = product_ok(n, k, element, gated);
    return st == kOk && (m > (1 << 20) || too_many(m, 0, n)) ? kUnsupported : st;
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
    if (m > 1 && (ldx > INT32_MAX || !extent_ok(256, ldx, k))) return kUnsupported;
    ProductArgs a{};
    a.x = (const uint16_t *)x, a.w = (const uint8_t *)packed, a.bias = bias, a.out = (uint16_t *)out;
    a.ldx = m > 1 ? ldx : 0, a.ldo = m > 1 ? ldo : 0, a.M = a.size_m = m;
    sizes(a, n, k);
    const bool bf16 = element == kv4::kBf16;
    return rows_pay(m, n) ? launch_rows(a, bf16, false, gated != 0, (hipStream_t)stream)
                          : launch_tiles(a, bf16, false, gated != 0, (hipStream_t)stream);
}

int32_t baracuda_kernels_moe_w4_grouped_gfx950_can_implement(int32_t num_experts, int32_t topk, int32_t size_m, int32_t n,
                                                             int32_t k, int32_t element, int32_t gated) {
    if (num_experts < 1 || topk < 1 || size_m < 0 || topk > num_experts) return kInvalid;
    const int32_t st = product_ok(n, k, element, gated);
    if (st != kOk) return st;
    if (num_experts > kMaxExperts || size_m > (1 << 20) || too_many(size_m, num_experts, n)) return kUnsupported;
    // with router weights x has a row for each pair, which `run` alone can tell
    if (size_m > 0 && !extent_ok(x_rows(size_m, topk), k, k)) return kUnsupported;
    return kOk;
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
    if (st != kOk) return st;
    if (!expert_counts || !expert_offsets) return kInvalid;
    if (size_m == 0) {      // no pair, but the counts are filled
        hipLaunchKernelGGL(moe_offsets_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, nullptr, 0, num_experts, expert_counts,
                           expert_offsets);
        return launch_status();
    }
    if (!x || !packed || !sorted_token_ids || !expert_ids || !out) return kInvalid;
    if ((uintptr_t)x % 16 || (uintptr_t)packed % 16 || (uintptr_t)out % 2 || (uintptr_t)bias % 4 || (uintptr_t)topk_weights % 4)
        return kMisaligned;
    const int32_t in_div = topk_weights ? 1 : topk;
    if (!extent_ok(x_rows(size_m, in_div), k, k)) return kUnsupported;
    ProductArgs a{};
    a.x = (const uint16_t *)x, a.w = (const uint8_t *)packed, a.bias = bias, a.out = (uint16_t *)out;
    a.ldx = k, a.ldo = gated ? n / 2 : n;
    const bool rows = moe_rows_pay(size_m, num_experts, n), few = size_m <= kFewPairs, bf16 = element == kv4::kBf16;
    a.order = sorted_token_ids, a.expert_ids = expert_ids, a.topk_weights = topk_weights;
    a.offsets = few ? nullptr : expert_offsets, a.counts_out = expert_counts, a.offsets_out = expert_offsets;
    a.E = num_experts, a.size_m = size_m, a.in_div = in_div;
    sizes(a, n, k);
    if (!few) {
        hipLaunchKernelGGL(moe_offsets_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, expert_ids, size_m, num_experts,
                           expert_counts, expert_offsets);
        if (hipPeekAtLastError() != hipSuccess) return kLaunch;
    }
    return rows ? launch_rows(a, bf16, true, gated != 0, (hipStream_t)stream)
                : launch_tiles(a, bf16, true, gated != 0, (hipStream_t)stream);
}

}  // extern "C"
