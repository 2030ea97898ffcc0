// w4_weights.hip -- weights into 4 bits under group scales, laid out as the
// products read them (w4.hpp), and back.
//
// All three kernels move pieces of 32 rows by 256 columns (four tiles and a word
// of scales a lane, 4352 bytes) through LDS: on the matrix's side a wave touches
// whole rows of 256 columns, on the packed side the piece's 4 KiB of codes are
// contiguous.  Nothing is computed but the group's largest magnitude and the
// hardware's conversions, so the float side's bytes bound them: 8 x 14336 x 4096 f32
// weights (1.9 GB) quantized in 413 us, 5.2 TB/s, read back in 475, 4.5; a large copy
// moves 5.0.  bf16 4096 x 4096: 8.5 and 8.0 us.
#include "w4.hpp"

namespace bk {
namespace w4 {
namespace {

using kv4::Bf16;
using kv4::F16;
using kv4::Raw;

constexpr int kThreads = 256;

struct WeightArgs {
    int64_t n, pieces;              // rows of a matrix; 32 x 256 pieces of all matrices
    int k, words, tiles, most;      // most: kv4::scale_byte
    int64_t blocks, matrix;         // row blocks and bytes of a matrix
    int64_t matrix_stride, row_stride;
    uint8_t *packed;
};

struct Piece {
    int64_t row0, matrix;           // first row, which matrix
    int word;                       // which 256 columns
    uint8_t *codes, *scales;        // its 4 KiB and 256 bytes
};

__device__ __forceinline__ Piece piece_of(const WeightArgs &a, int64_t i) {
    Piece p;
    p.word = (int)(i % a.words);
    const int64_t b = i / a.words, block = b % a.blocks;
    p.matrix = b / a.blocks;
    p.row0 = block * kRows;
    uint8_t *m = a.packed + p.matrix * a.matrix;
    p.codes = m + (block * a.tiles + 4 * p.word) * 1024;
    p.scales = m + a.blocks * a.tiles * 1024 + (block * a.words + p.word) * 256;
    return p;
}

// Place of group g (of eight) of row r in the piece: tile and lane.
__device__ __forceinline__ int lane_of(int r, int g) { return (g >> 1) * 64 + (g & 1) * 32 + r; }

// The piece in LDS to its place.  The last tiles of a matrix may be two.
__device__ __forceinline__ void put_piece(const WeightArgs &a, const Piece &p, const v4i *codes, const uint32_t *scales) {
    const int t = threadIdx.x;
    if (4 * p.word + t / 64 < a.tiles) *(v4i *)(p.codes + 16 * t) = codes[t];
    if (t < 64) *(uint32_t *)(p.scales + 4 * t) = scales[t];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const WeightArgs a, const void *__restrict__ w) {
    typedef typename Raw<T>::Mem Mem;
    constexpr int SIZE = sizeof(Mem) / 8;
    __shared__ v4i codes[256];
    __shared__ uint32_t scales[64];
    const int t = threadIdx.x, r0 = t / 32, u = t % 32;      // 32 lanes a row, eight values each
    for (int64_t i = blockIdx.x; i < a.pieces; i += gridDim.x) {
        const Piece p = piece_of(a, i);
        const int k = 256 * p.word + 8 * u;
        Mem raw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t row = p.row0 + r0 + 8 * j;
            raw[j] = Mem{};
            if (row < a.n && k < a.k)
                raw[j] = *(const Mem *)((const char *)w + (p.matrix * a.matrix_stride + row * a.row_stride + k) * SIZE);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float x[8];
            uint32_t top = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                x[q] = Raw<T>::get(raw[j], q);
                top = max(top, __float_as_uint(x[q]) & 0x7fffffffu);
            }
            // four lanes a group
            top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));
            top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));
            const bool good = top < 0x7f800000u;
            const int byte = good ? kv4::scale_byte(top, a.most) : 255;
            const int lane = lane_of(r0 + 8 * j, u / 4);
            ((uint32_t *)codes)[4 * lane + u % 4] = good ? kv4::encode8(x, byte) : 0u;
            if (u % 4 == 0) ((uint8_t *)scales)[4 * (lane % 64) + lane / 64] = (uint8_t)byte;
        }
        __syncthreads();
        put_piece(a, p, codes, scales);
        __syncthreads();
    }
}

struct __attribute__((packed, aligned(1))) Group {
    v4i w;
};

__global__ __launch_bounds__(kThreads) void pack_kernel(const WeightArgs a, const uint8_t *__restrict__ codes,
                                                        const uint8_t *__restrict__ scales) {
    __shared__ v4i lds[256];
    __shared__ uint32_t lds_s[64];
    const int t = threadIdx.x, r = t / 8, g = t % 8, groups = a.k / kGroup;
    for (int64_t i = blockIdx.x; i < a.pieces; i += gridDim.x) {
        const Piece p = piece_of(a, i);
        const int64_t at = (p.matrix * a.n + p.row0 + r) * groups + 8 * p.word + g;
        const bool here = p.row0 + r < a.n && 8 * p.word + g < groups;
        const int lane = lane_of(r, g);
        lds[lane] = here ? ((const Group *)(codes + 16 * at))->w : v4i{0, 0, 0, 0};
        ((uint8_t *)lds_s)[4 * (lane % 64) + lane / 64] = here ? scales[at] : 2;
        __syncthreads();
        put_piece(a, p, lds, lds_s);
        __syncthreads();
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void read_kernel(const WeightArgs a, void *__restrict__ out) {
    typedef typename Raw<T>::Mem Mem;
    constexpr int SIZE = sizeof(Mem) / 8;
    __shared__ v4i codes[256];
    __shared__ uint32_t scales[64];
    const int t = threadIdx.x, r0 = t / 32, u = t % 32;
    for (int64_t i = blockIdx.x; i < a.pieces; i += gridDim.x) {
        const Piece p = piece_of(a, i);
        if (4 * p.word + t / 64 < a.tiles) codes[t] = *(const v4i *)(p.codes + 16 * t);
        if (t < 64) scales[t] = *(const uint32_t *)(p.scales + 4 * t);
        __syncthreads();
        const int k = 256 * p.word + 8 * u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t row = p.row0 + r0 + 8 * j;
            if (row < a.n && k < a.k) {
                const int lane = lane_of(r0 + 8 * j, u / 4);
                float x[8];
                kv4::decode8(((const uint32_t *)codes)[4 * lane + u % 4], ((const uint8_t *)scales)[4 * (lane % 64) + lane / 64],
                             x);
                Mem m;
                Raw<T>::put(m, x);
                *(Mem *)((char *)out + (p.matrix * a.matrix_stride + row * a.row_stride + k) * SIZE) = m;
            }
        }
        __syncthreads();
    }
}

int32_t weights_ok(int32_t matrices, int32_t n, int32_t k, int32_t element) {
    if (matrices < 0 || n < 1 || k < 1) return kInvalid;
    if (element < kv4::kF32 || element > kv4::kBf16 || k % kGroup) return kUnsupported;
    if ((int64_t)matrices * row_blocks(n) > INT32_MAX / 4 || n > INT32_MAX - 64 || k > INT32_MAX - 512) return kUnsupported;
    return kOk;
}

WeightArgs weight_args(int32_t matrices, int32_t n, int32_t k, int32_t element, void *packed) {
    WeightArgs a{};
    a.n = n, a.k = k, a.words = scale_words(k), a.tiles = tiles(k);
    a.blocks = row_blocks(n), a.matrix = matrix_bytes(n, k);
    a.pieces = (int64_t)matrices * a.blocks * a.words;
    a.most = element == kv4::kF16 ? 13 : 125;
    a.packed = (uint8_t *)packed;
    return a;
}

// At most this many workgroups walk the pieces.
dim3 grid_of(const WeightArgs &a) { return dim3((unsigned)(a.pieces < 16384 ? a.pieces : 16384)); }

// Rows of an output that share elements, whichever of the two strides is the wider.
bool overlap(int64_t matrices, int64_t n, int64_t k, int64_t matrix_stride, int64_t row_stride) {
    const bool rows_first = (n == 1 || row_stride >= k) && (matrices == 1 || matrix_stride >= (n - 1) * row_stride + k);
    const bool matrices_first =
        (matrices == 1 || matrix_stride >= k) && (n == 1 || row_stride >= (matrices - 1) * matrix_stride + k);
    return !rows_first && !matrices_first;
}

}  // namespace
}  // namespace w4
}  // namespace bk

using namespace bk;
using namespace bk::w4;

extern "C" {

size_t baracuda_kernels_w4_packed_bytes_gfx950(int32_t n, int32_t k) {
    return n < 1 || k < 1 || k > INT32_MAX - 512 ? 0 : (size_t)matrix_bytes(n, k);
}

int32_t baracuda_kernels_w4_weights_gfx950_can_implement(int32_t matrices, int32_t n, int32_t k, int32_t element) {
    return weights_ok(matrices, n, k, element);
}

int32_t baracuda_kernels_w4_quantize_gfx950_run(int32_t matrices, int32_t n, int32_t k, int32_t element, const void *weights,
                                                int64_t matrix_stride, int64_t row_stride, void *packed, void *stream) {
    const int32_t st = weights_ok(matrices, n, k, element);
    if (st != kOk || matrices == 0) return st;
    if (!weights || !packed) return kInvalid;
    if ((uintptr_t)packed % 16 || (uintptr_t)weights % (element == kv4::kF32 ? 4 : 2)) return kMisaligned;
    WeightArgs a = weight_args(matrices, n, k, element, packed);
    a.matrix_stride = matrix_stride, a.row_stride = row_stride;
    const auto s = (hipStream_t)stream;
    if (element == kv4::kF32) hipLaunchKernelGGL(quantize_kernel<float>, grid_of(a), dim3(kThreads), 0, s, a, weights);
    else if (element == kv4::kF16) hipLaunchKernelGGL(quantize_kernel<F16>, grid_of(a), dim3(kThreads), 0, s, a, weights);
    else hipLaunchKernelGGL(quantize_kernel<Bf16>, grid_of(a), dim3(kThreads), 0, s, a, weights);
    return launch_status();
}

int32_t baracuda_kernels_w4_pack_gfx950_run(int32_t matrices, int32_t n, int32_t k, const void *codes, const void *scales,
                                            void *packed, void *stream) {
    const int32_t st = weights_ok(matrices, n, k, kv4::kBf16);
    if (st != kOk || matrices == 0) return st;
    if (!codes || !scales || !packed) return kInvalid;
    if ((uintptr_t)packed % 16) return kMisaligned;
    const WeightArgs a = weight_args(matrices, n, k, kv4::kBf16, packed);
    hipLaunchKernelGGL(pack_kernel, grid_of(a), dim3(kThreads), 0, (hipStream_t)stream, a, (const uint8_t *)codes,
                       (const uint8_t *)scales);
    return launch_status();
}

int32_t baracuda_kernels_w4_read_gfx950_run(int32_t matrices, int32_t n, int32_t k, int32_t element, const void *packed,
                                            void *weights, int64_t matrix_stride, int64_t row_stride, void *stream) {
    const int32_t st = weights_ok(matrices, n, k, element);
    if (st != kOk || matrices == 0) return st;
    if (!weights || !packed || overlap(matrices, n, k, matrix_stride, row_stride)) return kInvalid;
    if ((uintptr_t)packed % 16 || (uintptr_t)weights % (element == kv4::kF32 ? 4 : 2)) return kMisaligned;
    WeightArgs a = weight_args(matrices, n, k, element, const_cast<void *>(packed));
    a.matrix_stride = matrix_stride, a.row_stride = row_stride;
    const auto s = (hipStream_t)stream;
    if (element == kv4::kF32) hipLaunchKernelGGL(read_kernel<float>, grid_of(a), dim3(kThreads), 0, s, a, weights);
    else if (element == kv4::kF16) hipLaunchKernelGGL(read_kernel<F16>, grid_of(a), dim3(kThreads), 0, s, a, weights);
    else hipLaunchKernelGGL(read_kernel<Bf16>, grid_of(a), dim3(kThreads), 0, s, a, weights);
    return launch_status();
}

}  // extern "C"
