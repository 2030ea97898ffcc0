// w4.hpp -- matrices of 4-bit weights under group scales, as the products read
// them.
//
// A weight is code * 2^(byte - 127): a code is sign, two exponent bits and one
// mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6: the OCP E2M1 values), a byte is shared
// by the 32 consecutive weights of a group (the OCP E8M0 scale; 255 marks a group
// that held an infinity or a NaN and reads as NaN).  A matrix [N, K] lies as
//   codes   [ceil(N / 32)][tiles][64][16]    tiles = 2 ceil(K / 128)
//   scales  [ceil(N / 32)][ceil(K / 256)][64][4]
// bytes.  Lane l of a tile is row l % 32 of its block of rows and group l / 32 of
// the tile's two, 16 bytes with the lower index in the lower four bits; byte j of
// a lane's four scales is that of tile 4 s + j.  Past N or K codes are 0 and scale bytes
// 2.  (The products multiply weights by zeros of x there, also those of other tiles under
// such a byte, so that it has to leave them finite: 0 does as well, 255 does not.)
// So a tile is one kilobyte that a wave reads in one piece, 16 bytes a lane, and
// what a lane gets are the words of the matrix operands that it supplies: row l %
// 32 and eight values of K a word for the 32x32x16 product, or, from two tiles,
// row l % 16 and a quarter of 128 values for the 16x16x32 one.
#pragma once

#include "kv4.hpp"

namespace bk {
namespace w4 {

constexpr int kRows = 32, kGroup = 32, kTile = 64;     // rows of a block; weights of a group, of a tile's row

__host__ __device__ inline int64_t row_blocks(int64_t n) { return (n + kRows - 1) / kRows; }
__host__ __device__ inline int tiles(int k) { return (k + 127) / 128 * 2; }
__host__ __device__ inline int scale_words(int k) { return (k + 255) / 256; }
__host__ __device__ inline int64_t code_bytes(int64_t n, int k) { return row_blocks(n) * tiles(k) * 1024; }
__host__ __device__ inline int64_t matrix_bytes(int64_t n, int k) {
    return code_bytes(n, k) + row_blocks(n) * scale_words(k) * 256;
}

// Eight weights of a word as elements, the scale with them.  Exact where the
// element's type holds the weight: bf16 always but at the ends of its exponent
// range, f16 for scales of 2^-23 to 2^13 (else rounded to it).
template <bool BF16>
__device__ __forceinline__ v4i elements8(uint32_t w, float scale) {
    v4i r;
    if constexpr (BF16) {
        r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
        r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
        r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
        r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    } else {
        r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0));
        r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1));
        r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2));
        r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
    }
    return r;
}

// The scale of byte j of a word of four, in the exponent field that the
// conversions read.
__device__ __forceinline__ float scale_of(uint32_t four, int j) {
    return __uint_as_float(((four >> (8 * j)) & 0xffu) << 23);
}

}  // namespace w4
}  // namespace bk
