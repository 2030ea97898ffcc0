// kv4.hpp -- a key-value cache in pages, two 4-bit codes a byte.
//
// The cache is uint8 [pages, kv heads, head bytes].  A code is sign, two
// exponent bits and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6: the OCP E2M1
// values); 32 consecutive values of a head share a scale 2^(byte - 127), byte
// 255 stands for a group that holds an infinity or a NaN and reads as NaN.
// The head bytes of a page of PS tokens and a head of D values, in order:
//   K codes   [PS][D / 2]
//   V codes   [PS / 4][16][4][D / 32]
//   K scales  [PS][D / 32]
//   V scales  [PS / 4][D / 32][4]
// K lies token after token, as the rows of a 16x16 MFMA operand read it.  V
// lies four tokens together in 16 runs of D / 16 values: lane r of a matrix
// operand whose rows are values of a head finds its run of four tokens in one
// load, and its four scales in one 32-bit word.
#pragma once

#include "bk_common.hpp"

namespace bk {
namespace kv4 {

enum Element : int { kF32 = 0, kF16 = 1, kBf16 = 2 };

__host__ __device__ inline int64_t head_bytes(int ps, int D) { return (int64_t)ps * (D + D / 16); }
__host__ __device__ inline int v_codes(int ps, int D) { return ps * D / 2; }
__host__ __device__ inline int k_scales(int ps, int D) { return ps * D; }
__host__ __device__ inline int v_scales(int ps, int D) { return ps * D + ps * D / 32; }

// Two f32 -> packed f16x2, each rounded to nearest even.
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t f32x2_to_f16x2(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, f16x2_t));
}

inline bool page_size_ok(int ps) { return ps >= 16 && ps <= 1024 && (ps & (ps - 1)) == 0; }
inline bool head_dim_ok(int D) { return D == 64 || D == 128 || D == 256; }
inline int log2i(int x) { return 31 - __builtin_clz((unsigned)x); }

// Eight values from memory of any alignment that the element has.
template <typename T>
struct Raw;
template <>
struct Raw<float> {
    struct __attribute__((packed, aligned(4))) Mem { uint32_t w[8]; };
    static __device__ __forceinline__ float get(const Mem &m, int i) { return __uint_as_float(m.w[i]); }
    static __device__ __forceinline__ void put(Mem &m, const float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m.w[i] = __float_as_uint(x[i]);
    }
    static __device__ __forceinline__ float round(float x) { return x; }
};
struct Bf16 {};
struct F16 {};
template <>
struct Raw<Bf16> {
    struct __attribute__((packed, aligned(2))) Mem { uint32_t w[4]; };
    static __device__ __forceinline__ float get(const Mem &m, int i) {
        return __uint_as_float(i & 1 ? m.w[i / 2] & 0xffff0000u : m.w[i / 2] << 16);
    }
    static __device__ __forceinline__ void put(Mem &m, const float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m.w[i] = f32x2_to_bf16x2(x[2 * i], x[2 * i + 1]);
    }
    static __device__ __forceinline__ float round(float x) { return __uint_as_float(f32x2_to_bf16x2(x, x) << 16); }
};
template <>
struct Raw<F16> {
    struct __attribute__((packed, aligned(2))) Mem { uint32_t w[4]; };
    static __device__ __forceinline__ float get(const Mem &m, int i) {
        return f16_to_f32((uint16_t)(m.w[i / 2] >> (16 * (i & 1))));
    }
    static __device__ __forceinline__ void put(Mem &m, const float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m.w[i] = f32x2_to_f16x2(x[2 * i], x[2 * i + 1]);
    }
    static __device__ __forceinline__ float round(float x) { return (float)(_Float16)x; }
};

// The scale byte of a group whose largest magnitude has the bits `top`: the
// power of two that brings it below 7, which rounds to the largest code 6.
// 2^most keeps six times the scale a number of the stored type.
__device__ __forceinline__ int scale_byte(uint32_t top, int most) {
    const int byte = (int)((top + 0x200000u) >> 23) - 2;
    return min(max(byte, 2), most + 127);
}

// Eight values to eight codes under 2^(byte - 127), nearest, ties to the even
// code (v_cvt_scalef32_pk_fp4_f32 divides by the scale's power of two).
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], int byte) {
    const float s = __uint_as_float((uint32_t)byte << 23);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
    return w;
}

// Eight values from their codes and scale byte.  The conversion reads the scale's
// exponent alone, and 255 there gives NaN.
__device__ __forceinline__ void decode8(uint32_t w, uint32_t byte, float (&x)[8]) {
    const float s = __uint_as_float(byte << 23);
    const f32x2_t p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1),
                          __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3)};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = p[i][0], x[2 * i + 1] = p[i][1];
}

}  // namespace kv4
}  // namespace bk
