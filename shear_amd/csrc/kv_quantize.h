// kv_quantize.h -- 16-bit rows as the cache's codes, for the kernels that write
// new rows (kv_append.hip, kv_rotate.hip).  A row lies in 2^k neighbouring lanes,
// 8 values each.
#pragma once

#include "kv_device.h"

namespace tessa {

// Rows whose largest magnitude has at least these bits (2^-63) are divided by way of one
// reciprocal: x * (1/scale), corrected once by its remainder (Markstein's method),
// is the rounded quotient for every pair of 11-bit significands of the maximum and
// of x (tests/test_kv_quotient.py goes through all of them; powers of two change
// nothing in this range), at half the instructions: with a division each, an append
// of 4 prompts of up to 4,096 tokens, 8 heads of 128, took 27 us, so 21.
constexpr uint32_t kQuickTop = 0x20000000u;

// A lane's 8 values as SQ8: the codes, and the row's scale (a row of 2^lanes_log2 lanes).
template <typename T>
__device__ __forceinline__ kv_u2 quantize_row(kv_u4 x, uint32_t lanes_log2, float &scale) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[2 * e] = KvElem<T>::low(x[e]);
        f[2 * e + 1] = KvElem<T>::high(x[e]);
    }
    // the largest magnitude's bits as an integer: infinities and NaN are larger than every finite one
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
    for (uint32_t off = 1; off < (1u << lanes_log2); off <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, (int)off));
    const bool finite = top < 0x7f800000u;
    scale = __uint_as_float(top) * (1.0f / 127.0f);
    const bool zero = !finite || scale == 0.0f;  // a row of zeros, or of values whose scale is below f32's smallest
    if (zero) scale = 1.0f;
    uint32_t w[2] = {0, 0};
    if (__all(top == 0 || (top >= kQuickTop && finite))) {
        const float inverse = __fdiv_rn(1.0f, scale);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float q = f[e] * inverse;
            q = fmaf(fmaf(-q, scale, f[e]), inverse, q);
            const int code = (int)(q + copysignf(0.49999997f, q));  // half away: 0.5 less its last place
            w[e / 4] |= (uint32_t)(uint8_t)code << (8 * (e & 3));
        }
    } else if (!zero) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float q = fminf(fmaxf(roundf(__fdiv_rn(f[e], scale)), -127.0f), 127.0f);
            w[e / 4] |= (uint32_t)(uint8_t)(int8_t)(int)q << (8 * (e & 3));
        }
    }
    if (!finite) scale = __uint_as_float(0x7fc00000u);
    return kv_u2{w[0], w[1]};
}

// A lane's 8 values as 4-bit codes (one sign, two exponent, one fraction bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), and
// the scale byte of its group of 32 dims, 4 lanes.  The scale is the power of two that puts the
// largest magnitude between 3.5 and 7, which rounds to at most 6: one that left
// 7 to 8 to saturate would be off by up to a quarter of the value.  Its byte is held in 2..252: below, values are rounded
// to multiples of 2^-126 (bf16's smallest normal number, which attention reads), above, 4 * scale would be infinite.
template <typename T>
__device__ __forceinline__ uint32_t quantize_mx4(kv_u4 x, uint32_t &byte) {
    using E = KvElem<T>;
    // magnitudes as integers: infinities and NaN are larger than every finite one
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        top = max(max(top, __float_as_uint(E::low(x[e])) & 0x7fffffffu), __float_as_uint(E::high(x[e])) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    const bool finite = top < 0x7f800000u;
    // the exponent, one more from a significand of 1.75 on
    byte = (uint32_t)min(max((int)((top + 0x200000u) >> 23) - 2, 2), 252);
    const float scale = kv_mx_scale(byte);
    uint32_t codes = E::template to_mx4<0>(0u, x[0], scale);
    codes = E::template to_mx4<1>(codes, x[1], scale);
    codes = E::template to_mx4<2>(codes, x[2], scale);
    codes = E::template to_mx4<3>(codes, x[3], scale);
    if (!finite) byte = kMxNan;
    return finite ? codes : 0u;
}

// Writes a lane's 8 values of a row to the row's place in the cache (`place` units of 16 bytes with the head's, `scale_place` the
// place of its scales); every lane of the row takes part, those that are not `mine` write nothing.
template <typename T, int kRows>
__device__ __forceinline__ void kv_store_row(const KvArray &a, uint64_t place, uint64_t scale_place, kv_u4 x, uint32_t lane,
                                             uint32_t lanes_log2, bool mine) {
    char *to = a.rows + place * 16u;
    if constexpr (kRows == kRowsPlain) {
        if (mine) *reinterpret_cast<kv_u4 *>(to + 16u * lane) = x;
    } else if constexpr (kRows == kRowsSq8) {
        float scale;
        const kv_u2 codes = quantize_row<T>(x, lanes_log2, scale);
        if (mine) {
            *reinterpret_cast<kv_u2 *>(to + 8u * lane) = codes;
            if (lane == 0) kv_row_scales(a)[scale_place] = scale;
        }
    } else {
        uint32_t byte;
        const uint32_t codes = quantize_mx4<T>(x, byte);
        if (mine) {
            *reinterpret_cast<uint32_t *>(to + 4u * lane) = codes;
            if (lane % 4u == 0u) kv_group_scales(a)[scale_place + lane / 4u] = (uint8_t)byte;
        }
    }
}

}  // namespace tessa
