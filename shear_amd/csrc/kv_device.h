// kv_device.h -- device helpers of the attention kernels over the paged
// key-value cache: 16-bit element types on the matrix instructions, exchanges
// between the 16- and 32-lane groups of a wave, the table lookup.
#pragma once

#include <type_traits>
#include <utility>

#include "kv_kernels.h"

namespace tessa {

using kv_f4 = float __attribute__((ext_vector_type(4)));
using kv_f16 = float __attribute__((ext_vector_type(16)));
using kv_u4 = uint32_t __attribute__((ext_vector_type(4)));
using kv_u2 = uint32_t __attribute__((ext_vector_type(2)));

// A running maximum before any visible row: above no finite logit, and
// exp2(-inf - kKvNone) is 0 where exp2(-inf - -inf) would be NaN.
constexpr float kKvNone = -3.402823466e38f;
// Weights are exp2(logit - m) with m near the running maximum, which m follows only now and
// then, so that almost no tile pays for rescaling the output: it is set 2^kv_lift below
// the largest weight and stays until one (prompts of 16-bit rows: a tile's sum of them) passes
// 2^kv_top.  bf16 has f32's range and weights of at most 1 keep the sums of the largest
// values finite; fp16 has its range above 1 as well as below it, and uses all of it.
constexpr float kv_lift(bool half, bool prompt) { return half ? (prompt ? 9.0f : 7.0f) : (prompt ? -15.0f : -8.0f); }
constexpr float kv_top(bool half) { return half ? 15.0f : 0.0f; }

template <typename T>
struct KvElem;

template <>
struct KvElem<__bf16> {
    using v8 = __bf16 __attribute__((ext_vector_type(8)));
    using v2 = __bf16 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ kv_f4 mma16(kv_u4 a, kv_u4 b, kv_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ kv_f16 mma32(kv_u4 a, kv_u4 b, kv_f16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const v2 x = {(__bf16)lo, (__bf16)hi};
        return __builtin_bit_cast(uint32_t, x);
    }
    static __device__ __forceinline__ float low(uint32_t x) { return __uint_as_float(x << 16); }
    static __device__ __forceinline__ float high(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
    // two whole numbers of at most 8 bits: their bf16 is the upper half of the f32
    static __device__ __forceinline__ uint32_t pack_codes(float lo, float hi) {
        return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
    }
    static constexpr uint32_t kExponent = 0x7f80u;  // all ones: infinity or NaN
    // two 4-bit codes (byte kByte of x) times the power of two `scale`: exact unless below 2^-126
    template <int kByte>
    static __device__ __forceinline__ uint32_t from_mx4(uint32_t x, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, kByte));
    }
    // byte kByte of old: two values over `scale`, rounded to the nearest codes, ties to the even one, at most 6
    template <int kByte>
    static __device__ __forceinline__ uint32_t to_mx4(uint32_t old, uint32_t x, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(v2, x), scale, kByte);
    }
};

template <>
struct KvElem<_Float16> {
    using v8 = _Float16 __attribute__((ext_vector_type(8)));
    using v2 = _Float16 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ kv_f4 mma16(kv_u4 a, kv_u4 b, kv_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ kv_f16 mma32(kv_u4 a, kv_u4 b, kv_f16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const v2 x = {(_Float16)lo, (_Float16)hi};
        return __builtin_bit_cast(uint32_t, x);
    }
    static __device__ __forceinline__ float low(uint32_t x) { return (float)__builtin_bit_cast(v2, x)[0]; }
    static __device__ __forceinline__ float high(uint32_t x) { return (float)__builtin_bit_cast(v2, x)[1]; }
    static __device__ __forceinline__ uint32_t pack_codes(float lo, float hi) { return pack(lo, hi); }
    static constexpr uint32_t kExponent = 0x7c00u;
    template <int kByte>
    static __device__ __forceinline__ uint32_t from_mx4(uint32_t x, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, scale, kByte));
    }
    template <int kByte>
    static __device__ __forceinline__ uint32_t to_mx4(uint32_t old, uint32_t x, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(v2, x), scale, kByte);
    }
};

// byte e of x as a signed code
__device__ __forceinline__ float kv_code(uint32_t x, int e) { return (float)(int8_t)(x >> (8 * e)); }

// 4-bit rows: 32 dims share a scale 2^(byte - 127); 255 says that one of them is not finite.  As
// the exponent of an f32 the byte is what the conversions want, 255 (an infinity) included: they make it NaN.
constexpr uint32_t kMxGroup = 32;
constexpr uint32_t kMxNan = 255;
__device__ __forceinline__ float kv_mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes as values.
template <typename T>
__device__ __forceinline__ kv_u4 kv_mx_values(uint32_t codes, float scale) {
    using E = KvElem<T>;
    return kv_u4{E::template from_mx4<0>(codes, scale), E::template from_mx4<1>(codes, scale), E::template from_mx4<2>(codes, scale),
                 E::template from_mx4<3>(codes, scale)};
}

__device__ __forceinline__ float kv_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// log of the sum of exp from m and the sum of weights, which is near 2^lift: two numbers of the result's size are added
__device__ __forceinline__ float kv_lse(float m, float sum, float lift) {
    return sum == 0.0f ? -INFINITY : ((m + lift) + log2f(sum * kv_exp2(-lift))) * 0.69314718056f;
}

// max / sum of x over the lanes that differ in bit 5, in bits 4 and 5
__device__ __forceinline__ float kv_max32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float kv_sum32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float kv_max16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return kv_max32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float kv_sum16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return kv_sum32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Infinities and NaN among the values: p * inf is an infinity, but a weight too small for its type
// gives 0 * inf and parts of different sign inf - inf.  A sum that has become NaN
// under weights that are numbers is formed again from such values alone, whose sum s the
// finite ones cannot change; 0 says that there was none.
__device__ __forceinline__ float kv_not_finite(float x) { return fabsf(x) < INFINITY ? 0.0f : x; }
__device__ __forceinline__ float kv_settled(float sum, float s) { return s == 0.0f ? sum : s; }
__device__ __forceinline__ kv_f4 kv_not_finite(kv_f4 x) {
    return kv_f4{kv_not_finite(x[0]), kv_not_finite(x[1]), kv_not_finite(x[2]), kv_not_finite(x[3])};
}
__device__ __forceinline__ kv_f4 kv_settled(kv_f4 x, kv_f4 s) {
    return kv_f4{kv_settled(x[0], s[0]), kv_settled(x[1], s[1]), kv_settled(x[2], s[2]), kv_settled(x[3], s[3])};
}
__device__ __forceinline__ bool kv_nan(kv_f4 x) { return !(x[0] == x[0] && x[1] == x[1] && x[2] == x[2] && x[3] == x[3]); }

// Orders a wave's LDS writes before its own later reads by other lanes.
__device__ __forceinline__ void kv_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Rows of sequence b: its length, clipped to what the tables can hold.
__device__ __forceinline__ uint32_t kv_length(const KvCacheParams &c, uint32_t b) {
    const int32_t n = c.lengths[b];
    return n <= 0 ? 0u : min((uint32_t)n, c.max_length);
}

// Place of a row in 16-byte units (without the head), or kKvNoOffset where the
// table names no page of the cache.
__device__ __forceinline__ uint32_t kv_place(const KvCacheParams &c, const KvArray &a, int32_t page, uint32_t row) {
    if ((uint32_t)page >= c.pages) return kKvNoOffset;
    return (uint32_t)page * a.page_units + (row & ((1u << c.page_shift) - 1u)) * a.row_units;
}

__device__ __forceinline__ uint64_t kv_scale_place(const KvCacheParams &c, const KvArray &a, int32_t page, uint32_t row,
                                                   uint32_t head) {
    return (uint64_t)(uint32_t)page * a.scale_page + (uint64_t)head * a.scale_head +
           (uint64_t)(row & ((1u << c.page_shift) - 1u)) * a.scale_row;
}

__device__ __forceinline__ float *kv_row_scales(const KvArray &a) { return static_cast<float *>(a.scales); }
__device__ __forceinline__ uint8_t *kv_group_scales(const KvArray &a) { return static_cast<uint8_t *>(a.scales); }

// f(integral_constant i) for i below kCount, in order: for builtins that want constants.
template <typename F, int... i>
__device__ __forceinline__ void kv_each_of(F &&f, std::integer_sequence<int, i...>) {
    (f(std::integral_constant<int, i>{}), ...);
}
template <int kCount, typename F>
__device__ __forceinline__ void kv_each(F &&f) {
    kv_each_of(f, std::make_integer_sequence<int, kCount>{});
}

// The visible rows of a single token: [0, first), [last_begin, length) and the
// listed ones strictly between; index i of [0, count) names one of them.
struct KvVisible {
    uint32_t first, last_begin, before_list, count;
};

__device__ __forceinline__ KvVisible kv_visible(const KvAttendParams &p, uint32_t length) {
    KvVisible v;
    if (p.window == 0xffffffffu) {
        v.first = 0;
        v.last_begin = 0;
    } else {
        v.first = min(p.sinks, length);
        v.last_begin = max(v.first, length > p.window ? length - p.window : 0u);
    }
    v.before_list = v.first + (length - v.last_begin);
    v.count = v.before_list + (length ? p.listed_count : 0u);
    return v;
}

}  // namespace tessa
