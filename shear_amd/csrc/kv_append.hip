// kv_append.hip -- new keys and values into the pages of the cache.
//
// Token t of sequence b goes to row start_b + (t - offsets[b]) of that
// sequence: page table[b][row / page_rows], slot row % page_rows.  Into a
// cache of the tokens' own type the values are copied; into an SQ8 cache each
// (token, head) row is quantized as the package does it, symmetrically by row:
// scale = max|x| * (1/127) in f32 (1 for a row of zeros), code = x / scale rounded
// half away from zero.  The scale is within a unit in the last place of the
// quotient that the set quantizer takes; the codes are the nearest for it.  A row
// with a value that is not finite keeps codes of 0 and a scale of NaN, so that
// whatever attends over it gets NaN, as it would from the value itself.
//
// Copy-bound: 2^k lanes take one (token, head) row of keys and of values, 16 bytes each,
// and a workgroup's rows are tokens side by side, whose rows and scales follow each
// other in a page.  4 prompts of up to 4,096 tokens, 8 heads of 128, into SQ8 (76 MB):
// 21 us (3.7 TB/s; 4 of 16,384 tokens, 405 MB, 81 us, 5.0 TB/s); two tokens a lane 23.
// One token for each of 64 sequences: 2.7 us, a launch.
#include "kv_device.h"

namespace tessa {

namespace {

constexpr int kThreads = 256;

// Rows whose largest magnitude has at least these bits (2^-63) are divided by way of one
// reciprocal: x * (1/scale), corrected once by its remainder (Markstein's method),
// is the rounded quotient for every pair of 11-bit significands of the maximum and
// of x (tests/test_kv_quotient.py goes through all of them; powers of two change
// nothing in this range), at half the instructions: with a division each the
// prompts above took 27 us.
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

template <typename T, bool kSq8>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvAppendParams p, uint32_t lanes_log2, uint32_t tokens_log2) {
    const uint32_t lane = threadIdx.x & ((1u << lanes_log2) - 1u);
    const uint32_t b = blockIdx.y;
    const KvCacheParams &c = p.c;
    int64_t first = b, n = 1;
    if (p.offsets) {
        first = p.offsets[b];
        n = (int64_t)p.offsets[b + 1] - first;
    }
    n = min(n, (int64_t)p.max_new);
    const int64_t start = c.lengths[b];
    // the workgroup's rows: 2^tokens_log2 tokens of each of some heads
    const uint32_t own = threadIdx.x >> lanes_log2, heads_here = (kThreads >> lanes_log2) >> tokens_log2;
    const uint32_t head_blocks = (c.heads + heads_here - 1) / heads_here, token_block = blockIdx.x / head_blocks;
    const uint32_t head = (blockIdx.x - token_block * head_blocks) * heads_here + (own >> tokens_log2);
    const uint32_t i = (token_block << tokens_log2) + (own & ((1u << tokens_log2) - 1u));
    const int64_t t = first + i, r = start + i;
    const bool ok = (int64_t)i < n && head < c.heads && t >= 0 && (uint64_t)t < p.tokens && r >= 0 && r < (int64_t)c.max_length;
    const uint32_t row = ok ? (uint32_t)r : 0u;
    const int32_t page = ok ? c.table[(uint64_t)b * c.table_stride + (row >> c.page_shift)] : -1;
    kv_u4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
    if (ok && 8u * lane < c.dim) {
        k = *reinterpret_cast<const kv_u4 *>(p.k + (uint64_t)t * p.k_token + (uint64_t)head * p.k_head + 16u * lane);
        v = *reinterpret_cast<const kv_u4 *>(p.v + (uint64_t)t * p.v_token + (uint64_t)head * p.v_head + 16u * lane);
    }
    const uint32_t kp = kv_place(c, c.keys, page, row), vp = kv_place(c, c.values, page, row);
    const bool mine = kp != kKvNoOffset && 8u * lane < c.dim;
    char *kd = c.keys.rows + ((uint64_t)kp + (uint64_t)head * c.keys.head_units) * 16u;
    char *vd = c.values.rows + ((uint64_t)vp + (uint64_t)head * c.values.head_units) * 16u;
    if constexpr (!kSq8) {
        if (mine) {
            *reinterpret_cast<kv_u4 *>(kd + 16u * lane) = k;
            *reinterpret_cast<kv_u4 *>(vd + 16u * lane) = v;
        }
    } else {
        float ks, vs;
        const kv_u2 kc = quantize_row<T>(k, lanes_log2, ks), vc = quantize_row<T>(v, lanes_log2, vs);
        if (mine) {
            *reinterpret_cast<kv_u2 *>(kd + 8u * lane) = kc;
            *reinterpret_cast<kv_u2 *>(vd + 8u * lane) = vc;
            if (lane == 0) {
                c.keys.scales[kv_scale_place(c, c.keys, page, row, head)] = ks;
                c.values.scales[kv_scale_place(c, c.values, page, row, head)] = vs;
            }
        }
    }
}

}  // namespace

int launch_kv_append(const KvAppendParams &p, uint32_t source, bool sq8, hipStream_t stream) {
    if (p.c.batch == 0 || p.max_new == 0 || p.tokens == 0) return 0;
    uint32_t lanes_log2 = 1;
    while ((8u << lanes_log2) < p.c.dim) ++lanes_log2;
    // tokens side by side, as their rows and scales are in a page; heads too where there are few
    const uint32_t rows = (uint32_t)kThreads >> lanes_log2;
    uint32_t tokens_log2 = 0;
    while ((1u << tokens_log2) < rows && (1u << tokens_log2) < p.max_new) ++tokens_log2;
    const uint32_t heads_here = rows >> tokens_log2;
    const uint64_t blocks = ((uint64_t)p.max_new + (1u << tokens_log2) - 1) >> tokens_log2;
    const dim3 grid((uint32_t)(blocks * ((p.c.heads + heads_here - 1) / heads_here)), p.c.batch);
    if (source == kKvBf16) {
        if (sq8)
            kv_append_kernel<__bf16, true><<<grid, kThreads, 0, stream>>>(p, lanes_log2, tokens_log2);
        else
            kv_append_kernel<__bf16, false><<<grid, kThreads, 0, stream>>>(p, lanes_log2, tokens_log2);
    } else {
        if (sq8)
            kv_append_kernel<_Float16, true><<<grid, kThreads, 0, stream>>>(p, lanes_log2, tokens_log2);
        else
            kv_append_kernel<_Float16, false><<<grid, kThreads, 0, stream>>>(p, lanes_log2, tokens_log2);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tessa
