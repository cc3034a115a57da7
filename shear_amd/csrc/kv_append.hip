// kv_append.hip -- new keys and values into the pages of the cache.
//
// Token t of sequence b goes to row start_b + (t - offsets[b]) of that
// sequence: page table[b][row / page_rows], slot row % page_rows.  Into a
// cache of the tokens' own type the values are copied; into an SQ8 cache each
// (token, head) row is quantized as the package does it, symmetrically by row:
// scale = max|x| * (1/127) in f32 (1 for a row of zeros), code = x / scale rounded
// half away from zero.  The scale is within a unit in the last place of the
// quotient that the set quantizer takes; the codes are the nearest for it.  A row with a value that is not finite keeps codes of 0 and a
// scale of NaN, so that whatever attends over it gets NaN, as it would from the
// value itself.
//
// Copy-bound: 2^k lanes take one row, 16 bytes each, keys and values side by
// side in the grid; the table is read once per row.
#include "kv_device.h"

namespace tessa {

namespace {

constexpr int kThreads = 256;

// kLanes: lanes of a row (a power of two, at least dim / 8).
template <typename T, bool kSq8>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvAppendParams p, uint32_t lanes_log2) {
    const uint32_t lane = threadIdx.x & ((1u << lanes_log2) - 1u);
    const uint64_t slot = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) >> lanes_log2;
    const uint32_t b = blockIdx.y;
    const bool values = blockIdx.z != 0;
    const KvCacheParams &c = p.c;
    const uint32_t i = (uint32_t)(slot / c.heads), head = (uint32_t)(slot - (uint64_t)i * c.heads);
    int64_t t = b, n = 1;
    if (p.offsets) {
        t = p.offsets[b];
        n = (int64_t)p.offsets[b + 1] - t;
    }
    const int64_t row64 = (int64_t)c.lengths[b] + i;
    t += i;
    bool ok = (int64_t)i < n && i < p.max_new && t >= 0 && (uint64_t)t < p.tokens && row64 >= 0 && row64 < (int64_t)c.max_length;
    const uint32_t row = ok ? (uint32_t)row64 : 0u;
    const int32_t page = ok ? c.table[(uint64_t)b * c.table_stride + (row >> c.page_shift)] : -1;
    const KvArray &a = values ? c.values : c.keys;
    const uint32_t place = kv_place(c, a, page, row);
    ok = ok && place != kKvNoOffset;
    const bool mine = ok && 8u * lane < c.dim;
    kv_u4 x = {0, 0, 0, 0};
    if (mine) {
        const char *src = (values ? p.v : p.k) + (uint64_t)t * (values ? p.v_token : p.k_token) +
                          (uint64_t)head * (values ? p.v_head : p.k_head);
        x = *reinterpret_cast<const kv_u4 *>(src + 16u * lane);
    }
    char *dst = a.rows + ((uint64_t)place + (uint64_t)head * a.head_units) * 16u;
    if constexpr (!kSq8) {
        if (mine) *reinterpret_cast<kv_u4 *>(dst + 16u * lane) = x;
    } else {
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
        float scale = __uint_as_float(top) * (1.0f / 127.0f);
        const bool zero = !finite || scale == 0.0f;  // a row of zeros, or of values whose scale is below f32's smallest
        if (zero) scale = 1.0f;
        uint32_t w[2] = {0, 0};
        if (!zero) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = fminf(fmaxf(roundf(__fdiv_rn(f[e], scale)), -127.0f), 127.0f);
                w[e / 4] |= (uint32_t)(uint8_t)(int8_t)(int)q << (8 * (e & 3));
            }
        }
        if (mine) {
            const kv_u2 codes = {w[0], w[1]};
            *reinterpret_cast<kv_u2 *>(dst + 8u * lane) = codes;
            if (lane == 0) a.scales[kv_scale_place(c, a, page, row, head)] = finite ? scale : __uint_as_float(0x7fc00000u);
        }
    }
}

}  // namespace

int launch_kv_append(const KvAppendParams &p, uint32_t source, bool sq8, hipStream_t stream) {
    if (p.c.batch == 0 || p.max_new == 0 || p.tokens == 0) return 0;
    uint32_t lanes_log2 = 1;
    while ((8u << lanes_log2) < p.c.dim) ++lanes_log2;
    const uint64_t threads = ((uint64_t)p.max_new * p.c.heads) << lanes_log2;
    const dim3 grid((uint32_t)((threads + kThreads - 1) / kThreads), p.c.batch, 2);
    if (source == kKvBf16) {
        if (sq8)
            kv_append_kernel<__bf16, true><<<grid, kThreads, 0, stream>>>(p, lanes_log2);
        else
            kv_append_kernel<__bf16, false><<<grid, kThreads, 0, stream>>>(p, lanes_log2);
    } else {
        if (sq8)
            kv_append_kernel<_Float16, true><<<grid, kThreads, 0, stream>>>(p, lanes_log2);
        else
            kv_append_kernel<_Float16, false><<<grid, kThreads, 0, stream>>>(p, lanes_log2);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tessa
