// kv_read.hip -- rows of the cache by place, as values: 2^k lanes take a (slot, head) row, 16 bytes of the output each.
// Codes become values on the way: SQ8 code * scale in f32, MX4 code * 2^e exactly
// (bf16 and f32 hold every one); each is rounded to the output's type once.
#include "kv_device.h"

namespace tessa {

namespace {

constexpr int kThreads = 256;
constexpr int kFlight = 4;  // rows of a lane in flight

// A lane's dims: 16 bytes of the output, so that a store is whole cache lines (f32 as 8 dims, two stores with gaps:
// 72 us for 60,001 x 8 rows of 128, 245 MB; as 4 dims 57, both through the caches).
template <typename Out>
constexpr int kPer = 16 / (int)sizeof(Out);

// Results larger than all L2 caches together do not stay there anyway, and stores that do not pass through them are
// faster (245 MB of f32 42.6 us, 6.5 TB/s, through them 57.7; 102 MB of bf16 and an append before it 27.5, 30.0).  Smaller ones are left
// to whoever reads them next.
constexpr uint64_t kStreamed = 32ull << 20;

template <bool kStream>
__device__ __forceinline__ void put(char *to, kv_u4 x) {
    if constexpr (kStream)
        __builtin_nontemporal_store(x, reinterpret_cast<kv_u4 *>(to));
    else
        *reinterpret_cast<kv_u4 *>(to) = x;
}

// T: a plain row's type.  Out: float, __bf16 or _Float16.
template <typename T, int kRows, typename Out, bool kStream>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvReadParams p, uint32_t lanes_log2) {
    constexpr int kDims = kPer<Out>;
    constexpr int kBytes = kRows == kRowsPlain ? 2 * kDims : kRows == kRowsSq8 ? kDims : kDims / 2;  // of a lane's load
    const KvCacheParams &c = p.c;
    const KvArray &a = blockIdx.y ? c.values : c.keys;
    char *out = blockIdx.y ? p.v : p.k;
    const uint32_t lane = threadIdx.x & ((1u << lanes_log2) - 1u), d = kDims * lane, per = kThreads >> lanes_log2;
    const uint32_t rows = (uint32_t)p.count * c.heads, first = blockIdx.x * per * kFlight + (threadIdx.x >> lanes_log2);
    if (d >= c.dim) return;
    int64_t slot[kFlight];
    uint32_t head[kFlight];
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
        const uint32_t r = min(first + (uint32_t)j * per, rows - 1u), i = r / c.heads;
        head[j] = r - i * c.heads;
        slot[j] = p.slots[i];
    }
    uint32_t x[kFlight][(kBytes + 3) / 4];
    float scale[kFlight];
    bool there[kFlight];
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
        const uint64_t page = (uint64_t)slot[j] >> c.page_shift;
        there[j] = page < c.pages;
        const int32_t id = there[j] ? (int32_t)page : 0;  // row 0 of page 0 is there to read
        const uint32_t at = there[j] ? (uint32_t)slot[j] : 0u;
        const char *src = a.rows + ((uint64_t)kv_place(c, a, id, at) + (uint64_t)head[j] * a.head_units) * 16u + kBytes * lane;
        if constexpr (kBytes == 2) {
            x[j][0] = *reinterpret_cast<const uint16_t *>(src);
        } else if constexpr (kBytes == 4) {
            x[j][0] = *reinterpret_cast<const uint32_t *>(src);
        } else if constexpr (kBytes == 8) {
            const kv_u2 y = *reinterpret_cast<const kv_u2 *>(src);
            x[j][0] = y[0];
            x[j][1] = y[1];
        } else {
            const kv_u4 y = *reinterpret_cast<const kv_u4 *>(src);
#pragma unroll
            for (int w = 0; w < 4; ++w) x[j][w] = y[w];
        }
        scale[j] = 1.0f;
        if constexpr (kRows == kRowsSq8) scale[j] = kv_row_scales(a)[kv_scale_place(c, a, id, at, head[j])];
        if constexpr (kRows == kRowsMx4) scale[j] = kv_mx_scale(kv_group_scales(a)[kv_scale_place(c, a, id, at, head[j]) + d / kMxGroup]);
    }
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
        const uint32_t r = first + (uint32_t)j * per;
        if (r >= rows) return;
        char *to = out + ((uint64_t)r * c.dim + d) * sizeof(Out);
        if constexpr (kRows == kRowsMx4 && sizeof(Out) == 2) {
            const kv_u4 y = kv_mx_values<Out>(x[j][0], scale[j]);
            put<kStream>(to, there[j] ? y : kv_u4{0, 0, 0, 0});
        } else {
            float f[kDims];
            if constexpr (kRows == kRowsMx4) {
                kv_each<kDims / 2>([&](auto e) {
                    const auto y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x[j][0], scale[j], decltype(e)::value);
                    f[2 * e] = y[0];
                    f[2 * e + 1] = y[1];
                });
            } else {
#pragma unroll
                for (int e = 0; e < kDims; ++e) {
                    if constexpr (kRows == kRowsSq8)
                        f[e] = kv_code(x[j][e / 4], e & 3) * scale[j];
                    else
                        f[e] = e & 1 ? KvElem<T>::high(x[j][e / 2]) : KvElem<T>::low(x[j][e / 2]);
                }
            }
#pragma unroll
            for (int e = 0; e < kDims; ++e) f[e] = there[j] ? f[e] : 0.0f;
            if constexpr (sizeof(Out) == 4) {
                put<kStream>(to, __builtin_bit_cast(kv_u4, kv_f4{f[0], f[1], f[2], f[3]}));
            } else {
                using E = KvElem<Out>;
                put<kStream>(to, kv_u4{E::pack(f[0], f[1]), E::pack(f[2], f[3]), E::pack(f[4], f[5]), E::pack(f[6], f[7])});
            }
        }
    }
}

template <typename T, int kRows, typename Out>
int launch_out(const KvReadParams &p, hipStream_t stream) {
    uint32_t lanes_log2 = 1;
    while (((uint32_t)kPer<Out> << lanes_log2) < p.c.dim) ++lanes_log2;
    const uint32_t per = ((uint32_t)kThreads >> lanes_log2) * kFlight, rows = (uint32_t)p.count * p.c.heads;
    const dim3 grid((rows + per - 1u) / per, p.v ? 2u : 1u);
    if ((uint64_t)rows * p.c.dim * sizeof(Out) * grid.y > kStreamed)
        kv_read_kernel<T, kRows, Out, true><<<grid, kThreads, 0, stream>>>(p, lanes_log2);
    else
        kv_read_kernel<T, kRows, Out, false><<<grid, kThreads, 0, stream>>>(p, lanes_log2);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <typename T, int kRows>
int launch(const KvReadParams &p, uint32_t type, hipStream_t stream) {
    switch (type) {
        case kKvBf16: return launch_out<T, kRows, __bf16>(p, stream);
        case kKvF16: return launch_out<T, kRows, _Float16>(p, stream);
        default: return launch_out<T, kRows, float>(p, stream);
    }
}

}  // namespace

int launch_kv_read(const KvReadParams &p, uint32_t cache, uint32_t type, hipStream_t stream) {
    if (p.count == 0) return 0;
    switch (cache) {
        case kKvBf16: return launch<__bf16, kRowsPlain>(p, type, stream);
        case kKvF16: return launch<_Float16, kRowsPlain>(p, type, stream);
        case kKvSq8: return launch<__bf16, kRowsSq8>(p, type, stream);
        default: return launch<__bf16, kRowsMx4>(p, type, stream);
    }
}

}  // namespace tessa
