// kv_read.hip -- rows of the cache by place, as values: 2^k lanes take a (slot, head) row, 8 dims each.
// Codes become values on the way: SQ8 code * scale in f32, MX4 code * 2^e exactly
// (bf16 and f32 hold every one); each is rounded to the output's type once.
#include "kv_device.h"

namespace tessa {

namespace {

constexpr int kThreads = 256;
constexpr int kFlight = 4;  // rows of a lane in flight

struct Codes {  // what a lane loads of a row
    kv_u4 x;
    float scale;
};

// Out: float, __bf16 or _Float16.  T: a plain row's type.
template <typename Out>
__device__ __forceinline__ void put(char *to, const float (&f)[8]) {
    if constexpr (sizeof(Out) == 4) {
        reinterpret_cast<kv_f4 *>(to)[0] = kv_f4{f[0], f[1], f[2], f[3]};
        reinterpret_cast<kv_f4 *>(to)[1] = kv_f4{f[4], f[5], f[6], f[7]};
    } else {
        using E = KvElem<Out>;
        *reinterpret_cast<kv_u4 *>(to) = kv_u4{E::pack(f[0], f[1]), E::pack(f[2], f[3]), E::pack(f[4], f[5]), E::pack(f[6], f[7])};
    }
}

template <typename T, int kRows, typename Out>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvReadParams p, uint32_t lanes_log2) {
    const KvCacheParams &c = p.c;
    const KvArray &a = blockIdx.y ? c.values : c.keys;
    char *out = blockIdx.y ? p.v : p.k;
    const uint32_t lane = threadIdx.x & ((1u << lanes_log2) - 1u), d = 8u * lane, per = kThreads >> lanes_log2;
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
    Codes x[kFlight];
    bool there[kFlight];
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
        const uint64_t page = (uint64_t)slot[j] >> c.page_shift;
        there[j] = page < c.pages;
        const int32_t id = there[j] ? (int32_t)page : 0;  // row 0 of page 0 is there to read
        const uint32_t at = there[j] ? (uint32_t)slot[j] : 0u;
        const char *src = a.rows + ((uint64_t)kv_place(c, a, id, at) + (uint64_t)head[j] * a.head_units) * 16u;
        x[j].scale = 1.0f;
        if constexpr (kRows == kRowsPlain) {
            x[j].x = *reinterpret_cast<const kv_u4 *>(src + 2u * d);
        } else if constexpr (kRows == kRowsSq8) {
            const kv_u2 y = *reinterpret_cast<const kv_u2 *>(src + d);
            x[j].x = kv_u4{y[0], y[1], 0, 0};
            x[j].scale = kv_row_scales(a)[kv_scale_place(c, a, id, at, head[j])];
        } else {
            x[j].x = kv_u4{*reinterpret_cast<const uint32_t *>(src + d / 2u), 0, 0, 0};
            x[j].scale = kv_mx_scale(kv_group_scales(a)[kv_scale_place(c, a, id, at, head[j]) + d / kMxGroup]);
        }
    }
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
        const uint32_t r = first + (uint32_t)j * per;
        if (r >= rows) return;
        char *to = out + ((uint64_t)r * c.dim + d) * sizeof(Out);
        if constexpr (kRows == kRowsMx4 && sizeof(Out) == 2) {
            const kv_u4 y = kv_mx_values<Out>(x[j].x[0], x[j].scale);
            *reinterpret_cast<kv_u4 *>(to) = there[j] ? y : kv_u4{0, 0, 0, 0};
        } else {
            float f[8];
            if constexpr (kRows == kRowsMx4) {
                kv_each<4>([&](auto e) {
                    const auto y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x[j].x[0], x[j].scale, decltype(e)::value);
                    f[2 * e] = y[0];
                    f[2 * e + 1] = y[1];
                });
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (kRows == kRowsSq8)
                        f[e] = kv_code(x[j].x[e / 4], e & 3) * x[j].scale;
                    else
                        f[e] = e & 1 ? KvElem<T>::high(x[j].x[e / 2]) : KvElem<T>::low(x[j].x[e / 2]);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = there[j] ? f[e] : 0.0f;
            put<Out>(to, f);
        }
    }
}

template <typename T, int kRows>
int launch(const KvReadParams &p, uint32_t type, hipStream_t stream) {
    uint32_t lanes_log2 = 1;
    while ((8u << lanes_log2) < p.c.dim) ++lanes_log2;
    const uint32_t per = ((uint32_t)kThreads >> lanes_log2) * kFlight, rows = (uint32_t)p.count * p.c.heads;
    const dim3 grid((rows + per - 1u) / per, p.v ? 2u : 1u);
    if (type == kKvBf16)
        kv_read_kernel<T, kRows, __bf16><<<grid, kThreads, 0, stream>>>(p, lanes_log2);
    else if (type == kKvF16)
        kv_read_kernel<T, kRows, _Float16><<<grid, kThreads, 0, stream>>>(p, lanes_log2);
    else
        kv_read_kernel<T, kRows, float><<<grid, kThreads, 0, stream>>>(p, lanes_log2);
    return hipGetLastError() == hipSuccess ? 0 : -1;
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
