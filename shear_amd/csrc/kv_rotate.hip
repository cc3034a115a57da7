// kv_rotate.hip -- new tokens on their way into the cache: queries and keys are
// normalized by head, turned by their position, and keys and values written to
// their places.
//
//   y = x * rsqrt(mean x^2 + eps) * w
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * frequency_i
// for each pair i of dims, (i, i + r/2) or (2i, 2i + 1).  The angle is formed in 64 bits, in turns, and only its
// fraction becomes an f32: a position of 10^6 in f32 would leave the sine 4 bits of it.  Norm and rotation are in
// f32 and the result is rounded to the tokens' type once; an SQ8 or MX4 row is made of the rounded values, so that
// it is what append makes of them.
//
// Weight and rotation are two factors a dim, y_d = f (x_d w_d cos + x_p (-+ w_p sin)), p the other dim of the pair,
// formed once for a token in LDS.  A lane has 8 dims of a row, 16 bytes; its pairs' other dims lie in
// another lane (halves) or its own (neighbours).
//
// Bound by its bytes: 12,001 tokens of 32 + 2 * 8 heads of 128 dims (295 MB) take 53 us, 5.6 TB/s, four tokens a workgroup, the
// next one's rows on their way while one is worked on.  48 tokens take 4.7 us, a launch and a chain of reads.
#include "kv_quantize.h"

namespace tessa {

namespace {

constexpr int kThreads = 256;
constexpr int kFlight = 3;  // rows of a lane in flight
constexpr uint32_t kMostPasses = 4;
constexpr uint32_t kFullCard = 5;  // workgroups that a compute unit holds

// Where the other dim of a pair lies: beside it, in a lane `half / 8` away, or in the other half of the row's lanes.
enum { kNeighbours = 0, kHalves = 1, kWholeHalves = 2 };

template <int kControl>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kControl, 0xf, 0xf, true);
}
template <int kControl>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(dpp<kControl>(__float_as_uint(x)));
}

// Sum over the 2^kLog2 neighbouring lanes of a row: exchanges in pairs and quads, mirrors of 8 and 16.
template <int kLog2>
__device__ __forceinline__ float row_sum(float x) {
    x += dpp<0xb1>(x);
    x += dpp<0x4e>(x);
    x += dpp<0x141>(x);
    if constexpr (kLog2 >= 4) x += dpp<0x140>(x);
    if constexpr (kLog2 >= 5) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return x;
}

// x of the lane in the other half of a row's lanes.
template <int kLog2>
__device__ __forceinline__ uint32_t other_half(uint32_t x) {
    if constexpr (kLog2 == 3) {  // from 4 lanes on, and in the second and fourth 4 of 16 from 4 lanes back
        const uint32_t up = dpp<0x104>(x);
        return (uint32_t)__builtin_amdgcn_update_dpp((int)up, (int)x, 0x114, 0xf, 0xa, false);
    } else if constexpr (kLog2 == 4) {
        return dpp<0x128>(x);
    } else {
        return (uint32_t)__shfl_xor((int)x, 16);
    }
}

// A workgroup takes `passes` times `here` tokens, one after the other, or one of `parts` parts of a token's rows;
// 2^kLog2 lanes a row.
template <typename T, int kRows, int kLog2, int kPairs>
__global__ __launch_bounds__(kThreads) void kv_rotate_kernel(KvRotateParams p, uint32_t here, uint32_t passes, uint32_t parts) {
    using E = KvElem<T>;
    constexpr uint32_t kLanes = 1u << kLog2, kPer = kThreads >> kLog2, kDims = 8u * kLanes;
    // [passes * here][query, key][4 pieces of 2 dims][lane][2]: of the dim, of its partner (a lane's pieces side by side would
    // meet in a quarter of the banks)
    extern __shared__ __align__(16) float2 sh_factor[];
    auto place_of = [](uint32_t dim) { return ((dim % 8u / 2u) * kLanes + dim / 8u) * 2u + (dim & 1u); };
    const KvCacheParams &c = p.c;
    const uint32_t t = threadIdx.x, group = blockIdx.x / parts, part = blockIdx.x - group * parts;
    const uint64_t first = (uint64_t)group * here * passes;
    const uint32_t n = (uint32_t)min((uint64_t)here * passes, p.tokens - first), rows = p.q_heads + 2u * c.heads;
    const uint32_t lane = t & (kLanes - 1u), own = t >> kLog2;
    // the lane's token of a pass and its rows of it: row, row + kPer, .. below end
    const uint32_t mine = here > 1u ? own / rows : 0u, part_begin = rows * part / parts, part_end = rows * (part + 1u) / parts;
    const uint32_t begin = here > 1u ? own - mine * rows : part_begin + own;
    const uint32_t end = here == 1u ? part_end : mine < here ? begin + 1u : 0u;
    const uint32_t chunks = here > 1u ? 1u : (part_end - part_begin + kFlight * kPer - 1u) / (kFlight * kPer);
    const uint32_t items = (n + here - 1u) / here * chunks;
    const uint32_t d = 8u * lane;
    const bool inside = d < c.dim;
    // (copied again where they are chosen between: of two of the arguments' fields, or two variables that a lambda
    // refers to, the compiler chooses an address and loads from it, with a wait, for each row)
    const uint32_t q_head = (uint32_t)p.q_head, k_head = (uint32_t)p.k_head, v_head = (uint32_t)p.v_head, out_head = (uint32_t)p.out_head;
    const bool q_norm = p.q_weight != nullptr, k_norm = p.k_weight != nullptr;
    const uint32_t k_units = c.keys.head_units, v_units = c.values.head_units;
    char *const k_rows = c.keys.rows, *const v_rows = c.values.rows;
    struct Item {
        kv_u4 x[kFlight];
        int32_t position;
        int64_t slot;
        uint32_t token, row;  // of the workgroup's tokens; first row
    };
    auto load = [&](uint32_t i, Item &w) __attribute__((always_inline)) {
        const uint32_t pass = i / chunks, token = pass * here + mine;
        w.token = min(token, n - 1u);
        w.row = token < n ? begin + (i - pass * chunks) * kFlight * kPer : end;
        const uint64_t at = first + w.token;
        w.position = p.positions[at];
        w.slot = p.slots[at];
        const uint32_t q_bytes = q_head, k_bytes = k_head, v_bytes = v_head;
        const char *q = p.q + at * p.q_token, *k = p.k + at * p.k_token, *v = p.v + at * p.v_token;
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            const uint32_t r = w.row + (uint32_t)j * kPer;
            const bool is_q = r < p.q_heads, is_v = r >= p.q_heads + c.heads;
            const uint32_t head = is_q ? r : r - p.q_heads - (is_v ? c.heads : 0u);
            const char *src = (is_q ? q : is_v ? v : k) + (uint64_t)head * (is_q ? q_bytes : is_v ? v_bytes : k_bytes);
            w.x[j] = kv_u4{0, 0, 0, 0};
            if (r < end && inside) w.x[j] = *reinterpret_cast<const kv_u4 *>(src + 2u * d);
        }
    };
    Item even, odd;
    load(0, even);  // on their way while the factors are formed
    const bool wide_weights = p.wide_weights;
    auto weight = [=](const void *w, uint32_t i) {
        if (!w) return 1.0f;
        return wide_weights ? static_cast<const float *>(w)[i] : E::low(static_cast<const uint16_t *>(w)[i]);
    };
    for (uint32_t i = t; i < n * p.half; i += kThreads) {  // a pair of a token
        const uint32_t k = i / p.half, pair = i - k * p.half;
        const uint32_t da = kPairs == kNeighbours ? 2u * pair : pair, db = kPairs == kNeighbours ? da + 1u : da + p.half;
        const double turns = (double)p.positions[first + k] * (p.frequencies[pair] * 0.15915494309189533577);
        float sine, cosine;
        sincospif(2.0f * (float)(turns - rint(turns)), &sine, &cosine);
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            const void *w = kind ? p.k_weight : p.q_weight;
            const float wa = weight(w, da), wb = weight(w, db);
            float2 *f = sh_factor + (2u * k + kind) * kDims;
            f[place_of(da)] = float2{wa * cosine, -(wb * sine)};
            f[place_of(db)] = float2{wb * cosine, wa * sine};
        }
    }
    // dims that do not turn, and those of the lanes past the row: an SQ8 row's scale is made of all its lanes, so these must be
    // zeros and not what an earlier kernel left here
    const uint32_t still = kDims - 2u * p.half;
    for (uint32_t i = t; i < n * still; i += kThreads) {
        const uint32_t k = i / still, at = 2u * p.half + i - k * still;
#pragma unroll
        for (int kind = 0; kind < 2; ++kind)
            sh_factor[(2u * k + kind) * kDims + place_of(at)] =
                float2{at < c.dim ? weight(kind ? p.k_weight : p.q_weight, at) : 0.0f, 0.0f};
    }
    __syncthreads();
    const bool turned = inside && d < 2u * p.half;
    const uint32_t step = p.half / 8u;
    const uint32_t partner = (t & 63u) + (!turned ? 0u : d >= p.half ? 0u - step : step);  // (kHalves)
    const float inverse = 1.0f / (float)c.dim;
    auto work = [&](Item &w) __attribute__((always_inline)) {
        const uint64_t at = first + w.token, page = (uint64_t)w.slot >> c.page_shift;
        const bool real = w.position >= 0, there = real && page < c.pages;
        const int32_t id = there ? (int32_t)page : 0;
        const uint32_t ku = k_units, vu = v_units;
        char *const kr = k_rows, *const vr = v_rows;
        const uint32_t k_place = kv_place(c, c.keys, id, (uint32_t)w.slot), v_place = kv_place(c, c.values, id, (uint32_t)w.slot);
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            const uint32_t r = w.row + (uint32_t)j * kPer;
            const bool is_q = r < p.q_heads, is_k = !is_q && r < p.q_heads + c.heads;
            const kv_u4 x = w.x[j];
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float lo = E::low(x[e]), hi = E::high(x[e]);
                sum = fmaf(hi, hi, fmaf(lo, lo, sum));
            }
            const bool norm = (is_q && q_norm) || (!is_q && k_norm);
            const float scale = norm ? rsqrtf(fmaf(row_sum<kLog2>(sum), inverse, p.eps)) : 1.0f;
            const kv_f4 *f = reinterpret_cast<const kv_f4 *>(sh_factor + (2u * w.token + (is_q ? 0u : 1u)) * kDims) + lane;
            kv_u4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t other;
                if constexpr (kPairs == kNeighbours)
                    other = __builtin_amdgcn_alignbit(x[e], x[e], 16);
                else if constexpr (kPairs == kWholeHalves)
                    other = other_half<kLog2>(x[e]);
                else
                    other = (uint32_t)__shfl((int)x[e], (int)partner);
                if constexpr (kPairs != kWholeHalves) other = turned ? other : 0u;  // (0 * infinity would be NaN)
                const kv_f4 g = f[e * kLanes];  // of two dims
                const float lo = fmaf(E::low(other), g[1], E::low(x[e]) * g[0]);
                const float hi = fmaf(E::high(other), g[3], E::high(x[e]) * g[2]);
                y[e] = E::pack(lo * scale, hi * scale);
            }
            const uint32_t head = r - p.q_heads - (is_k ? 0u : c.heads);
            const uint64_t place = (uint64_t)(is_k ? k_place : v_place) + (uint64_t)head * (is_k ? ku : vu);
            const bool mine_too = r < end && inside;
            if constexpr (kRows == kRowsPlain) {
                char *to = is_q ? p.out + at * p.out_token + (uint64_t)r * out_head : (is_k ? kr : vr) + place * 16u;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = is_q ? (real ? y[e] : 0u) : is_k ? y[e] : x[e];
                if (mine_too && (is_q || there)) *reinterpret_cast<kv_u4 *>(to + 2u * d) = y;
            } else if (is_q) {
                if (mine_too)
                    *reinterpret_cast<kv_u4 *>(p.out + at * p.out_token + (uint64_t)r * out_head + 2u * d) =
                        real ? y : kv_u4{0, 0, 0, 0};
            } else {
                if (is_k)
                    kv_store_row<T, kRows>(c.keys, place, kv_scale_place(c, c.keys, id, (uint32_t)w.slot, head), y, lane, kLog2,
                                           mine_too && there);
                else
                    kv_store_row<T, kRows>(c.values, place, kv_scale_place(c, c.values, id, (uint32_t)w.slot, head), x, lane, kLog2,
                                           mine_too && there);
            }
        }
    };
    for (uint32_t i = 0; i < items; i += 2) {
        if (i + 1 < items) load(i + 1, odd);
        work(even);
        if (i + 1 >= items) break;
        if (i + 2 < items) load(i + 2, even);
        work(odd);
    }
}

struct Split {
    uint32_t blocks, here, passes, parts;
    hipStream_t stream;
};

template <typename T, int kRows, int kLog2>
int launch_pairs(const KvRotateParams &p, const Split &s) {
    const size_t lds = (size_t)s.here * s.passes * 2u * (8u << kLog2) * sizeof(float2);
    if (p.interleaved || p.half == 0u)
        kv_rotate_kernel<T, kRows, kLog2, kNeighbours><<<s.blocks, kThreads, lds, s.stream>>>(p, s.here, s.passes, s.parts);
    else if (p.half == 4u << kLog2)
        kv_rotate_kernel<T, kRows, kLog2, kWholeHalves><<<s.blocks, kThreads, lds, s.stream>>>(p, s.here, s.passes, s.parts);
    else
        kv_rotate_kernel<T, kRows, kLog2, kHalves><<<s.blocks, kThreads, lds, s.stream>>>(p, s.here, s.passes, s.parts);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <typename T, int kRows>
int launch_lanes(const KvRotateParams &p, uint32_t lanes_log2, const Split &s) {
    switch (lanes_log2) {
        case 3: return launch_pairs<T, kRows, 3>(p, s);
        case 4: return launch_pairs<T, kRows, 4>(p, s);
        default: return launch_pairs<T, kRows, 5>(p, s);
    }
}

template <typename T>
int launch_rows(const KvRotateParams &p, KvRows rows, uint32_t lanes_log2, const Split &s) {
    switch (rows) {
        case kRowsPlain: return launch_lanes<T, kRowsPlain>(p, lanes_log2, s);
        case kRowsSq8: return launch_lanes<T, kRowsSq8>(p, lanes_log2, s);
        default: return launch_lanes<T, kRowsMx4>(p, lanes_log2, s);
    }
}

}  // namespace

int launch_kv_rotate(const KvRotateParams &p, uint32_t source, KvRows rows, hipStream_t stream) {
    if (p.tokens == 0) return 0;
    uint32_t lanes_log2 = 3;
    while ((8u << lanes_log2) < p.c.dim) ++lanes_log2;
    const uint32_t threads = (p.q_heads + 2u * p.c.heads) << lanes_log2;  // of a token
    Split s{0, threads < (uint32_t)kThreads ? (uint32_t)kThreads / threads : 1u, 1, 1, stream};
    // many tokens: one after the other, so that the next one's rows come while one is worked on
    while (s.passes < kMostPasses && p.tokens > (uint64_t)kFullCard * kv_compute_units() * s.here * s.passes) s.passes *= 2;
    const uint64_t groups = (p.tokens + s.here * s.passes - 1) / (s.here * s.passes);
    // few tokens: their rows are shared out until the compute units have two workgroups each
    while (s.here == 1u && s.parts * kThreads < threads && groups * s.parts < 2u * (uint64_t)kv_compute_units()) ++s.parts;
    s.blocks = (uint32_t)(groups * s.parts);
    return source == kKvBf16 ? launch_rows<__bf16>(p, rows, lanes_log2, s) : launch_rows<_Float16>(p, rows, lanes_log2, s);
}

}  // namespace tessa
