// kv_rotate.hip -- new tokens on their way into the cache: queries and keys are
// normalized by head, turned by their position, and keys and values written to
// their places.
//
//   y = x * rsqrt(mean x^2 + eps) * w
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * frequency_i
// for each pair i of dims, (i, i + r/2) or (2i, 2i + 1).  The angle is formed in 64 bits, in turns: of a
// position of 10^6 f32 keeps 4 bits of a turn's fraction less than of 10^5, so it keeps none of what the
// sine needs.  Norm and rotation are in f32 and the result is rounded to the tokens' type once; an SQ8 or
// MX4 row is made of the rounded values, so that it is what append makes of them.
#include "kv_quantize.h"

namespace tessa {

namespace {

constexpr int kThreads = 256;
constexpr int kFlight = 2;  // rows of a lane in flight

// Sum over the 2^lanes_log2 lanes of a row.
__device__ __forceinline__ float row_sum(float x, uint32_t lanes_log2) {
    for (uint32_t off = 1; off < (1u << lanes_log2); off <<= 1) x += __shfl_xor(x, (int)off);
    return x;
}

template <typename T>
__device__ __forceinline__ void load_weights(const void *w, bool wide, uint32_t dim, float (&to)[8]) {
    if (wide) {
        const float *at = static_cast<const float *>(w) + dim;
#pragma unroll
        for (int e = 0; e < 8; ++e) to[e] = at[e];
    } else {
        const kv_u4 x = *reinterpret_cast<const kv_u4 *>(static_cast<const char *>(w) + 2u * dim);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            to[2 * e] = KvElem<T>::low(x[e]);
            to[2 * e + 1] = KvElem<T>::high(x[e]);
        }
    }
}

// A workgroup takes `here` tokens, or one of `parts` parts of a token's rows; 2^lanes_log2 lanes a row, 8 dims each.
template <typename T, int kRows>
__global__ __launch_bounds__(kThreads) void kv_rotate_kernel(KvRotateParams p, uint32_t lanes_log2, uint32_t here, uint32_t parts) {
    using E = KvElem<T>;
    extern __shared__ __align__(16) float2 sh_turn[];  // [here][half]: cosine, sine
    const KvCacheParams &c = p.c;
    const uint32_t t = threadIdx.x, part = blockIdx.x % parts;
    const uint64_t first = (uint64_t)(blockIdx.x / parts) * here;
    const uint32_t n = (uint32_t)min((uint64_t)here, p.tokens - first), rows = p.q_heads + 2u * c.heads;
    for (uint32_t i = t; i < n * p.half; i += kThreads) {
        const uint32_t token = i / p.half;
        const double turns = (double)p.positions[first + token] * (p.frequencies[i - token * p.half] * 0.15915494309189533577);
        float s, k;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &k);
        sh_turn[i] = float2{k, s};
    }
    __syncthreads();
    const uint32_t lane = t & ((1u << lanes_log2) - 1u), own = t >> lanes_log2, per = kThreads >> lanes_log2;
    const uint32_t d = 8u * lane;
    const bool inside = d < c.dim;
    // the lane's pairs: in halves its partner has the other dim of each
    const bool turned = inside && d < 2u * p.half, second = d >= p.half;
    const uint32_t step = p.half / 8u;
    const uint32_t partner = turned && !p.interleaved ? (second ? lane - step : lane + step) : lane;
    const uint32_t pair = p.interleaved ? d / 2u : second ? d - p.half : d;
    float wq[8], wk[8], pq[8], pk[8];  // weights of the lane's dims and of its partner's
#pragma unroll
    for (int e = 0; e < 8; ++e) wq[e] = wk[e] = pq[e] = pk[e] = 1.0f;
    if (p.q_weight && inside) {
        load_weights<T>(p.q_weight, p.wide_weights, d, wq);
        load_weights<T>(p.q_weight, p.wide_weights, 8u * partner, pq);
    }
    if (p.k_weight && inside) {
        load_weights<T>(p.k_weight, p.wide_weights, d, wk);
        load_weights<T>(p.k_weight, p.wide_weights, 8u * partner, pk);
    }
    const uint32_t begin = n * rows * part / parts, end = n * rows * (part + 1u) / parts;
    for (uint32_t r0 = begin; r0 < end; r0 += kFlight * per) {
        kv_u4 x[kFlight];
        uint32_t token[kFlight], row[kFlight];
        int32_t position[kFlight];
        int64_t slot[kFlight];
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            const uint32_t r = r0 + (uint32_t)j * per + own;
            token[j] = min(r, end - 1u) / rows;
            row[j] = min(r, end - 1u) - token[j] * rows;
            const uint64_t at = first + token[j];
            position[j] = p.positions[at];
            slot[j] = p.slots[at];
            const char *src = row[j] < p.q_heads ? p.q + at * p.q_token + (uint64_t)row[j] * p.q_head
                              : row[j] < p.q_heads + c.heads
                                  ? p.k + at * p.k_token + (uint64_t)(row[j] - p.q_heads) * p.k_head
                                  : p.v + at * p.v_token + (uint64_t)(row[j] - p.q_heads - c.heads) * p.v_head;
            x[j] = kv_u4{0, 0, 0, 0};
            if (inside) x[j] = *reinterpret_cast<const kv_u4 *>(src + 2u * d);
        }
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            const uint32_t r = r0 + (uint32_t)j * per + own;
            const bool ok = r < end, is_q = row[j] < p.q_heads, is_k = !is_q && row[j] < p.q_heads + c.heads;
            float y[8];
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[2 * e] = E::low(x[j][e]);
                y[2 * e + 1] = E::high(x[j][e]);
                sum = fmaf(y[2 * e], y[2 * e], sum);
                sum = fmaf(y[2 * e + 1], y[2 * e + 1], sum);
            }
            sum = row_sum(sum, lanes_log2);
            const bool norm = is_q ? p.q_weight != nullptr : p.k_weight != nullptr;
            const float f = norm ? rsqrtf(sum / (float)c.dim + p.eps) : 1.0f;
            kv_u4 other;  // the partner's values
#pragma unroll
            for (int e = 0; e < 4; ++e) other[e] = (uint32_t)__shfl((int)x[j][e], (int)((t & 63u) - lane + partner));
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = y[e] * f * (is_q ? wq[e] : wk[e]);
            if (turned) {
                const float2 *turn = sh_turn + token[j] * p.half + pair;
                if (p.interleaved) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float2 cs = turn[e / 2];
                        const float a = y[e], b = y[e + 1];
                        y[e] = a * cs.x - b * cs.y;
                        y[e + 1] = a * cs.y + b * cs.x;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 cs = turn[e];
                        const float z = (e & 1 ? E::high(other[e / 2]) : E::low(other[e / 2])) * f * (is_q ? pq[e] : pk[e]);
                        y[e] = second ? z * cs.y + y[e] * cs.x : y[e] * cs.x - z * cs.y;
                    }
                }
            }
            kv_u4 out = x[j];  // values as they are
            if (is_q || is_k) {
#pragma unroll
                for (int e = 0; e < 4; ++e) out[e] = E::pack(y[2 * e], y[2 * e + 1]);
            }
            const bool real = position[j] >= 0;
            if (is_q) {
                char *to = p.out + (first + token[j]) * p.out_token + (uint64_t)row[j] * p.out_head;
                if (ok && inside) *reinterpret_cast<kv_u4 *>(to + 2u * d) = real ? out : kv_u4{0, 0, 0, 0};
            } else {
                const KvArray &a = is_k ? c.keys : c.values;
                const uint32_t head = row[j] - p.q_heads - (is_k ? 0u : c.heads);
                const uint64_t page = (uint64_t)slot[j] >> c.page_shift;
                const bool mine = ok && inside && real && page < c.pages;
                const int32_t id = mine ? (int32_t)page : 0;
                const uint32_t at = (uint32_t)slot[j];
                kv_store_row<T, kRows>(a, (uint64_t)kv_place(c, a, id, at) + (uint64_t)head * a.head_units,
                                       kv_scale_place(c, a, id, at, head), out, lane, lanes_log2, mine);
            }
        }
    }
}

template <typename T>
int launch_rows(const KvRotateParams &p, KvRows rows, uint32_t blocks, size_t lds, uint32_t lanes_log2, uint32_t here, uint32_t parts,
                hipStream_t stream) {
    switch (rows) {
        case kRowsPlain: kv_rotate_kernel<T, kRowsPlain><<<blocks, kThreads, lds, stream>>>(p, lanes_log2, here, parts); break;
        case kRowsSq8: kv_rotate_kernel<T, kRowsSq8><<<blocks, kThreads, lds, stream>>>(p, lanes_log2, here, parts); break;
        default: kv_rotate_kernel<T, kRowsMx4><<<blocks, kThreads, lds, stream>>>(p, lanes_log2, here, parts);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace

int launch_kv_rotate(const KvRotateParams &p, uint32_t source, KvRows rows, hipStream_t stream) {
    if (p.tokens == 0) return 0;
    uint32_t lanes_log2 = 1;
    while ((8u << lanes_log2) < p.c.dim) ++lanes_log2;
    const uint32_t threads = (p.q_heads + 2u * p.c.heads) << lanes_log2;  // of a token
    const uint32_t here = threads < (uint32_t)kThreads ? (uint32_t)kThreads / threads : 1u;
    const uint64_t groups = (p.tokens + here - 1) / here;
    // few tokens: their rows are shared out until the compute units have two workgroups each
    uint32_t parts = 1;
    while (here == 1u && parts * kThreads < threads && groups * parts < 2u * (uint64_t)kv_compute_units()) ++parts;
    const size_t lds = (size_t)here * p.half * sizeof(float2);
    const uint32_t blocks = (uint32_t)(groups * parts);
    return source == kKvBf16 ? launch_rows<__bf16>(p, rows, blocks, lds, lanes_log2, here, parts, stream)
                             : launch_rows<_Float16>(p, rows, blocks, lds, lanes_log2, here, parts, stream);
}

}  // namespace tessa
