// kv_token.hip -- attention of one new token for each sequence over the paged
// cache, split over the cache's rows and joined.
//
// For head h of the cache and its G query heads:
//   s_j = scale * q . k_j,  p_j = exp(s_j - m),  out = sum p_j v_j / sum p_j
// over the visible rows j, in base 2 throughout (scale * log2(e) is one factor).
// Each wave keeps a running maximum m, sum l and output O; the waves of a
// workgroup are joined through LDS, workgroups of one (sequence, head) by
// kv_finish_kernel.
//
// The rows of all sequences and heads, in units of 128, are one line that as many
// workgroups as the card holds at once share out evenly, whatever the sequences'
// lengths: each takes a contiguous range, often the end of one column of rows
// (a sequence's rows of one head) and the beginning of the next.  Part (column g,
// worker i) has place g + i, which no other part has, since along the line
// every next part is of a later column or a later worker.
//
// Every visible row is read once for up to 16 query heads, so the cache's
// bytes bound it; nothing is staged in LDS but row places.  Measured, 32 heads over 8
// of 128 dims (4 for the third), kernel and join:
//   48 sequences of up to 4,100 rows, with weights   533 MB   115 + 14 us   4.1 TB/s
//   8 of up to 40,000 SQ8 rows, with weights         522 MB   122 + 15 us   3.8 TB/s
//   one of 131,071 rows                              268 MB    52 +  7 us   4.5 TB/s
//   16, 2,016 rows each of which 1,500 are listed     49 MB    17 +  5 us   2.3 TB/s
// (a copy reaches 4.9 to 5.5 TB/s here).  The last is a chain of dependent
// reads, length, list, page, row, and then only two units a workgroup.
//  * S^T = K Q^T on 16x16x32 instructions: the K operand is 16 bytes of a row
//    per lane, straight from memory.  Query heads are the columns, so a lane
//    holds logits of one head and the maximum, sum and rescaling are its own.
//  * O^T = V^T P^T: the sum over rows may run in any order as long as both
//    operands agree, so the logits' registers are the P^T operand as they
//    stand.  V comes as whole rows (16 lanes a row, head_dim / 16 values each,
//    eight rows a lane); the operand of instruction c is value c of each of
//    the eight, one byte permute per two values.
//  * P is given to the matrix instructions as the sum of three bf16 parts (the
//    rounded value, the rounded rest and the rest of that: f32's 24 bits) or two of
//    fp16, because a single rounding of P would add an error as large as that of
//    rounding the result, and two bf16 parts 2^-18 of the sum of |p v|, which shows
//    where that cancels.  The instructions they cost are idle otherwise (the second
//    SQ8 case above 137.4 us with two parts, 138.3 with three).  fp16 has nothing between 0 and 2^-24: there the
//    largest weight lies between 2^7 and 2^15, and the rest is multiplied by
//    2^12 and summed by itself, so that a weight is right to 2^-44 of the largest and
//    many small ones beside a large one (a first row that takes the attention) add up.
//  * SQ8 rows: codes are whole numbers that both 16-bit types hold exactly.
//    The key's scale multiplies the logit, the value's the weight, after l has
//    summed it; O is formed in bf16 whatever q's type is, because the scales of
//    a cache can lie further apart than fp16 reaches (a row of zeros has scale 1).
//  * A row that the table leaves without a page, and a place of the list that
//    names no further visible row, weighs nothing; its values are replaced by zeros
//    (0 * NaN would be NaN).
#include <type_traits>

#include "kernel_attr.h"
#include "kv_device.h"

namespace tessa {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kTile = 32;  // rows of a wave's step

template <int N>
struct KvWords;  // N 32-bit words in one load
template <>
struct KvWords<1> {
    uint32_t w[1];
};
template <>
struct alignas(8) KvWords<2> {
    uint32_t w[2];
};
template <>
struct alignas(16) KvWords<4> {
    uint32_t w[4];
};
template <>
struct alignas(16) KvWords<8> {
    uint32_t w[8];
};

// Row id of visible index i < v.count, or -1 (a place of the list that names no further row).
__device__ __forceinline__ int32_t visible_row(const KvVisible &v, uint32_t i, const int32_t *list) {
    if (i < v.first) return (int32_t)i;
    if (i < v.before_list) return (int32_t)(v.last_begin + (i - v.first));
    const int32_t r = list[i - v.before_list];
    return r >= (int32_t)v.first && r < (int32_t)v.last_begin ? r : -1;
}

constexpr uint32_t kUnit = 128;  // rows: a tile for each wave

__device__ __forceinline__ uint32_t units_of(const KvAttendParams &p, uint32_t b) {
    return (kv_visible(p, kv_length(p.c, b)).count + kUnit - 1) / kUnit;
}

// The workers of a line: no more than it has units, so that all of them have some.
__device__ __forceinline__ uint32_t workers_of(const KvAttendParams &p, uint64_t total) {
    return (uint32_t)min((uint64_t)p.workers, total * p.columns);
}

// Where unit u lies on the line of `total` units: the worker that has it.
__device__ __forceinline__ uint32_t worker_of(uint64_t u, uint64_t total, uint32_t workers) {
    return (uint32_t)(((u + 1) * workers - 1) / total);
}
__device__ __forceinline__ uint64_t first_unit(uint32_t worker, uint64_t total, uint32_t workers) {
    return total * worker / workers;
}

// Sums over the batch by a workgroup: units of all sequences, and of those
// before `until`.
__device__ __forceinline__ void sum_units(const KvAttendParams &p, uint32_t until, uint64_t *sh, uint64_t &total, uint64_t &before) {
    uint64_t a = 0, c = 0;
    for (uint32_t b = threadIdx.x; b < p.c.batch; b += kThreads) {
        const uint32_t n = units_of(p, b);
        a += n;
        c += b < until ? n : 0u;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        a += __shfl_xor(a, off);
        c += __shfl_xor(c, off);
    }
    if ((threadIdx.x & 63u) == 0u) {
        sh[threadIdx.x >> 6] = a;
        sh[kWaves + (threadIdx.x >> 6)] = c;
    }
    __syncthreads();
    total = sh[0] + sh[1] + sh[2] + sh[3];
    before = sh[4] + sh[5] + sh[6] + sh[7];
    static_assert(kWaves == 4, "");
}

// The sequence that has unit `u` of the columns' lines (u < total units of the
// batch, not times columns) and the units before it.
__device__ __forceinline__ void find_sequence(const KvAttendParams &p, uint64_t u, uint64_t *sh, uint32_t &b, uint64_t &before) {
    uint64_t base = 0;
    for (uint32_t b0 = 0;; b0 += kThreads) {
        const uint32_t mine = b0 + threadIdx.x;
        const uint64_t n = mine < p.c.batch ? units_of(p, mine) : 0u;
        uint64_t x = n;  // inclusive sum over the wave, then over the waves
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint64_t y = __shfl_up(x, off);
            if ((threadIdx.x & 63u) >= (uint32_t)off) x += y;
        }
        __syncthreads();  // sh has been read
        if ((threadIdx.x & 63u) == 63u) sh[threadIdx.x >> 6] = x;
        if (threadIdx.x == 0) sh[kWaves] = ~0ull;
        __syncthreads();
        uint64_t all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            if ((uint32_t)w < threadIdx.x >> 6) x += sh[w];
            all += sh[w];
        }
        if (u >= base + x - n && u < base + x) {
            sh[kWaves] = mine;
            sh[kWaves + 1] = base + x - n;
        }
        __syncthreads();
        if (sh[kWaves] != ~0ull) {
            b = (uint32_t)sh[kWaves];
            before = sh[kWaves + 1];
            return;
        }
        base += all;
        if (b0 + kThreads >= p.c.batch) {  // (u is not on the line: no sequence)
            b = p.c.batch;
            before = base;
            return;
        }
    }
}

// kDirect: one workgroup for each column of rows, which writes the result; else
// workers and parts.
template <typename T, bool kSq8, int DP, bool kDirect>
__global__ __launch_bounds__(kThreads, DP == 256 ? 1 : 2) void kv_token_kernel(KvAttendParams p) {
    using E = KvElem<T>;
    using P = KvElem<std::conditional_t<kSq8, __bf16, T>>;  // of the weights and the values
    constexpr bool kHalf = !kSq8 && std::is_same_v<T, _Float16>;  // fp16 weights
    constexpr float kLift = kv_lift(kHalf, false), kTop = kv_top(kHalf), kRest = kHalf ? 4096.0f : 1.0f;
    constexpr int kSteps = DP / 32;                 // matrix instructions of 16 logits
    constexpr int kPer = DP / 16;                   // values of a row that a lane holds
    constexpr int kKWords = kSq8 ? DP / 16 : DP / 8;  // words of a K row that a lane holds
    constexpr int kVWords = kSq8 ? kPer / 4 : kPer / 2;
    constexpr int kKLoads = kKWords / 4;
    __shared__ __align__(16) uint32_t sh_place[kWaves][2][kTile];  // (read four at a time)
    __shared__ __align__(16) float sh_scale[kSq8 ? kWaves : 1][2][kTile];
    __shared__ float sh_ml[kWaves][2][16];
    extern __shared__ __align__(16) float sh_out[];  // [waves][heads of the block][DP]

    const KvCacheParams &c = p.c;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t n = lane & 15u, g = lane >> 4;
    const uint32_t blocks = (p.group + 15u) / 16u, block_heads = min(16u, p.group);
    // the workgroup's range of units; lines lie sequence by sequence, column by column
    uint32_t b = blockIdx.y, column = blockIdx.x;
    uint64_t unit = 0, unit_end = 1, line = 0;  // line: first unit of the column at hand
    if constexpr (!kDirect) {
        __shared__ uint64_t sh_sum[2 * kWaves];
        uint64_t total, before;
        uint32_t n;
        if (c.batch <= kThreads) {  // the lengths are read once: a thread has one sequence's
            const uint32_t mine = threadIdx.x < c.batch ? units_of(p, threadIdx.x) : 0u;
            uint32_t upto = mine;  // (the host keeps a batch under 2^32 units)
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t y = __shfl_up(upto, off);
                if (lane >= (uint32_t)off) upto += y;
            }
            if (lane == 63u) sh_sum[wave] = upto;
            __syncthreads();
            total = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                if ((uint32_t)w < wave) upto += (uint32_t)sh_sum[w];
                total += sh_sum[w];
            }
            const uint32_t workers = workers_of(p, total);
            if (blockIdx.x >= workers) return;
            unit = first_unit(blockIdx.x, total * p.columns, workers);
            unit_end = first_unit(blockIdx.x + 1, total * p.columns, workers);
            const uint64_t u = unit / p.columns;
            if (u >= upto - mine && u < upto) {
                sh_sum[kWaves] = threadIdx.x;
                sh_sum[kWaves + 1] = upto - mine;
                sh_sum[kWaves + 2] = mine;
            }
            __syncthreads();
            b = (uint32_t)sh_sum[kWaves];
            before = sh_sum[kWaves + 1];
            n = (uint32_t)sh_sum[kWaves + 2];
        } else {
            sum_units(p, 0, sh_sum, total, before);
            const uint32_t workers = workers_of(p, total);
            if (blockIdx.x >= workers) return;
            unit = first_unit(blockIdx.x, total * p.columns, workers);
            unit_end = first_unit(blockIdx.x + 1, total * p.columns, workers);
            find_sequence(p, unit / p.columns, sh_sum, b, before);
            n = units_of(p, b);
        }
        // a sequence's columns follow each other, each of its units
        line = before * p.columns;
        column = (uint32_t)((unit - line) / n);
        line += (uint64_t)column * n;
    }
    bool again = false;
    while (unit < unit_end) {
    const uint32_t h = column / blocks, first_q = (column - h * blocks) * 16u;
    const uint32_t heads = min(16u, p.group - first_q);
    const KvVisible vis = kv_visible(p, kv_length(c, b));
    const uint32_t units = (vis.count + kUnit - 1) / kUnit;
    const uint32_t begin = kDirect ? 0u : (uint32_t)(unit - line) * kUnit;
    const uint32_t end = kDirect ? vis.count : min(vis.count, begin + (uint32_t)min(unit_end - unit, (uint64_t)units) * kUnit);
    const uint32_t rows = end > begin ? end - begin : 0u;
    const uint32_t tiles = (rows + kTile - 1) / kTile;
    const int32_t *list = p.listed ? p.listed + ((uint64_t)b * c.heads + h) * p.listed_count : nullptr;
    const int32_t *table = c.table + (uint64_t)b * c.table_stride;
    if (again) __syncthreads();  // the last part's sums have been read
    again = true;

    // Q operand: heads are columns; dims of step s as K's lanes hold them
    const bool head_ok = n < heads;
    // beside the second sum of 256 dims the queries would not fit the registers (48 sequences of up to 4,100 rows,
    // 32 heads over 2 of 256 dims: 72 us, in registers with spills 77, bf16 65)
    constexpr bool kQueryInLds = kHalf && DP == 256;
    __shared__ kv_u4 sh_q[kQueryInLds ? kSteps : 1][64];
    kv_u4 qf[kQueryInLds ? 1 : kSteps];
    {
        const char *q = p.q + (uint64_t)b * p.q_token + (uint64_t)(h * p.group + first_q + (head_ok ? n : 0u)) * p.q_head;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = kSq8 ? (uint32_t)(s / 2) * 64u + g * 16u + (uint32_t)(s & 1) * 8u : (uint32_t)s * 32u + g * 8u;
            const kv_u4 zero = {0, 0, 0, 0};
            const kv_u4 x = head_ok && d < c.dim ? *reinterpret_cast<const kv_u4 *>(q + 2u * d) : zero;
            if constexpr (!kQueryInLds)
                qf[s] = x;
            else if (wave == 0)
                sh_q[s][lane] = x;
        }
        if constexpr (kQueryInLds) __syncthreads();
    }
    const char *kbase = c.keys.rows + (uint64_t)h * c.keys.head_units * 16u;
    const char *vbase = c.values.rows + (uint64_t)h * c.values.head_units * 16u;
    // byte of the lane's values in a row (lanes past the row repeat its start; their outputs are not stored)
    const uint32_t vbyte = (n * kPer < c.dim ? n * kPer : 0u) * (kSq8 ? 1u : 2u);

    float m = kKvNone, l = 0.0f;
    kv_f4 acc[kPer], rest[kHalf ? kPer : 1];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        acc[i] = kv_f4{0, 0, 0, 0};
        if constexpr (kHalf) rest[i] = acc[i];
    }

    // row of the tile after next, page of the next tile: each load waits a whole step
    const uint32_t l32 = lane & 31u;
    auto row_of = [&](uint32_t tile) -> int32_t {
        const uint32_t i = tile * kTile + l32;
        return i < rows ? visible_row(vis, begin + i, list) : -1;
    };
    auto page_of = [&](int32_t row) -> int32_t { return row >= 0 ? table[(uint32_t)row >> c.page_shift] : -1; };
    int32_t row = row_of(wave);
    int32_t page = page_of(row);
    int32_t next_row = row_of(wave + kWaves);

    for (uint32_t tile = wave; tile < tiles; tile += kWaves) {
        const uint32_t kplace = kv_place(c, c.keys, page, (uint32_t)row);
        const uint32_t vplace = kv_place(c, c.values, page, (uint32_t)row);
        const bool mine = kplace != kKvNoOffset;
        const uint32_t valid = (uint32_t)__ballot(mine);  // lanes 32..63 repeat 0..31
        // a row's scales, by lanes 0..31 of the key, by lanes 32..63 of the value (its place: used after the rows' loads are out)
        float scale = lane < kTile ? 0.0f : 1.0f;
        if constexpr (kSq8) {
            const KvArray &array = lane < kTile ? c.keys : c.values;
            if (mine) scale = array.scales[kv_scale_place(c, array, page, (uint32_t)row, h)];
        }
        sh_place[wave][lane >> 5][l32] = mine ? (lane < kTile ? kplace : vplace) : 0u;  // row 0 of page 0 is there to read
        kv_wave_sync();
        row = next_row;
        page = page_of(row);
        next_row = row_of(tile + 2 * kWaves);

        // K: rows n and 16 + n
        KvWords<4> kw[2][kKLoads];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const char *src = kbase + (uint64_t)sh_place[wave][0][16 * t + n] * 16u;
#pragma unroll
            for (int s = 0; s < kKLoads; ++s) {
                const uint32_t d = kSq8 ? (uint32_t)s * 64u + g * 16u : (uint32_t)s * 32u + g * 8u;
                kw[t][s] = *reinterpret_cast<const KvWords<4> *>(src + (d < c.dim ? d : 0u) * (kSq8 ? 1u : 2u));
            }
        }
        // V: rows 16 (j / 4) + 4 g + j % 4
        KvWords<kVWords> vw[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const kv_u4 place = *reinterpret_cast<const kv_u4 *>(&sh_place[wave][1][16 * t + 4 * g]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                vw[4 * t + j] = *reinterpret_cast<const KvWords<kVWords> *>(vbase + (uint64_t)place[j] * 16u + vbyte);
        }
        if constexpr (kSq8) {
            sh_scale[wave][lane >> 5][l32] = lane < kTile ? scale * p.scale_log2 : scale;
            kv_wave_sync();
        }
        if (DP != c.dim) {  // dims past the row meet zeros of Q and must be finite
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int s = 0; s < kKLoads; ++s) {
                    const uint32_t d = kSq8 ? (uint32_t)s * 64u + g * 16u : (uint32_t)s * 32u + g * 8u;
#pragma unroll
                    for (int w = 0; w < 4; ++w) kw[t][s].w[w] = d < c.dim ? kw[t][s].w[w] : 0u;
                }
        }
        // logits of rows 16 t + 4 g + i
        float x[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            kv_f4 sacc = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                kv_u4 a;
                if constexpr (kSq8) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t word = kw[t][s / 2].w[2 * (s & 1) + e / 2];
                        a[e] = E::pack_codes(kv_code(word, 2 * (e & 1)), kv_code(word, 2 * (e & 1) + 1));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] = kw[t][s].w[e];
                }
                sacc = E::mma16(a, kQueryInLds ? sh_q[kQueryInLds ? s : 0][lane] : qf[kQueryInLds ? 0 : s], sacc);
            }
            if constexpr (kSq8) {
                const kv_f4 ks = *reinterpret_cast<const kv_f4 *>(&sh_scale[wave][0][16 * t + 4 * g]);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[t][i] = sacc[i] * ks[i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[t][i] = sacc[i] * p.scale_log2;
            }
        }
        if (valid != 0xffffffffu) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool ok = valid >> (16 * t + 4 * g + i) & 1u;
                    if (!ok) x[t][i] = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kVWords; ++w) vw[4 * t + i].w[w] = ok ? vw[4 * t + i].w[w] : 0u;
                }
        }
        if (p.logits) {
            float *at = p.logits + (((uint64_t)b * c.heads + h) * p.max_visible + begin + tile * kTile) * p.group + first_q + n;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t r = 16 * t + 4 * g + i;
                    if (head_ok && tile * kTile + r < rows) at[(uint64_t)r * p.group] = x[t][i];
                }
        }
        float top = kKvNone;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, x[t][i]);
        top = kv_max16(top);
        if (__any(top > m + kTop)) {
            const float higher = fmaxf(m, top - kLift);
            const float f = kv_exp2(m - higher);
            m = higher;
            l *= f;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                acc[i] *= f;
                if constexpr (kHalf) rest[i] *= f;
            }
        }
        kv_u4 hi, lo, least;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            kv_f4 vs = {1, 1, 1, 1};
            if constexpr (kSq8) vs = *reinterpret_cast<const kv_f4 *>(&sh_scale[wave][1][16 * t + 4 * g]);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                float w0 = kv_exp2(x[t][i] - m), w1 = kv_exp2(x[t][i + 1] - m);
                l += w0 + w1;
                if constexpr (kSq8) {
                    w0 *= vs[i];
                    w1 *= vs[i + 1];
                }
                const uint32_t r = P::pack(w0, w1);
                hi[2 * t + i / 2] = r;
                const float r0 = (w0 - P::low(r)) * kRest, r1 = (w1 - P::high(r)) * kRest;
                const uint32_t y = P::pack(r0, r1);
                lo[2 * t + i / 2] = y;
                if constexpr (!kHalf) least[2 * t + i / 2] = P::pack(r0 - P::low(y), r1 - P::high(y));
            }
        }
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            kv_u4 a;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (kSq8)
                    a[j] = P::pack_codes(kv_code(vw[2 * j].w[e / 4], e & 3), kv_code(vw[2 * j + 1].w[e / 4], e & 3));
                else
                    a[j] = __builtin_amdgcn_perm(vw[2 * j + 1].w[e / 2], vw[2 * j].w[e / 2], e & 1 ? 0x07060302u : 0x05040100u);
            }
            acc[e] = P::mma16(a, hi, acc[e]);
            if constexpr (kHalf)
                rest[e] = P::mma16(a, lo, rest[e]);
            else
                acc[e] = P::mma16(a, least, P::mma16(a, lo, acc[e]));
        }
    }
    l = kv_sum16(l);
    if constexpr (kHalf) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] += rest[i] * (1.0f / kRest);
    }

    // join the waves: sums relative to the largest maximum
    if (g == 0) {
        sh_ml[wave][0][n] = m;
        sh_ml[wave][1][n] = l;
    }
    __syncthreads();
    float top = sh_ml[0][0][n];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sh_ml[w][0][n]);
    const float f = kv_exp2(m - top);
    if (head_ok) {
        // the lane's values are dims kPer * 4 g .. of head n, in the order of the rows of the accumulators
        float *o = sh_out + ((uint64_t)wave * heads + n) * DP + kPer * 4 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < kPer; e += 4)
                *reinterpret_cast<kv_f4 *>(o + kPer * i + e) =
                    kv_f4{acc[e][i] * f, acc[e + 1][i] * f, acc[e + 2][i] * f, acc[e + 3][i] * f};
    }
    __syncthreads();
    const uint64_t q0 = (uint64_t)b * p.q_heads + h * p.group + first_q;
    for (uint32_t at = threadIdx.x; at < heads * (DP / 4); at += kThreads) {
        const uint32_t head = at / (DP / 4), d = (at % (DP / 4)) * 4;
        kv_f4 o = {0, 0, 0, 0};
        float big = kKvNone, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            o += *reinterpret_cast<const kv_f4 *>(sh_out + ((uint64_t)w * heads + head) * DP + d);
            big = fmaxf(big, sh_ml[w][0][head]);
        }
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += sh_ml[w][1][head] * kv_exp2(sh_ml[w][0][head] - big);
        if constexpr (!kSq8) {
            if (kv_nan(o) && sum == sum && d < c.dim) {  // values that are not finite, under weights that are
                kv_f4 s = {0, 0, 0, 0};
                for (uint32_t i = begin; i < end; ++i) {
                    const int32_t r = visible_row(vis, i, list);
                    const uint32_t place = kv_place(c, c.values, page_of(r), (uint32_t)r);
                    if (place == kKvNoOffset) continue;
                    const kv_u2 y = *reinterpret_cast<const kv_u2 *>(vbase + (uint64_t)place * 16u + 2u * d);
                    s += kv_not_finite(kv_f4{E::low(y[0]), E::high(y[0]), E::low(y[1]), E::high(y[1])});
                }
                o = kv_settled(o, s);
            }
        }
        if constexpr (!kDirect) {
            const uint64_t part = ((uint64_t)b * p.columns + column + blockIdx.x) * block_heads + head;
            *reinterpret_cast<kv_f4 *>(p.part_o + part * DP + d) = o;
            if (d == 0) {
                p.part_ml[part * 2] = big;
                p.part_ml[part * 2 + 1] = sum;
            }
        } else {
            const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
            if (d < c.dim) {
                const kv_u2 y = {E::pack(o[0] * r, o[1] * r), E::pack(o[2] * r, o[3] * r)};
                *reinterpret_cast<kv_u2 *>(p.out + (uint64_t)b * p.out_token + (uint64_t)(h * p.group + first_q + head) * p.out_head +
                                           2u * d) = y;
            }
            if (d == 0) p.lse[q0 + head] = kv_lse(big, sum, kLift);
        }
    }
    if constexpr (kDirect) break;
    // the next column, of this sequence or of the next that has rows
    unit = line + units;
    line = unit;
    if (++column == p.columns) {
        column = 0;
        do ++b;
        while (b < c.batch && unit < unit_end && units_of(p, b) == 0u);
    }
    }
}

// Joins the partial results of a query, out = sum_c exp2(m_c - m) O_c / sum_c
// exp2(m_c - m) l_c: blocks below `joins`, one for join_dims dims of a query, whose
// parts it reads 1,024 / join_dims side by side.  Where there are fewer than
// kJoinBlocks queries a block has fewer dims, 64 at the least, so that few queries with
// many parts use many compute units (32 queries of 128 dims over 131,071 rows: 59.6 us, with
// whole queries 62.4; 1,536 queries over 4,100 rows: 131.5, with whole queries 128).  With weights the other blocks turn the
// logits of 1,024 visible rows into weights and add them, summed over the group's
// heads, to the caller's.
constexpr int kWeightPer = 4;  // rows of a thread
constexpr uint32_t kWeightRows = kThreads * kWeightPer;
constexpr uint32_t kJoinDims = 64;
constexpr uint64_t kJoinBlocks = 1024;

// With join_dims 0 (prompts of at least kJoinBlocks queries) a wave takes a query: 16,384 queries
// of 128 dims over 512 rows in two parts each, the whole call 26 us, and 44 with a block a query.

// Largest maximum and sum of a query's parts, in all lanes of a wave.
__device__ __forceinline__ void join_parts(const KvAttendParams &p, uint64_t first, uint32_t step, uint32_t count, float &m, float &l) {
    m = kKvNone;
    l = 0.0f;
    for (uint32_t i = threadIdx.x & 63u; i < count; i += 64) {
        const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + (first + (uint64_t)i * step) * 2);
        const float big = fmaxf(m, ml.x);
        l = l * kv_exp2(m - big) + ml.y * kv_exp2(ml.x - big);
        m = big;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const float m2 = __shfl_xor(m, off), l2 = __shfl_xor(l, off);
        const float big = fmaxf(m, m2);
        l = l * kv_exp2(m - big) + l2 * kv_exp2(m2 - big);
        m = big;
    }
}

// The parts of a column of rows: those of the workers that have units of it.
__device__ __forceinline__ void column_parts(const KvAttendParams &p, uint32_t b, uint32_t column, uint64_t *sh, uint64_t &first,
                                             uint32_t &count) {
    uint64_t total, before;
    sum_units(p, b, sh, total, before);
    const uint32_t n = units_of(p, b);
    const uint64_t line = before * p.columns + (uint64_t)column * n;
    first = (uint64_t)b * p.columns + column;
    count = 0;
    if (n) {
        const uint32_t workers = workers_of(p, total), w0 = worker_of(line, total * p.columns, workers);
        first += w0;
        count = worker_of(line + n - 1, total * p.columns, workers) - w0 + 1;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void kv_finish_kernel(KvAttendParams p, uint32_t dp, uint32_t join_dims, uint32_t joins,
                                                             uint32_t row_blocks, bool prompt) {
    using E = KvElem<T>;
    const KvCacheParams &c = p.c;
    __shared__ __align__(16) float sh[kThreads * 4];  // [groups][dims of the block]
    __shared__ float sh_m[kThreads], sh_l[kThreads];
    __shared__ uint64_t sh_sum[2 * kWaves];
    const uint32_t t = threadIdx.x;
    if (join_dims == 0) {  // a wave for a query, a lane for each 64th dim
        const uint64_t query = (uint64_t)blockIdx.x * kWaves + (t >> 6);
        if (query >= p.tokens * p.q_heads) return;
        const uint64_t first = query * p.chunks;
        const uint32_t lane = t & 63u;
        float m, l;
        join_parts(p, first, 1, p.chunks, m, l);
        constexpr int kMost = 4;  // 256 dims
        kv_f4 o = {0, 0, 0, 0};
        const uint32_t per = dp / 64, d = lane * per;
#pragma unroll 4
        for (uint32_t i = 0; i < p.chunks; ++i) {
            const float f = kv_exp2(p.part_ml[(first + i) * 2] - m);
            const float *x = p.part_o + (first + i) * dp + d;
            if (per == kMost) {
                o += *reinterpret_cast<const kv_f4 *>(x) * f;
            } else if (per == 2) {
                const float2 y = *reinterpret_cast<const float2 *>(x);
                o[0] = fmaf(y.x, f, o[0]);
                o[1] = fmaf(y.y, f, o[1]);
            } else {
                o[0] = fmaf(x[0], f, o[0]);
            }
        }
        if (kv_nan(o) && l == l) {
            kv_f4 s = {0, 0, 0, 0};
            for (uint32_t i = 0; i < p.chunks; ++i)
#pragma unroll
                for (int e = 0; e < kMost; ++e)
                    if ((uint32_t)e < per) s[e] += kv_not_finite(p.part_o[(first + i) * dp + d + e]);
            o = kv_settled(o, s);
        }
        const uint32_t token = (uint32_t)(query / p.q_heads), head = (uint32_t)(query - (uint64_t)token * p.q_heads);
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        char *to = p.out + (uint64_t)token * p.out_token + (uint64_t)head * p.out_head + 2u * d;
        if (d < c.dim) {
            if (per == kMost)
                *reinterpret_cast<kv_u2 *>(to) = kv_u2{E::pack(o[0] * r, o[1] * r), E::pack(o[2] * r, o[3] * r)};
            else if (per == 2)
                *reinterpret_cast<uint32_t *>(to) = E::pack(o[0] * r, o[1] * r);
            else
                *reinterpret_cast<uint16_t *>(to) = (uint16_t)E::pack(o[0] * r, 0.0f);
        }
        if (lane == 0) p.lse[query] = kv_lse(m, l, p.lift);
        return;
    }
    if (blockIdx.x < joins) {
        const uint32_t slices = (c.dim + join_dims - 1) / join_dims, groups = kThreads * 4 / join_dims;
        const uint64_t query = blockIdx.x / slices;
        const uint32_t slice = blockIdx.x - (uint32_t)query * slices;
        const uint32_t token = (uint32_t)(query / p.q_heads), head = (uint32_t)(query - (uint64_t)token * p.q_heads);
        uint64_t first = query * p.chunks;
        uint32_t count = p.chunks, step = 1;
        if (!prompt) {
            const uint32_t h = head / p.group, q = head - h * p.group;
            step = min(16u, p.group);
            column_parts(p, token, h * ((p.group + 15u) / 16u) + q / 16u, sh_sum, first, count);
            first = first * step + (q & 15u);
        }
        float m, l;
        join_parts(p, first, step, count, m, l);
        const uint32_t grp = t * 4 / join_dims, d4 = t * 4 % join_dims, d = slice * join_dims + d4;
        kv_f4 o = {0, 0, 0, 0};
        constexpr int kFlight = 4;
        for (uint32_t i0 = grp; i0 < count; i0 += kFlight * groups) {
            kv_f4 x[kFlight];
            float f[kFlight];
#pragma unroll
            for (int j = 0; j < kFlight; ++j) {
                const uint32_t i = i0 + (uint32_t)j * groups;
                const uint64_t at = first + (uint64_t)(i < count ? i : i0) * step;
                x[j] = *reinterpret_cast<const kv_f4 *>(p.part_o + at * dp + d);
                f[j] = i < count ? kv_exp2(p.part_ml[at * 2] - m) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < kFlight; ++j)
                if (i0 + (uint32_t)j * groups < count) o += x[j] * f[j];
        }
        *reinterpret_cast<kv_f4 *>(&sh[t * 4]) = o;
        __syncthreads();
        if (grp == 0 && d < c.dim) {
            for (uint32_t i = 1; i < min(groups, count); ++i) o += *reinterpret_cast<const kv_f4 *>(&sh[i * join_dims + d4]);
            if (kv_nan(o) && l == l) {
                kv_f4 s = {0, 0, 0, 0};
                for (uint32_t i = 0; i < count; ++i)
                    s += kv_not_finite(*reinterpret_cast<const kv_f4 *>(p.part_o + (first + (uint64_t)i * step) * dp + d));
                o = kv_settled(o, s);
            }
            const float r = l == 0.0f ? 0.0f : 1.0f / l;
            const kv_u2 y = {E::pack(o[0] * r, o[1] * r), E::pack(o[2] * r, o[3] * r)};
            *reinterpret_cast<kv_u2 *>(p.out + (uint64_t)token * p.out_token + (uint64_t)head * p.out_head + 2u * d) = y;
        }
        if (t == 0 && slice == 0) p.lse[query] = kv_lse(m, l, p.lift);
        return;
    }
    // weights of kWeightRows visible rows of one (sequence, head)
    const uint32_t item = blockIdx.x - joins;
    const uint32_t part = item % row_blocks, bh = item / row_blocks;
    const uint32_t b = bh / c.heads, h = bh - b * c.heads;
    const KvVisible vis = kv_visible(p, kv_length(c, b));
    const uint32_t i0 = part * kWeightRows + t;
    if (part * kWeightRows >= vis.count) return;
    const float *x = p.logits + ((uint64_t)b * c.heads + h) * p.max_visible * p.group;
    const bool fours = p.group % 4u == 0u;
    // the first logits and the weights travel while the parts are joined
    kv_f4 first4[kWeightPer];
    int32_t row[kWeightPer];
    float old[kWeightPer];
    const int32_t *list = p.listed ? p.listed + ((uint64_t)b * c.heads + h) * p.listed_count : nullptr;
    float *weights = p.weights + (uint64_t)b * p.weight_batch + (uint64_t)h * p.weight_head;
#pragma unroll
    for (int j = 0; j < kWeightPer; ++j) {
        const uint32_t i = i0 + (uint32_t)j * kThreads;
        row[j] = i < vis.count ? visible_row(vis, i, list) : -1;
        first4[j] = kv_f4{0, 0, 0, 0};
        if (fours && i < vis.count) first4[j] = *reinterpret_cast<const kv_f4 *>(x + (uint64_t)i * p.group);
        old[j] = row[j] >= 0 && i < vis.before_list ? weights[row[j]] : 0.0f;
    }
    // a wave joins one query head at a time
    const uint32_t step = min(16u, p.group);
    for (uint32_t q0 = 0; q0 < p.group; q0 += 16u) {
        uint64_t first;
        uint32_t count;
        if (q0) __syncthreads();
        column_parts(p, b, h * ((p.group + 15u) / 16u) + q0 / 16u, sh_sum, first, count);
        for (uint32_t q = q0 + (t >> 6); q < min(q0 + 16u, p.group); q += kWaves) {
            float m, l;
            join_parts(p, first * step + (q - q0), step, count, m, l);
            if ((t & 63u) == 0u) {
                sh_m[q] = m;
                sh_l[q] = l == 0.0f ? 0.0f : 1.0f / l;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kWeightPer; ++j) {
        const uint32_t i = i0 + (uint32_t)j * kThreads;
        if (row[j] < 0) continue;
        const float *y = x + (uint64_t)i * p.group;
        float sum = 0.0f;  // (a row without a page has logits of -inf: no weight)
        if (fours) {
            for (uint32_t q = 0; q < p.group; q += 4) {
                const kv_f4 z = q ? *reinterpret_cast<const kv_f4 *>(y + q) : first4[j];
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += kv_exp2(z[e] - sh_m[q + e]) * sh_l[q + e];
            }
        } else {
            for (uint32_t q = 0; q < p.group; ++q) sum += kv_exp2(y[q] - sh_m[q]) * sh_l[q];
        }
        if (sum != sum) {  // a query's sum is NaN: its weights are, but that of a logit of -inf is none
            sum = 0.0f;
            for (uint32_t q = 0; q < p.group; ++q) sum += y[q] == -INFINITY ? 0.0f : kv_exp2(y[q] - sh_m[q]) * sh_l[q];
        }
        if (i < vis.before_list)
            weights[row[j]] = old[j] + sum;
        else
            unsafeAtomicAdd(weights + row[j], sum);  // a row that the list names twice counts twice
    }
}

template <typename T, bool kSq8, int DP>
int launch(const KvAttendParams &p, hipStream_t stream) {
    const size_t lds = (size_t)kWaves * (p.group < 16u ? p.group : 16u) * DP * sizeof(float);
    auto *kernel = p.workers ? &kv_token_kernel<T, kSq8, DP, false> : &kv_token_kernel<T, kSq8, DP, true>;
    // 16 heads of 256 dims are 64 KiB, beside up to 10 KiB that the kernel has anyway: above the default limit
    if (lds > 32768 && ensure_lds_limit(reinterpret_cast<const void *>(kernel), (int)lds) != 0) return -1;
    kernel<<<p.workers ? dim3(p.workers) : dim3(p.columns, p.c.batch), kThreads, lds, stream>>>(p);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <typename T, bool kSq8>
int launch_dim(const KvAttendParams &p, hipStream_t stream) {
    switch (kv_padded_dim(p.c.dim)) {
        case 64: return launch<T, kSq8, 64>(p, stream);
        case 128: return launch<T, kSq8, 128>(p, stream);
        default: return launch<T, kSq8, 256>(p, stream);
    }
}

}  // namespace

uint32_t kv_padded_dim(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Up to 512 rows, or 8 for each column of rows of the batch and up to 2,048, one
// workgroup takes a column and writes the result: a join's launch costs more than
// the rows do, and many columns fill the card by themselves.  Otherwise, and
// where weights are wanted, as many workgroups as the registers of the compute units
// hold share the rows out, or fewer where there are fewer units.
// Measured, groups of 4 heads of 128 dims, whole columns against shared rows, us:
//   64 columns of 512 rows    9.8, 11.7    of 1,024   16.9, 14.4
//   256 columns of 512 rows  15.2, 21.1    of 1,024   24.2, 29.9    of 2,048   43.3, 49.8
//   512 columns of 1,024     42.7, 52.6    of 2,048   98.9, 109     of 4,096   190, 199
// and with lengths far apart (the squares of even ones) 256 columns of up to 2,048
// rows 26.2, 25.3, 512 of up to 4,096 117, 101.
void kv_token_split(KvAttendParams &p) {
    constexpr uint64_t kWhole = 512, kMostWhole = 2048, kWholeOfColumn = 8;
    p.columns = p.c.heads * ((p.group + 15u) / 16u);
    p.workers = 0;
    const uint64_t most = (uint64_t)kv_compute_units() * (kv_padded_dim(p.c.dim) == 256 ? 1u : 2u);
    const uint64_t whole = kWholeOfColumn * p.columns * p.c.batch;
    if (p.max_visible <= (whole < kWhole ? kWhole : whole < kMostWhole ? whole : kMostWhole) && !p.weights) return;
    const uint64_t units = (uint64_t)(p.max_visible + kUnit - 1) / kUnit * p.columns * p.c.batch;
    p.workers = (uint32_t)(units < most ? units : most);
    if (!p.workers) p.workers = 1;
}

int launch_kv_token(const KvAttendParams &p, uint32_t type, bool sq8, hipStream_t stream) {
    if (type == kKvBf16) return sq8 ? launch_dim<__bf16, true>(p, stream) : launch_dim<__bf16, false>(p, stream);
    return sq8 ? launch_dim<_Float16, true>(p, stream) : launch_dim<_Float16, false>(p, stream);
}

int launch_kv_finish(const KvAttendParams &params, uint32_t type, bool sq8, bool prompt, hipStream_t stream) {
    KvAttendParams p = params;
    p.lift = kv_lift(!sq8 && type == kKvF16, prompt);
    const uint64_t queries = p.tokens * p.q_heads;
    const uint32_t dp = kv_padded_dim(p.c.dim);
    uint32_t dims = dp;
    while (dims > kJoinDims && queries * (dp / dims) < kJoinBlocks) dims /= 2;
    uint32_t joins = (uint32_t)queries * ((p.c.dim + dims - 1) / dims);
    if (prompt && queries >= kJoinBlocks) {
        dims = 0;
        joins = (uint32_t)((queries + kWaves - 1) / kWaves);
    }
    const uint32_t row_blocks = p.weights && !prompt ? (p.max_visible + kWeightRows - 1) / kWeightRows : 0u;
    const uint32_t blocks = joins + row_blocks * p.c.heads * p.c.batch;
    if (type == kKvBf16)
        kv_finish_kernel<__bf16><<<blocks, kThreads, 0, stream>>>(p, dp, dims, joins, row_blocks, prompt);
    else
        kv_finish_kernel<_Float16><<<blocks, kThreads, 0, stream>>>(p, dp, dims, joins, row_blocks, prompt);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tessa
