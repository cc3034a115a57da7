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
//   64 of up to 8,200 rows of 4 bits                 372 MB    76 +  9 us   4.4 TB/s
//   3 of up to 131,071, 4 bits, 4 heads, weights     170 MB    49 + 16 us   2.6 TB/s
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
//  * 4-bit rows: a conversion makes two codes and their group's scale two bf16 values, exactly.  Four lanes take the
//    four quarters of a key's row (dims are then summed in an order of their own, the query's with them), so that a lane has
//    one group.  The weight's three parts are cut, not rounded: 8 bits each are all that f32 has.
//    fp16 queries are two bf16 parts, exactly.
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

// kOnce: rows that no other workgroup reads need no place in the caches.
template <int N, bool kOnce>
__device__ __forceinline__ KvWords<N> load_words(const char *from) {
    if constexpr (!kOnce) {
        return *reinterpret_cast<const KvWords<N> *>(from);
    } else {
        KvWords<N> x;
        if constexpr (N == 1) {
            x.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(from));
        } else {
            using V = uint32_t __attribute__((ext_vector_type(N)));
            const V y = __builtin_nontemporal_load(reinterpret_cast<const V *>(from));
#pragma unroll
            for (int i = 0; i < N; ++i) x.w[i] = y[i];
        }
        return x;
    }
}

// Row id of visible index i < v.count, or -1 (a place of the list that names no further row).
__device__ __forceinline__ int32_t visible_row(const KvVisible &v, uint32_t i, const int32_t *list) {
    if (i < v.first) return (int32_t)i;
    if (i < v.before_list) return (int32_t)(v.last_begin + (i - v.first));
    const int32_t r = list[i - v.before_list];
    return r >= (int32_t)v.first && r < (int32_t)v.last_begin ? r : -1;
}

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
    return (uint64_t)uniform((uint32_t)(x >> 32)) << 32 | uniform((uint32_t)x);
}

// x of the lane kBy before in a ring of 16.
template <int kBy>
__device__ __forceinline__ float turned(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x120 + kBy, 0xf, 0xf, true));
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

// Forms of the kernel over 4-bit rows.  A wave issues an instruction each 5 cycles at most and waits for its own
// results, so two waves of a SIMD, all that the registers of kFormAny leave, take as long for the instructions
// alone (70 us for the batch of 64 above, its rows in the cache) as the memory does (72), and 100 for both.
// Where 16 rows of a tile lie in one page, one after the other (all rows visible, pages of at least 16), addresses are a
// scalar and a lane's constant, and up to 4 or 8 query heads are repeated over the 16 columns of the instructions, so that the
// parts of a weight (and of an fp16 query) have columns of their own, one or two products instead of three.
//  * kFormColumns4: with the registers that this saves three waves fit a SIMD (two at 256 dims).
//  * kFormColumns8: likewise at 128 dims.
// These pass the caches by (of 8 heads the keys alone: the values too cost 2 us).
// Microseconds of a call, bf16, in columns and in kFormAny (a window that shows every row):
//                                           64 dims       128 dims      256 dims
//   64 sequences of up to 8,200 rows,  4 heads  65, 66    82, 92        81, 103 (32 sequences)
//                                      8        74, 72    90, 100      128, 109
//   3 of up to 131,071,                4        48, 50    60, 66       105, 133
//                                      8        51, 50    64, 67       174, 136
// Past 8 heads the scalar addresses alone took as long as kFormAny or up to a tenth longer.  Rows that no other workgroup
// reads need no place in the caches: 64 sequences of 8,200 rows each 117 us, through the caches 126.  Sequences that share pages
// read them from memory more often for it: 98 and 94 with all of them in common, 105 and 102 with half.
enum { kFormAny = 0, kFormColumns4 = 1, kFormColumns8 = 2 };
// Waves of a SIMD, by registers.
constexpr int token_waves(int dp, int form) { return dp == 256 ? (form != kFormAny ? 2 : 1) : form != kFormAny ? 3 : 2; }

// kDirect: one workgroup for each column of rows, which writes the result; else
// workers and parts.
template <typename T, int kRowsKind, int DP, bool kDirect, int kForm>
__global__ __launch_bounds__(kThreads, token_waves(DP, kForm)) void kv_token_kernel(KvAttendParams p) {
    constexpr bool kColumns = kForm != kFormAny;
    constexpr uint32_t kColumnHeads = kForm == kFormColumns4 ? 4 : kForm == kFormColumns8 ? 8 : 16;
    constexpr bool kSq8 = kRowsKind == kRowsSq8, kMx4 = kRowsKind == kRowsMx4;
    using E = KvElem<T>;
    using K = KvElem<std::conditional_t<kMx4, __bf16, T>>;  // of the logits' products
    using P = KvElem<std::conditional_t<kSq8 || kMx4, __bf16, T>>;  // of the weights and the values
    constexpr bool kHalf = !kSq8 && !kMx4 && std::is_same_v<T, _Float16>;  // fp16 weights
    constexpr bool kSplitQuery = kMx4 && std::is_same_v<T, _Float16>;  // an fp16 query is two bf16 parts, exactly,
    constexpr int kQueryParts = kSplitQuery && !kColumns ? 2 : 1;      // each a product (kColumns: of columns of its own)
    constexpr float kLift = kv_lift(kHalf, false), kTop = kv_top(kHalf), kRest = kHalf ? 4096.0f : 1.0f;
    constexpr int kSteps = DP / 32;                 // matrix instructions of 16 logits
    constexpr int kPer = DP / 16;                   // values of a row that a lane holds
    constexpr int kKWords = kMx4 ? DP / 32 : kSq8 ? DP / 16 : DP / 8;  // words of a K row that a lane holds
    constexpr int kVWords = kMx4 ? (kPer + 7) / 8 : kSq8 ? kPer / 4 : kPer / 2;
    constexpr int kKLoad = kKWords < 4 ? kKWords : 4;  // words of one load
    constexpr int kKLoads = kKWords / kKLoad;
    constexpr uint32_t kKDims = DP / 4 / kKLoads;      // dims of a lane's load, which four lanes share out
    constexpr int kMxGroups = DP / (int)kMxGroup;
    // 4-bit rows: the next tiles' loads are out while one is worked on, which costs few registers
    constexpr int kTurns = kMx4 && !kColumns ? 2 : 1;
    struct Tile {  // what a lane has of a tile's rows
        KvWords<kKLoad> kw[2][kKLoads];
        KvWords<kVWords> vw[8];
        float scale;
        uint32_t bytes[kMx4 ? (kMxGroups + 3) / 4 : 1];
        uint32_t valid;  // rows that are there
    };
    __shared__ __align__(16) uint32_t sh_place[kWaves][2][kTile];  // (read four at a time)
    __shared__ __align__(16) float sh_scale[kSq8 ? kWaves : 1][2][kTile];
    __shared__ __align__(16) float sh_group[kMx4 ? kWaves : 1][2][kMx4 ? kMxGroups : 1][kTile];  // scales of 32 dims
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
    if constexpr (kColumns) {  // the same for all lanes, which the compiler cannot see: scalar registers
        b = uniform(b);
        column = uniform(column);
        unit = uniform(unit);
        unit_end = uniform(unit_end);
        line = uniform(line);
    }
    const uint32_t h = kColumns ? uniform(column / blocks) : column / blocks, first_q = (column - h * blocks) * 16u;
    const uint32_t heads = min(16u, p.group - first_q);
    const KvVisible vis = kv_visible(p, kv_length(c, b));
    const uint32_t units = (vis.count + kUnit - 1) / kUnit;
    const uint32_t begin0 = kDirect ? 0u : (uint32_t)(unit - line) * kUnit;
    const uint32_t begin = kColumns ? uniform(begin0) : begin0;
    const uint32_t end0 = kDirect ? vis.count : min(vis.count, begin + (uint32_t)min(unit_end - unit, (uint64_t)units) * kUnit);
    const uint32_t end = kColumns ? uniform(end0) : end0;
    const uint32_t rows = end > begin ? end - begin : 0u;
    const uint32_t tiles = (rows + kTile - 1) / kTile;
    const int32_t *list = p.listed ? p.listed + ((uint64_t)b * c.heads + h) * p.listed_count : nullptr;
    const int32_t *table = c.table + (uint64_t)b * c.table_stride;
    if (again) __syncthreads();  // the last part's sums have been read
    again = true;

    // Q operand: heads are columns; dims of step s as K's lanes hold them
    const uint32_t my_head = n & (kColumnHeads - 1u);
    const bool head_ok = my_head < heads;
    // beside the second sum of 256 dims the queries would not fit the registers (48 sequences of up to 4,100 rows,
    // 32 heads over 2 of 256 dims: 72 us, in registers with spills 77, bf16 65)
    constexpr bool kQueryInLds = kHalf && DP == 256;
    __shared__ kv_u4 sh_q[kQueryInLds ? kSteps : 1][64];
    kv_u4 qf[kQueryParts][kQueryInLds ? 1 : kSteps];
    {
        const char *q = p.q + (uint64_t)b * p.q_token + (uint64_t)(h * p.group + first_q + (head_ok ? my_head : 0u)) * p.q_head;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            constexpr int kHere = kMx4 ? kKWords / kKLoads : kSq8 ? 2 : 1;  // steps of a load
            const uint32_t d = (uint32_t)(s / kHere) * 4u * kKDims + g * kKDims + (uint32_t)(s % kHere) * 8u;
            const kv_u4 zero = {0, 0, 0, 0};
            const kv_u4 x = head_ok && d < c.dim ? *reinterpret_cast<const kv_u4 *>(q + 2u * d) : zero;
            if constexpr (kSplitQuery) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float lo = E::low(x[e]), hi = E::high(x[e]);
                    const uint32_t first = K::pack(lo, hi);
                    auto rest_of = [](float w, float part) { return fabsf(w) < INFINITY ? w - part : 0.0f; };
                    const uint32_t second = K::pack(rest_of(lo, K::low(first)), rest_of(hi, K::high(first)));
                    qf[0][s][e] = kColumns && n >= 8u ? second : first;
                    if constexpr (!kColumns) qf[1][s][e] = second;
                }
            } else if constexpr (!kQueryInLds)
                qf[0][s] = x;
            else if (wave == 0)
                sh_q[s][lane] = x;
        }
        if constexpr (kQueryInLds) __syncthreads();
    }
    const char *kbase = c.keys.rows + (uint64_t)h * c.keys.head_units * 16u;
    const char *vbase = c.values.rows + (uint64_t)h * c.values.head_units * 16u;
    // byte of the lane's values in a row (lanes past the row repeat its start; their outputs are not stored)
    const uint32_t vdim = n * kPer < c.dim ? n * kPer : 0u;
    const uint32_t vbyte = kMx4 ? vdim / 2u : kSq8 ? vdim : 2u * vdim;

    // kColumns: what the parts after the first leave off (of 4 heads columns 12 .. 15 are left out)
    const uint32_t first_cut = n >= kColumnHeads ? 0xffff0000u : 0u, second_cut = n >= 2u * kColumnHeads ? 0xffff0000u : 0u;
    const uint32_t third_cut = n >= kColumnHeads ? 0xffffffffu : 0xffff0000u;
    float m = kKvNone, l = 0.0f;
    kv_f4 acc[kPer], rest[kHalf ? kPer : 1];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        acc[i] = kv_f4{0, 0, 0, 0};
        if constexpr (kHalf) rest[i] = acc[i];
    }

    // row of the tile after next, page of the next tile: each load waits a whole step
    const uint32_t l32 = lane & 31u;
    // the tile's row in place r of the instructions: 4-bit rows are half a cache line, so that a load of V, places j, 4 + j, 8 + j and
    // 12 + j, takes neighbouring rows
    auto row_in = [](uint32_t r) { return kMx4 ? (r & 16u) + 4u * (r & 3u) + (r >> 2 & 3u) : r; };
    auto row_of = [&](uint32_t tile) -> int32_t {
        const uint32_t i = tile * kTile + row_in(l32);
        return i < rows ? visible_row(vis, begin + i, list) : -1;
    };
    auto page_of = [&](int32_t row) -> int32_t { return row >= 0 ? table[(uint32_t)row >> c.page_shift] : -1; };
    int32_t row = -1, page = -1, next_row = -1;
    // kColumns: page of the lane's half of a tile; the lane's place in 16 rows
    auto tile_page = [&](uint32_t tile) { return table[min(begin + tile * kTile + (l32 & 16u), end - 1u) >> c.page_shift]; };
    uint32_t koffset[kColumns ? kKLoads : 1], voffset = 0, soffset = 0;
    const uint8_t *sbase = nullptr;
    const uint32_t wave0 = kColumns ? uniform(wave) : wave;
    if constexpr (kColumns) {
#pragma unroll
        for (int s = 0; s < kKLoads; ++s) {
            const uint32_t d = (uint32_t)s * 4u * kKDims + g * kKDims;
            koffset[s] = row_in(n) * c.keys.row_units * 16u + (d < c.dim ? d : 0u) / 2u;
        }
        voffset = g * c.values.row_units * 16u + vbyte;
        const KvArray &array = lane < kTile ? c.keys : c.values;
        sbase = kv_group_scales(array);
        soffset = h * (uint32_t)array.scale_head + (row_in(l32) & 15u) * (uint32_t)array.scale_row;
        if (wave0 < tiles) page = tile_page(wave0);
    } else {
        row = row_of(wave);
        page = page_of(row);
        next_row = row_of(wave + kWaves);
    }

    // The scale bytes of a row's groups.
    auto group_scales = [&](const uint8_t *at, uint32_t (&bytes)[kMx4 ? (kMxGroups + 3) / 4 : 1]) {
        if (c.scales_together) {  // as one word
            if constexpr (DP == 64) bytes[0] = *reinterpret_cast<const uint16_t *>(at);
            if constexpr (DP == 128) bytes[0] = *reinterpret_cast<const uint32_t *>(at);
            if constexpr (DP == 256) {
                const kv_u2 both = *reinterpret_cast<const kv_u2 *>(at);
                bytes[0] = both[0];
                bytes[kMx4 ? kMxGroups / 4 - 1 : 0] = both[1];
            }
        } else {
#pragma unroll
            for (int w = 0; w < (kMxGroups + 3) / 4; ++w) {
                uint32_t word = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * w + i < kMxGroups) word |= (uint32_t)at[kMxGroup * (4 * w + i) < c.dim ? 4 * w + i : 0] << (8 * i);
                bytes[kMx4 ? w : 0] = word;
            }
        }
    };
    // Starts the loads of a tile.
    auto fetch = [&](uint32_t tile, Tile &x) __attribute__((always_inline)) {
      if constexpr (kColumns) {
        const uint32_t at = begin + tile * kTile, slots = 1u << c.page_shift;
        const bool there = (uint32_t)page < c.pages;
        x.valid = (uint32_t)__ballot(there && tile * kTile + row_in(l32) < rows);
        const int32_t mine = there ? page : 0;  // row 0 of page 0 is there to read
        uint32_t scales[2];                     // places of the halves' scales, of the lane's array
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t id = (uint32_t)__builtin_amdgcn_readlane(mine, 16 * t), slot = (at + 16u * t) & (slots - 1u);
            const char *k = kbase + (uint64_t)(id * c.keys.page_units + slot * c.keys.row_units) * 16u;
            const char *v = vbase + (uint64_t)(id * c.values.page_units + slot * c.values.row_units) * 16u;
            scales[t] = lane < kTile ? id * (uint32_t)c.keys.scale_page + slot * (uint32_t)c.keys.scale_row
                                     : id * (uint32_t)c.values.scale_page + slot * (uint32_t)c.values.scale_row;
#pragma unroll
            for (int s = 0; s < kKLoads; ++s) x.kw[t][s] = load_words<kKLoad, kColumns>(k + koffset[s]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const char *src = v + j * 4u * c.values.row_units * 16u + voffset;
                if constexpr (kPer == 4)
                    x.vw[4 * t + j].w[0] = *reinterpret_cast<const uint16_t *>(src);
                else
                    x.vw[4 * t + j] = load_words<kVWords, kForm == kFormColumns4>(src);
            }
        }
        group_scales(sbase + (soffset + (l32 & 16u ? scales[1] : scales[0])), x.bytes);
        if (tile + kWaves < tiles) page = tile_page(tile + kWaves);
      } else {
        const uint32_t kplace = kv_place(c, c.keys, page, (uint32_t)row);
        const uint32_t vplace = kv_place(c, c.values, page, (uint32_t)row);
        const bool mine = kplace != kKvNoOffset;
        x.valid = (uint32_t)__ballot(mine);  // lanes 32..63 repeat 0..31
        // a row's scales, by lanes 0..31 of the key, by lanes 32..63 of the value (its place: used after the rows' loads are out)
        x.scale = lane < kTile ? 0.0f : 1.0f;
        if constexpr (kSq8) {
            const KvArray &array = lane < kTile ? c.keys : c.values;
            if (mine) x.scale = kv_row_scales(array)[kv_scale_place(c, array, page, (uint32_t)row, h)];
        }
        // MX4: a byte of each group, of the same rows by the same lanes (1 where there is no row: 0 * NaN would be NaN)
        if constexpr (kMx4) {
            const KvArray &array = lane < kTile ? c.keys : c.values;
            const uint8_t *at = kv_group_scales(array);
#pragma unroll
            for (int w = 0; w < (kMxGroups + 3) / 4; ++w) x.bytes[w] = 0x7f7f7f7fu;
            if (mine) {
                at += kv_scale_place(c, array, page, (uint32_t)row, h);
                group_scales(at, x.bytes);
            }
        }
        sh_place[wave][lane >> 5][l32] = mine ? (lane < kTile ? kplace : vplace) : 0u;  // row 0 of page 0 is there to read
        kv_wave_sync();
        row = next_row;
        page = page_of(row);
        next_row = row_of(tile + 2 * kWaves);

        // K: rows n and 16 + n
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const char *src = kbase + (uint64_t)sh_place[wave][0][16 * t + n] * 16u;
#pragma unroll
            for (int s = 0; s < kKLoads; ++s) {
                const uint32_t d = (uint32_t)s * 4u * kKDims + g * kKDims, there = d < c.dim ? d : 0u;
                x.kw[t][s] = *reinterpret_cast<const KvWords<kKLoad> *>(src + (kMx4 ? there / 2u : kSq8 ? there : 2u * there));
            }
        }
        // V: rows 16 (j / 4) + 4 g + j % 4
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const kv_u4 place = *reinterpret_cast<const kv_u4 *>(&sh_place[wave][1][16 * t + 4 * g]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const char *src = vbase + (uint64_t)place[j] * 16u + vbyte;
                if constexpr (kMx4 && kPer == 4)
                    x.vw[4 * t + j].w[0] = *reinterpret_cast<const uint16_t *>(src);
                else
                    x.vw[4 * t + j] = *reinterpret_cast<const KvWords<kVWords> *>(src);
            }
        }
      }
    };
    auto attend = [&](uint32_t tile, Tile &here) __attribute__((always_inline)) {
        auto &kw = here.kw;
        auto &vw = here.vw;
        const uint32_t valid = here.valid;
        if constexpr (kMx4) {
            if (kColumns && valid != 0xffffffffu) {  // what lies where no row is: 0 * NaN would be NaN
                asm volatile("");
#pragma unroll
                for (int w = 0; w < (kMxGroups + 3) / 4; ++w) here.bytes[w] = valid >> l32 & 1u ? here.bytes[w] : 0x7f7f7f7fu;
            }
#pragma unroll
            for (int i = 0; i < kMxGroups; ++i)
                sh_group[wave][lane >> 5][i][l32] = kv_mx_scale(here.bytes[i / 4] >> (8 * (i & 3)) & 255u);
            kv_wave_sync();
        }
        if constexpr (kSq8) {
            sh_scale[wave][lane >> 5][l32] = lane < kTile ? here.scale * p.scale_log2 : here.scale;
            kv_wave_sync();
        }
        if (!kMx4 && DP != c.dim) {  // (codes of 4 bits are) dims past the row meet zeros of Q and must be finite
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int s = 0; s < kKLoads; ++s) {
                    const uint32_t d = (uint32_t)s * 4u * kKDims + g * kKDims;
#pragma unroll
                    for (int w = 0; w < kKLoad; ++w) kw[t][s].w[w] = d < c.dim ? kw[t][s].w[w] : 0u;
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
                if constexpr (kMx4) {
                    const uint32_t d = (uint32_t)(s / kKLoad) * 4u * kKDims + g * kKDims;
                    a = kv_mx_values<__bf16>(kw[t][s / kKLoad].w[s % kKLoad], sh_group[wave][0][d / kMxGroup][16 * t + n]);
                } else if constexpr (kSq8) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t word = kw[t][s / 2].w[2 * (s & 1) + e / 2];
                        a[e] = E::pack_codes(kv_code(word, 2 * (e & 1)), kv_code(word, 2 * (e & 1) + 1));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] = kw[t][s].w[e];
                }
                sacc = K::mma16(a, kQueryInLds ? sh_q[kQueryInLds ? s : 0][lane] : qf[0][kQueryInLds ? 0 : s], sacc);
                if constexpr (kQueryParts == 2) sacc = K::mma16(a, qf[1][s], sacc);
            }
            if constexpr (kSq8) {
                const kv_f4 ks = *reinterpret_cast<const kv_f4 *>(&sh_scale[wave][0][16 * t + 4 * g]);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[t][i] = sacc[i] * ks[i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float logit = sacc[i];
                    if constexpr (kSplitQuery && kColumns) logit += turned<8>(logit);
                    // rounded once: the maximum, the weights and the stored logits are of one number.  (With the scale in the weight's
                    // own difference a large logit's rounding became a factor of its weight; 4-bit rows are no faster so.)
                    x[t][i] = logit * p.scale_log2;
                }
            }
        }
        if (valid != 0xffffffffu) {
            asm volatile("");  // a branch: as selections it costs every tile 32 instructions
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
                    const uint32_t r = row_in(16 * t + 4 * g + i);
                    if (head_ok && n < kColumnHeads && tile * kTile + r < rows) at[(uint64_t)r * p.group] = x[t][i];
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
        kv_u4 hi, lo = {0, 0, 0, 0}, least = {0, 0, 0, 0};
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
                if constexpr (kColumns) {  // the column's part
                    auto rest_of = [](float w, uint32_t cut) { return w - __uint_as_float(__float_as_uint(w) & cut); };
                    float r0 = rest_of(w0, first_cut), r1 = rest_of(w1, first_cut);
                    if constexpr (kColumnHeads == 4) {
                        r0 = rest_of(r0, second_cut);
                        r1 = rest_of(r1, second_cut);
                    }
                    hi[2 * t + i / 2] = __builtin_amdgcn_perm(__float_as_uint(r1), __float_as_uint(r0), 0x07060302u);
                    if constexpr (kColumnHeads == 8) {  // the third part beside the first, nothing beside the second
                        r0 = rest_of(rest_of(r0, 0xffff0000u), third_cut);
                        r1 = rest_of(rest_of(r1, 0xffff0000u), third_cut);
                        lo[2 * t + i / 2] = __builtin_amdgcn_perm(__float_as_uint(r1), __float_as_uint(r0), 0x07060302u);
                    }
                    continue;
                }
                if constexpr (kMx4) {  // cut, not rounded: three parts of 8 bits are all that f32 has
                    constexpr uint32_t kUpper = 0x07060302u;  // the upper halves of both
                    auto rest_of = [](float w) { return w - __uint_as_float(__float_as_uint(w) & 0xffff0000u); };
                    const float r0 = rest_of(w0), r1 = rest_of(w1), y0 = rest_of(r0), y1 = rest_of(r1);
                    hi[2 * t + i / 2] = __builtin_amdgcn_perm(__float_as_uint(w1), __float_as_uint(w0), kUpper);
                    lo[2 * t + i / 2] = __builtin_amdgcn_perm(__float_as_uint(r1), __float_as_uint(r0), kUpper);
                    least[2 * t + i / 2] = __builtin_amdgcn_perm(__float_as_uint(y1), __float_as_uint(y0), kUpper);
                    continue;
                }
                const uint32_t r = P::pack(w0, w1);
                hi[2 * t + i / 2] = r;
                const float r0 = (w0 - P::low(r)) * kRest, r1 = (w1 - P::high(r)) * kRest;
                const uint32_t y = P::pack(r0, r1);
                lo[2 * t + i / 2] = y;
                if constexpr (!kHalf) least[2 * t + i / 2] = P::pack(r0 - P::low(y), r1 - P::high(y));
            }
        }
        if constexpr (kMx4) {
            // two dims at a time: each row's pair of codes in one conversion, then rows beside each other
            float vs[8];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const kv_f4 s4 = *reinterpret_cast<const kv_f4 *>(&sh_group[wave][1][vdim / kMxGroup][16 * t + 4 * g]);
#pragma unroll
                for (int i = 0; i < 4; ++i) vs[4 * t + i] = s4[i];
            }
            kv_each<kPer / 2>([&](auto at) {
                constexpr int e = 2 * decltype(at)::value;
                kv_u4 a0, a1;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t x = P::template from_mx4<(e % 8) / 2>(vw[2 * j].w[e / 8], vs[2 * j]);
                    const uint32_t y = P::template from_mx4<(e % 8) / 2>(vw[2 * j + 1].w[e / 8], vs[2 * j + 1]);
                    a0[j] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                    a1[j] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                }
                acc[e] = P::mma16(a0, hi, acc[e]);
                acc[e + 1] = P::mma16(a1, hi, acc[e + 1]);
                if constexpr (kColumnHeads >= 8) {
                    acc[e] = P::mma16(a0, lo, acc[e]);
                    acc[e + 1] = P::mma16(a1, lo, acc[e + 1]);
                }
                if constexpr (kColumnHeads == 16) {
                    acc[e] = P::mma16(a0, least, acc[e]);
                    acc[e + 1] = P::mma16(a1, least, acc[e + 1]);
                }
            });
        }
#pragma unroll
        for (int e = 0; e < (kMx4 ? 0 : kPer); ++e) {
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
    };
    if constexpr (kTurns == 2) {  // by turns: in one set of registers moved on, each tile would wait for the next one's loads
        Tile even, odd;
        uint32_t tile = wave0;
        if (tile < tiles) fetch(tile, even);
        for (; tile < tiles; tile += 2 * kWaves) {
            if (tile + kWaves < tiles) fetch(tile + kWaves, odd);
            attend(tile, even);
            if (tile + kWaves >= tiles) break;
            if (tile + 2 * kWaves < tiles) fetch(tile + 2 * kWaves, even);
            attend(tile + kWaves, odd);
        }
    } else {
        for (uint32_t tile = wave; tile < tiles; tile += kWaves) {  // (wave0 would take scalar registers that are not left)
            Tile here;
            fetch(tile, here);
            attend(tile, here);
        }
    }
    l = kv_sum16(l);
    if constexpr (kHalf) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] += rest[i] * (1.0f / kRest);
    }

    if constexpr (kColumns) {  // the parts of a head
#pragma unroll
        for (int e = 0; e < kPer; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float y = kColumnHeads == 8 || n < 12u ? acc[e][i] : 0.0f;
                y += turned<8>(y);
                acc[e][i] = kColumnHeads == 8 ? y : y + turned<4>(y);
            }
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
    if (head_ok && n < kColumnHeads) {
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
        if constexpr (kRowsKind == kRowsPlain) {
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

template <typename T, int kRowsKind, int DP, int kForm>
int launch_form(const KvAttendParams &p, hipStream_t stream) {
    const size_t lds = (size_t)kWaves * (p.group < 16u ? p.group : 16u) * DP * sizeof(float);
    auto *kernel = p.workers ? &kv_token_kernel<T, kRowsKind, DP, false, kForm> : &kv_token_kernel<T, kRowsKind, DP, true, kForm>;
    // 16 heads of 256 dims are 64 KiB, beside up to 10 KiB that the kernel has anyway: above the default limit
    if (lds > 32768 && ensure_lds_limit(reinterpret_cast<const void *>(kernel), (int)lds) != 0) return -1;
    kernel<<<p.workers ? dim3(p.workers) : dim3(p.columns, p.c.batch), kThreads, lds, stream>>>(p);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// The form that a call takes.
int token_form(const KvAttendParams &p) {
    // (16 rows within 2^28 bytes: their offsets are 32-bit)
    if (!p.c.mx4 || p.window != 0xffffffffu || p.c.page_shift < 4u || p.c.keys.row_units > 1u << 20 || p.c.values.row_units > 1u << 20)
        return kFormAny;
    if (p.group <= 4u) return kFormColumns4;
    return p.group <= 8u && kv_padded_dim(p.c.dim) == 128u ? kFormColumns8 : kFormAny;
}

template <typename T, int kRowsKind, int DP>
int launch(const KvAttendParams &p, hipStream_t stream) {
    if constexpr (kRowsKind == kRowsMx4) {
        const int form = token_form(p);
        if (form == kFormColumns4) return launch_form<T, kRowsKind, DP, kFormColumns4>(p, stream);
        if constexpr (DP == 128)
            if (form == kFormColumns8) return launch_form<T, kRowsKind, DP, kFormColumns8>(p, stream);
    }
    return launch_form<T, kRowsKind, DP, kFormAny>(p, stream);
}

template <typename T, int kRowsKind>
int launch_dim(const KvAttendParams &p, hipStream_t stream) {
    switch (kv_padded_dim(p.c.dim)) {
        case 64: return launch<T, kRowsKind, 64>(p, stream);
        case 128: return launch<T, kRowsKind, 128>(p, stream);
        default: return launch<T, kRowsKind, 256>(p, stream);
    }
}

template <typename T>
int launch_rows(const KvAttendParams &p, KvRows rows, hipStream_t stream) {
    switch (rows) {
        case kRowsPlain: return launch_dim<T, kRowsPlain>(p, stream);
        case kRowsSq8: return launch_dim<T, kRowsSq8>(p, stream);
        default: return launch_dim<T, kRowsMx4>(p, stream);
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
    const uint64_t most = (uint64_t)kv_compute_units() * token_waves((int)kv_padded_dim(p.c.dim), token_form(p));
    const uint64_t whole = kWholeOfColumn * p.columns * p.c.batch;
    if (p.max_visible <= (whole < kWhole ? kWhole : whole < kMostWhole ? whole : kMostWhole) && !p.weights) return;
    const uint64_t units = (uint64_t)(p.max_visible + kUnit - 1) / kUnit * p.columns * p.c.batch;
    p.workers = (uint32_t)(units < most ? units : most);
    if (!p.workers) p.workers = 1;
}

int launch_kv_token(const KvAttendParams &p, uint32_t type, KvRows rows, hipStream_t stream) {
    return type == kKvBf16 ? launch_rows<__bf16>(p, rows, stream) : launch_rows<_Float16>(p, rows, stream);
}

int launch_kv_finish(const KvAttendParams &params, uint32_t type, KvRows rows, bool prompt, hipStream_t stream) {
    KvAttendParams p = params;
    p.lift = kv_lift(rows == kRowsPlain && type == kKvF16, prompt);
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
