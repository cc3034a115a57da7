// kv_evict.hip -- eviction from the paged cache by accumulated attention weight.
//
// Of the n rows of a (sequence, head) with n > keep, the first `sinks` and the
// last `recent` stay, and of the others the keep - sinks - recent with the
// largest weights, equal weights by the lower row, NaN below everything.  The
// kept rows, in ascending order, become rows 0.. of the destination pages.  A row
// whose page id names no page is not there: it is never kept, so that no row of the
// destination is counted without having been written.
//
// kv_select_kernel: one workgroup per (sequence, head).  The weights, as
// integers of the same order, go through three histograms in LDS (11, 11 and 10
// bits from the top); the last leaves the exact value of the last kept row and
// how many rows of that value are kept.  A wave owns a contiguous range of rows, so
// ballots and one sum over the waves give each kept row its place, in order
// and without a sort.  Up to 32,768 candidates stay in LDS from one read.  A chain
// of passes over few bytes, latency-bound: 8 sequences of up to 32,768 rows, 8 heads,
// 28 us.  (Weights that are all equal meet in one bin: 68 us more.)
//
// kv_move_kernel: copy-bound (8 x 8,000 rows kept of 8 heads, 128 dims, 16 bits: 524 MB
// read and written in 109 us, 4.8 TB/s).  Into other pages, workgroups share the kept rows
// out; in place, the destination of a row is never after its source, so one
// workgroup walks the rows of one 64-byte column of a (sequence, head) in order,
// reading a batch of rows into registers, waiting for all of it, and writing:
// what a batch writes lies before every source of the later ones.  Columns
// are independent, which is where the parallelism comes from.
#include "kernel_attr.h"
#include "kv_device.h"

namespace tessa {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr uint32_t kSelHeld = 32768;  // candidates held in LDS
constexpr int kSelGroup = 8;      // loads in flight
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;
constexpr int kMovePer = 8;       // rows of a thread in flight
constexpr uint64_t kMoveHere = 65536;

// An integer that orders as the weight does; NaN is 0.
__device__ __forceinline__ uint32_t order_of(float w) {
    uint32_t u = __float_as_uint(w);
    if (w != w) return 0u;
    if (w == 0.0f) u = 0u;  // -0 and 0 are equal
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Sum of sh[i] over i < wave.
__device__ __forceinline__ uint32_t before_wave(const uint32_t *sh, uint32_t wave) {
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves - 1; ++i) sum += (uint32_t)i < wave ? sh[i] : 0u;
    return sum;
}

// The weight of a key (-0 as 0).
__device__ __forceinline__ float weight_of(uint32_t u) {
    return __uint_as_float(u == 0u ? 0x7fc00000u : u >> 31 ? u ^ 0x80000000u : ~u);
}

// The `need` candidates of the largest weights, fewer than there are: places `place`.. of `kept`
// and `out`.  Candidates are the middle rows [sinks, n - recent); with kHoles (a page is
// missing) all rows, of which the first and the last are above every weight and
// those that are not there below NaN.
// Lanes past a wave's last candidate hold the lowest value.  They can at most
// add to the lowest bin and to the ties of the lowest value, after every real
// candidate of theirs, where no row is left to place.
template <bool kHeld, bool kHoles>
__device__ __forceinline__ void select_rows(const KvEvictParams &p, const float *w, const int32_t *table, uint32_t n, uint32_t need,
                                            uint32_t place, int32_t *kept, float *out, uint32_t *held, uint32_t *hist,
                                            uint32_t (*sh_wave)[kSelWaves], uint32_t *sh_pick) {
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const uint32_t skipped = kHoles ? 0u : p.sinks;
    const uint32_t candidates = kHoles ? n : n - p.sinks - p.recent;
    if (need == 0) return;
    // contiguous rows of a wave, whole groups of 64
    const uint32_t span = ((candidates + kSelWaves - 1) / kSelWaves + 63u) / 64u * 64u;
    const uint32_t lo = wave * span, hi = min(lo + span, candidates);
    const uint32_t steps = __builtin_amdgcn_readfirstlane(lo < hi ? (hi - lo + 63u) / 64u : 0u);
    // (loads without a branch, so that a group of them is out at once)
    const float *middle = w + skipped;
    auto load = [&](uint32_t s) { return __float_as_uint(middle[min(lo + s * 64u + lane, candidates - 1u)]); };
    auto order = [&](uint32_t s, uint32_t x) {
        const uint32_t i = lo + s * 64u + lane;
        if (i >= hi) return 0u;
        const uint32_t u = order_of(__uint_as_float(x));
        if constexpr (kHoles) {
            if ((uint32_t)table[i >> p.c.page_shift] >= p.c.pages) return 0u;
            return i < p.sinks || i >= n - p.recent ? 0xffffffffu : max(u, 1u);
        }
        return u;
    };
    // f(step, value) for each of the lane's candidates.  The loops stay loops: unrolled
    // over the 32 steps of 32,768 candidates, each instruction runs once a wave and fetching them takes
    // longer than the work.
    auto each = [&](auto &&value, auto &&f) {
#pragma unroll 1
        for (uint32_t s0 = 0; s0 < steps; s0 += kSelGroup) {
            uint32_t x[kSelGroup];
#pragma unroll
            for (int s = 0; s < kSelGroup; ++s) x[s] = value(s0 + s);
#pragma unroll
            for (int s = 0; s < kSelGroup; ++s) f(s0 + s, x[s]);
        }
    };
    uint32_t *own = held + lo + lane;  // (whole groups of 64 of each wave: span * waves <= kSelHeld)
    auto again = [&](uint32_t s) { return kHeld ? own[min(s, steps - 1u) * 64u] : load(s); };
    auto known = [&](uint32_t s, uint32_t x) { return s >= steps ? 0u : kHeld ? x : order(s, x); };
    // the need-th largest value: three digits from the top
    uint32_t least = 0, left = need;  // digits known so far, kept rows still to place among them
    auto pick = [&](int bits) {       // the digit of the left-th largest value in `hist`
        // bins from the top: thread t has bins 2047 - 2t and 2046 - 2t
        const uint32_t a = hist[kBins - 1 - 2 * t], c = hist[kBins - 2 - 2 * t];
        uint32_t sum = a + c;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t y = __shfl_up(sum, off);
            if (lane >= (uint32_t)off) sum += y;
        }
        if (lane == 63u) sh_wave[0][wave] = sum;
        __syncthreads();
        hist[kBins - 1 - 2 * t] = hist[kBins - 2 - 2 * t] = 0u;  // for the next digit
        const uint32_t before = sum - a - c + before_wave(sh_wave[0], wave);
        if (before < left && left <= before + a + c) {
            const bool first = left <= before + a;
            sh_pick[0] = kBins - 1 - 2 * t - (first ? 0u : 1u);
            sh_pick[1] = left - before - (first ? 0u : a);
        }
        __syncthreads();
        least = (least << bits) | sh_pick[0];
        left = sh_pick[1];
    };
    for (uint32_t i = t; i < kBins; i += kSelThreads) hist[i] = 0u;
    __syncthreads();
    each(load, [&](uint32_t s, uint32_t x) {
        const uint32_t u = order(s, x);
        if (s < steps) {
            if constexpr (kHeld) own[s * 64u] = u;
            atomicAdd(&hist[u >> 21], 1u);
        }
    });
    __syncthreads();
    pick(11);
    each(again, [&](uint32_t s, uint32_t x) {
        const uint32_t u = known(s, x);
        if (s < steps && u >> 21 == least) atomicAdd(&hist[u >> 10 & 2047u], 1u);
    });
    __syncthreads();
    pick(11);
    each(again, [&](uint32_t s, uint32_t x) {
        const uint32_t u = known(s, x);
        if (s < steps && u >> 10 == least) atomicAdd(&hist[u & 1023u], 1u);
    });
    __syncthreads();
    pick(10);

    // rows above it, and equal to it, before each wave's
    uint32_t above = 0, equal = 0;
    each(again, [&](uint32_t s, uint32_t x) {
        const uint32_t u = known(s, x);
        above += __popcll(__ballot(u > least));
        equal += __popcll(__ballot(s < steps && u == least));
    });
    if (lane == 0) {
        sh_wave[0][wave] = above;
        sh_wave[1][wave] = equal;
    }
    __syncthreads();
    const uint32_t equal_before = before_wave(sh_wave[1], wave);
    place += before_wave(sh_wave[0], wave) + min(equal_before, left);
    uint32_t room = left > equal_before ? left - equal_before : 0u;  // ties of this wave that stay
    each(again, [&](uint32_t s, uint32_t x) {
        const uint32_t u = known(s, x);
        uint64_t keep = __ballot(u > least);
        if (room && s < steps) {
            const uint64_t ties = __ballot(u == least);
            if (ties) {
                const uint32_t mine_th = __builtin_amdgcn_mbcnt_hi((uint32_t)(ties >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ties, 0u));
                keep |= __ballot(u == least && mine_th < room);
                const uint32_t used = (uint32_t)__popcll(ties);
                room = room > used ? room - used : 0u;
            }
        }
        if (keep >> lane & 1u) {
            const uint32_t at = place + __builtin_amdgcn_mbcnt_hi((uint32_t)(keep >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)keep, 0u));
            const uint32_t i = lo + s * 64u + lane;
            kept[at] = (int32_t)(skipped + i);
            out[at] = kHoles ? w[i] : weight_of(u);
        }
        place += (uint32_t)__popcll(keep);
    });
}

// Moves rows [first, last) of the kept ones of one (sequence, head): of the keys or the
// values, pieces of 16 bytes from `unit0` on, `units` of them by 2^lanes_log2 lanes of a row.
template <int kThreads>
__device__ __forceinline__ void move_rows(const KvEvictParams &p, const KvArray &a, uint32_t b, uint32_t h, uint32_t first, uint32_t last,
                                          uint32_t row_units, uint32_t unit0, uint32_t units, uint32_t lanes_log2, bool in_place) {
    const KvCacheParams &c = p.c;
    const uint32_t t = threadIdx.x;
    const int32_t *kept = p.kept + ((uint64_t)b * c.heads + h) * p.keep;
    const int32_t *from = c.table + (uint64_t)b * c.table_stride, *to = p.into + (uint64_t)b * p.into_stride;
    const uint32_t lane = t & ((1u << lanes_log2) - 1u), per = kThreads >> lanes_log2;
    const uint32_t unit = unit0 + lane;
    const bool mine = lane < units && unit < row_units;
    const bool scales = a.scales != nullptr && unit == 0;
    char *base = a.rows + ((uint64_t)h * a.head_units + (mine ? unit : 0u)) * 16u;
    const uint32_t into_rows = p.into_columns << c.page_shift;
    last = min(last, into_rows);
    for (uint32_t j0 = first; j0 < last; j0 += per * kMovePer) {
        // one load after the other for all rows of the batch, without a branch between: what
        // is not moved reads the last row's entries and row 0 of page 0
        uint32_t row[kMovePer], dst[kMovePer];
        int32_t src_page[kMovePer], dst_page[kMovePer];
        kv_u4 x[kMovePer];
        float sx[kMovePer];
#pragma unroll
        for (int i = 0; i < kMovePer; ++i) row[i] = (uint32_t)kept[min(j0 + i * per + (t >> lanes_log2), last - 1u)];
#pragma unroll
        for (int i = 0; i < kMovePer; ++i) {
            src_page[i] = from[row[i] >> c.page_shift];
            dst_page[i] = to[min(j0 + i * per + (t >> lanes_log2), last - 1u) >> c.page_shift];
        }
#pragma unroll
        for (int i = 0; i < kMovePer; ++i) {
            const uint32_t j = j0 + i * per + (t >> lanes_log2), src = kv_place(c, a, src_page[i], row[i]);
            dst[i] = j < last && !(in_place && row[i] == j) && src != kKvNoOffset ? kv_place(c, a, dst_page[i], j) : kKvNoOffset;
            x[i] = *reinterpret_cast<const kv_u4 *>(base + (uint64_t)(dst[i] != kKvNoOffset ? src : 0u) * 16u);
            sx[i] = 0.0f;
            if (scales && dst[i] != kKvNoOffset) sx[i] = a.scales[kv_scale_place(c, a, src_page[i], row[i], h)];
        }
        if (in_place) {
            // every row of the batch has arrived before any is written
#pragma unroll
            for (int i = 0; i < kMovePer; ++i) asm volatile("" : "+v"(x[i]), "+v"(sx[i]));
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < kMovePer; ++i) {
            if (dst[i] != kKvNoOffset) {
                if (mine) *reinterpret_cast<kv_u4 *>(base + (uint64_t)dst[i] * 16u) = x[i];
                if (scales) a.scales[kv_scale_place(c, a, dst_page[i], j0 + i * per + (t >> lanes_log2), h)] = sx[i];
            }
        }
    }
}

__global__ __launch_bounds__(kSelThreads) void kv_select_kernel(KvEvictParams p, uint32_t row_units, uint32_t lanes_log2, bool move) {
    extern __shared__ uint32_t sh_held[];
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t sh_wave[2][kSelWaves];
    __shared__ uint32_t sh_pick[2];
    __shared__ uint32_t sh_missing;
    const uint32_t h = blockIdx.x, b = blockIdx.y, t = threadIdx.x;
    const uint32_t n = kv_length(p.c, b);
    const uint64_t bh = (uint64_t)b * p.c.heads + h;
    const float *w = p.weights + (uint64_t)b * p.weight_batch + (uint64_t)h * p.weight_head;
    int32_t *kept = p.kept + bh * p.keep;
    float *out = p.new_weights + bh * p.weight_rows;
    // rows whose page is none
    const int32_t *table = p.c.table + (uint64_t)b * p.c.table_stride;
    const uint32_t table_pages = n ? ((n - 1u) >> p.c.page_shift) + 1u : 0u, page_rows = 1u << p.c.page_shift;
    uint32_t missing = 0;
    for (uint32_t i = t; i < table_pages; i += kSelThreads)
        if ((uint32_t)table[i] >= p.c.pages) missing += min(page_rows, n - i * page_rows);
    const bool holes = __syncthreads_or(missing != 0);
    uint32_t count = min(n, p.keep);
    if (holes) {
        if (t == 0) sh_missing = 0u;
        __syncthreads();
        if (missing) atomicAdd(&sh_missing, missing);
        __syncthreads();
        count = min(n - sh_missing, p.keep);
        select_rows<false, true>(p, w, table, n, count, 0u, kept, out, sh_held, hist, sh_wave, sh_pick);
    } else if (n > p.keep) {
        const uint32_t need = p.keep - p.sinks - p.recent;
        if (n - p.sinks - p.recent <= kSelHeld)
            select_rows<true, false>(p, w, table, n, need, p.sinks, kept, out, sh_held, hist, sh_wave, sh_pick);
        else
            select_rows<false, false>(p, w, table, n, need, p.sinks, kept, out, sh_held, hist, sh_wave, sh_pick);
    }
    // the rows that stay without being asked, and what follows the kept ones (after the
    // selection, whose loads would wait for these stores)
    if (h == 0 && t == 0) p.new_lengths[b] = (int32_t)count;
    const uint32_t first = holes ? 0u : n > p.keep ? p.sinks : n, last = holes || n <= p.keep ? 0u : p.recent;
    for (uint32_t i = t; i < first + last; i += kSelThreads) {
        const uint32_t from = i < first ? i : n - last + (i - first), to = i < first ? i : count - last + (i - first);
        kept[to] = (int32_t)from;
        out[to] = w[from];
    }
    for (uint32_t i = count + t; i < p.keep; i += kSelThreads) kept[i] = -1;
    for (uint32_t i = count + t; i < p.weight_rows; i += kSelThreads) out[i] = 0.0f;
    if (move) {  // few rows: here, without another launch
        const bool in_place = p.into == p.c.table;
        if (in_place && count == n) return;
        __syncthreads();  // the kept rows are listed
        move_rows<kSelThreads>(p, p.c.keys, b, h, 0, count, row_units, 0, row_units, lanes_log2, in_place);
        move_rows<kSelThreads>(p, p.c.values, b, h, 0, count, row_units, 0, row_units, lanes_log2, in_place);
    }
}

// span: rows of a workgroup (in place: all); `columns` workgroups share a row out.
__global__ __launch_bounds__(kMoveThreads) void kv_move_kernel(KvEvictParams p, uint32_t row_units, uint32_t columns, uint32_t units,
                                                               uint32_t lanes_log2, uint32_t span, bool in_place) {
    const uint32_t h = blockIdx.y / (2 * columns), rest = blockIdx.y - h * 2 * columns, b = blockIdx.z;
    const uint32_t n = kv_length(p.c, b), count = (uint32_t)p.new_lengths[b];
    const uint32_t first = blockIdx.x * span, last = min(first + span, count);
    if (first >= last || (in_place && count == n)) return;
    move_rows<kMoveThreads>(p, (rest & 1u) ? p.c.values : p.c.keys, b, h, first, last, row_units, (rest >> 1) * units, units, lanes_log2,
                            in_place);
}

}  // namespace

int launch_kv_evict(const KvEvictParams &p, uint32_t type, hipStream_t stream) {
    if (p.c.batch == 0) return 0;
    // candidates of the longest sequence that lets them be held, in whole groups of 64 a wave
    const uint32_t most = p.c.max_length > p.keep ? p.c.max_length - p.sinks - p.recent : 0u;
    const uint32_t held = most < kSelHeld ? (most + kSelThreads - 1) / kSelThreads * kSelThreads : kSelHeld;
    if (ensure_lds_limit(reinterpret_cast<const void *>(&kv_select_kernel), (int)(kSelHeld * sizeof(uint32_t))) != 0) return -1;
    const bool in_place = p.into == p.c.table;
    const uint32_t row_units = p.c.dim * (type == kKvSq8 ? 1u : 2u) / 16u;
    uint32_t row_lanes_log2 = 0;
    while ((1u << row_lanes_log2) < row_units) ++row_lanes_log2;
    // up to kMoveHere bytes of keys the workgroup that selected the rows moves them too, which saves the
    // host a launch: 256 of 700 rows of 128 bytes, two kernels 7.7 + 7.5 us, one 11.0.  Of 4,096 rows, 8 heads,
    // replayed from a graph, two kernels and one: 2 sequences 512 rows of 128 bytes 14.1, 15.3 us, 16 sequences 18.7,
    // 17.0; at four times the bytes 17.5, 37.0 and 50.5, 80.8
    const bool here = (uint64_t)p.keep * row_units * 16u <= kMoveHere;
    kv_select_kernel<<<dim3(p.c.heads, p.c.batch), kSelThreads, held * sizeof(uint32_t), stream>>>(p, row_units, row_lanes_log2, here);
    if (hipGetLastError() != hipSuccess) return -1;
    if (here) return 0;
    const uint32_t units = in_place ? 4u : row_units;  // 64-byte columns in place, else whole rows
    const uint32_t columns = (row_units + units - 1) / units;
    uint32_t lanes_log2 = 0;
    while ((1u << lanes_log2) < units) ++lanes_log2;
    const uint32_t span = in_place ? p.keep : (uint32_t)(kMoveThreads >> lanes_log2) * kMovePer;
    const dim3 grid((p.keep + span - 1) / span, p.c.heads * 2 * columns, p.c.batch);
    kv_move_kernel<<<grid, kMoveThreads, 0, stream>>>(p, row_units, columns, units, lanes_log2, span, in_place);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tessa
