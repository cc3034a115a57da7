// kv_plan.hip -- the pages and places of a step: which pages sequences give back
// and get, and for each new token its position, sequence and place.
//
// Sequences depend on each other through three running sums (tokens, pages given
// back, pages needed).  Up to 1,024 of them every workgroup forms the sums for itself, in LDS, and takes a
// share of the ids that move and of the tokens: no workgroup waits for what another writes,
// because the stack below its old count and the pages that were held are only read, and an id that this step pushes is found
// where it comes from.  More sequences go through one workgroup 1,024 at a time, and a second launch maps the
// tokens.  A chain of a few reads and scans: 200 sequences
// of one new token each 7.6 us, 96 with 300,000 tokens 12.
#include "kv_device.h"

namespace tessa {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kTokensPer = 4;    // of a thread
constexpr int kMapThreads = 256;
constexpr int kMapPer = 4;            // tokens of a thread
constexpr uint32_t kMapHeld = 4096;   // offsets in LDS
constexpr uint64_t kMostRows = 0x3fffffffu;

// Sum of x over the threads up to this one; total: over all.
__device__ __forceinline__ uint64_t block_sum(uint64_t x, uint64_t *sh, uint64_t &total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint64_t y = __shfl_up(x, off);
        if (lane >= (uint32_t)off) x += y;
    }
    __syncthreads();  // sh has been read
    if (lane == 63u) sh[wave] = x;
    __syncthreads();
    total = 0;
    for (uint32_t w = 0; w < blockDim.x / 64u; ++w) {
        if (w < wave) x += sh[w];
        total += sh[w];
    }
    return x;
}

// The first of `n` ascending sums that is above i.
template <typename S>
__device__ __forceinline__ uint32_t above(const S *sums, uint32_t n, uint64_t i) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2u;
        if ((uint64_t)sums[mid] > i)
            hi = mid;
        else
            lo = mid + 1u;
    }
    return lo;
}

// A token's places, from its index in the step.
__device__ __forceinline__ void map_token(const KvPlanParams &p, uint64_t i, const int32_t *ends, uint32_t b) {
    int32_t position = -1;
    int64_t slot = -1;
    if (b < p.batch) {
        const int64_t at = (int64_t)i - (b ? ends[b - 1] : 0);
        if (at < p.granted[b]) {
            position = p.new_lengths[b] - p.granted[b] + (int32_t)at;
            const int32_t page = p.table[(uint64_t)b * p.table_stride + ((uint32_t)position >> p.page_shift)];
            if (page >= 0) slot = ((int64_t)page << p.page_shift) + (position & ((1 << p.page_shift) - 1));
        }
    }
    p.positions[i] = position;
    p.sequences[i] = b < p.batch ? (int32_t)b : -1;
    p.slots[i] = slot;
}

// Up to kThreads sequences, one of a thread; as few threads as that takes (200 sequences: 9.1 us with 1,024, 7.6 with 256).
__global__ __launch_bounds__(kThreads) void kv_plan_kernel(KvPlanParams p) {
    __shared__ uint64_t sh[2 * kWaves];
    __shared__ uint64_t sh_gives[kThreads], sh_needs[kThreads];  // pages of the sequences up to each
    __shared__ uint64_t sh_taken;
    __shared__ uint32_t sh_end[kThreads];                        // tokens
    __shared__ uint32_t sh_rows[kThreads], sh_granted[kThreads], sh_held[kThreads], sh_target[kThreads];
    const uint32_t t = threadIdx.x;
    const uint64_t covers = min((uint64_t)p.columns << p.page_shift, kMostRows), page_rows = 1ull << p.page_shift;
    const bool mine = t < p.batch;
    const int32_t fresh = mine ? p.fresh[t] : 0;
    const uint64_t rows = mine ? min((uint64_t)max(0, p.lengths[t]), covers) : 0u;
    const uint32_t held = mine ? min((uint32_t)max(0, p.held[t]), p.columns) : 0u;
    const uint64_t count = (uint64_t)max(0, min(*p.count, (int32_t)p.pages));
    const uint64_t n = (uint64_t)max(0, fresh);
    if (t == 0) sh_taken = 0;
    uint64_t all, given, needed;
    const uint64_t upto = block_sum(n, sh, all);
    const uint64_t grow = rows + n <= covers && upto <= p.tokens ? n : 0u;
    const uint32_t target = fresh < 0 ? 0u : (uint32_t)((rows + grow + page_rows - 1u) >> p.page_shift);
    const uint64_t needs = target > held ? target - held : 0u;
    const uint64_t gives_upto = block_sum(held > target ? held - target : 0u, sh, given);
    const uint64_t needs_upto = block_sum(needs, sh, needed);
    const uint64_t available = count + given;
    const bool served = needs == 0u || needs_upto <= available;
    // (who is served is served with all before it, so its pages follow theirs)
    if (served && needs) atomicMax(reinterpret_cast<unsigned long long *>(&sh_taken), (unsigned long long)needs_upto);
    sh_end[t] = (uint32_t)min(upto, (uint64_t)0x7fffffff);
    sh_rows[t] = (uint32_t)rows;
    sh_granted[t] = served ? (uint32_t)grow : 0u;
    sh_held[t] = held;
    sh_target[t] = target;
    sh_gives[t] = gives_upto;
    __syncthreads();
    const uint64_t taken = sh_taken;
    sh_needs[t] = min(needs_upto, taken);
    __syncthreads();
    // the id at place i of the stack after what is given back
    auto page_at = [&](uint64_t i) -> int32_t {
        if (i >= p.pages) return -1;
        if (i < count) return p.free[i];
        const uint32_t x = above(sh_gives, p.batch, i - count);
        return p.table[(uint64_t)x * p.table_stride + sh_target[x] + (i - count - (x ? sh_gives[x - 1] : 0u))];
    };
    const uint64_t first = (uint64_t)blockIdx.x * blockDim.x + t, step = (uint64_t)gridDim.x * blockDim.x;
    if (blockIdx.x == 0) {
        if (mine) {
            p.granted[t] = (int32_t)sh_granted[t];
            p.new_lengths[t] = fresh < 0 ? 0 : (int32_t)(rows + sh_granted[t]);
            p.new_held[t] = (int32_t)(served ? target : held);
            p.offsets[t + 1] = (int32_t)sh_end[t];
        }
        if (t == 0) {
            p.offsets[0] = 0;
            *p.new_count = (int32_t)min(available - taken, (uint64_t)p.pages);
        }
    }
    for (uint64_t i = first; i < given; i += step)
        if (count + i < p.pages) p.free[count + i] = page_at(count + i);
    for (uint64_t i = first; i < taken; i += step) {
        const uint32_t x = above(sh_needs, p.batch, i);
        p.table[(uint64_t)x * p.table_stride + sh_held[x] + (i - (x ? sh_needs[x - 1] : 0u))] = page_at(available - 1u - i);
    }
    for (uint64_t i = first; i < p.tokens; i += step) {
        const uint32_t b = above(sh_end, p.batch, i);
        int32_t position = -1;
        int64_t slot = -1;
        if (b < p.batch) {
            const uint32_t at = (uint32_t)i - (b ? sh_end[b - 1] : 0u);
            if (at < sh_granted[b]) {
                position = (int32_t)(sh_rows[b] + at);
                const uint32_t column = (uint32_t)position >> p.page_shift;
                const int32_t page = column < sh_held[b]
                                         ? p.table[(uint64_t)b * p.table_stride + column]
                                         : page_at(available - 1u - ((b ? sh_needs[b - 1] : 0u) + column - sh_held[b]));
                if (page >= 0) slot = ((int64_t)page << p.page_shift) + (position & ((1 << p.page_shift) - 1));
            }
        }
        p.positions[i] = position;
        p.sequences[i] = b < p.batch ? (int32_t)b : -1;
        p.slots[i] = slot;
    }
}

// Any number of sequences.
__global__ __launch_bounds__(kThreads) void kv_plan_many_kernel(KvPlanParams p) {
    __shared__ uint64_t sh[kWaves];
    __shared__ uint64_t sh_sums[kThreads];  // pages of the sequences up to each
    __shared__ uint32_t sh_from[kThreads];  // the first of its columns that moves
    const uint32_t t = threadIdx.x;
    const uint64_t covers = min((uint64_t)p.columns << p.page_shift, kMostRows), page_rows = 1ull << p.page_shift;
    const uint64_t count = (uint64_t)max(0, min(*p.count, (int32_t)p.pages));
    struct Sequence {
        uint64_t rows, grow, target, held;
        bool ends;
    } s;
    uint64_t tokens = 0;  // before the sequences at hand
    auto look = [&](uint32_t b) {
        const bool there = b < p.batch;
        const int32_t fresh = there ? p.fresh[b] : 0;
        const uint64_t n = (uint64_t)max(0, fresh);
        s.rows = there ? min((uint64_t)max(0, p.lengths[b]), covers) : 0u;
        s.held = there ? (uint64_t)min((uint32_t)max(0, p.held[b]), p.columns) : 0u;
        s.ends = fresh < 0;
        uint64_t all;
        const uint64_t upto = tokens + block_sum(n, sh, all);
        tokens += all;
        s.grow = s.rows + n <= covers && upto <= p.tokens ? n : 0u;
        s.target = s.ends ? 0u : (s.rows + s.grow + page_rows - 1u) >> p.page_shift;
        return upto;
    };
    // pages that are given back
    if (t == 0) p.offsets[0] = 0;
    uint64_t available = count;
    for (uint32_t b0 = 0; b0 < p.batch; b0 += kThreads) {
        const uint32_t b = b0 + t;
        const uint64_t upto = look(b);
        if (b < p.batch) p.offsets[b + 1] = (int32_t)min(upto, (uint64_t)0x7fffffff);
        const uint64_t gives = s.held > s.target ? s.held - s.target : 0u;
        uint64_t all;
        sh_sums[t] = block_sum(gives, sh, all);
        sh_from[t] = (uint32_t)s.target;
        __syncthreads();
        for (uint64_t i = t; i < all; i += kThreads) {
            const uint32_t x = above(sh_sums, kThreads, i);
            const uint64_t column = sh_from[x] + (i - (x ? sh_sums[x - 1] : 0u));
            if (available + i < p.pages) p.free[available + i] = p.table[(uint64_t)(b0 + x) * p.table_stride + column];
        }
        available += all;
        __syncthreads();  // the sums have been read; the ids are written
    }
    // pages that are got
    uint64_t needed = 0, taken = 0;
    tokens = 0;
    for (uint32_t b0 = 0; b0 < p.batch; b0 += kThreads) {
        const uint32_t b = b0 + t;
        look(b);
        const uint64_t needs = s.target > s.held ? s.target - s.held : 0u;
        uint64_t all, got;
        const uint64_t upto = needed + block_sum(needs, sh, all);
        needed += all;
        const bool served = needs == 0u || upto <= available;
        sh_sums[t] = block_sum(served ? needs : 0u, sh, got);
        sh_from[t] = (uint32_t)s.held;
        if (b < p.batch) {
            p.granted[b] = served ? (int32_t)s.grow : 0;
            p.new_lengths[b] = s.ends ? 0 : (int32_t)(s.rows + (served ? s.grow : 0u));
            p.new_held[b] = (int32_t)(served ? s.target : s.held);
        }
        __syncthreads();
        for (uint64_t i = t; i < got; i += kThreads) {
            const uint32_t x = above(sh_sums, kThreads, i);
            const uint64_t column = sh_from[x] + (i - (x ? sh_sums[x - 1] : 0u)), from = available - 1u - taken - i;
            p.table[(uint64_t)(b0 + x) * p.table_stride + column] = from < p.pages ? p.free[from] : -1;
        }
        taken += got;
        __syncthreads();
    }
    if (t == 0) *p.new_count = (int32_t)min(available - taken, (uint64_t)p.pages);
}

// Tokens of the whole card; the offsets lie in LDS where they fit.
__global__ __launch_bounds__(kMapThreads) void kv_map_kernel(KvPlanParams p) {
    __shared__ int32_t sh_ends[kMapHeld];
    const int32_t *ends = p.offsets + 1;
    if (p.batch <= kMapHeld) {
        for (uint32_t b = threadIdx.x; b < p.batch; b += kMapThreads) sh_ends[b] = ends[b];
        __syncthreads();
    }
    for (int j = 0; j < kMapPer; ++j) {
        const uint64_t i = ((uint64_t)blockIdx.x * kMapPer + j) * kMapThreads + threadIdx.x;
        if (i >= p.tokens) return;
        map_token(p, i, ends, p.batch <= kMapHeld ? above(sh_ends, p.batch, i) : above(ends, p.batch, i));
    }
}

}  // namespace

int launch_kv_plan(const KvPlanParams &p, hipStream_t stream) {
    if (p.batch <= (uint32_t)kThreads) {
        const uint32_t threads = p.batch <= 256u ? 256u : p.batch <= 512u ? 512u : (uint32_t)kThreads;
        const uint64_t per = (uint64_t)kTokensPer * threads, blocks = (p.tokens + per - 1) / per, most = 2u * (uint64_t)kv_compute_units();
        kv_plan_kernel<<<(uint32_t)(blocks < 1 ? 1 : blocks < most ? blocks : most), threads, 0, stream>>>(p);
        return hipGetLastError() == hipSuccess ? 0 : -1;
    }
    kv_plan_many_kernel<<<1, kThreads, 0, stream>>>(p);
    if (hipGetLastError() != hipSuccess) return -1;
    if (p.tokens == 0) return 0;
    constexpr uint64_t kPer = (uint64_t)kMapThreads * kMapPer;
    kv_map_kernel<<<(uint32_t)((p.tokens + kPer - 1) / kPer), kMapThreads, 0, stream>>>(p);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tessa
