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
// Into a cache of 4-bit rows each 32 dims of a row get a scale of their own (kv_quantize.h).
//
// Copy-bound: 2^k lanes take one (token, head) row of keys and of values, 16 bytes each,
// and a workgroup's rows are tokens side by side, whose rows and scales follow each
// other in a page.  4 prompts of up to 4,096 tokens, 8 heads of 128, into SQ8 (76 MB):
// 21 us (3.7 TB/s; 4 of 16,384 tokens, 405 MB, 81 us, 5.0 TB/s); two tokens a lane 23.
// One token for each of 64 sequences: 2.7 us, a launch.  The prompts into 4-bit rows (54 MB): 13.6 us.
#include "kv_quantize.h"

namespace tessa {

namespace {

constexpr int kThreads = 256;

template <typename T, int kRows>
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
    const uint64_t ks = mine ? kv_scale_place(c, c.keys, page, row, head) : 0, vs = mine ? kv_scale_place(c, c.values, page, row, head) : 0;
    kv_store_row<T, kRows>(c.keys, (uint64_t)kp + (uint64_t)head * c.keys.head_units, ks, k, lane, lanes_log2, mine);
    kv_store_row<T, kRows>(c.values, (uint64_t)vp + (uint64_t)head * c.values.head_units, vs, v, lane, lanes_log2, mine);
}

template <typename T, int kRows>
int launch(const KvAppendParams &p, dim3 grid, uint32_t lanes_log2, uint32_t tokens_log2, hipStream_t stream) {
    kv_append_kernel<T, kRows><<<grid, kThreads, 0, stream>>>(p, lanes_log2, tokens_log2);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <typename T>
int launch_rows(const KvAppendParams &p, KvRows rows, dim3 grid, uint32_t lanes_log2, uint32_t tokens_log2, hipStream_t stream) {
    switch (rows) {
        case kRowsPlain: return launch<T, kRowsPlain>(p, grid, lanes_log2, tokens_log2, stream);
        case kRowsSq8: return launch<T, kRowsSq8>(p, grid, lanes_log2, tokens_log2, stream);
        default: return launch<T, kRowsMx4>(p, grid, lanes_log2, tokens_log2, stream);
    }
}

}  // namespace

int launch_kv_append(const KvAppendParams &p, uint32_t source, KvRows rows, hipStream_t stream) {
    if (p.c.batch == 0 || p.max_new == 0 || p.tokens == 0) return 0;
    uint32_t lanes_log2 = 1;
    while ((8u << lanes_log2) < p.c.dim) ++lanes_log2;
    // tokens side by side, as their rows and scales are in a page; heads too where there are few
    const uint32_t here = (uint32_t)kThreads >> lanes_log2;
    uint32_t tokens_log2 = 0;
    while ((1u << tokens_log2) < here && (1u << tokens_log2) < p.max_new) ++tokens_log2;
    const uint32_t heads_here = here >> tokens_log2;
    const uint64_t blocks = ((uint64_t)p.max_new + (1u << tokens_log2) - 1) >> tokens_log2;
    const dim3 grid((uint32_t)(blocks * ((p.c.heads + heads_here - 1) / heads_here)), p.c.batch);
    return source == kKvBf16 ? launch_rows<__bf16>(p, rows, grid, lanes_log2, tokens_log2, stream)
                             : launch_rows<_Float16>(p, rows, grid, lanes_log2, tokens_log2, stream);
}

}  // namespace tessa
