// kv_prompt.hip -- attention of prompts over the paged cache: the new tokens of
// each sequence, its last rows, attend causally over all of its rows, or over
// the first `sinks` and the last `window` of them.
//
// Per head h of the cache the queries are the pairs (token, one of the G query
// heads), token-major, 128 to a workgroup and 32 to a wave, so that the heads
// of a group share every K and V tile and a short prompt still fills the
// instructions' columns.  Tiles of 64 rows (32 at 256 dims of 16 bits) are staged in LDS twice over: while
// one is worked on, the next comes from memory (its page ids were read a tile
// earlier): 16-bit rows go to the other half without a register, codes through registers.
//
// Bound by the issue of instructions: beside 32 matrix instructions of a wave and
// tile (128 dims) stand some 185 vector ones, most of them the weights', and 130 scalar
// ones (with a window 235 and 155: masks).  No LDS bank conflict was counted.  Two
// prompts of 4,096 tokens, 16 heads over 4 of 128 dims, causal: 154 us,
// 893 TFLOP/s of 1,207 that a product of 8,192^3 reaches; 12,001 tokens with a
// window of 1,024 and 4 first rows: 145 us, 667 TFLOP/s (a workgroup's 32
// tokens see 1,060 rows, its tiles have 1,216).
//  * S^T = K Q^T on 32x32x16 instructions (rows are the tile's, columns the
//    queries): a lane has half of the logits of one query, its partner lane (+- 32) the other
//    half, so the running maximum and sum cost one exchange a tile.
//  * O^T = V^T P^T: the logits' registers are the P^T operand as they
//    stand; V^T comes from LDS by transposing reads of 4 rows x 16 values.
//  * The maximum follows only where a tile's weights would sum to 2^15 times the
//    largest that it was set for (fp16 2^6 times; SQ8: a weight would be that),
//    and tiles that every query of the workgroup sees in full carry no mask.
//  * P is rounded to the queries' type once (an error of the size of the
//    result's own rounding); sums are in f32.  fp16 has nothing between 0 and 2^-24: there
//    the largest weight lies between 2^9 and 2^15, so a weight is right to 11 bits
//    or to 2^-34 of the largest, and many small ones beside a large one add up.
//  * SQ8 rows become 16-bit whole numbers on the way into LDS, exactly; scales
//    enter as in kv_token.hip, the weights in bf16, for fp16 queries as the sum of
//    two parts (one alone would be rounded to 8 bits, the result to 11).
//  * 4-bit rows become 16-bit values on the way into LDS: bf16 with their scales, exactly, and no factor is left for logits
//    or weights.  For fp16 queries keys are fp16 relative to the largest scale of their row, which multiplies the
//    logit; values stay bf16, under weights of two parts.  The two prompts above take 168 us, 84 vector
//    instructions of a wave and tile more than 16-bit rows.
//  * A row that only some queries see may hold infinities or NaN, which would
//    reach the others as 0 * inf.  In tiles with a mask such values go to LDS as zeros,
//    and come back at the end for the queries that see them.
#include <cmath>
#include <type_traits>

#include "kernel_attr.h"
#include "kv_device.h"

namespace tessa {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kQueries = 128;  // of a workgroup

using lds_ptr = __attribute__((address_space(3))) void *;
typedef short kv_s4 __attribute__((ext_vector_type(4)));

// Piece (16 bytes) of an LDS row in which piece c of row r lies: the K reads
// (16 rows, one piece) and the V reads (4 rows, 64 bytes) then meet all banks.
template <int DP>
__device__ __forceinline__ uint32_t k_piece(uint32_t r, uint32_t c) {
    return DP == 64 ? c ^ ((r >> 1) & 7u) : c ^ (r & 15u);
}
template <int DP>
__device__ __forceinline__ uint32_t v_piece(uint32_t r, uint32_t c) {
    return DP == 64 ? c ^ (((r >> 1) & 1u) << 2) : c ^ ((r & 3u) << 2);
}

// 16 bytes a lane from base + offset to LDS, lane after lane from `to` on.  The base is a scalar
// resource and the offset a register of the lane, so no vector instruction forms an
// address.
__device__ __forceinline__ void lds_load(const char *base, uint32_t offset, uint32_t scalar_offset, char *to) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int kReach = 0x7fffffff, kRaw = 0x00027000;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, kReach, kRaw),
                                             (lds_ptr)to, 16, offset, scalar_offset, 0, 0);
#endif
}

// Reads of LDS.  Their pointers are `restrict`, which tells the compiler that no
// load to LDS in flight writes there; through plain pointers it would wait for
// the next tile's loads before the first read of this one.  The kernel itself waits
// for a tile's loads before the barrier after which the tile is read.
template <typename V>
__device__ __forceinline__ V lds_read(const V *__restrict__ at) {
    return *at;
}
__device__ __forceinline__ kv_u2 lds_read_transposed(const char *__restrict__ at) {
    const kv_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) kv_s4 *)const_cast<char *>(at));
    return __builtin_bit_cast(kv_u2, x);
}

template <typename T>
__device__ __forceinline__ bool special_half(uint32_t x) {
    return (x & KvElem<T>::kExponent) == KvElem<T>::kExponent;
}

// Rows of a tile: at 256 dims of 16-bit rows half as many, for the registers' sake.  (Two
// prompts of 4,096 tokens, 16 heads over 4 of 256: 549 us, with 64 rows and spills 1,390;
// SQ8 609 with 64 rows, 742 with 32.  fp16 queries over 4-bit rows spill with 64: 2,449, with 32 821.)
template <typename T, int kRowsKind, int DP>
constexpr uint32_t prompt_rows() {
    return DP == 256 && (kRowsKind == kRowsPlain || (kRowsKind == kRowsMx4 && !std::is_same_v<T, __bf16>)) ? 32u : 64u;
}

template <typename T, int kRowsKind, int DP>
struct PromptLds {
    static constexpr uint32_t kRows = prompt_rows<T, kRowsKind, DP>();
    static constexpr bool kCodes = kRowsKind != kRowsPlain;
    alignas(16) char k[2][kRows * DP * 2];
    alignas(16) char v[2][kRows * DP * 2];
    alignas(16) float scale[kCodes ? 2 : 1][2][kCodes ? kRows : 4];  // of keys (a logit's factor) and values
    // of tile i at i % 4: whether a value was replaced, and the rows without a page.
    // Cleared two tiles ahead, when nothing reads or sets them.
    uint32_t marks[4][1 + kRows / 32];
};

// Zeros that lanes read in the place of rows and dims that are not there.
__device__ __attribute__((aligned(16))) const uint32_t kv_zeros[4] = {0, 0, 0, 0};

// kWhole: each load of the workgroup lies in one page and rows have DP dims, so
// that addresses are one scalar and a lane's constant; chosen where page_rows
// is at least kRowsPer.  (The prompts above: 208 us, with an address of each lane's own 233, before
// the later steps.)
template <typename T, int kRowsKind, int DP, bool kWhole>
__global__ __launch_bounds__(kThreads, DP == 256 ? 1 : 2) void kv_prompt_kernel(KvAttendParams p, uint32_t query_tiles) {
    using E = KvElem<T>;
    constexpr bool kSq8 = kRowsKind == kRowsSq8, kMx4 = kRowsKind == kRowsMx4, kCodes = kSq8 || kMx4;
    using V = std::conditional_t<kCodes, __bf16, T>;  // type of the weights and the values
    using P = KvElem<V>;
    constexpr bool kTwoParts = kCodes && !std::is_same_v<T, __bf16>;
    constexpr bool kHalf = !kCodes && std::is_same_v<T, _Float16>;  // fp16 weights
    // logits get a factor of their row: an SQ8 row's scale, the largest scale of an MX4 row where keys are fp16
    constexpr bool kRowScale = kSq8 || (kMx4 && !std::is_same_v<T, __bf16>);
    // (32 alike rows at the lift sum to 2^5 times it, below the top)
    constexpr float kLift = kv_lift(kHalf, true), kTop = kv_top(kHalf), kMost = kHalf ? 32768.0f : 1.0f;  // kMost = 2^kTop
    using Lds = PromptLds<T, kRowsKind, DP>;
    constexpr uint32_t kRows = Lds::kRows;
    constexpr int kSubs = (int)kRows / 32;       // 32 rows of logits each
    constexpr int kSteps = DP / 16;              // instructions along the dims
    constexpr int kBlocks = DP / 32;             // blocks of 32 dims of the output
    constexpr uint32_t kWide = kMx4 ? 32u : kSq8 ? 16u : 8u;  // dims of a 16-byte piece
    constexpr uint32_t kPieces = DP / kWide;                  // of a row in memory
    // loads of a thread, for K and for V each (MX4, 64 dims: of half of the threads)
    constexpr int kLoads = kRows * kPieces < (uint32_t)kThreads ? 1 : (int)(kRows * kPieces) / kThreads;
    constexpr uint32_t kRowsPer = kThreads / kPieces;  // rows of one load of the workgroup
    constexpr bool kSomeThreads = kRowsPer > kRows;    // (threads past the tile load nothing)
    extern __shared__ __align__(16) char smem[];
    Lds &lds = *reinterpret_cast<Lds *>(smem);

    const KvCacheParams &c = p.c;
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const uint32_t n = lane & 31u, half = lane >> 5;
    // (sequence, head) pairs by eights, one for each XCD, whose L2 then holds its
    // rows; within a pair the last queries, which see most rows, come first
    const uint32_t pairs = c.heads * c.batch, per = query_tiles * p.chunks;
    const uint32_t together = pairs % 8u == 0u ? 8u : pairs;
    const uint32_t group = blockIdx.x / (together * per), in_group = blockIdx.x - group * together * per;
    const uint32_t pair = group * together + in_group % together, item = in_group / together;
    const uint32_t split = item % p.chunks, query_tile = query_tiles - 1u - item / p.chunks;
    const uint32_t b = pair / c.heads, h = pair - b * c.heads;
    const uint32_t length = kv_length(c, b);
    const int64_t first_token = p.offsets[b];
    int64_t new64 = (int64_t)p.offsets[b + 1] - first_token;
    if (first_token < 0 || new64 <= 0 || first_token + new64 > (int64_t)p.tokens) return;
    const uint32_t fresh = min((uint32_t)min(new64, (int64_t)0x7fffffff), p.max_new);
    const uint32_t queries = fresh * p.group;
    const uint32_t q0 = query_tile * kQueries;
    if (q0 >= queries) return;
    // a token's row: those of a sequence are its last; before row 0 (fewer rows than tokens) nothing is seen
    const int32_t row0 = (int32_t)length - (int32_t)fresh;
    const uint32_t my_q = q0 + wave * 32u + n;
    const bool query_ok = my_q < queries;
    const uint32_t my_token = min(my_q, queries - 1u) / p.group;
    const uint32_t my_head = h * p.group + min(my_q, queries - 1u) - my_token * p.group;
    const int32_t pos = row0 + (int32_t)my_token;
    const int32_t pos_first = row0 + (int32_t)(q0 / p.group);
    const int32_t pos_last = row0 + (int32_t)((min(q0 + kQueries, queries) - 1u) / p.group);
    const int32_t wave_last = __builtin_amdgcn_readfirstlane(row0 + (int32_t)(min(q0 + wave * 32u + 31u, queries - 1u) / p.group));
    // rows [0, sinks) and (pos - window, pos]
    const bool windowed = p.window != 0xffffffffu;
    const int32_t window = windowed ? (int32_t)p.window : 0;
    const int32_t sinks = windowed ? (int32_t)p.sinks : 0;
    const int32_t row_end = max(0, pos_last + 1);
    const int32_t row_begin = windowed ? max(0, pos_first - window + 1) : 0;
    const uint32_t sink_tiles = ((uint32_t)min(sinks, row_end) + kRows - 1u) / kRows;
    const uint32_t window_tile = max(sink_tiles, (uint32_t)row_begin / kRows);
    const uint32_t end_tile = ((uint32_t)row_end + kRows - 1u) / kRows;
    const uint32_t all_tiles = sink_tiles + (end_tile > window_tile ? end_tile - window_tile : 0u);
    const uint32_t first_it = (uint32_t)((uint64_t)all_tiles * split / p.chunks);
    const uint32_t last_it = (uint32_t)((uint64_t)all_tiles * (split + 1u) / p.chunks);
    auto tile_row = [&](uint32_t it) { return (it < sink_tiles ? it : window_tile + it - sink_tiles) * kRows; };
    auto masked = [&](uint32_t r0) {  // whether some query of the workgroup does not see all of the tile
        const int32_t lo = (int32_t)r0, hi = lo + (int32_t)kRows - 1;
        return hi > pos_first || (windowed && hi >= sinks && lo <= pos_last - window);
    };

    const int32_t *table = c.table + (uint64_t)b * c.table_stride;
    const char *kbase = c.keys.rows + (uint64_t)h * c.keys.head_units * 16u;
    const char *vbase = c.values.rows + (uint64_t)h * c.values.head_units * 16u;
    // the thread's place in a load of the workgroup: row i * kRowsPer + load_row, piece load_piece of the
    // row in LDS (codes: of the row in memory)
    const uint32_t load_piece = t % kPieces, load_row = t / kPieces;

    kv_u4 qf[kSteps];
    {
        const char *q = p.q + (uint64_t)(first_token + my_token) * p.q_token + (uint64_t)my_head * p.q_head;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = (uint32_t)s * 16u + half * 8u;
            const kv_u4 zero = {0, 0, 0, 0};
            qf[s] = query_ok && d < c.dim ? *reinterpret_cast<const kv_u4 *>(q + 2u * d) : zero;
        }
    }
    float m = kKvNone, l = 0.0f;
    kv_f16 acc[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;

    // bytes of the thread's piece in a load (kWhole); K's order of pieces repeats after 16 rows
    constexpr int kOffsets = kRowsPer >= 16 ? 1 : 16 / (int)kRowsPer;
    uint32_t koffset[kOffsets];
#pragma unroll
    for (int i = 0; i < kOffsets; ++i)
        koffset[i] = (load_row * c.keys.row_units + k_piece<DP>((uint32_t)i * kRowsPer + load_row, load_piece)) * 16u;
    const uint32_t voffset = (load_row * c.values.row_units + v_piece<DP>(load_row, load_piece)) * 16u;

    int32_t pages[kLoads];
    kv_u4 kr[kCodes ? kLoads : 1], vr[kCodes ? kLoads : 1];  // codes on their way to LDS
    float ks = 0.0f, vs = 1.0f;
    const uint32_t kgroup = h * (uint32_t)c.keys.scale_head + load_piece, vgroup = h * (uint32_t)c.values.scale_head + load_piece;
    uint32_t kb[kMx4 ? kLoads : 1], vb[kMx4 ? kLoads : 1];  // scale bytes of the pieces
    bool special = false;  // some value or scale was replaced
    // some maximum is so large that its rounding is felt (from 2^23 on it would be binades of a
    // weight): logits are then rounded as it was, before it is taken from them
    bool huge = false;
    constexpr float kHuge = 4194304.0f;  // 2^22, rounded to a quarter

    // 4-bit rows: a piece becomes four of LDS, which a thread writes from its k_turn-th and v_turn-th on, so that 16 threads'
    // writes meet all banks (a row's order of pieces alone left every fourth of them: two prompts of 4,096 tokens of 256 dims
    // 562 us, so 537; of 128 170 and 168)
    const uint32_t k_turn = DP == 256 ? load_piece >> 2 << 1 : 0u;
    const uint32_t v_turn = (DP == 64 ? load_row >> 1 : DP == 128 ? load_row : (load_piece >> 2) + 2u * load_row) & 3u;
    auto turned_by = [](kv_u4 x, uint32_t by) {
        const kv_u4 y = by & 1u ? kv_u4{x[1], x[2], x[3], x[0]} : x;
        return by & 2u ? kv_u4{y[2], y[3], y[0], y[1]} : y;
    };
    // Page ids for a tile (past the end: those of the last row), read a tile before they are used.
    auto read_pages = [&](uint32_t it) {
        const uint32_t r0 = tile_row(min(it, last_it - 1u));
#pragma unroll
        for (int i = 0; i < kLoads; ++i)  // kWhole: one page for all threads
            pages[i] = table[min(r0 + (uint32_t)i * kRowsPer + (kWhole ? 0u : load_row), length - 1u) >> c.page_shift];
    };
    // Starts the loads of a tile; 16-bit rows go to LDS without a register.
    auto read_rows = [&](uint32_t it, uint32_t buf) {
        const uint32_t r0 = tile_row(it);
        if constexpr (kWhole) {
            const uint32_t page0 = __builtin_amdgcn_readfirstlane(pages[0]);
            if ((1u << c.page_shift) >= kRows && page0 < c.pages) {  // the whole tile lies in one page
                const uint32_t slot = r0 & ((1u << c.page_shift) - 1u);
                const char *kpage = kbase + (uint64_t)(page0 * c.keys.page_units + slot * c.keys.row_units) * 16u;
                const char *vpage = vbase + (uint64_t)(page0 * c.values.page_units + slot * c.values.row_units) * 16u;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const uint32_t at = ((uint32_t)i * kThreads + wave * 64u) * 16u, rows = (uint32_t)i * kRowsPer * 16u;
                    lds_load(kpage, koffset[i & (kOffsets - 1)], rows * c.keys.row_units, lds.k[buf] + at);
                    lds_load(vpage, voffset, rows * c.values.row_units, lds.v[buf] + at);
                }
                return;
            }
            bool all = true;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) all &= (uint32_t)__builtin_amdgcn_readfirstlane(pages[i]) < c.pages;
            if (all) {  // a page for each load; rows past the length are read too: finish_rows() clears their values
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const uint32_t page = __builtin_amdgcn_readfirstlane(pages[i]);
                    const uint32_t slot = (r0 + (uint32_t)i * kRowsPer) & ((1u << c.page_shift) - 1u);
                    const char *kpage = kbase + (uint64_t)(page * c.keys.page_units + slot * c.keys.row_units) * 16u;
                    const char *vpage = vbase + (uint64_t)(page * c.values.page_units + slot * c.values.row_units) * 16u;
                    const uint32_t at = ((uint32_t)i * kThreads + wave * 64u) * 16u;
                    lds_load(kpage, koffset[i & (kOffsets - 1)], 0, lds.k[buf] + at);
                    lds_load(vpage, voffset, 0, lds.v[buf] + at);
                }
                return;
            }
        }
        uint32_t missing = 0;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t r = (uint32_t)i * kRowsPer + load_row;
            const uint32_t row = r0 + r;
            const bool there = row < length && (!kSomeThreads || r < kRows) && (uint32_t)pages[i] < c.pages;
            missing |= (uint32_t)(!there && row < length && (!kSomeThreads || r < kRows)) << i;
            const uint32_t slot = row & ((1u << c.page_shift) - 1u), page = (uint32_t)pages[i];
            const uint64_t kp = (uint64_t)(page * c.keys.page_units + slot * c.keys.row_units);
            const uint64_t vp = (uint64_t)(page * c.values.page_units + slot * c.values.row_units);
            const uint32_t kpiece = kCodes ? load_piece : k_piece<DP>(r, load_piece);
            const uint32_t vpiece = kCodes ? load_piece : v_piece<DP>(r, load_piece);
            const char *zeros = reinterpret_cast<const char *>(kv_zeros);
            const char *ksrc = there && kpiece * kWide < c.dim ? kbase + (kp + kpiece) * 16u : zeros;
            const char *vsrc = there && vpiece * kWide < c.dim ? vbase + (vp + vpiece) * 16u : zeros;
            if constexpr (kMx4) {  // a piece is a group
                kb[i] = vb[i] = 0u;
                if (there && load_piece * kWide < c.dim) {
                    // (scales span less than 4 GiB)
                    kb[i] = kv_group_scales(c.keys)[kgroup + page * (uint32_t)c.keys.scale_page + slot * (uint32_t)c.keys.scale_row];
                    vb[i] = kv_group_scales(c.values)[vgroup + page * (uint32_t)c.values.scale_page + slot * (uint32_t)c.values.scale_row];
                }
            }
            if constexpr (kCodes) {
                kr[i] = *reinterpret_cast<const kv_u4 *>(ksrc);
                vr[i] = *reinterpret_cast<const kv_u4 *>(vsrc);
            } else if constexpr (kWhole) {
                const uint32_t at = ((uint32_t)i * kThreads + t) * 16u;
                *reinterpret_cast<kv_u4 *>(lds.k[buf] + at) = *reinterpret_cast<const kv_u4 *>(ksrc);
                *reinterpret_cast<kv_u4 *>(lds.v[buf] + at) = *reinterpret_cast<const kv_u4 *>(vsrc);
            } else {
                // the wave's 64 pieces land one after the other
                const uint32_t at = ((uint32_t)i * kThreads + wave * 64u) * 16u;
                __builtin_amdgcn_global_load_lds(static_cast<const void *>(ksrc), (lds_ptr)(lds.k[buf] + at), 16, 0, 0);
                __builtin_amdgcn_global_load_lds(static_cast<const void *>(vsrc), (lds_ptr)(lds.v[buf] + at), 16, 0, 0);
            }
        }
        if (missing) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t r = (uint32_t)i * kRowsPer + load_row;
                if (missing >> i & 1u) atomicOr(&lds.marks[it & 3u][1 + r / 32u], 1u << (r & 31u));
            }
        }
        if constexpr (kSq8) {
            if (t < kRows) {
                const uint32_t row = r0 + t;
                const int32_t page = row < length ? table[row >> c.page_shift] : -1;
                ks = 0.0f;
                vs = 1.0f;
                if ((uint32_t)page < c.pages) {
                    ks = kv_row_scales(c.keys)[kv_scale_place(c, c.keys, page, row, h)];
                    vs = kv_row_scales(c.values)[kv_scale_place(c, c.values, page, row, h)];
                }
            }
        }
    };
    // Completes a tile whose loads were started: codes become 16-bit values; in a
    // tile with a mask infinities and NaN become zeros.
    auto finish_rows = [&](uint32_t it, uint32_t buf) {
        if constexpr (kMx4) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t r = (uint32_t)i * kRowsPer + load_row;
                float kscale = kv_mx_scale(kb[i]);
                if constexpr (kRowScale) {
                    // fp16 holds no scale of any size: the row's largest goes to the logit, keys are
                    // relative to it (below 2^-24 of it they vanish: 2^-26 of the row's largest value)
                    uint32_t most = kb[i];
#pragma unroll
                    for (uint32_t off = 1; off < kPieces; off <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, (int)off));
                    const bool nan = most == kMxNan;
                    kscale = kv_mx_scale(nan ? 0x7fu : (uint32_t)max(127 - (int)(most - kb[i]), 0));
                    if (load_piece == 0 && r < kRows)
                        lds.scale[buf][0][r] = nan ? NAN : (most ? kv_mx_scale(most) : __uint_as_float(0x400000u)) * p.scale_log2;
                }
                // NaN would reach those that do not see the row as 0 * NaN
                const bool bad = vb[i] == kMxNan && masked(tile_row(it));
                if (bad) lds.marks[it & 3u][0] = 1u;
                const float vscale = kv_mx_scale(bad ? 0x7fu : vb[i]);
                if (r < kRows) {
                    const kv_u4 kx = turned_by(kr[i], k_turn), vx = turned_by(vr[i], v_turn);
#pragma unroll
                    for (uint32_t w = 0; w < 4; ++w) {
                        const uint32_t kto = 4u * load_piece + ((w + k_turn) & 3u), vto = 4u * load_piece + ((w + v_turn) & 3u);
                        *reinterpret_cast<kv_u4 *>(&lds.k[buf][r * DP * 2 + k_piece<DP>(r, kto) * 16u]) = kv_mx_values<T>(kx[w], kscale);
                        *reinterpret_cast<kv_u4 *>(&lds.v[buf][r * DP * 2 + v_piece<DP>(r, vto) * 16u]) =
                            kv_mx_values<V>(bad ? 0u : vx[w], vscale);
                    }
                }
            }
        } else if constexpr (kSq8) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t r = (uint32_t)i * kRowsPer + load_row;
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    kv_u4 k4, v4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t kw = kr[i][2 * part + e / 2], vw = vr[i][2 * part + e / 2];
                        k4[e] = E::pack_codes(kv_code(kw, 2 * (e & 1)), kv_code(kw, 2 * (e & 1) + 1));
                        v4[e] = P::pack_codes(kv_code(vw, 2 * (e & 1)), kv_code(vw, 2 * (e & 1) + 1));
                    }
                    const uint32_t to = 2u * load_piece + (uint32_t)part;
                    *reinterpret_cast<kv_u4 *>(&lds.k[buf][r * DP * 2 + k_piece<DP>(r, to) * 16u]) = k4;
                    *reinterpret_cast<kv_u4 *>(&lds.v[buf][r * DP * 2 + v_piece<DP>(r, to) * 16u]) = v4;
                }
            }
            if (t < kRows) {
                // a value's NaN scale would reach those that do not see the row as 0 * NaN
                const bool bad = vs != vs && masked(tile_row(it));
                lds.scale[buf][0][t] = ks * p.scale_log2;
                lds.scale[buf][1][t] = bad ? 1.0f : vs;
                if (bad) lds.marks[it & 3u][0] = 1u;
            }
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (masked(tile_row(it))) {
                bool found = false;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    kv_u4 *at = reinterpret_cast<kv_u4 *>(lds.v[buf] + ((uint32_t)i * kThreads + t) * 16u);
                    kv_u4 x = *at;
                    bool hit = false;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const bool lo = special_half<T>(x[w]), hi = special_half<T>(x[w] >> 16);
                        if (lo) x[w] &= 0xffff0000u;
                        if (hi) x[w] &= 0xffffu;
                        hit |= lo | hi;
                    }
                    if (hit) *at = x;
                    found |= hit && tile_row(it) + (uint32_t)i * kRowsPer + load_row < length;
                }
                if (found) lds.marks[it & 3u][0] = 1u;
            }
        }
    };

    if (first_it < last_it) {
        if (t < 4u * (1u + kRows / 32u)) lds.marks[0][t] = 0u;
        read_pages(first_it);
        __syncthreads();  // the marks are cleared
        read_rows(first_it, 0);
        read_pages(first_it + 1);
        finish_rows(first_it, 0);
        __syncthreads();
#pragma unroll
        for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(qf[s]));  // has arrived: no wait for it in the loop
    }
    for (uint32_t it = first_it; it < last_it; ++it) {
        const uint32_t buf = (it - first_it) & 1u;
        const uint32_t r0 = tile_row(it);
        const bool more = it + 1 < last_it;
        if (more) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) asm volatile("" : "+v"(pages[i]));  // their reads had a tile's time
            read_rows(it + 1, buf ^ 1u);
            read_pages(it + 2);
        }
        const bool mask = masked(r0);
        const uint32_t *marks = lds.marks[it & 3u];
        if (t < 1u + kRows / 32u) lds.marks[(it + 2u) & 3u][t] = 0u;
        if ((int32_t)r0 <= wave_last) {  // else the wave's queries see nothing of it
            // logits of rows 32 u + 8 (e / 4) + 4 half + e % 4
            kv_f16 x[kSubs];
#pragma unroll
            for (int u = 0; u < kSubs; ++u) {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[u][e] = 0.0f;
                const uint32_t r = 32u * u + n;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    const kv_u4 a = lds_read(reinterpret_cast<const kv_u4 *>(&lds.k[buf][r * DP * 2 + k_piece<DP>(r, 2u * s + half) * 16u]));
                    x[u] = E::mma32(a, qf[s], x[u]);
                }
            }
            if constexpr (kRowScale) {
#pragma unroll
                for (int u = 0; u < kSubs; ++u)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const uint32_t r = 32u * u + 2u * e + 4u * half;
                        const kv_f4 k4 = lds_read(reinterpret_cast<const kv_f4 *>(&lds.scale[buf][0][r]));
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[u][e + i] *= k4[i];
                    }
            }
            if (mask) {
                // rows relative to the lane's first; opaque, so that the comparisons stay in this branch
                int32_t last = pos - (int32_t)r0 - 4 * (int32_t)half;  // r is seen if last - width < r <= last,
                int32_t shown = min(sinks - (int32_t)r0 - 4 * (int32_t)half, last + 1);  // or below this
                const uint32_t width = windowed ? (uint32_t)window : 0x80000000u;
                asm volatile("" : "+v"(last), "+v"(shown));
                if ((int32_t)r0 < sinks) {
#pragma unroll
                    for (int u = 0; u < kSubs; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int32_t r = 32 * u + 8 * (e / 4) + e % 4;
                            if ((uint32_t)(last - r) >= width && r >= shown) x[u][e] = -INFINITY;
                        }
                } else {
#pragma unroll
                    for (int u = 0; u < kSubs; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int32_t r = 32 * u + 8 * (e / 4) + e % 4;
                            if ((uint32_t)(last - r) >= width) x[u][e] = -INFINITY;
                        }
                }
            }
#pragma unroll
            for (int u = 0; u < kSubs; ++u) {
                uint32_t gone = lds_read(&marks[1 + u]);
                if (__builtin_amdgcn_readfirstlane(gone)) {
                    gone >>= 4u * half;
                    asm volatile("" : "+v"(gone));
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (gone >> (8 * (e / 4) + e % 4) & 1u) x[u][e] = -INFINITY;
                }
            }
            float factor = kRowScale ? 1.0f : p.scale_log2;
            auto scale_first = [&] {
#pragma unroll
                for (int u = 0; u < kSubs; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[u][e] *= factor;
                factor = 1.0f;
            };
            if (!kRowScale && huge) scale_first();
            // The running maximum follows the largest logit.
            auto follow = [&] {
                float top = x[0][0];
#pragma unroll
                for (int u = 0; u < kSubs; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = fmaxf(top, x[u][e]);
                const float higher = fmaxf(m, kv_max32(fmaxf(top * factor - kLift, kKvNone)));
                const float f = kv_exp2(m - higher);
                m = higher;
                l *= f;
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) acc[i] *= f;
            };
            kv_u4 pf[2 * kSubs], rest[kTwoParts ? 2 * kSubs : 1];  // P^T operands of 16 rows each
            float sum;
            if constexpr (kSq8) {
                float top = x[0][0];
#pragma unroll
                for (int u = 0; u < kSubs; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = fmaxf(top, x[u][e]);
                if (__any(kv_max32(top) > m + kTop)) follow();
            }
            // 16-bit rows: the weights are formed with the old maximum, and their sum tells
            // whether it still served (it does but for a sequence's first tiles): a search for
            // the largest logit of every tile would stand between the products and the weights
            for (bool again = false;; again = true) {
                sum = 0.0f;
#pragma unroll
                for (int u = 0; u < kSubs; ++u)
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        float w0 = kv_exp2(fmaf(x[u][e], factor, -m)), w1 = kv_exp2(fmaf(x[u][e + 1], factor, -m));
                        sum += w0 + w1;
                        if constexpr (kSq8) {
                            const uint32_t r = 32u * u + 8u * (e / 4) + 4u * half + e % 4;
                            w0 *= lds_read(&lds.scale[buf][1][r]);
                            w1 *= lds_read(&lds.scale[buf][1][r + 1]);
                        }
                        const uint32_t both = P::pack(w0, w1);
                        pf[2 * u + e / 8][(e % 8) / 2] = both;
                        if constexpr (kTwoParts) rest[2 * u + e / 8][(e % 8) / 2] = P::pack(w0 - P::low(both), w1 - P::high(both));
                    }
                if (kSq8 || again || !__any(!(sum < kMost))) break;
                follow();
                if (!kRowScale && !huge && __any(fabsf(m) >= kHuge && m > kKvNone)) {
                    huge = true;
                    scale_first();
                }
            }
            l += sum;
            // V^T of dims 32 i + n: rows 16 k + 4 half + {0..3}, + 8; read a block ahead
            {
                kv_u4 a[kBlocks][2 * kSubs];
                auto read = [&](int i) {
#pragma unroll
                    for (int k = 0; k < 2 * kSubs; ++k)
#pragma unroll
                        for (int part = 0; part < 2; ++part) {
                            // of its 16-lane group, lane 4 j + q reads values 4 q .. of row j
                            const uint32_t r = 16u * k + 8u * part + 4u * half + ((lane & 15u) >> 2);
                            const uint32_t d = 32u * i + 16u * ((lane >> 4) & 1u) + 4u * (lane & 3u);
                            const kv_u2 y = lds_read_transposed(
                                &lds.v[buf][r * DP * 2 + v_piece<DP>(r, d / 8u) * 16u + (d & 7u) * 2u]);
                            a[i][k][2 * part] = y[0];
                            a[i][k][2 * part + 1] = y[1];
                        }
                };
                read(0);
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) {
                    if (i + 1 < kBlocks) read(i + 1);
#pragma unroll
                    for (int k = 0; k < 2 * kSubs; ++k) {
                        acc[i] = P::mma32(a[i][k], pf[k], acc[i]);
                        if constexpr (kTwoParts) acc[i] = P::mma32(a[i][k], rest[k], acc[i]);
                    }
                }
            }
            if (mask) special |= lds_read(&marks[0]) != 0u;
        }
        if (more) finish_rows(it + 1, buf ^ 1u);
        __syncthreads();
    }
    l = kv_sum32(l);

    // values (SQ8: scales) that were replaced in tiles with a mask, for the queries that see their
    // rows; all tiles' where a sum became NaN under weights that are numbers
    bool lost = false;
    if constexpr (!kCodes) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) lost |= acc[i][e] != acc[i][e];
        lost = __any(lost && l == l);
    }
    if (lost || __any(special)) {
        auto seen = [&](uint32_t row) {
            const int32_t r = (int32_t)row;
            return r <= pos && (!windowed || r < sinks || r > pos - window);
        };
#pragma unroll
        for (int i = 0; i < (kSq8 ? 1 : kBlocks); ++i) {  // (MX4: a block's dims are a group)
            float s[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll 1
            for (uint32_t it = first_it; it < last_it; ++it) {
                const uint32_t r0 = tile_row(it);
                if (!lost && !masked(r0)) continue;
                // the rows that have such values in these dims, a lane for a row
                const uint32_t mine = r0 + lane;
                bool odd = false;
                if (lane < kRows && mine < length) {
                    const int32_t page = table[mine >> c.page_shift];
                    const uint32_t place = kv_place(c, c.values, page, mine);
                    if constexpr (kSq8) {
                        if (place != kKvNoOffset) {
                            const float scale = kv_row_scales(c.values)[kv_scale_place(c, c.values, page, mine, h)];
                            odd = scale != scale;
                        }
                    } else if constexpr (kMx4) {
                        if (place != kKvNoOffset && 32u * i < c.dim)
                            odd = kv_group_scales(c.values)[kv_scale_place(c, c.values, page, mine, h) + i] == kMxNan;
                    } else {
#pragma unroll 1
                        for (uint32_t d = 32u * i; d < min(32u * i + 32u, c.dim) && place != kKvNoOffset; d += 8) {
                            const kv_u4 x = *reinterpret_cast<const kv_u4 *>(vbase + (uint64_t)place * 16u + 2u * d);
#pragma unroll
                            for (int w = 0; w < 4; ++w) odd |= special_half<T>(x[w]) || special_half<T>(x[w] >> 16);
                        }
                    }
                }
                for (uint64_t rows = __ballot(odd); rows; rows &= rows - 1) {
                    const uint32_t row = r0 + (uint32_t)__builtin_ctzll(rows);
                    if constexpr (kCodes) {
                        s[0] = seen(row) ? NAN : s[0];
                    } else {
                        const uint64_t place = kv_place(c, c.values, table[row >> c.page_shift], row);
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const uint32_t d = 32u * i + 2u * (uint32_t)e + 4u * half;
                            const kv_u2 x = *reinterpret_cast<const kv_u2 *>(d < c.dim ? vbase + place * 16u + 2u * d
                                                                                        : reinterpret_cast<const char *>(kv_zeros));
#pragma unroll
                            for (int w = 0; w < 4; ++w) {
                                const float y = kv_not_finite(w & 1 ? E::high(x[w / 2]) : E::low(x[w / 2]));
                                s[e + w] += seen(row) ? y : 0.0f;
                            }
                        }
                    }
                }
            }
            if constexpr (kSq8) {
#pragma unroll
                for (int j = 0; j < kBlocks; ++j) acc[j] += s[0];
            } else if constexpr (kMx4) {
                acc[i] += s[0];
            } else if (l == l) {
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][e] = kv_settled(acc[i][e], s[e]);
            }
        }
    }

    if (!query_ok) return;
    const uint64_t token = (uint64_t)first_token + my_token;
    const uint64_t query = token * p.q_heads + my_head;
    if (p.chunks > 1) {
        float *o = p.part_o + (query * p.chunks + split) * DP;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<kv_f4 *>(o + 32 * i + 2 * e + 4 * half) =
                    kv_f4{acc[i][e], acc[i][e + 1], acc[i][e + 2], acc[i][e + 3]};
        if (half == 0) {
            p.part_ml[(query * p.chunks + split) * 2] = m;
            p.part_ml[(query * p.chunks + split) * 2 + 1] = l;
        }
        return;
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    char *o = p.out + token * p.out_token + (uint64_t)my_head * p.out_head;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const uint32_t d = 32u * i + 2u * e + 4u * half;
            if (d < c.dim) {
                const kv_u2 y = {E::pack(acc[i][e] * r, acc[i][e + 1] * r), E::pack(acc[i][e + 2] * r, acc[i][e + 3] * r)};
                *reinterpret_cast<kv_u2 *>(o + 2u * d) = y;
            }
        }
    if (half == 0) p.lse[query] = kv_lse(m, l, kLift);
}

template <typename T, int kRowsKind, int DP, bool kWhole>
int launch(const KvAttendParams &p, hipStream_t stream) {
    const uint32_t tiles = (uint32_t)(((uint64_t)p.max_new * p.group + kQueries - 1) / kQueries);
    const int lds = (int)sizeof(PromptLds<T, kRowsKind, DP>);
    auto *kernel = &kv_prompt_kernel<T, kRowsKind, DP, kWhole>;
    if (ensure_lds_limit(reinterpret_cast<const void *>(kernel), lds) != 0) return -1;
    kernel<<<tiles * p.chunks * p.c.heads * p.c.batch, kThreads, lds, stream>>>(p, tiles);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <typename T, int kRowsKind, int DP>
int launch_pages(const KvAttendParams &p, hipStream_t stream) {
    if constexpr (kRowsKind == kRowsPlain)
        // (a tile's rows within 2^30 bytes: their offsets are 32-bit)
        if (p.c.dim == DP && (1u << p.c.page_shift) >= kThreads * 8u / DP && p.c.keys.row_units <= 1u << 20 &&
            p.c.values.row_units <= 1u << 20)
            return launch<T, kRowsKind, DP, true>(p, stream);
    return launch<T, kRowsKind, DP, false>(p, stream);
}

template <typename T, int kRowsKind>
int launch_dim(const KvAttendParams &p, hipStream_t stream) {
    switch (kv_padded_dim(p.c.dim)) {
        case 64: return launch_pages<T, kRowsKind, 64>(p, stream);
        case 128: return launch_pages<T, kRowsKind, 128>(p, stream);
        default: return launch_pages<T, kRowsKind, 256>(p, stream);
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

// One workgroup for all rows of its queries where the queries fill the card or the
// rows are few; else the rows are split, into as many parts as keep the card in one
// round and at least 256 rows (4 tiles) each, and the partial results joined.
// Where that saves most: a workgroup alone takes 18.5, 26.5 and 53 ns a row
// at 64, 128 and 256 dims, a join 4 us and 3 ps for each dim of a query's part.
// Measured, 32 heads of 128 dims over 8, us without and with it:
//   1 token over 512 rows 17.7, 13.6; over 4,096 106, 14.6; over 32,768 915, 32.6
//   2 x 256 tokens over 512 rows 20.8, 26.0 (not split); over 2,048 58.8, 49.8; over 4,096 121, 62
void kv_prompt_split(KvAttendParams &p) {
    constexpr float kPartCost = 3e-6f, kJoinCost = 4.0f;  // us
    uint64_t tiles = ((uint64_t)p.max_new * p.group + kQueries - 1) / kQueries * p.c.heads * p.c.batch;
    // 4-bit rows: no more than the tokens there are fill, which are fewer where prompts differ in length (5 of 30 to 301 tokens
    // over a window of 1,500, 24 heads over 8 of 96 dims, fp16: 93 us in whole columns, 61 in two parts)
    if (p.c.mx4) {
        const uint64_t real = ((p.tokens * p.group + kQueries - 1) / kQueries + p.c.batch) * p.c.heads;
        tiles = real < tiles ? real : tiles;
    }
    const uint32_t visible = p.window == 0xffffffffu
                                 ? p.c.max_length
                                 : (uint32_t)min((uint64_t)p.c.max_length, (uint64_t)p.sinks + p.window + kQueries / p.group);
    const uint32_t dp = kv_padded_dim(p.c.dim);
    const uint64_t fill = tiles ? (uint64_t)kv_compute_units() * (dp == 256 ? 1u : 2u) / tiles : 1;
    const uint64_t most = fill < visible / 256u ? fill : visible / 256u;
    const float rows = (dp == 64 ? 0.0185f : dp == 128 ? 0.0265f : 0.053f) * (float)visible;
    const float part = (float)(p.tokens * p.q_heads) * (float)dp * kPartCost, best = std::sqrt(rows / part);
    const uint64_t chunks = best < (float)most ? (uint64_t)best : most;
    p.chunks = chunks > 1 && rows / (float)chunks + (float)chunks * part + kJoinCost < rows ? (uint32_t)chunks : 1u;
}

int launch_kv_prompt(const KvAttendParams &p, uint32_t type, KvRows rows, hipStream_t stream) {
    if (p.tokens == 0 || p.max_new == 0 || p.c.batch == 0) return 0;
    return type == kKvBf16 ? launch_rows<__bf16>(p, rows, stream) : launch_rows<_Float16>(p, rows, stream);
}

}  // namespace tessa
