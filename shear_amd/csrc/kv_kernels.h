// kv_kernels.h -- launch interface of the paged key-value cache's kernels
// (kv_append.hip, kv_token.hip, kv_prompt.hip, kv_evict.hip), shared with the
// ABI (kv_abi.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tessa {

constexpr uint32_t kKvNoOffset = 0xffffffffu;

// One of the cache's two page arrays.  Strides count 16-byte units (rows are
// 16-byte aligned), so that a row's place fits 32 bits in arrays of up to 64 GiB.
struct KvArray {
    char *rows;
    float *scales;                                // SQ8 only
    uint32_t page_units, head_units, row_units;   // 16-byte units between pages, heads, rows
    uint64_t scale_page, scale_head, scale_row;   // floats between them
};

struct KvCacheParams {
    KvArray keys, values;
    const int32_t *table;      // batch x table_stride page ids
    uint64_t table_stride;
    const int32_t *lengths;    // rows of each sequence
    uint32_t batch;
    uint32_t max_length;       // lengths are clipped to it (at most table columns * page rows)
    uint32_t pages, heads, dim, page_shift;
};

struct KvAppendParams {
    KvCacheParams c;           // c.lengths: first row of each sequence's new ones; max_length: rows that the table covers
    const char *k, *v;         // tokens x heads rows of dim 16-bit values
    uint64_t k_token, k_head, v_token, v_head;  // bytes
    const int32_t *offsets;    // batch + 1, or null: one token each
    uint64_t tokens;
    uint32_t max_new;
};

struct KvAttendParams {
    KvCacheParams c;
    const char *q;
    char *out;
    float *lse;                // tokens x q_heads
    uint64_t q_token, q_head, out_token, out_head;  // bytes
    uint32_t q_heads, group;   // group: query heads of a key head
    float scale_log2;          // scale * log2(e)
    float lift;                // of the partial sums: kv_lift()
    uint32_t sinks, window;    // window 0xffffffff: none
    const int32_t *listed;     // batch x heads x listed_count, or null
    uint32_t listed_count;
    float *weights;            // batch x heads x weight_row, or null
    uint64_t weight_batch, weight_head;
    // prompts
    const int32_t *offsets;    // batch + 1
    uint32_t max_new;
    uint64_t tokens;
    // the split over the rows
    uint32_t workers;          // token: workgroups that share all rows out evenly (0: one for each column of rows)
    uint32_t columns;          // token: (head, block of 16 query heads) pairs
    uint32_t chunks;           // prompt: partial results of a query
    uint32_t max_visible;      // token: most visible rows of a sequence
    float *part_o;             // [part][padded dim]; prompt: part = query * chunks + chunk,
                               // token: (column + worker) * query heads of a block + head
    float *part_ml;            // [part][2]: running maximum (base 2), sum
    float *logits;             // token with weights: [batch][heads][max_visible][group], base 2
};

struct KvEvictParams {
    KvCacheParams c;
    const int32_t *into;       // destination table; c.table: in place
    uint64_t into_stride;
    uint32_t into_columns;     // pages of a destination row
    uint32_t keep, sinks, recent;
    const float *weights;      // batch x heads x weight rows
    uint64_t weight_batch, weight_head;
    float *new_weights;        // batch x heads x weight_rows, contiguous
    uint32_t weight_rows;      // columns of new_weights (>= keep)
    int32_t *kept;             // batch x heads x keep
    int32_t *new_lengths;      // batch
};

enum KvType : uint32_t { kKvBf16 = 1, kKvF16 = 2, kKvSq8 = 3 };

uint32_t kv_padded_dim(uint32_t dim);  // 64, 128 or 256
int kv_compute_units();

int launch_kv_append(const KvAppendParams &p, uint32_t source, bool sq8, hipStream_t stream);
void kv_token_split(KvAttendParams &p);
int launch_kv_token(const KvAttendParams &p, uint32_t type, bool sq8, hipStream_t stream);
int launch_kv_finish(const KvAttendParams &params, uint32_t type, bool sq8, bool prompt, hipStream_t stream);
void kv_prompt_split(KvAttendParams &p);
int launch_kv_prompt(const KvAttendParams &p, uint32_t type, bool sq8, hipStream_t stream);
int launch_kv_evict(const KvEvictParams &p, uint32_t type, hipStream_t stream);

}  // namespace tessa
