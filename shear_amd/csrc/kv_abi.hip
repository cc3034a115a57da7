// kv_abi.hip -- the extern "C" entry points of the paged key-value cache
// (include/tessa_hip.h, tessa_kv_*): arguments are checked here, before any
// device work, so that the kernels meet only shapes they are written for.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/tessa_hip.h"
#include "kv_kernels.h"

using namespace tessa;

namespace tessa {

// Compute units of the first device (256 where it cannot be asked): what splits are planned for.
int kv_compute_units() {
    static const int units = [] {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, 0) == hipSuccess && n > 0) return n;
        (void)hipGetLastError();
        return 256;
    }();
    return units;
}

}  // namespace tessa

namespace {

constexpr uint32_t kMaxGrid = 65535;
constexpr uint32_t kMaxGroup = 256;
constexpr uint32_t kMaxRows = 0x3fffffffu;  // rows, new tokens and windows: differences of them fit 32 bits
constexpr uint64_t kScratchAlign = 256;

__attribute__((format(printf, 2, 3))) tessa_status status(int32_t code, const char *fmt, ...) {
    tessa_status s;
    std::memset(&s, 0, sizeof(s));
    s.code = code;
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(s.msg, sizeof(s.msg), fmt, ap);
    va_end(ap);
    return s;
}

tessa_status fine() {
    tessa_status s;
    std::memset(&s, 0, sizeof(s));
    return s;
}

#define KV_INVALID(...) return status(TESSA_ERR_INVALID_ARGUMENT, __VA_ARGS__)
#define KV_UNSUPPORTED(...) return status(TESSA_ERR_UNSUPPORTED, __VA_ARGS__)

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

KvRows rows_kind(uint32_t cache) {
    return cache == TESSA_KV_SQ8 ? kRowsSq8 : cache == TESSA_KV_MX4 ? kRowsMx4 : kRowsPlain;
}

// One page array in 16-byte units; false where a row is misaligned or its place
// would not fit 32 bits.
tessa_status page_array(const tessa_kv_cache &k, const char *what, void *rows, const uint64_t (&strides)[3], void *scales,
                        const uint64_t (&scale_strides)[3], KvArray &out) {
    const uint64_t unit = k.type == TESSA_KV_MX4 ? 32 : k.type == TESSA_KV_SQ8 ? 16 : 8;  // elements of 16 bytes
    if (!rows) KV_INVALID("kv cache: null %s", what);
    if (!aligned16(rows)) KV_INVALID("kv cache: %s are not 16-byte aligned", what);
    uint64_t units[3];
    for (int i = 0; i < 3; ++i) {
        if (strides[i] >= (1ull << 40) || strides[i] % unit != 0)
            KV_INVALID("kv cache: %s stride %llu is not a multiple of 16 bytes", what, (unsigned long long)strides[i]);
        units[i] = strides[i] / unit;
    }
    const uint64_t counts[3] = {k.pages, k.heads, k.page_rows};
    // units are below 2^37 and counts below 2^32: sum them as doubles first
    double last = (double)k.head_dim / (double)unit;
    for (int i = 0; i < 3; ++i) last += (double)units[i] * (double)(counts[i] - 1);
    if (last >= 4294967295.0 || units[0] > 0xffffffffull || units[1] > 0xffffffffull || units[2] > 0xffffffffull)
        KV_UNSUPPORTED("kv cache: %s span more than 64 GiB", what);
    out.rows = static_cast<char *>(rows);
    out.page_units = (uint32_t)units[0];
    out.head_units = (uint32_t)units[1];
    out.row_units = (uint32_t)units[2];
    out.scales = nullptr;
    out.scale_page = out.scale_head = out.scale_row = 0;
    if (k.type == TESSA_KV_SQ8 || k.type == TESSA_KV_MX4) {
        if (!scales) KV_INVALID("kv cache: %s %s need scales", k.type == TESSA_KV_SQ8 ? "SQ8" : "MX4", what);
        double bytes = k.head_dim / 32;
        for (int i = 0; i < 3 && k.type == TESSA_KV_MX4; ++i) {
            if (scale_strides[i] >= (1ull << 40)) KV_INVALID("kv cache: scale stride of %s", what);
            bytes += (double)scale_strides[i] * (double)(counts[i] - 1);
        }
        if (bytes >= 4294967296.0) KV_UNSUPPORTED("kv cache: scales of %s span more than 4 GiB", what);
        out.scales = scales;
        out.scale_page = scale_strides[0];
        out.scale_head = scale_strides[1];
        out.scale_row = scale_strides[2];
    }
    return fine();
}

// Whether an MX4 row's scales lie together in a word that may be read as one.
bool word_scales(const tessa_kv_cache &k, const void *scales, const uint64_t (&strides)[3]) {
    const uint64_t word = k.head_dim / 32;
    if (word != 2 && word != 4 && word != 8) return false;
    return ((reinterpret_cast<uintptr_t>(scales) | strides[0] | strides[1] | strides[2]) & (word - 1)) == 0;
}

tessa_status pages_of(const tessa_kv_cache *k, KvCacheParams &c) {
    if (!k) KV_INVALID("kv cache: null pointer");
    if (k->type != TESSA_KV_MX4 && (k->type < TESSA_KV_BF16 || k->type > TESSA_KV_SQ8))
        KV_INVALID("kv cache: unknown type %u", k->type);
    if (!k->pages || !k->heads) KV_INVALID("kv cache: %u pages, %u heads", k->pages, k->heads);
    if (k->pages > 0x7fffffffu || k->heads > 1024u) KV_UNSUPPORTED("kv cache: %u pages, %u heads", k->pages, k->heads);
    if (!k->page_rows || (k->page_rows & (k->page_rows - 1u)) || k->page_rows > 65536u)
        KV_INVALID("kv cache: page_rows must be a power of two in 1..=65536, got %u", k->page_rows);
    if (!k->head_dim || k->head_dim % 16u || k->head_dim > 256u)
        KV_UNSUPPORTED("kv cache: head_dim must be a multiple of 16 in 16..=256, got %u", k->head_dim);
    if (k->type == TESSA_KV_MX4 && k->head_dim % 32u)
        KV_UNSUPPORTED("kv cache: MX4 head_dim must be a multiple of 32, got %u", k->head_dim);
    tessa_status st = page_array(*k, "keys", k->keys, k->key_strides, k->key_scales, k->key_scale_strides, c.keys);
    if (st.code) return st;
    st = page_array(*k, "values", k->values, k->value_strides, k->value_scales, k->value_scale_strides, c.values);
    if (st.code) return st;
    c.pages = k->pages;
    c.heads = k->heads;
    c.dim = k->head_dim;
    c.page_shift = (uint32_t)__builtin_ctz(k->page_rows);
    c.mx4 = k->type == TESSA_KV_MX4;
    c.scales_together = c.mx4 && word_scales(*k, k->key_scales, k->key_scale_strides) &&
                        word_scales(*k, k->value_scales, k->value_scale_strides);
    return fine();
}

tessa_status cache_of(const tessa_kv_cache *k, const tessa_kv_sequences *s, KvCacheParams &c) {
    if (!k || !s) KV_INVALID("kv cache: null pointer");
    const tessa_status st = pages_of(k, c);
    if (st.code) return st;
    if (s->batch > kMaxGrid) KV_UNSUPPORTED("kv cache: batch %u over %u", s->batch, kMaxGrid);
    if (s->batch && (!s->lengths || (s->columns && !s->table))) KV_INVALID("kv cache: null table or lengths");
    if (s->batch > 1 && s->table_stride < s->columns)
        KV_INVALID("kv cache: table stride %llu below %u columns", (unsigned long long)s->table_stride, s->columns);
    const uint64_t covers = (uint64_t)s->columns * k->page_rows;
    if (s->max_length > kMaxRows) KV_UNSUPPORTED("kv cache: max_length %u over %u", s->max_length, kMaxRows);
    if (s->max_length > covers)
        KV_INVALID("kv cache: max_length %u over the %llu rows that the table covers", s->max_length, (unsigned long long)covers);
    c.table = s->table;
    c.table_stride = s->table_stride;
    c.lengths = s->lengths;
    c.batch = s->batch;
    c.max_length = s->max_length;
    return fine();
}

// The 16-bit type of q, k, v: the cache's own, or either for a cache of codes.
tessa_status own_type(uint32_t cache, uint32_t type) {
    if (type != TESSA_KV_BF16 && type != TESSA_KV_F16) KV_INVALID("kv: type %u is neither bf16 nor fp16", type);
    if (rows_kind(cache) == kRowsPlain && cache != type) KV_INVALID("kv: type %u over a cache of type %u", type, cache);
    return fine();
}

tessa_status rows_of(const char *what, const void *rows, const uint64_t (&strides)[2], uint64_t (&bytes)[2]) {
    if (!rows) KV_INVALID("kv: null %s", what);
    if (!aligned16(rows) || strides[0] % 8 || strides[1] % 8) KV_INVALID("kv: rows of %s are not 16-byte aligned", what);
    if (strides[0] >= (1ull << 60) || strides[1] >= (1ull << 60)) KV_INVALID("kv: stride of %s", what);
    bytes[0] = strides[0] * 2;
    bytes[1] = strides[1] * 2;
    return fine();
}

uint64_t round_up(uint64_t n) { return (n + kScratchAlign - 1) / kScratchAlign * kScratchAlign; }

// Arguments of both attention calls and the split that they will run with.
tessa_status attend_of(const tessa_kv_cache *cache, const tessa_kv_sequences *seq, const tessa_kv_attend *a, bool prompt,
                       KvAttendParams &p, uint64_t &part_o, uint64_t &part_ml, uint64_t &logits) {
    std::memset(&p, 0, sizeof(p));
    part_o = part_ml = logits = 0;
    if (!a) KV_INVALID("kv attend: null pointer");
    tessa_status st = cache_of(cache, seq, p.c);
    if (st.code) return st;
    st = own_type(cache->type, a->type);
    if (st.code) return st;
    if (!a->q_heads || a->q_heads % p.c.heads) KV_INVALID("kv attend: %u query heads over %u heads", a->q_heads, p.c.heads);
    p.q_heads = a->q_heads;
    p.group = a->q_heads / p.c.heads;
    if (p.group > kMaxGroup) KV_UNSUPPORTED("kv attend: %u query heads share one head, at most %u", p.group, kMaxGroup);
    if (!(a->scale > 0.0f) || !std::isfinite(a->scale)) KV_INVALID("kv attend: scale must be positive and finite");
    p.scale_log2 = a->scale * 1.44269504088896341f;
    if (!(p.scale_log2 > 0.0f) || !std::isfinite(p.scale_log2)) KV_INVALID("kv attend: scale %g", (double)a->scale);
    p.sinks = a->sinks;
    p.window = a->window == TESSA_KV_ALL || a->window < kMaxRows ? a->window : kMaxRows;
    if (p.sinks > kMaxRows) KV_INVALID("kv attend: %u sinks", p.sinks);
    p.tokens = a->tokens;
    if (a->tokens) {
        uint64_t b[2];
        st = rows_of("q", a->q, a->q_strides, b);
        if (st.code) return st;
        p.q = static_cast<const char *>(a->q);
        p.q_token = b[0];
        p.q_head = b[1];
        st = rows_of("out", a->out, a->out_strides, b);
        if (st.code) return st;
        p.out = static_cast<char *>(a->out);
        p.out_token = b[0];
        p.out_head = b[1];
        if (!a->lse) KV_INVALID("kv attend: null lse");
        p.lse = a->lse;
    }
    if (a->tokens * a->q_heads > 0x7fffffffull || a->tokens > kMaxRows)
        KV_UNSUPPORTED("kv attend: %llu tokens of %u heads", (unsigned long long)a->tokens, a->q_heads);
    const uint64_t dp = kv_padded_dim(p.c.dim);
    if (!prompt && a->tokens != p.c.batch)
        KV_INVALID("kv attend: %llu tokens for %u sequences", (unsigned long long)a->tokens, p.c.batch);
    if (a->tokens && !p.c.batch) KV_INVALID("kv attend: %llu tokens of no sequence", (unsigned long long)a->tokens);
    p.chunks = 1;
    if (!a->tokens || !p.c.batch) return fine();
    if (prompt) {
        if (a->listed || a->listed_count || a->weights) KV_INVALID("kv attend: a prompt takes no list and no weights");
        if (!a->offsets) KV_INVALID("kv attend: null offsets");
        p.offsets = a->offsets;
        p.max_new = a->max_new < a->tokens ? a->max_new : (uint32_t)a->tokens;
        kv_prompt_split(p);
        if ((double)((uint64_t)p.max_new * p.group / 128 + 1) * p.chunks * p.c.heads * p.c.batch >= 2147483647.0)
            KV_UNSUPPORTED("kv attend: %u new tokens for each of %u sequences", p.max_new, p.c.batch);
    } else {
        if (a->offsets) KV_INVALID("kv attend: single tokens take no offsets");
        if ((a->listed == nullptr) != (a->listed_count == 0)) KV_INVALID("kv attend: listed and listed_count go together");
        if (a->listed && p.window == TESSA_KV_ALL) KV_INVALID("kv attend: a list needs a window (every row is visible)");
        p.listed = a->listed;
        p.listed_count = a->listed_count;
        p.weights = a->weights;
        p.weight_batch = a->weight_strides[0];
        p.weight_head = a->weight_strides[1];
        if (a->weights) {  // sums are read and written back: no two rows may be one place
            const uint64_t n[2] = {p.c.batch, p.c.heads}, rows = p.c.max_length;
            const int inner = n[1] <= 1 || (n[0] > 1 && a->weight_strides[0] < a->weight_strides[1]) ? 0 : 1;
            const uint64_t near = a->weight_strides[inner], far = a->weight_strides[1 - inner];
            if (near >= (1ull << 40) || far >= (1ull << 40) || (n[inner] > 1 && near < rows) ||
                (n[1 - inner] > 1 && far < near * (n[inner] - 1) + rows))
                KV_INVALID("kv attend: weight strides %llu and %llu for %u rows", (unsigned long long)a->weight_strides[0],
                           (unsigned long long)a->weight_strides[1], p.c.max_length);
        }
        const uint64_t shown = p.window == TESSA_KV_ALL ? p.c.max_length : (uint64_t)p.sinks + p.window;
        const uint64_t visible = (shown < p.c.max_length ? shown : p.c.max_length) + p.listed_count;
        if (visible > 0x7fffffffull) KV_UNSUPPORTED("kv attend: %llu visible rows", (unsigned long long)visible);
        p.max_visible = (uint32_t)visible;
        kv_token_split(p);
        const uint64_t blocks = (visible + 255) / 256 * p.c.heads * p.c.batch + a->tokens * a->q_heads * 4u;
        if (blocks > 0x7fffffffull) KV_UNSUPPORTED("kv attend: batch %u of %llu rows", p.c.batch, (unsigned long long)visible);
        if (p.weights) logits = round_up(visible * p.c.heads * p.c.batch * p.group * sizeof(float));
    }
    uint64_t parts = prompt && p.chunks > 1 ? a->tokens * a->q_heads * p.chunks : 0;
    if (!prompt && p.workers)
        parts = ((uint64_t)p.columns * p.c.batch + p.workers) * (p.group < 16u ? p.group : 16u);
    if (parts) {
        part_o = round_up(parts * dp * sizeof(float));
        part_ml = round_up(parts * 2 * sizeof(float));
    }
    return fine();
}

tessa_status attend_scratch(const tessa_kv_cache *cache, const tessa_kv_sequences *seq, const tessa_kv_attend *a, bool prompt,
                            uint64_t *bytes) {
    if (!bytes) KV_INVALID("kv attend: null pointer");
    *bytes = 0;
    KvAttendParams p;
    uint64_t o, ml, logits;
    const tessa_status st = attend_of(cache, seq, a, prompt, p, o, ml, logits);
    if (!st.code) *bytes = o + ml + logits;
    return st;
}

tessa_status attend(const tessa_kv_cache *cache, const tessa_kv_sequences *seq, const tessa_kv_attend *a, bool prompt, void *scratch,
                    uint64_t bytes, void *stream) {
    KvAttendParams p;
    uint64_t o, ml, logits;
    const tessa_status st = attend_of(cache, seq, a, prompt, p, o, ml, logits);
    if (st.code) return st;
    if (!a->tokens || !p.c.batch) return fine();
    if (bytes < o + ml + logits) {
        return status(TESSA_ERR_INVALID_ARGUMENT, "kv attend: %llu bytes of scratch, %llu needed", (unsigned long long)bytes,
                      (unsigned long long)(o + ml + logits));
    }
    if (o) {
        if (!scratch || !aligned16(scratch)) KV_INVALID("kv attend: scratch is null or not 16-byte aligned");
        char *at = static_cast<char *>(scratch);
        p.part_o = reinterpret_cast<float *>(at);
        p.part_ml = reinterpret_cast<float *>(at + o);
        if (logits) p.logits = reinterpret_cast<float *>(at + o + ml);
    }
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const KvRows rows = rows_kind(cache->type);
    int rc = prompt ? launch_kv_prompt(p, a->type, rows, s) : launch_kv_token(p, a->type, rows, s);
    if (rc == 0 && o) rc = launch_kv_finish(p, a->type, rows, prompt, s);
    if (rc) return status(TESSA_ERR_HIP, "kv attend: launch failed");
    return fine();
}

// Whether the arrays of a step lie apart: workgroups read the arguments, and the table's held pages and the stack,
// while others write, so what is written may share no memory with anything else.
tessa_status apart(const tessa_kv_step &s) {
    struct Array {
        const char *name;
        const void *at;
        uint64_t bytes;
    };
    const uint64_t each = 4ull * s.batch, places = 4ull * s.tokens;
    constexpr int kWritten = 9;
    const Array arrays[] = {{"free", s.free, 4ull * s.pages},       {"new_lengths", s.new_lengths, each},
                            {"new_held", s.new_held, each},         {"new_count", s.new_count, 4},
                            {"granted", s.granted, each},           {"offsets", s.offsets, each + 4},
                            {"positions", s.positions, places},     {"sequences", s.sequences, places},
                            {"slots", s.slots, 2 * places},         {"lengths", s.lengths, each},
                            {"held", s.held, each},                 {"fresh", s.fresh, each},
                            {"count", s.count, 4}};
    constexpr int kArrays = sizeof(arrays) / sizeof(arrays[0]);
    const uintptr_t table = reinterpret_cast<uintptr_t>(s.table);
    const uint64_t row = 4ull * s.columns, stride = 4ull * s.table_stride;
    if (s.batch > 1 && s.table_stride >= (1ull << 40)) KV_INVALID("kv plan: table stride %llu", (unsigned long long)s.table_stride);
    for (int i = 0; i < kArrays; ++i) {
        const uintptr_t from = reinterpret_cast<uintptr_t>(arrays[i].at), to = from + arrays[i].bytes;
        if (!arrays[i].bytes) continue;
        for (int j = 0; j < i && j < kWritten; ++j) {
            const uintptr_t other = reinterpret_cast<uintptr_t>(arrays[j].at);
            if (from < other + arrays[j].bytes && other < to)
                KV_INVALID("kv plan: %s overlap %s: results may not be the arguments", arrays[j].name, arrays[i].name);
        }
        if (!row) continue;
        // (other arrays may lie between the table's rows) the first of them that ends behind the array's begin
        const uint64_t first = from < table + row || s.batch <= 1 ? 0 : (from - table - row) / stride + 1;
        if (first < s.batch && table + first * stride < to && from < table + first * stride + row)
            KV_INVALID("kv plan: the table overlaps %s: results may not be the arguments", arrays[i].name);
    }
    return fine();
}

// The C boundary: nothing is thrown across it.
template <typename F>
tessa_status guarded(F &&f) {
    try {
        return f();
    } catch (...) {
        return status(TESSA_ERR_OUT_OF_MEMORY, "kv: no host memory");
    }
}

}  // namespace

extern "C" {

tessa_status tessa_kv_append(const tessa_kv_cache *cache, const tessa_kv_sequences *seq, const tessa_kv_tokens *tokens, void *stream) {
    return guarded([&]() -> tessa_status {
        if (!tokens) KV_INVALID("kv append: null pointer");
        KvAppendParams p;
        std::memset(&p, 0, sizeof(p));
        tessa_status st = cache_of(cache, seq, p.c);
        if (st.code) return st;
        st = own_type(cache->type, tokens->type);
        if (st.code) return st;
        if (!tokens->offsets && tokens->tokens != seq->batch)
            KV_INVALID("kv append: %llu tokens for %u sequences without offsets", (unsigned long long)tokens->tokens, seq->batch);
        if (!tokens->tokens || !seq->batch) return fine();
        if (tokens->tokens > 0x7fffffffull) KV_UNSUPPORTED("kv append: %llu tokens", (unsigned long long)tokens->tokens);
        uint64_t b[2];
        st = rows_of("k", tokens->k, tokens->k_strides, b);
        if (st.code) return st;
        p.k = static_cast<const char *>(tokens->k);
        p.k_token = b[0];
        p.k_head = b[1];
        st = rows_of("v", tokens->v, tokens->v_strides, b);
        if (st.code) return st;
        p.v = static_cast<const char *>(tokens->v);
        p.v_token = b[0];
        p.v_head = b[1];
        p.offsets = tokens->offsets;
        p.tokens = tokens->tokens;
        p.max_new = tokens->offsets ? tokens->max_new : 1u;
        if (p.max_new > tokens->tokens) p.max_new = (uint32_t)tokens->tokens;
        // 2^5 lanes a row at most, 256 threads a workgroup
        if ((uint64_t)p.max_new * p.c.heads / 8 + 1 > 0x7fffffffull) KV_UNSUPPORTED("kv append: %u new tokens", p.max_new);
        if (launch_kv_append(p, tokens->type, rows_kind(cache->type), reinterpret_cast<hipStream_t>(stream)))
            return status(TESSA_ERR_HIP, "kv append: launch failed");
        return fine();
    });
}

tessa_status tessa_kv_attend_token_scratch(const tessa_kv_cache *cache, const tessa_kv_sequences *seq, const tessa_kv_attend *a,
                                           uint64_t *bytes) {
    return guarded([&] { return attend_scratch(cache, seq, a, false, bytes); });
}

tessa_status tessa_kv_attend_token(const tessa_kv_cache *cache, const tessa_kv_sequences *seq, const tessa_kv_attend *a, void *scratch,
                                   uint64_t bytes, void *stream) {
    return guarded([&] { return attend(cache, seq, a, false, scratch, bytes, stream); });
}

tessa_status tessa_kv_attend_prompt_scratch(const tessa_kv_cache *cache, const tessa_kv_sequences *seq, const tessa_kv_attend *a,
                                            uint64_t *bytes) {
    return guarded([&] { return attend_scratch(cache, seq, a, true, bytes); });
}

tessa_status tessa_kv_attend_prompt(const tessa_kv_cache *cache, const tessa_kv_sequences *seq, const tessa_kv_attend *a, void *scratch,
                                    uint64_t bytes, void *stream) {
    return guarded([&] { return attend(cache, seq, a, true, scratch, bytes, stream); });
}

tessa_status tessa_kv_evict(const tessa_kv_cache *cache, const tessa_kv_sequences *seq, const tessa_kv_eviction *e, void *stream) {
    return guarded([&]() -> tessa_status {
        if (!e) KV_INVALID("kv evict: null pointer");
        KvEvictParams p;
        std::memset(&p, 0, sizeof(p));
        const tessa_status st = cache_of(cache, seq, p.c);
        if (st.code) return st;
        if (!e->keep || (uint64_t)e->sinks + e->recent > e->keep)
            KV_INVALID("kv evict: keep %u must be positive and at least sinks %u + recent %u", e->keep, e->sinks, e->recent);
        if (e->keep > 0x7fffffffu) KV_UNSUPPORTED("kv evict: keep %u", e->keep);
        if (!seq->batch) return fine();
        if (!e->weights || !e->new_weights || !e->kept || !e->new_lengths) KV_INVALID("kv evict: null pointer");
        if (e->weights == e->new_weights) KV_INVALID("kv evict: new_weights are the weights");
        if (e->new_lengths == seq->lengths) KV_INVALID("kv evict: new_lengths are the lengths");
        if (e->weight_rows < e->keep) KV_INVALID("kv evict: %u weight rows below keep %u", e->weight_rows, e->keep);
        if (e->into) {
            if (seq->batch > 1 && e->into_stride < e->into_columns)
                KV_INVALID("kv evict: table stride %llu below %u columns", (unsigned long long)e->into_stride, e->into_columns);
            const uint64_t need = e->keep < seq->max_length ? e->keep : seq->max_length;
            if ((uint64_t)e->into_columns * cache->page_rows < need)
                KV_INVALID("kv evict: %u pages of %u rows for %llu kept rows", e->into_columns, cache->page_rows,
                           (unsigned long long)need);
        }
        p.into = e->into ? e->into : seq->table;
        p.into_stride = e->into ? e->into_stride : seq->table_stride;
        // (pages past the kept rows' are not used; their rows need not fit 32 bits)
        const uint32_t used = (e->keep - 1u) / cache->page_rows + 1u, given = e->into ? e->into_columns : seq->columns;
        p.into_columns = used < given ? used : given;
        p.keep = e->keep;
        p.sinks = e->sinks;
        p.recent = e->recent;
        p.weights = e->weights;
        p.weight_batch = e->weight_strides[0];
        p.weight_head = e->weight_strides[1];
        p.new_weights = e->new_weights;
        p.weight_rows = e->weight_rows;
        p.kept = e->kept;
        p.new_lengths = e->new_lengths;
        if (launch_kv_evict(p, cache->type, reinterpret_cast<hipStream_t>(stream)))
            return status(TESSA_ERR_HIP, "kv evict: launch failed");
        return fine();
    });
}

tessa_status tessa_kv_append_rotated(const tessa_kv_cache *cache, const tessa_kv_rotated *t, void *stream) {
    return guarded([&]() -> tessa_status {
        if (!t) KV_INVALID("kv append rotated: null pointer");
        KvRotateParams p;
        std::memset(&p, 0, sizeof(p));
        tessa_status st = pages_of(cache, p.c);
        if (st.code) return st;
        st = own_type(cache->type, t->type);
        if (st.code) return st;
        if (!t->q_heads || t->q_heads > kMaxGroup * 1024u) KV_INVALID("kv append rotated: %u query heads", t->q_heads);
        if (t->rotated % 16u || t->rotated > p.c.dim)
            KV_INVALID("kv append rotated: rotated dims must be a multiple of 16 up to %u, got %u", p.c.dim, t->rotated);
        if (t->rotated && !t->frequencies) KV_INVALID("kv append rotated: null frequencies");
        if ((reinterpret_cast<uintptr_t>(t->frequencies) & 7u) != 0) KV_INVALID("kv append rotated: frequencies are not 8-byte aligned");
        if (t->weight_type != t->type && t->weight_type != TESSA_KV_F32)
            KV_INVALID("kv append rotated: weights of type %u for tokens of type %u", t->weight_type, t->type);
        if (!aligned16(t->q_weight) || !aligned16(t->k_weight)) KV_INVALID("kv append rotated: weights are not 16-byte aligned");
        if (!(t->eps >= 0.0f) || !std::isfinite(t->eps)) KV_INVALID("kv append rotated: eps must be finite and not negative");
        if (!t->tokens) return fine();
        const uint64_t rows = (uint64_t)t->q_heads + 2u * p.c.heads;
        if (t->tokens > kMaxRows || t->tokens * rows > 0x7fffffffull)
            KV_UNSUPPORTED("kv append rotated: %llu tokens of %llu rows", (unsigned long long)t->tokens, (unsigned long long)rows);
        uint64_t b[2];
        st = rows_of("q", t->q, t->q_strides, b);
        if (st.code) return st;
        p.q = static_cast<const char *>(t->q);
        p.q_token = b[0];
        p.q_head = b[1];
        st = rows_of("k", t->k, t->k_strides, b);
        if (st.code) return st;
        p.k = static_cast<const char *>(t->k);
        p.k_token = b[0];
        p.k_head = b[1];
        st = rows_of("v", t->v, t->v_strides, b);
        if (st.code) return st;
        p.v = static_cast<const char *>(t->v);
        p.v_token = b[0];
        p.v_head = b[1];
        st = rows_of("out", t->out, t->out_strides, b);
        if (st.code) return st;
        p.out = static_cast<char *>(t->out);
        p.out_token = b[0];
        p.out_head = b[1];
        // (a row of out may be written before another workgroup has read its rows of k and v)
        if (t->out == t->k || t->out == t->v) KV_INVALID("kv append rotated: out may be q, but not k or v");
        if (t->out == t->q && (p.out_token != p.q_token || (t->q_heads > 1 && p.out_head != p.q_head)))
            KV_INVALID("kv append rotated: out is q with other strides");
        if (p.q_head > 0xffffffffull || p.k_head > 0xffffffffull || p.v_head > 0xffffffffull || p.out_head > 0xffffffffull)
            KV_UNSUPPORTED("kv append rotated: heads lie more than 4 GiB apart");
        if (!t->positions || !t->slots) KV_INVALID("kv append rotated: null positions or slots");
        p.positions = t->positions;
        p.slots = t->slots;
        p.frequencies = t->frequencies;
        p.q_weight = t->q_weight;
        p.k_weight = t->k_weight;
        p.tokens = t->tokens;
        p.q_heads = t->q_heads;
        p.half = t->rotated / 2;
        p.eps = t->eps;
        p.interleaved = t->interleaved != 0;
        p.wide_weights = t->weight_type == TESSA_KV_F32;
        if (launch_kv_rotate(p, t->type, rows_kind(cache->type), reinterpret_cast<hipStream_t>(stream)))
            return status(TESSA_ERR_HIP, "kv append rotated: launch failed");
        return fine();
    });
}

tessa_status tessa_kv_read(const tessa_kv_cache *cache, const tessa_kv_rows *r, void *stream) {
    return guarded([&]() -> tessa_status {
        if (!r) KV_INVALID("kv read: null pointer");
        KvReadParams p;
        std::memset(&p, 0, sizeof(p));
        const tessa_status st = pages_of(cache, p.c);
        if (st.code) return st;
        if (r->type != TESSA_KV_BF16 && r->type != TESSA_KV_F16 && r->type != TESSA_KV_F32)
            KV_INVALID("kv read: type %u is neither bf16, fp16 nor f32", r->type);
        if (!r->count) return fine();
        if (r->count > kMaxRows || r->count * p.c.heads > 0x7fffffffull)
            KV_UNSUPPORTED("kv read: %llu rows of %u heads", (unsigned long long)r->count, p.c.heads);
        if (!r->slots || !r->k) KV_INVALID("kv read: null pointer");
        if (!aligned16(r->k) || !aligned16(r->v)) KV_INVALID("kv read: k and v are not 16-byte aligned");
        const uint64_t bytes = r->count * p.c.heads * p.c.dim * (r->type == TESSA_KV_F32 ? 4u : 2u);
        const uintptr_t k = reinterpret_cast<uintptr_t>(r->k), v = reinterpret_cast<uintptr_t>(r->v);
        if (v && k < v + bytes && v < k + bytes) KV_INVALID("kv read: k and v overlap");
        p.slots = r->slots;
        p.k = static_cast<char *>(r->k);
        p.v = static_cast<char *>(r->v);
        p.count = r->count;
        if (launch_kv_read(p, cache->type, r->type, reinterpret_cast<hipStream_t>(stream)))
            return status(TESSA_ERR_HIP, "kv read: launch failed");
        return fine();
    });
}

tessa_status tessa_kv_plan(const tessa_kv_step *s, void *stream) {
    return guarded([&]() -> tessa_status {
        if (!s) KV_INVALID("kv plan: null pointer");
        if (!s->page_rows || (s->page_rows & (s->page_rows - 1u)) || s->page_rows > 65536u)
            KV_INVALID("kv plan: page_rows must be a power of two in 1..=65536, got %u", s->page_rows);
        if (s->batch > kMaxGrid) KV_UNSUPPORTED("kv plan: batch %u over %u", s->batch, kMaxGrid);
        if (s->pages > 0x7fffffffu || s->columns > 0x7fffffffu) KV_UNSUPPORTED("kv plan: %u pages, %u columns", s->pages, s->columns);
        if (s->tokens > 0x7fffffffull) KV_UNSUPPORTED("kv plan: %llu tokens", (unsigned long long)s->tokens);
        if (!s->count || !s->new_count || !s->offsets || (s->pages && !s->free)) KV_INVALID("kv plan: null pointer");
        if (s->batch && (!s->lengths || !s->held || !s->fresh || !s->new_lengths || !s->new_held || !s->granted ||
                         (s->columns && !s->table)))
            KV_INVALID("kv plan: null pointer");
        if (s->batch > 1 && s->table_stride < s->columns)
            KV_INVALID("kv plan: table stride %llu below %u columns", (unsigned long long)s->table_stride, s->columns);
        if (s->tokens && (!s->positions || !s->sequences || !s->slots)) KV_INVALID("kv plan: null pointer");
        const tessa_status st = apart(*s);
        if (st.code) return st;
        KvPlanParams p;
        std::memset(&p, 0, sizeof(p));
        p.table = s->table;
        p.table_stride = s->table_stride;
        p.lengths = s->lengths;
        p.held = s->held;
        p.fresh = s->fresh;
        p.free = s->free;
        p.count = s->count;
        p.new_lengths = s->new_lengths;
        p.new_held = s->new_held;
        p.new_count = s->new_count;
        p.granted = s->granted;
        p.offsets = s->offsets;
        p.positions = s->positions;
        p.sequences = s->sequences;
        p.slots = s->slots;
        p.tokens = s->tokens;
        p.batch = s->batch;
        p.columns = s->columns;
        p.pages = s->pages;
        p.page_shift = (uint32_t)__builtin_ctz(s->page_rows);
        if (launch_kv_plan(p, reinterpret_cast<hipStream_t>(stream))) return status(TESSA_ERR_HIP, "kv plan: launch failed");
        return fine();
    });
}

}  // extern "C"
