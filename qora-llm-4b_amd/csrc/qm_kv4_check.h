// qm_kv4_check.h -- what the host can tell of a call on the paged 4-bit KV
// cache: a status code and its message before anything is enqueued.  Host
// code without HIP, so that it is tested on the CPU.
#pragma once
#include "qora_mixer.h"
#include "qm_kv4.h"

#include <cstdarg>
#include <cstdio>
#include <initializer_list>

namespace qm_kv4 {

static_assert(QMK_KV4_PAGE_TOKENS == QM_KV4_PAGE_TOKENS && QMK_KV4_PAGE_BYTES == QM_KV4_PAGE_BYTES,
              "the public constants are the layout's");

struct Fault {
    int32_t code = QM_OK;
    char text[256] = "";
};

inline Fault fault(int32_t code, const char* fmt, ...) {
    Fault f;
    f.code = code;
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(f.text, sizeof(f.text), fmt, ap);
    va_end(ap);
    return f;
}

inline bool off_grid(uintptr_t grid, std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) & (grid - 1)) return true;
    return false;
}

inline Fault check_cache(const char* who, const qm_kv4_cache* c) {
    if (!c || !c->pages_dev || !c->table_dev || !c->lens_dev || !c->refs_dev)
        return fault(QM_ERR_INVALID_ARG, "%s: null cache or cache pointer", who);
    if (off_grid(16, {c->pages_dev}) || off_grid(4, {c->table_dev, c->lens_dev, c->refs_dev}))
        return fault(QM_ERR_INVALID_ARG, "%s: pages must be 16-byte aligned, table, lens and refs 4-byte", who);
    if (c->layers <= 0 || c->num_pages <= 0 || c->rows <= 0 || c->max_pages <= 0)
        return fault(QM_ERR_INVALID_ARG, "%s: cache of %d layers, %d pages, %d rows of %d pages", who, c->layers,
                     c->num_pages, c->rows, c->max_pages);
    if (c->num_pages > QMK_KV4_MAX_PAGES || c->rows > QMK_KV4_MAX_ROWS || c->max_pages > QMK_KV4_LEN_PAGES)
        return fault(QM_ERR_SHAPE, "%s: %d pages (at most %d), %d rows (at most %d) of %d pages (at most %d)", who,
                     c->num_pages, QMK_KV4_MAX_PAGES, c->rows, QMK_KV4_MAX_ROWS, c->max_pages, QMK_KV4_LEN_PAGES);
    return Fault{};
}

inline Fault check_list(const char* who, const qm_kv4_cache* c, int32_t count, std::initializer_list<const void*> lists,
                        const void* result) {
    Fault f = check_cache(who, c);
    if (f.code != QM_OK) return f;
    if (count <= 0 || count > QMK_KV4_MAX_COUNT || count > c->rows)
        return fault(QM_ERR_INVALID_ARG, "%s: %d rows listed (1 .. %d, of a cache of %d)", who, count, QMK_KV4_MAX_COUNT,
                     c->rows);
    for (const void* p : lists)
        if (!p) return fault(QM_ERR_INVALID_ARG, "%s: null list", who);
    if (!result) return fault(QM_ERR_INVALID_ARG, "%s: null result", who);
    if (off_grid(4, lists) || off_grid(4, {result}))
        return fault(QM_ERR_INVALID_ARG, "%s: lists and result must be 4-byte aligned", who);
    return Fault{};
}

inline Fault check_resize(const qm_kv4_cache* c, int32_t count, const int32_t* rows, const int32_t* lens, int32_t flags,
                          const int32_t* result) {
    Fault f = check_list("qm_kv4_resize", c, count, {lens}, result);
    if (f.code != QM_OK) return f;
    if (off_grid(4, {rows})) return fault(QM_ERR_INVALID_ARG, "qm_kv4_resize: lists and result must be 4-byte aligned");
    if (flags != QM_KV4_LENS && flags != QM_KV4_ADD) return fault(QM_ERR_INVALID_ARG, "qm_kv4_resize: flags %d", flags);
    return Fault{};
}

inline Fault check_rows(const char* who, const qm_kv4_cache* c, int32_t layer, int32_t row, int32_t batch,
                        const int32_t* first, int32_t n, const uint16_t* k, const uint16_t* v, int64_t capacity) {
    Fault f = check_cache(who, c);
    if (f.code != QM_OK) return f;
    if (layer < 0 || layer >= c->layers) return fault(QM_ERR_INVALID_ARG, "%s: layer %d of %d", who, layer, c->layers);
    if (batch <= 0 || row < 0 || row > c->rows - batch)
        return fault(QM_ERR_INVALID_ARG, "%s: rows %d .. + %d of %d", who, row, batch, c->rows);
    if (!k || !v) return fault(QM_ERR_INVALID_ARG, "%s: null pointer", who);
    if (off_grid(16, {k, v}) || off_grid(4, {first}))
        return fault(QM_ERR_INVALID_ARG, "%s: k and v must be 16-byte aligned, first 4-byte", who);
    if (n <= 0) return fault(QM_ERR_INVALID_ARG, "%s: %d tokens", who, n);
    if (n > capacity)
        return fault(QM_ERR_CAPACITY, "%s: %d tokens beyond the f16 rows' capacity %lld", who, n,
                     static_cast<long long>(capacity));
    return Fault{};
}

inline Fault check_decode(const qm_kv4_cache* c, int32_t layer, int32_t batch, const int32_t* slots,
                          std::initializer_list<const void*> data, int32_t rope_len, int32_t max_len,
                          const int32_t* result) {
    Fault f = check_cache("qm_gqa_decode_kv4", c);
    if (f.code != QM_OK) return f;
    if (layer < 0 || layer >= c->layers)
        return fault(QM_ERR_INVALID_ARG, "qm_gqa_decode_kv4: layer %d of %d", layer, c->layers);
    if (batch <= 0 || (!slots && batch > c->rows))
        return fault(QM_ERR_INVALID_ARG, "qm_gqa_decode_kv4: batch %d of a cache of %d rows", batch, c->rows);
    for (const void* p : data)
        if (!p) return fault(QM_ERR_INVALID_ARG, "qm_gqa_decode_kv4: null pointer");
    if (off_grid(16, data) || off_grid(4, {slots, result}))
        return fault(QM_ERR_INVALID_ARG, "qm_gqa_decode_kv4: device pointers must be 16-byte aligned (slots and result 4-byte)");
    if (max_len <= 0) return fault(QM_ERR_INVALID_ARG, "qm_gqa_decode_kv4: max_len %d", max_len);
    if (max_len > rope_len)
        return fault(QM_ERR_ROPE_RANGE, "length %d beyond RoPE table of %d rows", max_len, rope_len);
    if (max_len > static_cast<int64_t>(c->max_pages) * QMK_KV4_PAGE_TOKENS)
        return fault(QM_ERR_CAPACITY, "length %d beyond the %d pages of a row", max_len, c->max_pages);
    return Fault{};
}

// What append and chunk attention have in common: the batch's lists and bounds.
inline Fault check_ragged(const char* who, const qm_kv4_cache* c, int32_t layer, int32_t batch, const int32_t* slots,
                          const int32_t* begins, int32_t tokens, std::initializer_list<const void*> data,
                          int32_t rope_len, int32_t max_len, const int32_t* result) {
    Fault f = check_cache(who, c);
    if (f.code != QM_OK) return f;
    if (layer < 0 || layer >= c->layers) return fault(QM_ERR_INVALID_ARG, "%s: layer %d of %d", who, layer, c->layers);
    if (batch <= 0 || batch > QMK_KV4_MAX_ROWS || (!slots && batch > c->rows))
        return fault(QM_ERR_INVALID_ARG, "%s: batch %d of a cache of %d rows", who, batch, c->rows);
    if (tokens <= 0 || tokens > QMK_CHUNK_MAX_TOKENS)
        return fault(QM_ERR_INVALID_ARG, "%s: %d tokens (1 .. %d)", who, tokens, QMK_CHUNK_MAX_TOKENS);
    if (!begins) return fault(QM_ERR_INVALID_ARG, "%s: null begins", who);
    for (const void* p : data)
        if (!p) return fault(QM_ERR_INVALID_ARG, "%s: null pointer", who);
    if (off_grid(16, data) || off_grid(4, {slots, begins, result}))
        return fault(QM_ERR_INVALID_ARG, "%s: device pointers must be 16-byte aligned (slots, begins and result 4-byte)", who);
    if (max_len <= 0) return fault(QM_ERR_INVALID_ARG, "%s: max_len %d", who, max_len);
    if (max_len > rope_len) return fault(QM_ERR_ROPE_RANGE, "length %d beyond RoPE table of %d rows", max_len, rope_len);
    if (max_len > static_cast<int64_t>(c->max_pages) * QMK_KV4_PAGE_TOKENS)
        return fault(QM_ERR_CAPACITY, "length %d beyond the %d pages of a row", max_len, c->max_pages);
    return Fault{};
}
inline Fault check_append(const qm_kv4_cache* c, int32_t layer, int32_t batch, const int32_t* slots, const int32_t* begins,
                          int32_t tokens, int32_t dtype, std::initializer_list<const void*> data, int32_t rope_len,
                          int32_t max_len, const int32_t* result) {
    if (dtype != QM_F32 && dtype != QM_BF16)
        return fault(QM_ERR_INVALID_ARG, "qm_kv4_append: dtype %d (QM_F32 or QM_BF16)", dtype);
    return check_ragged("qm_kv4_append", c, layer, batch, slots, begins, tokens, data, rope_len, max_len, result);
}
inline Fault check_chunk(const qm_kv4_cache* c, int32_t layer, int32_t batch, const int32_t* slots, const int32_t* begins,
                         int32_t tokens, int32_t max_new, std::initializer_list<const void*> data, int32_t rope_len,
                         int32_t max_len, const int32_t* result) {
    if (max_new <= 0) return fault(QM_ERR_INVALID_ARG, "qm_gqa_chunk_kv4: max_new %d", max_new);
    return check_ragged("qm_gqa_chunk_kv4", c, layer, batch, slots, begins, tokens, data, rope_len, max_len, result);
}

// Half pages that `tokens` new tokens of `batch` rows touch at most: n of a row
// floor((n + 30) / 32) + 1.
inline int64_t append_halves(int32_t tokens, int32_t batch) {
    return (static_cast<int64_t>(tokens) + 30ll * batch) / QMK_KV4_HALF_TOKENS + batch;
}
// The chunk attention's shape: operand columns of a block of few tokens (4 new
// tokens each), whether there are blocks of many, the most row blocks of both
// kinds, workgroups per kv head (one a CU, or fewer where the blocks' pages are
// fewer) and whether blocks may be split over them.  One column where it has all
// of a row's new tokens (one / two, us: 1 token of 260 11.7 / 13.9, 4 of 4000
// 14.1 / 16.7, 24 x 4 of 12001 82 / 94).
struct Chunk {
    int32_t columns;
    bool many, split;
    int64_t most_many, most_few, groups;
};
inline Chunk chunk_shape_of(int32_t tokens, int32_t batch, int32_t max_new, int32_t max_len, int cus, bool many) {
    Chunk c{};
    c.columns = max_new <= 4 ? 1 : 2;
    c.many = many;
    // a row of n: ceil(n / tokens of a block) <= n / that + 1, and many is FEW + 1 at least;
    // one that is refused, whatever its n, is one block
    const int64_t t = tokens, b = batch, block = 4 * c.columns, with_many = t / (QMK_CHUNK_FEW + 1);
    const int64_t row = ((many ? QMK_CHUNK_FEW : max_new) + block - 1) / block;
    c.most_many = many ? t / QMK_CHUNK_TOKENS + (b < with_many ? b : with_many) : 0;
    c.most_few = t / block + b < b * row ? t / block + b : b * row;
    const int64_t tiles = (static_cast<int64_t>(max_len) + QMK_KV4_PAGE_TOKENS - 1) / QMK_KV4_PAGE_TOKENS;
    c.split = tiles > (many ? QMK_CHUNK_MANY_WHOLE : QMK_CHUNK_WHOLE);
    const int64_t blocks = c.most_few + c.most_many;
    const int64_t quarter = cus / 4 > 0 ? cus / 4 : 1, most = quarter < QMK_CHUNK_MAX_GROUPS ? quarter : QMK_CHUNK_MAX_GROUPS;
    const int64_t parts = c.split ? tiles : 1;
    c.groups = blocks >= most || blocks * parts >= most ? most : blocks * parts;
    if (c.groups < 1) c.groups = 1;
    c.split = c.split && c.groups > 1;
    return c;
}
// Whether a call has blocks of many tokens; max_new may be a loose bound, and no
// row has more new tokens than the call.
inline bool chunk_many(int32_t tokens, int32_t max_new, int32_t max_len) {
    const bool few = tokens <= QMK_CHUNK_SHORT_TOKENS && static_cast<int64_t>(tokens) * max_len <= QMK_CHUNK_SHORT;
    return max_new > QMK_CHUNK_FEW && tokens > QMK_CHUNK_FEW && !few;
}
inline Chunk chunk_shape(int32_t tokens, int32_t batch, int32_t max_new, int32_t max_len, int cus) {
    return chunk_shape_of(tokens, batch, max_new < tokens ? max_new : tokens, max_len, cus, chunk_many(tokens, max_new, max_len));
}
inline size_t chunk_partial_bytes(const Chunk& c) {
    const int64_t columns = c.many ? 16 : c.columns;
    return c.split ? static_cast<size_t>(c.groups) * 4 * 2 * columns * QMK_CHUNK_COLUMN * 4 : 0;
}
inline size_t chunk_ws(const Chunk& c) {
    return chunk_partial_bytes(c) + 16 + static_cast<size_t>(c.most_many + c.most_few) * sizeof(ChunkRecord);
}
// A bound of it for up to so many tokens, rows and lengths, whatever max_new is.
// Where the largest such call has no blocks of many tokens, no other has.
inline size_t chunk_reserve_ws(int32_t tokens, int32_t batch, int32_t max_len, int cus) {
    size_t ws = 0;
    const int forms = chunk_many(tokens, tokens, max_len) ? 3 : tokens > 4 ? 2 : 1;
    for (int form = 0; form < forms; ++form) {
        const size_t one = chunk_ws(chunk_shape_of(tokens, batch, form ? tokens : 4, max_len, cus, form == 2));
        if (one > ws) ws = one;
    }
    return ws;
}

// The decode's workgroups.  Short rows, and somewhat longer ones where there
// are enough of them, take one workgroup each per kv head and no merge
// (measured, one workgroup / dealt out, us: 1 row of 250 tokens 8.1 / 9.1, of
// 257 9.5 / 9.1, of 500 10.8 / 9.1; 16 rows of 400 11.1 / 9.5, of 512 11.0 /
// 10.0; 24 rows of 400 11.2 / 11.2, of 512 11.1 / 11.7; 32 rows of 512 11.1 /
// 12.7; 64 rows of 250 8.6 / 12.8, of 500 13.0 / 17.7; rows of one step may
// differ, so not much longer).  Others are dealt out by the kernel
// (deal_chunk): splits of 128 n tokens, at most QMK_KV4_MAX_SPLIT, n such that
// one or two workgroups a CU, or some full rounds of two, have about the same
// number.  max_splits bounds the splits of all rows: two workgroups a CU and
// round over the four kv heads and one per row, and cus / 16 for the errors of
// the f32 sum that the rounds are counted by (under 2^-7 of one); past
// QMK_KV4_ROUNDS rounds ceil(len / QMK_KV4_MAX_SPLIT) per row.
inline bool single(int64_t len, int64_t batch) { return len <= 256 || (len <= 512 && batch >= 24); }
inline int64_t max_splits(int64_t len, int64_t batch, int cus) {
    const int64_t least = (len + 127) / 128 * batch, longest = (len + QMK_KV4_MAX_SPLIT - 1) / QMK_KV4_MAX_SPLIT * batch;
    const int64_t rounds = len * batch / (static_cast<int64_t>(QMK_KV4_MAX_SPLIT) * cus / 2) + 1;
    int64_t n = cus / 2 * (rounds < QMK_KV4_ROUNDS ? rounds : QMK_KV4_ROUNDS) + batch + cus / 16 + 1;
    if (rounds >= QMK_KV4_ROUNDS && longest > n) n = longest;
    return least < n ? least : n;
}

// Workspace of each call, bytes.
inline size_t resize_ws(int32_t count) { return 4 * (4 + 4 * static_cast<size_t>(count)); }
inline size_t fork_ws(int32_t count, int32_t max_pages) {
    return 4 * (4 + static_cast<size_t>(count) * (1 + static_cast<size_t>(max_pages)));
}
inline size_t compact_ws(int32_t num_pages) { return 4 * (4 + 3 * static_cast<size_t>(num_pages)); }
inline size_t partial_bytes(int64_t splits) { return static_cast<size_t>(splits) * 4 * 4 * 260 * 4; }
inline size_t decode_ws(int64_t splits, int32_t batch) { return partial_bytes(splits) + static_cast<size_t>(batch) * 8; }

// A bound of all of them for batches up to `batch` over lengths up to `len`,
// a table of no more pages a row than those need, a pool of no more than
// `batch` such rows have, forks and resizes of at most `batch` rows.
inline size_t reserve_ws(int32_t batch, int32_t len, int cus) {
    const int64_t pages = (static_cast<int64_t>(len) + QMK_KV4_PAGE_TOKENS - 1) / QMK_KV4_PAGE_TOKENS;
    size_t ws = decode_ws(max_splits(len, batch, cus), batch);
    const size_t lists = resize_ws(batch), forks = fork_ws(batch, static_cast<int32_t>(pages));
    const size_t pool = 4 * (4 + 3 * static_cast<size_t>(pages) * static_cast<size_t>(batch));
    if (lists > ws) ws = lists;
    if (forks > ws) ws = forks;
    if (pool > ws) ws = pool;
    return ws;
}

}  // namespace qm_kv4
