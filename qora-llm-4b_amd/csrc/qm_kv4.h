// qm_kv4.h -- the paged 4-bit KV cache: its layout, for the host and the
// kernels, and the host's checks of a call's arguments.
//
// One layer's page holds QMK_KV4_PAGE_TOKENS tokens of the four kv heads' K
// and V.  Per token, head and group of 64 dims (group 0 are the rotary dims)
// the f16 values x are kept as
//   lo = min x,  s = f16(f32((max x - min x) / 15)),
//   q  = clamp(rne((x - lo) / s), 0, 15)  (0 where s = 0),   x ~ lo + s q,
// 4.5 bits a value.  A group with an infinity or a NaN keeps s = lo = NaN.
//
// The layout is the order in which the attention's matrix operands are
// loaded: half a page (32 tokens) of one head is 9216 contiguous bytes,
//   K codes  u32 [run 2][dim / 128][g 4][token 16][word 4]: dims
//            32 s + 8 g + e (s = 4 (dim / 128) + word) of token 16 run + c,
//   V codes  u32 [group 4][g 4][dim 16][word 4]: dim 64 group + 16 word + c of
//            the eight tokens 16 (e >> 2) + 4 g + (e & 3),
//   sK, loK, sV, loV  f16: s as [g][run][i][group], lo as [group][g][run][i]
//            of token 16 run + 4 g + i,
// so that every load of a wave is 1024 contiguous bytes and lane (g, c) gets
// its eight values of a matrix instruction's k-group in one word.  Element e
// of a word is nibble (e >> 1) + 4 (e & 1): masks alone put the elements in
// pairs (elements 2 i, 2 i + 1 in the halves of a register).
#pragma once
#include <stdint.h>

#define QMK_KV4_PAGE_TOKENS 64
#define QMK_KV4_HALF_TOKENS 32
#define QMK_KV4_HALF_BYTES 9216
#define QMK_KV4_HEAD_BYTES (2 * QMK_KV4_HALF_BYTES)
#define QMK_KV4_PAGE_BYTES (4 * QMK_KV4_HEAD_BYTES)
#define QMK_KV4_V_WORDS 1024        // first word of the V codes
#define QMK_KV4_META 8192           // first byte of the scales and minima
#define QMK_KV4_MAX_PAGES 4194303   // pages of a pool (309 GB a layer): 1024 rows' needs are a uint32
#define QMK_KV4_MAX_COUNT 1024      // rows of one resize or fork: one thread each
#define QMK_KV4_MAX_ROWS 65536      // table rows: the LDS bitmap of those seen
#define QMK_KV4_MAX_SPLIT 4096      // tokens of a decode workgroup: 64 pages
#define QMK_KV4_ROUNDS 64           // full rounds of decode workgroups that are dealt evenly
#define QMK_KV4_LEN_PAGES 33554431  // pages of a row: its length is an int32

#ifdef __HIPCC__
#define QMK_HD __host__ __device__ inline
#else
#define QMK_HD inline
#endif

// Word (of a half page) and nibble of the code of token t (0 .. 31), dim d.
QMK_HD int kv4_k_word(int t, int d) {
    return ((t >> 4) * 2 + (d >> 7)) * 256 + ((d >> 3) & 3) * 64 + (t & 15) * 4 + ((d >> 5) & 3);
}
QMK_HD int kv4_v_word(int t, int d) {
    return QMK_KV4_V_WORDS + (d >> 6) * 256 + ((t >> 2) & 3) * 64 + (d & 15) * 4 + ((d >> 4) & 3);
}
QMK_HD int kv4_nibble(int e) { return (e >> 1) + 4 * (e & 1); }
QMK_HD int kv4_k_nibble(int d) { return kv4_nibble(d & 7); }
QMK_HD int kv4_v_nibble(int t) { return kv4_nibble(4 * (t >> 4) + (t & 3)); }
// f16 (of the 128 of one of the four arrays) of the scale and of the minimum
// of token t, group.
QMK_HD int kv4_s_at(int t, int group) { return ((t >> 2) & 3) * 32 + (t >> 4) * 16 + (t & 3) * 4 + group; }
QMK_HD int kv4_lo_at(int t, int group) { return group * 32 + ((t >> 2) & 3) * 8 + (t >> 4) * 4 + (t & 3); }
QMK_HD int kv4_pages_of(int32_t len) { return (int)(((int64_t)len + QMK_KV4_PAGE_TOKENS - 1) / QMK_KV4_PAGE_TOKENS); }

// A cache as the kernels take it (qm_kv4_cache of the public header).
struct Kv4Cache {
    uint8_t* pages;          // [layers][num_pages][QMK_KV4_PAGE_BYTES]
    int32_t* table;          // [rows][max_pages]
    int32_t* lens;           // [rows]
    int32_t* refs;           // [num_pages]
    int32_t layers, num_pages, rows, max_pages;
};

// f16 rows [batch][4][cap][256] <-> the pages of table rows row ..
struct Kv4RowsArgs {
    Kv4Cache c;
    const int32_t* first;    // [batch] or null: 0
    uint16_t* k;
    uint16_t* v;
    int64_t cap;
    int32_t layer, row, batch, n;
    int32_t halves;          // half pages per (sequence, head) of the grid
};

// Workspace: state[0] verdict (0: go on), state[1] copies, then from
// state[4] count x {src, dst} (the copies), then count x {first, end} (table
// entries given up by list row i).
struct Kv4ResizeArgs {
    Kv4Cache c;
    const int32_t* list;     // [count] or null: rows 0 .. count - 1
    const int32_t* lens;     // [count]
    int32_t* result;
    int32_t* state;
    int32_t count;
    int32_t add;             // lens are added to the rows' lengths
};

// Workspace: state[0] verdict, state[4 + i] new length of pair i, then
// count x max_pages entries.
struct Kv4ForkArgs {
    Kv4Cache c;
    const int32_t* src;
    const int32_t* dst;
    int32_t* result;
    int32_t* state;
    int32_t count;
};

// Workspace: state[0] live pages, state[1] moves, then from state[4]
// num_pages each of movers, holes and new ids.
struct Kv4CompactArgs {
    Kv4Cache c;
    int32_t* live;
    int32_t* state;
};

// One attention step over the pages.
struct GqaKv4Args {
    Kv4Cache c;
    const int32_t* slots;    // [batch] or null: row b
    const float* q_gate;     // [B][16][512]
    const float* k_new;      // [B][4][256]
    const float* v_new;
    const uint16_t* q_norm;  // [256] f16
    const uint16_t* k_norm;
    const float* rope_cos;   // [rope_len][32]
    const float* rope_sin;
    const int32_t* result;   // null, or a resize's result
    float* out;              // [B][16][256]
    float* partial;          // [splits][4 kv heads][4 heads][260]: acc[256], m, l, pad
    int32_t* splits;         // [B] {first, splits}: for the merge
    int32_t layer, batch, max_len;
    int32_t cus;             // compute units of the device
    int32_t single;          // a workgroup per batch row and head, no merge
};
