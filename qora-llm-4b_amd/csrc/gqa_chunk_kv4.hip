// gqa_chunk_kv4.hip -- attention of chunks of new tokens over the paged 4-bit
// KV cache (qm_kv4.h) for gfx950: parts of prompts, drafted tokens, whole
// prompts, of several rows at once.
//
// Mathematics.  Token i of a batch row's n new ones stands at position
// pos = len - n + i.  With q its RMSNorm'd, rotated query (gemv.rs:586-627),
//   out = sigmoid(gate) sum_t p_t V_t / sum_t p_t,  p_t = exp(q . K_t / 16),
// over the cached tokens t <= pos, K and V as the cache keeps them: lo + s c,
// rounded to f16 once.  q, p (in base 2, counted from CHUNK_HEAD below a running
// maximum) and the operands are f16, all sums f32.
//
// Both products run transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane's
// scores, its running maximum and its outputs are all of one row, and its
// scores are, as they stand, the keys that a word of V codes holds: between the
// products nothing changes lanes.  The scores come out counted from the row's
// reference (the product begins at its negative), so that a weight is one exp2;
// the reference moves, and outputs are rescaled, only where a score passes it by
// CHUNK_HEAD + CHUNK_SLACK.
//
// Two forms, by the call's and a row's new tokens (QMK_CHUNK_FEW, _SHORT), one
// workgroup of 8 waves a CU in both:
//   few   blocks of 4 NF tokens x 4 heads, the columns of a 16 x 16 x 32 product.  A wave has half pages of its own, their codes by LDS DMA
//         two ahead, and makes operands of them in registers; the waves' sums
//         are joined at the end.  Bound by HBM once there is enough to read: 24
//         rows of up to 12001 tokens 44 us with the merge, 22 of it while the
//         codes stream (6 TB/s), 8 before the first of them (lengths -> deal ->
//         table -> page), the joins 9.  Vector unit 60% busy, matrix unit 11%.
//   many  blocks of 64 tokens: wave w has head w & 3 and 32 of them, the columns
//         of a 32 x 32 x 16 product.  A page is a tile: its codes come by LDS
//         DMA, each wave makes f16 operands of an eighth of them, which all
//         waves read, in between the second product's matrix instructions of the
//         tile before; a barrier a tile.  Bound by the matrix unit and what
//         issues beside it: 2048 tokens of 32768 1075 us, 0.99 PFLOP/s (a large
//         f16 product 1.19), matrix unit 51% busy at the clock that this load
//         leaves, vector unit 43%; a tile takes 3.3 us, 4.2 with every CU at it.
//         An operand a wave for itself, as above, would be made eight times over.
//         A block costs 18 us beside its pages, the latency of code and data that
//         come once (64 tokens of 64 27 us; few, in eight workgroups, 12).
//
// Row blocks are dealt over the workgroups, in pieces where one has too many
// pages (Deal); pieces leave partial sums, which qm_gqa_chunk_merge joins.
#include "qm_kv4_device.h"
#include "qm_kernel_args.h"

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

#define CHUNK_WAVES 8
// A row's reference is its largest score less CHUNK_HEAD (log2 units), and moves
// only where a score passes that by CHUNK_SLACK more, so that outputs are seldom
// rescaled.  Weights are thus up to 2^15 (f16's largest is 65504), and a key's
// is 2^-11 of itself off down to 2^-21 of the largest, and 2^-32 of that below
// (6000 keys 18 nats below one whose V is 0: outputs off by 0.2%, bf16's own
// rounding; with weights of 1 at most by 15%).
#define CHUNK_HEAD 7.0f
#define CHUNK_SLACK 8.0f
// What is seldom true stands away from the code that each workgroup runs: code
// comes from memory once a launch, and a short call waits for little else (700
// tokens 43.1 / 41.9 us).
#define CHUNK_SELDOM(x) __builtin_expect(!!(x), 0)

// ---- how the work is dealt --------------------------------------------------
// A batch row of the call.  A row that has no tokens to read (its slot is
// outside the table, or empty) or is refused (longer than max_len, more new
// tokens than max_new or than its length) is one block of a page's units, in
// which its outputs, 0 or NaN, are written.
enum { CHUNK_RUN = 0, CHUNK_NONE = 1, CHUNK_REFUSED = 2 };
struct ChunkRow {
    int row, len, n, begin, kind;
};
QM_DEV ChunkRow chunk_row(const GqaChunkArgs& A, int b) {
    ChunkRow r{0, 0, 0, 0, CHUNK_NONE};
    if (b >= A.batch) return r;
    const int begin = A.begins[b], end = A.begins[b + 1], row = A.slots ? A.slots[b] : b;
    if (begin < 0 || end < begin || end > A.tokens) return r;
    r.begin = begin;
    r.n = end - begin;
    if ((A.result && A.result[0] != 0) || (uint32_t)row >= (uint32_t)A.c.rows) return r;
    r.row = row;
    r.len = A.c.lens[row];
    if (r.len <= 0) return r;
    r.kind = r.len > A.max_len || r.n > A.max_new || r.n > r.len ? CHUNK_REFUSED : CHUNK_RUN;
    return r;
}

// NF: operand columns of a row block of few tokens (4 NF tokens of four heads).
template <int NF, bool MANY>
struct Deal {
    static constexpr int kFew = 4 * NF;
    const GqaChunkArgs& A;
    const int lane;
    ChunkRow mine;                     // batch row `lane`, if there are no more than 64
    // No more row blocks than workgroups: a workgroup has a piece of one, and
    // each block of the lane's row is cut into `cuts` of at most `piece` units.
    bool pieces;
    double piece;
    int cuts;
    // Otherwise equal runs of `each` of the `total` units of a kv head.
    double total, each;
    double incl, units;

    // Short rows' calls have no merge, and no block is cut (few tokens, 500 of them
    // cached: whole 14 us without a merge and 17 with its launch, cut 14; many
    // tokens: 12 x 60 of 291 whole without 39, cut where it pays 43, 9 x 64 of 512,
    // 8 pages, 49 and 40).
    static constexpr int kShort = MANY ? QMK_CHUNK_MANY_WHOLE : QMK_CHUNK_WHOLE;
    QM_DEV bool split() const { return A.max_len > kShort * QMK_KV4_PAGE_TOKENS; }
    // Pages up to which a block of few tokens is not cut, where others are.
    QM_DEV int whole() const { return split() ? QMK_CHUNK_FEW_PIECE : kShort; }
    QM_DEV static bool few(const ChunkRow& r) { return !MANY || r.n <= QMK_CHUNK_FEW; }
    QM_DEV static int tokens(const ChunkRow& r) { return few(r) ? kFew : QMK_CHUNK_TOKENS; }
    QM_DEV static int blocks(const ChunkRow& r) { return r.kind != CHUNK_RUN ? min(r.n, 1) : (r.n + tokens(r) - 1) / tokens(r); }
    QM_DEV static int weight(const ChunkRow& r) { return few(r) ? 1 : QMK_CHUNK_WEIGHT; }
    // Pages that block j reads, and that the blocks before it do.
    QM_DEV static int tiles(const ChunkRow& r, int j) {
        if (r.kind != CHUNK_RUN) return 1;
        return (r.len - r.n + min(r.n, tokens(r) * (j + 1)) - 1) / QMK_KV4_PAGE_TOKENS + 1;
    }
    QM_DEV static double before(const ChunkRow& r, int j) {
        if (r.kind != CHUNK_RUN) return j;
        // block i of T tokens, but the row's last, reads page (len - n + T (i + 1) - 1) / 64
        // and those before it: floor((c + i) / d) of them with d = 64 / T
        const int d = QMK_KV4_PAGE_TOKENS / tokens(r), c = (r.len - r.n + tokens(r) - 1) / tokens(r);
        auto sum = [&](int m) {                            // of floor(k / d), k < m
            const double q = m / d;
            return 0.5 * q * (q - 1.0) * d + q * (m % d);
        };
        return sum(c + j) - sum(c) + j;
    }
    // What a block costs beside its pages, in units; where block j begins among the
    // row's units, and its pages.
    QM_DEV static int entry(const ChunkRow& r) { return few(r) ? QMK_CHUNK_FEW_ENTRY : QMK_CHUNK_MANY_ENTRY; }
    QM_DEV static double start(const ChunkRow& r, int j) { return weight(r) * before(r, j) + (double)entry(r) * j; }
    QM_DEV static double row_units(const ChunkRow& r) {
        const int nb = blocks(r);
        return nb ? start(r, nb - 1) + entry(r) + (double)weight(r) * tiles(r, nb - 1) : 0.0;
    }
    template <int CTRL, int ROWS>
    QM_DEV static double step(double x) {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
        return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    }
    // Inclusive sum over the lanes, of whole numbers below 2^53.
    QM_DEV static double scan(double x) {
        x = step<0x111, 0xF>(x);
        x = step<0x112, 0xF>(x);
        x = step<0x114, 0xF>(x);
        x = step<0x118, 0xF>(x);
        x = step<0x142, 0xA>(x);
        return step<0x143, 0xC>(x);
    }
    QM_DEV static double lane_of(double x, int lane) { return readlane_f64(x, lane); }
    QM_DEV static ChunkRow lane_of(const ChunkRow& r, int lane) {
        return ChunkRow{__builtin_amdgcn_readlane(r.row, lane), __builtin_amdgcn_readlane(r.len, lane),
                        __builtin_amdgcn_readlane(r.n, lane), __builtin_amdgcn_readlane(r.begin, lane),
                        __builtin_amdgcn_readlane(r.kind, lane)};
    }

    QM_DEV static int cuts_of(double cost, double piece) { return (int)ceil(cost / piece); }
    // Blocks of many tokens, cut into k pieces each: a page takes 3.4 us of a
    // workgroup, a piece's partial sums (264 KB a kv head, written and read by
    // the merge) 0.3 us of all.  3.4 * pages / k + 0.3 * blocks * k is least at
    // pieces of sqrt(0.09 * blocks * pages) pages.  Measured, whole and cut so:
    // 64 tokens of 1000 80 / 34 us, 256 of 256 41 / 34, 700 of 700 63 / 43;
    // where it says whole, cut in two: 4 x 200 of 200 39 / 41, 16 x 128 of 400
    // 60 / 70.
    QM_DEV static float many_piece(float pages, float blocks) { return fmaxf(1.0f, __builtin_amdgcn_sqrtf(0.09f * blocks * pages)); }
    QM_DEV static bool many_cut(float pages, float blocks, float k) { return 3.4f * (pages - ceilf(pages / k)) > 0.3f * blocks * k; }

    // sums: what the first one of a workgroup found, null for that one.
    struct Sums {
        double total, each;
    };
    QM_DEV Deal(const GqaChunkArgs& args, int l, const Sums* sums) : A(args), lane(l), pieces(false), piece(0.0), cuts(0), total(0.0), each(0.0), incl(0.0), units(0.0) {
        if (sums) {
            total = sums->total, each = sums->each;
            if (A.batch > 64) return;
            mine = chunk_row(A, lane);
            units = row_units(mine);
            incl = scan(units);
            return;
        }
        mine = chunk_row(A, lane);
        if (!CHUNK_SELDOM(A.batch > 64)) {
            const int nb = blocks(mine);
            const uint32_t all = __builtin_amdgcn_readlane((int)wave_scan((uint32_t)min(nb, 1 << 20)), 63);
            if (!CHUNK_SELDOM(all > (uint32_t)A.groups)) {
                // the smallest piece with which they are no more than the
                // workgroups, from an equal share on, in steps of an eighth
                pieces = true;
                const int last = tiles(mine, max(nb - 1, 0));          // pages of the row's longest block
                const double most = nb ? (double)weight(mine) * last : 0.0;
                const double least = few(mine) ? QMK_CHUNK_FEW_PIECE : QMK_CHUNK_WEIGHT * (double)many_piece((float)last, (float)all);
                piece = lane_of(scan(nb * most), 63) / A.groups;
                for (;;) {
                    cuts = nb ? cuts_of(most, fmax(piece, least)) : 0;
                    if (last <= whole() && (few(mine) || !split())) cuts = min(cuts, 1);
                    else if (!few(mine) && !many_cut((float)last, (float)all, (float)cuts)) cuts = min(cuts, 1);
                    if (__builtin_amdgcn_readlane((int)wave_scan((uint32_t)(nb * cuts)), 63) <= A.groups) break;
                    piece = fmax(piece, 1.0) * 1.125;
                }
                return;
            }
        }
        for (int b0 = 0; b0 < A.batch; b0 += 64) {         // uniform
            if (A.batch > 64) mine = chunk_row(A, b0 + lane);
            units = row_units(mine);
            incl = scan(units);
            total += lane_of(incl, 63);
        }
        // (a page of many tokens at least: less, and shares inside a block would be empty)
        each = fmax(ceil(total / A.groups), (double)QMK_CHUNK_WEIGHT);
    }

    // A row block: its row, number among the row's, pages, number among the blocks
    // of few tokens, or of many, and the units before it and before its pages.
    struct Item {
        ChunkRow r;
        int block, tiles, number;
        double first, pages;
    };
    // Where to look from: the units and blocks of the batch rows before b0.
    struct Place {
        int b0, number[2];
        double past;
    };
    // The row block that unit u (< total) falls into, at `from` or behind it.
    QM_DEV Item find(double u, bool numbered, Place& from) const {
        Item it;
        double past = from.past;
        int number[2] = {from.number[0], from.number[1]};
        ChunkRow r = mine;
        double n = units, in = incl;
        for (int b0 = from.b0;; b0 += 64) {                // uniform
            from = Place{b0, {number[0], number[1]}, lane_of(past, 0)};
            if (A.batch > 64) {
                r = chunk_row(A, b0 + lane);
                n = row_units(r);
                in = scan(n);
            }
            const double all = lane_of(in, 63);
            const bool here = u < past + all;
            const int at = here ? __popcll(__ballot(past + in <= u)) : 64;
            if (numbered) {
                const int nb = lane < at ? blocks(r) : 0;
                const bool f = few(r);
                number[0] += __builtin_amdgcn_readlane((int)wave_scan(f ? 0u : (uint32_t)nb), 63);
                number[1] += __builtin_amdgcn_readlane((int)wave_scan(f ? (uint32_t)nb : 0u), 63);
            }
            if (here || b0 + 64 >= A.batch) {              // (u < total: here)
                it.r = lane_of(r, at);
                it.first = past + lane_of(in - n, at);
                break;
            }
            past += all;
        }
        // the last block that begins at or before u
        const double rest = u - it.first;
        int lo = 0, hi = blocks(it.r) - 1;
        while (lo < hi) {
            const int mid = lo + (hi - lo + 1) / 2;
            if (start(it.r, mid) <= rest) lo = mid;
            else hi = mid - 1;
        }
        it.block = __builtin_amdgcn_readfirstlane(lo);
        it.tiles = __builtin_amdgcn_readfirstlane(tiles(it.r, it.block));
        it.first = lane_of(it.first + start(it.r, it.block), 0);
        it.pages = it.first + entry(it.r);
        it.number = number[few(it.r)] + it.block;
        return it;
    }
    // Piece i: its row block, and which of its pages; false: there is none.
    QM_DEV bool find_piece(int i, Item& it, int& ta, int& tb, int& n) const {
        const int nb = blocks(mine), all = nb * cuts, in = (int)wave_scan((uint32_t)all);
        if (i >= __builtin_amdgcn_readlane(in, 63)) return false;
        const int at = __popcll(__ballot(in <= i));
        it.r = lane_of(mine, at);
        const int k = __builtin_amdgcn_readlane(cuts, at), rest = i - __builtin_amdgcn_readlane(in - all, at);
        it.block = __builtin_amdgcn_readfirstlane((int)((uint32_t)rest / (uint32_t)k));
        it.tiles = __builtin_amdgcn_readfirstlane(tiles(it.r, it.block));
        it.first = it.pages = 0.0;
        const uint32_t same = lane < at && few(mine) == few(it.r) ? (uint32_t)nb : 0u;
        it.number = __builtin_amdgcn_readlane((int)wave_scan(same), 63) + it.block;
        const int q = rest - it.block * k;
        n = min(k, it.tiles);                              // shorter blocks of the row are cut less finely
        // (at most 2^25 pages and QMK_CHUNK_MAX_GROUPS pieces)
        ta = __builtin_amdgcn_readfirstlane((int)((uint32_t)it.tiles * (uint32_t)q / (uint32_t)n));
        tb = __builtin_amdgcn_readfirstlane((int)((uint32_t)it.tiles * (uint32_t)(q + 1) / (uint32_t)n));
        return q < n;
    }
    // Where workgroup i begins (at `from` or behind it): a multiple of `each`, but
    // whole pages, and none inside a block of few pages.
    QM_DEV double begin(int i, Place from) const {
        const double u = each * i;
        if (u >= total) return total;
        const Item it = find(u, false, from);
        const int w = weight(it.r);
        int t = max(0, (int)floor((u - it.pages) / w));
        if (it.tiles <= whole()) t = 2 * (u - it.pages) < (double)it.tiles * w ? 0 : it.tiles;
        return t == 0 ? it.first : it.pages + (double)t * w;
    }
};

// Groups whose V is NaN, of the half page's tokens: bit 4 t + group.
struct ChunkNan {
    uint64_t low, high;
};
// Whether a row at pos sees one of them, of the half page's from k0 on.
QM_DEV bool chunk_sees(const ChunkNan& nan, int group, int pos, int k0) {
    const int n = min(max(pos - k0 + 1, 0), QMK_KV4_HALF_TOKENS);            // tokens that it sees
    const uint64_t low = n >= 16 ? ~0ull : (1ull << (4 * n)) - 1, high = n >= 32 ? ~0ull : n <= 16 ? 0ull : (1ull << (4 * n - 64)) - 1;
    return ((nan.low & low) | (nan.high & high)) & 0x1111111111111111ull << group;
}
// ---- a tile -------------------------------------------------------------------
// LDS: two buffers of f16 operands, block entry l the 16 bytes that lane l
// reads for a product:
//   K block h, s (16 h + s):             dims 16 s + 8 (l >> 5) .. + 7 of token many_token(l & 31) of half page h
//   V block h, dt, k (32 + 16 h + 2 dt + k): dim 32 dt + (l & 31), tokens 16 (e >> 2) + 4 (2 k + (l >> 5)) + (e & 3),
//                                        e < 8, of half page h
// and a wave's own part of the next tile's codes, K's and V's, each with its
// half page's scales and minima.  Wave w has half page w >> 2 and pieces
// i = w & 3: K's run i >> 1, dims 128 (i & 1) .., and V's group i.
#define CHUNK_TILE 65536
#define CHUNK_RAW 1536
struct ChunkLds {
    __attribute__((aligned(1024))) uint8_t tile[2][CHUNK_TILE];
    __attribute__((aligned(1024))) uint8_t raw[CHUNK_WAVES][2][CHUNK_RAW];
    __attribute__((aligned(16))) uint32_t nan[2][2][4];      // [buffer][half][group]: tokens whose V is NaN there
};

QM_DEV uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }

// The wave's K (is_v 0) or V codes of page id, and their scales and minima.
#define CHUNK_DMA 2
template <int IS_V>
QM_DEV void many_fetch(const GqaChunkArgs& A, ChunkLds& sh, int id, int head, int w, int lane) {
    const uint8_t* half = kv4_half(A.c, A.layer, id, head, w >> 2);
    const uint32_t raw = lds_addr(sh.raw[w][IS_V]);
    dma16_off(half + 4 * QMK_KV4_V_WORDS * IS_V + 1024 * (w & 3), 16 * lane, raw);
    if (lane < 32) dma16_off(half + QMK_KV4_META + 512 * IS_V, 16 * lane, raw + 1024);
}

// Token of score e of run r in lane group g.
QM_DEV int chunk_token(int r, int g, int e) { return 16 * r + 4 * g + e; }

// The lane, recomputed from: addresses that depend on it alone would be held
// in registers across a loop that has none to spare.
QM_DEV int chunk_lane(int lane) {
    asm volatile("" : "+v"(lane));
    return lane;
}

QM_DEV half2_t as_half2(uint32_t u) { return __builtin_bit_cast(half2_t, u); }
// The eight values of a word, s and lo in pairs of elements 2 i, 2 i + 1: a
// code c in the low bits of 1024 (16 c in bits 4..7) is 1024 + c exactly, so
// c is one exact packed step away and the value one rounding more.
QM_DEV half8 chunk_values(uint32_t word, const half2_t (&s)[4], const half2_t (&lo)[4]) {
    // in registers, opaque: the masking and the exponent are one instruction then
    uint32_t low = 0x000f000fu, high = 0x00f000f0u, one = 0x64006400u;
    asm("" : "+s"(low), "+s"(high), "+v"(one));
    const uint32_t v = word >> 8;
    const half2_t k1024 = {(_Float16)1024.0f, (_Float16)1024.0f}, k64 = {(_Float16)64.0f, (_Float16)64.0f},
                  sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    half2_t c[4];
    c[0] = as_half2((word & low) | one) - k1024;
    c[1] = __builtin_elementwise_fma(as_half2((word & high) | one), sixteenth, -k64);
    c[2] = as_half2((v & low) | one) - k1024;
    c[3] = __builtin_elementwise_fma(as_half2((v & high) | one), sixteenth, -k64);
    half8 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2_t x = __builtin_elementwise_fma(c[i], s[i], lo[i]);
        out[2 * i] = x[0];
        out[2 * i + 1] = x[1];
    }
    return out;
}

// V of the half page's tokens from `left` on is 0, whatever stands there.
QM_DEV void chunk_cut(half2_t (&s)[4], half2_t (&lo)[4], int left, int g) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (chunk_token(e >> 2, g, e & 3) >= left) s[e >> 1][e & 1] = lo[e >> 1][e & 1] = (_Float16)0.0f;
}

// Whether some of K's, or V's, scales and minima of a half page (at `meta`, 512
// bytes) are NaN, or so large that its values may not be finite (2^10 and 2^14:
// lo + 15 s is under 2^15).
QM_DEV bool chunk_odd(uint32_t s, uint32_t lo) {
    const uint32_t x = s & 0x7c007c00u, y = lo & 0x7c007c00u;
    return (x & 0xffffu) >= 0x6400u || x >= 0x64000000u || (y & 0xffffu) >= 0x7400u || y >= 0x74000000u;
}
QM_DEV bool chunk_odd(const uint8_t* meta, int lane) {
    const uint32_t* m = reinterpret_cast<const uint32_t*>(meta) + lane;
    return __any(chunk_odd(m[0], m[64]));
}
// Puts such scales right, in LDS.  One that takes the group past f16's largest
// value becomes the next lower one.  V that is NaN becomes 0, and is returned:
// the rows that see it are given the NaN beside the product, as a weight of 0
// times it would give it to the others too.
template <bool IS_V>
QM_DEV ChunkNan chunk_mend(uint8_t* meta, int lane) {
    uint64_t nan[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int t = 16 * k + (lane >> 2), group = lane & 3;
        uint16_t* s = reinterpret_cast<uint16_t*>(meta) + kv4_s_at(t, group);
        uint16_t* lo = reinterpret_cast<uint16_t*>(meta + 256) + kv4_lo_at(t, group);
        const float top = fmaf(15.0f, f16_to_f32(*s), f16_to_f32(*lo));
        if (top >= 65520.0f) *s = *s - 1;
        nan[k] = __ballot(IS_V && top != top);
        if (IS_V && top != top) *s = *lo = 0;
    }
    asm volatile("" ::: "memory");                         // read again as other types
    return ChunkNan{nan[0], nan[1]};
}

// The wave's part of a tile, from its codes into buffer `buf`, K and V each in
// steps that can stand between matrix instructions: the reads, then what is
// seldom, then a word at a time.
struct ManyK {
    uintx4 k;
    uint32_t s, lo;                    // of the lane's token, groups 2 dims and + 1

    QM_DEV void reads(const ChunkLds& sh, int w, int lane) {
        const uint8_t* raw = sh.raw[w][0];
        const int run = (w & 3) >> 1, dims = w & 1, c = lane & 15;
        k = *reinterpret_cast<const uintx4*>(raw + 16 * lane);
        scales(raw + 1024, 16 * run + c, 2 * dims);
    }
    QM_DEV void scales(const uint8_t* meta, int t, int group) {
        s = *reinterpret_cast<const uint32_t*>(meta + 2 * kv4_s_at(t, group));
        lo = (uint32_t)*reinterpret_cast<const uint16_t*>(meta + 256 + 2 * kv4_lo_at(t, group)) |
             (uint32_t)*reinterpret_cast<const uint16_t*>(meta + 256 + 2 * kv4_lo_at(t, group + 1)) << 16;
    }
    QM_DEV void seldom(ChunkLds& sh, int, int, int w, int lane) {
        if (__any(chunk_odd(s, lo))) {
            uint8_t* meta = sh.raw[w][0] + 1024;
            chunk_mend<false>(meta, lane);
            scales(meta, 16 * ((w & 3) >> 1) + (lane & 15), 2 * (w & 1));
        }
    }
    QM_DEV void word(ChunkLds& sh, int buf, int m, int w, int lane) const {
        // dims 128 dims + 32 m + 8 g .. of token 16 run + c: block 2 (4 dims + m) + (g >> 1), entry of its row and g & 1
        const int half = w >> 2, run = (w & 3) >> 1, dims = w & 1, c = lane & 15, g = lane >> 4, row = 16 * (c >> 3) + 8 * run + (c & 7);
        const half2_t ss = as_half2(s), ll = as_half2(lo), s2 = {ss[m >> 1], ss[m >> 1]}, l2 = {ll[m >> 1], ll[m >> 1]};
        const half2_t s4[4] = {s2, s2, s2, s2}, l4[4] = {l2, l2, l2, l2};
        *reinterpret_cast<half8*>(sh.tile[buf] + (16 * half + 8 * dims + (g >> 1)) * 1024 + 16 * (row + 32 * (g & 1)) + 2048 * m) = chunk_values(k[m], s4, l4);
    }
};
struct ManyV {
    uintx4 v, s, lo;                   // of the lane's eight tokens, in pairs

    QM_DEV void reads(const ChunkLds& sh, int w, int lane) {
        const uint8_t* raw = sh.raw[w][1];
        v = *reinterpret_cast<const uintx4*>(raw + 16 * lane);
        scales(raw + 1024, w & 3, lane >> 4);
    }
    QM_DEV void scales(const uint8_t* meta, int i, int g) {
        lo = *reinterpret_cast<const uintx4*>(meta + 256 + (4 * i + g) * 16);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const uint16_t* at = reinterpret_cast<const uint16_t*>(meta) + g * 32 + (n >> 1) * 16 + (n & 1) * 8 + i;
            s[n] = (uint32_t)at[0] | (uint32_t)at[4] << 16;
        }
    }
    // `left`: the row's tokens in the tile (64 and more: all); V of the others is 0.
    QM_DEV void seldom(ChunkLds& sh, int buf, int left, int w, int lane) {
        const int half = w >> 2, i = w & 3, g = lane >> 4;
        uint32_t nan = 0;
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 ms = {0, 0}, ml = {0, 0};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            ms = __builtin_elementwise_max(ms, __builtin_bit_cast(u16x2, s[n]));
            ml = __builtin_elementwise_max(ml, __builtin_bit_cast(u16x2, lo[n] & 0x7fff7fffu));
        }
        if (__any(chunk_odd(__builtin_bit_cast(uint32_t, ms), __builtin_bit_cast(uint32_t, ml)))) {
            uint8_t* meta = sh.raw[w][1] + 1024;
            const ChunkNan all = chunk_mend<true>(meta, lane);
#pragma clang loop unroll(disable)
            for (int t = 0; t < QMK_KV4_HALF_TOKENS; ++t) nan |= (uint32_t)((t < 16 ? all.low : all.high) >> (4 * (t & 15) + i) & 1) << t;
            scales(meta, i, g);
        }
        if (lane == 0) sh.nan[buf][half][i] = nan;
        if (left < QMK_KV4_PAGE_TOKENS) {                  // uniform
            half2_t a[4], b[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) a[n] = as_half2(s[n]), b[n] = as_half2(lo[n]);
            chunk_cut(a, b, left - 32 * half, g);
#pragma unroll
            for (int n = 0; n < 4; ++n) s[n] = __builtin_bit_cast(uint32_t, a[n]), lo[n] = __builtin_bit_cast(uint32_t, b[n]);
        }
    }
    QM_DEV void word(ChunkLds& sh, int buf, int m, int w, int lane) const {
        // dim 64 i + 16 m + c, tokens of g: block of dims 32 (2 i + (m >> 1)) .. and g >> 1
        const int half = w >> 2, i = w & 3, c = lane & 15, g = lane >> 4;
        const half2_t s4[4] = {as_half2(s[0]), as_half2(s[1]), as_half2(s[2]), as_half2(s[3])};
        const half2_t l4[4] = {as_half2(lo[0]), as_half2(lo[1]), as_half2(lo[2]), as_half2(lo[3])};
        *reinterpret_cast<half8*>(sh.tile[buf] + 32768 + (16 * half + 4 * i + (g >> 1)) * 1024 + 16 * (c + 32 * (g & 1)) + 2048 * (m >> 1) + 256 * (m & 1)) =
            chunk_values(v[m], s4, l4);
    }
};

// ---- a wave's rows ---------------------------------------------------------------
// A row's softmax: the reference m (-inf: none yet), from which its scores are
// counted (0 before there is one), and as an integer the score at which a new
// one is due.  A float's bits are in its order where it is positive, and
// negative where it is.  l: the lane's share of the sum.
struct ChunkSum {
    float m, l;
    int due;
};
QM_DEV ChunkSum chunk_sum() { return ChunkSum{-INFINITY, 0.0f, (int)0x80000000}; }
QM_DEV float chunk_base(const ChunkSum& s) { return s.m == -INFINITY ? 0.0f : s.m; }

// A new reference, where a row's largest score (of all its lanes) wants one;
// returned: what its scores drop by, and the factor of its sums.
QM_DEV float chunk_raise(ChunkSum& s, float mx, float& corr) {
    const bool first = s.m == -INFINITY;                   // sums there may be only of NaN scores
    const float to = mx - CHUNK_HEAD;
    const float up = first ? (mx == -INFINITY ? 0.0f : to) : mx >= CHUNK_HEAD + CHUNK_SLACK ? to : 0.0f;
    corr = first ? 1.0f : __builtin_amdgcn_exp2f(-up);
    s.m = first ? to : s.m + up;
    s.due = s.m == -INFINITY ? (int)0x80000000 : __float_as_int(CHUNK_HEAD + CHUNK_SLACK);
    s.l *= corr;
    return up;
}
// Two weights, in a word, and their sum.
QM_DEV uint32_t chunk_pair(ChunkSum& s, float a, float b) {
    typedef float float2_t __attribute__((ext_vector_type(2)));
    const half2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
    const half2_t h = __builtin_convertvector((float2_t){__builtin_amdgcn_exp2f(a), __builtin_amdgcn_exp2f(b)}, half2_t);
    s.l = __builtin_amdgcn_fdot2(h, ones, s.l, false);     // of what is multiplied
    return __builtin_bit_cast(uint32_t, h);
}
QM_DEV float4 bf16x4(uint2 u) {
    return make_float4(bf16_to_f32((uint16_t)(u.x & 0xffffu)), bf16_to_f32((uint16_t)(u.x >> 16)),
                       bf16_to_f32((uint16_t)(u.y & 0xffffu)), bf16_to_f32((uint16_t)(u.y >> 16)));
}
// Sum of squares of the bf16 pairs of four words.
QM_DEV float chunk_squares(uint4 u, float ss) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x2_t x = __builtin_bit_cast(bf16x2_t, w[i]);
        ss = __builtin_amdgcn_fdot2_f32_bf16(x, x, ss, false);
    }
    return ss;
}
// Eight bf16 values times inv (1 + gamma).
QM_DEV void chunk_normed(float (&x)[8], uint4 u, uint4 gamma, float inv) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w}, gw[4] = {gamma.x, gamma.y, gamma.z, gamma.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2_t gv = as_half2(gw[i]);
        const float a = __uint_as_float(w[i] << 16) * inv, b = __uint_as_float(w[i] & 0xffff0000u) * inv;
        x[2 * i] = fmaf(a, (float)gv[0], a);
        x[2 * i + 1] = fmaf(b, (float)gv[1], b);
    }
}
// 1 / rms of a row, and the softmax's scale in base 2 as well: the scores come
// out of the product in log2 units.
QM_DEV float chunk_inv(float ss) {
    return (1.4426950408889634f / 16.0f) * __builtin_amdgcn_rsqf(ss * (1.0f / QM_GQA_HD) + 1e-6f);
}

// The queries of a block's columns, RMSNorm (1 + gamma, eps 1e-6) and RoPE: 16
// lanes have a row, lane j dims 16 j .. + 15, so that a wave does four of them
// and the rotation's pairs (i, i + 32) are two lanes apart.
template <int NF>
struct FewQuery {
    uint4 u[2], gamma[2];
    float4 cs[4], sn[4];

    QM_DEV void load(const GqaChunkArgs& A, const ChunkRow& r, int i0, int kvh, int w, int lane) {
        const int j = lane & 15, col = 4 * w + (lane >> 4);
        if (4 * w >= 16 * NF) return;                      // uniform
        const int i = min(i0 + (col >> 2), r.n - 1);       // columns past the last token: any row, never written
        const uint16_t* row = A.q_gate + ((size_t)(r.begin + i) * QM_GQA_HEADS + 4 * kvh + (col & 3)) * (2 * QM_GQA_HD) + 16 * j;
        const size_t at = (size_t)(r.len - r.n + i) * (QM_GQA_ROT / 2) + 16 * (j & 1);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            u[k] = reinterpret_cast<const uint4*>(row)[k];
            gamma[k] = reinterpret_cast<const uint4*>(A.q_norm + 16 * j)[k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            cs[k] = ld4(A.rope_cos + at + 4 * k);
            sn[k] = ld4(A.rope_sin + at + 4 * k);
        }
        // here before the DMA that follows: the compiler's waits would take that for its own
        asm volatile("" ::"v"(u[1].x), "v"(gamma[1].x), "v"(cs[3].x), "v"(sn[3].x));
    }
    QM_DEV void store(uint8_t (&q)[NF][8][1024], int w, int lane) const {
        const int j = lane & 15, col = 4 * w + (lane >> 4);
        if (4 * w >= 16 * NF) return;
        const float inv = chunk_inv(row_sum16(chunk_squares(u[1], chunk_squares(u[0], 0.0f))));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float x[8];
            chunk_normed(x, u[k], gamma[k], inv);
            const float c8[8] = {cs[2 * k].x, cs[2 * k].y, cs[2 * k].z, cs[2 * k].w, cs[2 * k + 1].x, cs[2 * k + 1].y, cs[2 * k + 1].z, cs[2 * k + 1].w};
            const float s8[8] = {sn[2 * k].x, sn[2 * k].y, sn[2 * k].z, sn[2 * k].w, sn[2 * k + 1].x, sn[2 * k + 1].y, sn[2 * k + 1].z, sn[2 * k + 1].w};
            half8 out;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float p = dpp_f32<0x4E>(x[e]);
                out[e] = (_Float16)(j >= 4 ? x[e] : x[e] * c8[e] + (j < 2 ? -p : p) * s8[e]);
            }
            *reinterpret_cast<half8*>(&q[col >> 4][j >> 1][16 * ((col & 15) + 16 * (2 * (j & 1) + k))]) = out;
        }
    }
};

// The weights of a half page's scores (runs 0, 1 of 16 tokens), which come
// counted from the reference: the products' sums begin at its negative.
QM_DEV half8 few_weights(floatx4 (&x)[2], floatx4 (&o)[16], ChunkSum& s, int pos, int k0, bool edge, int g) {
    if (edge) {                                            // uniform: some row does not see all of it
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i >> 2][i & 3] = k0 + chunk_token(i >> 2, g, i & 3) > pos ? -INFINITY : x[i >> 2][i & 3];
    }
    int top = __float_as_int(x[0][0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) top = max(top, __float_as_int(x[i >> 2][i & 3]));
    if (__any(top >= s.due)) {                             // seldom after the first
        float mx = -INFINITY, corr;
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, x[i >> 2][i & 3]);
        const float up = chunk_raise(s, max_xor32(max_xor16(mx)), corr);
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) o[dt] *= corr;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i >> 2][i & 3] -= up;
    }
    uintx4 p;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = chunk_pair(s, x[i >> 1][2 * (i & 1)], x[i >> 1][2 * (i & 1) + 1]);
    return __builtin_bit_cast(half8, p);
}

// Four outputs, gated.
QM_DEV uint2 chunk_gated(floatx4 o, uint2 gate) {
    const float4 x = bf16x4(gate);
    return make_uint2(pack_bf16x2(o[0] * sigmoid_fast(x.x), o[1] * sigmoid_fast(x.y)), pack_bf16x2(o[2] * sigmoid_fast(x.z), o[3] * sigmoid_fast(x.w)));
}
QM_DEV uint4 chunk_gated8(floatx4 a, floatx4 b, uint4 gate) {
    const uint2 x = chunk_gated(a, make_uint2(gate.x, gate.y)), y = chunk_gated(b, make_uint2(gate.z, gate.w));
    return make_uint4(x.x, x.y, y.x, y.y);
}
QM_DEV float chunk_inverse(float l) { return l != 0.0f ? __builtin_amdgcn_rcpf(l) : 0.0f; }      // 0: nothing to see

// ---- few tokens ------------------------------------------------------------------
// Blocks of 4 NF tokens, an operand column 4 of them of the four heads.  Every wave has all columns and every
// eighth half page, whose codes come by LDS DMA, two ahead, and become operands
// in its registers; the waves' sums are joined at the end.
// The queries stand in LDS as operands, block 8 f + s: entry l the 16 bytes that
// lane l = (c, g) reads, dims 32 s + 8 g .. of column 16 f + c.
template <int NF>
struct FewLds {
    // later of each wave o [dim group][entry][4] f32, then (m, l)[16]
    __attribute__((aligned(1024))) uint8_t ring[CHUNK_WAVES][2][QMK_KV4_HALF_BYTES];
    __attribute__((aligned(1024))) uint8_t q[NF][8][1024];
};
template <int NF>
struct FewWave {
    floatx4 o[NF][16];
    ChunkSum sum[NF];
    int pos[NF];
};
#define FEW_DMA (QMK_KV4_HALF_BYTES / 1024)
QM_DEV void few_fetch(const uint8_t* half, uint32_t buf, int lane) {
#pragma unroll
    for (int i = 0; i < FEW_DMA; ++i) dma16_off(half + 1024 * i, 16 * lane, buf + 1024 * i);
}
// `left` tokens of the half page are the row's.
template <int NF>
QM_DEV void few_half(FewWave<NF>& st, uint8_t* buf, const uint8_t (&q)[NF][8][1024], int k0, int left, bool edge, int lane) {
    const int c = lane & 15, g = lane >> 4;
    uint8_t* meta = buf + QMK_KV4_META;
    ChunkNan nan{0, 0};
    if (CHUNK_SELDOM(chunk_odd(meta, lane))) chunk_mend<false>(meta, lane);
    if (CHUNK_SELDOM(chunk_odd(meta + 512, lane))) nan = chunk_mend<true>(meta + 512, lane);
    floatx4 x[NF][2];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        const float base = -chunk_base(st.sum[f]);
        x[f][0] = x[f][1] = floatx4{base, base, base, base};
    }
    half2_t s[2][2];                                       // of the lane's token of each run
    _Float16 lo[2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const uint2 s4 = *reinterpret_cast<const uint2*>(meta + 2 * kv4_s_at(16 * r + c, 0));
        s[r][0] = as_half2(s4.x), s[r][1] = as_half2(s4.y);
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[r][j] = *reinterpret_cast<const _Float16*>(meta + 256 + 2 * kv4_lo_at(16 * r + c, j));
    }
#pragma unroll
    for (int d = 0; d < 2; ++d) {
        uintx4 k[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) k[r] = *reinterpret_cast<const uintx4*>(buf + 1024 * (2 * r + d) + 16 * lane);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            half8 qf[NF];
#pragma unroll
            for (int f = 0; f < NF; ++f) qf[f] = *reinterpret_cast<const half8*>(&q[f][4 * d + m][16 * lane]);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int j = 2 * d + (m >> 1);            // the words' group
                const half2_t s2 = {s[r][d][m >> 1], s[r][d][m >> 1]}, l2 = {lo[r][j], lo[r][j]};
                const half2_t ss[4] = {s2, s2, s2, s2}, ll[4] = {l2, l2, l2, l2};
                const half8 a = chunk_values(k[r][m], ss, ll);
#pragma unroll
                for (int f = 0; f < NF; ++f) x[f][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[f], x[f][r], 0, 0, 0);
            }
        }
    }
    half8 p[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) p[f] = few_weights(x[f], st.o[f], st.sum[f], st.pos[f], k0, edge, g);
    // scales of the lane's eight tokens, all groups: [token][group]
    uintx4 sv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sv[i] = *reinterpret_cast<const uintx4*>(meta + 512 + 64 * g + 16 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uintx4 v = *reinterpret_cast<const uintx4*>(buf + 4 * QMK_KV4_V_WORDS + 1024 * j + 16 * lane);
        const uintx4 lo4 = *reinterpret_cast<const uintx4*>(meta + 768 + (4 * j + g) * 16);
        half2_t s[4], lo[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {                      // tokens 2 n, 2 n + 1: dwords 4 n + j / 2 and two on
            s[n] = as_half2(__builtin_amdgcn_perm(sv[n][2 + (j >> 1)], sv[n][j >> 1], j & 1 ? 0x07060302u : 0x05040100u));
            lo[n] = as_half2(lo4[n]);
        }
        if (left < QMK_KV4_HALF_TOKENS) chunk_cut(s, lo, left, g);      // uniform
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const half8 a = chunk_values(v[m], s, lo);
#pragma unroll
            for (int f = 0; f < NF; ++f) st.o[f][4 * j + m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p[f], st.o[f][4 * j + m], 0, 0, 0);
        }
    }
    if (CHUNK_SELDOM(nan.low | nan.high)) {                              // uniform
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float add = chunk_sees(nan, j, st.pos[f], k0) ? __builtin_nanf("") : 0.0f;
#pragma unroll
                for (int m = 0; m < 4; ++m) st.o[f][4 * j + m] += add;
            }
    }
}

template <int NF, bool MANY>
QM_DEV void few_item(const GqaChunkArgs& A, FewLds<NF>& sh, const typename Deal<NF, MANY>::Item& it, int ta, int tb, int kvh, float* part, int w, int lane) {
    const int c = lane & 15, g = lane >> 4;
    const int i0 = 4 * NF * it.block, first_pos = it.r.len - it.r.n + i0;
    const int end = it.r.len - it.r.n + min(it.r.n, i0 + 4 * NF);             // past the block's last token
    const int h0 = 2 * ta + w, h_end = min(2 * tb, (end + QMK_KV4_HALF_TOKENS - 1) / QMK_KV4_HALF_TOKENS);
    // page ids of the wave's rounds, one a lane, 64 rounds at a time
    const int32_t* table = A.c.table + (size_t)it.r.row * A.c.max_pages;
    auto load_ids = [&](int round) {
        const int t = ta + (w >> 1) + 4 * (round + lane);
        return t < tb ? table[t] : -1;
    };
    int ids = load_ids(0);
    FewQuery<NF> query;
    query.load(A, it.r, i0, kvh, w, lane);
    const uint32_t ring = lds_addr(sh.ring[w]);
    auto fetch = [&](int round, int h) {                   // the half page of that round, if there is one
        if (h >= h_end) return false;
        const int id = __builtin_amdgcn_readlane(ids, round & 63);
        if (!kv4_is_page(A.c, id)) return false;
        few_fetch(kv4_half(A.c, A.layer, id, kvh, h & 1), ring + QMK_KV4_HALF_BYTES * (round & 1), lane);
        return true;
    };
    FewWave<NF> st;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        const int i = i0 + 4 * f + (c >> 2);
        st.pos[f] = i < it.r.n ? it.r.len - it.r.n + i : -1;
    }
    bool now = fetch(0, h0), next = fetch(1, h0 + CHUNK_WAVES);
    query.store(sh.q, w, lane);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        st.sum[f] = chunk_sum();
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) st.o[f][dt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int round = 0;
    for (int h = h0; h < h_end; h += CHUNK_WAVES, ++round) {
        if (next) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(FEW_DMA) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        uint8_t* buf = sh.ring[w][round & 1];
        if (now) {
            const int k0 = QMK_KV4_HALF_TOKENS * h;
            const bool edge = k0 + QMK_KV4_HALF_TOKENS - 1 > first_pos;
            few_half<NF>(st, buf, sh.q, k0, it.r.len - k0, edge, lane);
        }
        if (((round + 2) & 63) == 0) ids = load_ids(round + 2);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // the buffer's reads are done
        now = next;
        next = fetch(round + 2, h + 2 * CHUNK_WAVES);
    }
    // The waves' sums, by way of LDS: columns 2 w, 2 w + 1 are this wave's to
    // join, 4 dims a lane.  (Entries are turned over so that neither the writes,
    // a dim group's, nor the reads, a column's, meet in a bank.)
    const bool whole = tb - ta == it.tiles;                // uniform
    auto row_of = [&](int f, int j) { return i0 + 4 * f + ((2 * w + j) >> 2); };
    auto at_of = [&](int f, int j) { return (size_t)(it.r.begin + min(row_of(f, j), it.r.n - 1)) * QM_GQA_HEADS + 4 * kvh + ((2 * w + j) & 3); };
    uint2 gate[NF][2];
    if (whole) {
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int j = 0; j < 2; ++j) gate[f][j] = *reinterpret_cast<const uint2*>(A.q_gate + at_of(f, j) * (2 * QM_GQA_HD) + QM_GQA_HD + 4 * lane);
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        const float l = sum_xor32(sum_xor16(st.sum[f].l));
        float* mine = reinterpret_cast<float*>(sh.ring[w][0]);
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) *reinterpret_cast<floatx4*>(mine + 256 * dt + 4 * ((c ^ (g + 4 * (dt & 1))) + 16 * g)) = st.o[f][dt];
        if (lane < 16) *reinterpret_cast<float2*>(mine + 4096 + 2 * lane) = make_float2(st.sum[f].m, l);
        // (LDS only: no wave waits for another's stores)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (row_of(f, j) >= it.r.n) continue;          // uniform
            const int col = 2 * w + j;
            // lane k, and every eighth from it: wave k's reference and sum
            const float2 ml = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(sh.ring[lane & 7][0]) + 4096 + 2 * col);
            floatx4 part_o[CHUNK_WAVES];
#pragma unroll
            for (int k = 0; k < CHUNK_WAVES; ++k)          // dims 4 lane ..: group lane >> 2, entry of the column and lane & 3
                part_o[k] = *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(sh.ring[k][0]) + 256 * (lane >> 2) +
                                                              4 * ((col ^ ((lane & 3) + (lane & 4))) + 16 * (lane & 3)));
            float M = fmaxf(ml.x, dpp_f32<0xB1>(ml.x));
            M = fmaxf(M, dpp_f32<0x4E>(M));
            M = fmaxf(M, dpp_f32<0x141>(M));
            const float e = ml.x == M ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
            float L = ml.y * e;
            L += dpp_f32<0xB1>(L);
            L += dpp_f32<0x4E>(L);
            L += dpp_f32<0x141>(L);
            floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < CHUNK_WAVES; ++k) o += part_o[k] * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(e), k));
            if (whole) {
                *reinterpret_cast<uint2*>(A.out + at_of(f, j) * QM_GQA_HD + 4 * lane) = chunk_gated(o * chunk_inverse(L), gate[f][j]);
            } else {
                float* to = part + f * QMK_CHUNK_COLUMN;
                *reinterpret_cast<floatx4*>(to + 256 * col + 4 * lane) = o;
                if (lane == 0) {
                    to[4096 + col] = M;
                    to[4112 + col] = L;
                }
            }
        }
        // before the next column's, or the next block's pages
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
}

// ---- many tokens ------------------------------------------------------------------
typedef float floatx16 __attribute__((ext_vector_type(16)));
// Lane (c, h) = (l & 31, l >> 5) has row c: o[dt][i] is dim
// 32 dt + 8 (i >> 2) + 4 h + (i & 3) of it.
struct ManyWave {
    half8 q[16];                       // dims 16 s + 8 h + e
    floatx16 o[8];
    ChunkSum sum;
    int pos;                           // -1: no row
};
// Token (of a half page) of score i: what stands at rows 8 (i >> 2) + 4 h +
// (i & 3) of the product.  Scores 8 k .. 8 k + 7 are those of a V operand.
QM_DEV int many_token(int i, int h) { return 16 * ((i >> 2) & 1) + 8 * (i >> 3) + 4 * h + (i & 3); }

// A product's 16 operand reads, CHUNK_AHEAD ahead of their use, so that LDS's
// latency passes under the matrix instructions before.  The order is pinned:
// the compiler's own had none ahead, where registers are short.  (Three ahead are
// no faster, and may cost a spill in the loop: 2048 tokens of 32768 1072 / 1039.)
#define CHUNK_AHEAD 2
template <class Read, class Use>
QM_DEV void many_product(Read read, Use use) {
    half8 a[CHUNK_AHEAD + 1];
#pragma unroll
    for (int i = 0; i < CHUNK_AHEAD; ++i) a[i] = read(i);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (i + CHUNK_AHEAD < 16) a[(i + CHUNK_AHEAD) % (CHUNK_AHEAD + 1)] = read(i + CHUNK_AHEAD);
        __builtin_amdgcn_sched_barrier(0);
        use(i, a[i % (CHUNK_AHEAD + 1)]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// The rows' queries, RMSNorm (1 + gamma, eps 1e-6) and RoPE straight into the
// operand: a row is in lanes c and c + 32, and the rotation's pairs (i, i + 32)
// in one.
QM_DEV void many_query(const GqaChunkArgs& A, half8 (&q)[16], const ChunkRow& r, int i, int head, int h) {
    const uint16_t* row = A.q_gate + ((size_t)(r.begin + i) * QM_GQA_HEADS + head) * (2 * QM_GQA_HD) + 8 * h;
    const size_t at = (size_t)(r.len - r.n + i) * (QM_GQA_ROT / 2) + 8 * h;
    uint4 u[16], gq[16];
    float4 cs[4], sn[4];
#pragma unroll
    for (int s = 0; s < 16; ++s) u[s] = *reinterpret_cast<const uint4*>(row + 16 * s);
#pragma unroll
    for (int s = 0; s < 16; ++s) gq[s] = *reinterpret_cast<const uint4*>(A.q_norm + 16 * s + 8 * h);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        cs[j] = ld4(A.rope_cos + at + 16 * (j >> 1) + 4 * (j & 1));
        sn[j] = ld4(A.rope_sin + at + 16 * (j >> 1) + 4 * (j & 1));
    }
    float ss = 0.0f;
#pragma unroll
    for (int s = 0; s < 16; ++s) ss = chunk_squares(u[s], ss);
    const float inv = chunk_inv(sum_xor32(ss));
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        float x1[8], x2[8];
        chunk_normed(x1, u[s], gq[s], inv);
        chunk_normed(x2, u[s + 2], gq[s + 2], inv);
        const float c8[8] = {cs[2 * s].x, cs[2 * s].y, cs[2 * s].z, cs[2 * s].w, cs[2 * s + 1].x, cs[2 * s + 1].y, cs[2 * s + 1].z, cs[2 * s + 1].w};
        const float s8[8] = {sn[2 * s].x, sn[2 * s].y, sn[2 * s].z, sn[2 * s].w, sn[2 * s + 1].x, sn[2 * s + 1].y, sn[2 * s + 1].z, sn[2 * s + 1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            q[s][e] = (_Float16)(x1[e] * c8[e] - x2[e] * s8[e]);
            q[s + 2][e] = (_Float16)(x2[e] * c8[e] + x1[e] * s8[e]);
        }
    }
#pragma unroll
    for (int s = 4; s < 16; ++s) {
        float x[8];
        chunk_normed(x, u[s], gq[s], inv);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[s][e] = (_Float16)x[e];
    }
}

// Half a tile, the 32 tokens from k0 on; meanwhile a part E of the next tile is
// made, for buffer buf ^ 1 of which `left` tokens are the row's.
template <class E>
QM_DEV void many_half(ManyWave& st, ChunkLds& sh, int buf, int half, int k0, bool edge, int left, int w, int lane) {
    const uint8_t* K = sh.tile[buf] + 16 * lane + 16384 * half;
    const uint8_t* V = K + 32768;
    const int h = lane >> 5;
    const float base = -chunk_base(st.sum);                // scores are counted from the reference
    floatx16 x;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = base;
    many_product([&](int s) { return *reinterpret_cast<const half8*>(K + 1024 * s); },
                 [&](int s, half8 a) { x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, st.q[s], x, 0, 0, 0); });
    E part;
    part.reads(sh, w, lane);
    if (edge) {                                            // uniform: some row does not see all of it
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = k0 + many_token(i, h) > st.pos ? -INFINITY : x[i];
    }
    int top = __float_as_int(x[0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) top = max(top, __float_as_int(x[i]));
    if (__any(top >= st.sum.due)) {                        // seldom after the first
        float mx = -INFINITY, corr;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[i]);
        const float up = chunk_raise(st.sum, max_xor32(mx), corr);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) st.o[dt] *= corr;
        x -= up;
    }
    half8 p[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        uintx4 w4;
#pragma unroll
        for (int i = 0; i < 4; ++i) w4[i] = chunk_pair(st.sum, x[8 * k + 2 * i], x[8 * k + 2 * i + 1]);
        p[k] = __builtin_bit_cast(half8, w4);
    }
    part.seldom(sh, buf ^ 1, left, w, lane);
    many_product([&](int i) { return *reinterpret_cast<const half8*>(V + 1024 * i); },
                 [&](int i, half8 a) {
                     st.o[i >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, p[i & 1], st.o[i >> 1], 0, 0, 0);
                     if ((i & 3) == 1) part.word(sh, buf ^ 1, i >> 2, w, lane);
                 });
    const uintx4 nan = *reinterpret_cast<const uintx4*>(sh.nan[buf][half]);
    if (__builtin_amdgcn_readfirstlane((int)(nan[0] | nan[1] | nan[2] | nan[3]))) {
        const int seen = st.pos - k0;                      // the last of the half's tokens that the row sees
        const uint32_t mask = seen < 0 ? 0u : seen >= 31 ? ~0u : (2u << seen) - 1;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) st.o[dt] += nan[dt >> 1] & mask ? __builtin_nanf("") : 0.0f;
    }
}
// A part of a tile by itself.
template <class E>
QM_DEV void many_make(ChunkLds& sh, int buf, int left, int w, int lane) {
    E part;
    part.reads(sh, w, lane);
    part.seldom(sh, buf, left, w, lane);
#pragma unroll
    for (int m = 0; m < 4; ++m) part.word(sh, buf, m, w, lane);
}

QM_DEV floatx4 many_four(const ManyWave& st, int j) {
    const int i = 4 * (j & 3);
    return floatx4{st.o[j >> 2][i], st.o[j >> 2][i + 1], st.o[j >> 2][i + 2], st.o[j >> 2][i + 3]};
}

template <int NF, bool MANY>
QM_DEV void many_item(const GqaChunkArgs& A, ChunkLds& sh, const typename Deal<NF, MANY>::Item& it, int ta, int tb, int kvh, float* part, int w, int lane) {
    const int c = lane & 31, h = lane >> 5, head = 4 * kvh + (w & 3);
    const int i0 = QMK_CHUNK_TOKENS * it.block + 32 * (w >> 2), i = i0 + c;      // the wave's first row, the lane's
    const int32_t* table = A.c.table + (size_t)it.r.row * A.c.max_pages;
    // page ids, one a lane, 64 at a time
    auto load_ids = [&](int t) { return t + lane < tb ? table[t + lane] : -1; };
    int ids = load_ids(ta);
    auto page_of = [&](int t) { return __builtin_amdgcn_readlane(ids, (t - ta) & 63); };
    int id = -1, next = page_of(ta);                       // of tiles t, t + 1
    if (kv4_is_page(A.c, next)) {
        many_fetch<0>(A, sh, next, kvh, w, lane);
        many_fetch<1>(A, sh, next, kvh, w, lane);
    }
    ManyWave st;
    st.pos = i < it.r.n ? it.r.len - it.r.n + i : -1;      // rows past the last: any row, never written
    many_query(A, st.q, it.r, min(i, it.r.n - 1), head, h);
    st.sum = chunk_sum();
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) st.o[dt] = floatx16{};
    const int first_pos = it.r.len - it.r.n + i0;
    // Tile t is multiplied while tile t + 1 is made of its codes, and those of
    // tile t + 2 come as soon as theirs are read.  A tile that is none (a page
    // that is none of the pool, past the last) is made of whatever stands there
    // and not multiplied.
    for (int t = ta - 1; t < tb; ++t) {
        if (t >= ta && ((t + 2 - ta) & 63) == 0) ids = load_ids(t + 2);
        const int after = t + 2 < tb ? page_of(t + 2) : -1;
        const int left = it.r.len - QMK_KV4_PAGE_TOKENS * (t + 1), k0 = QMK_KV4_PAGE_TOKENS * t, ln = chunk_lane(lane);
        const bool active = kv4_is_page(A.c, id) && i0 < it.r.n, more = kv4_is_page(A.c, after);
        const bool edge = k0 + QMK_KV4_PAGE_TOKENS - 1 > first_pos;
        // K's codes are here when only V's, which came after, are out
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(CHUNK_DMA) : "memory");
        if (active) many_half<ManyK>(st, sh, t & 1, 0, k0, edge, left, w, ln);
        else many_make<ManyK>(sh, (t + 1) & 1, left, w, ln);
        if (more) {
            many_fetch<0>(A, sh, after, kvh, w, ln);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(CHUNK_DMA) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if (active) many_half<ManyV>(st, sh, t & 1, 1, k0 + QMK_KV4_HALF_TOKENS, edge, left, w, ln);
        else many_make<ManyV>(sh, (t + 1) & 1, left, w, ln);
        if (more) many_fetch<1>(A, sh, after, kvh, w, ln);
        id = next;
        next = after;
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    // The rows by way of LDS (the tiles are read), 128 dims at a time, so that
    // memory sees whole runs of them.  Quad k of a row stands at k ^ row.
    const float l = sum_xor32(st.sum.l);
    const bool whole = tb - ta == it.tiles;
    const float inv = whole ? chunk_inverse(l) : 1.0f;
    const int ln = chunk_lane(lane), col = ln & 31;
    uint4 gate[2][8];                                      // in place of the queries: their latency passes once
    if (whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int row = min(i0 + 4 * j + (ln >> 4), it.r.n - 1);
            const uint16_t* at = A.q_gate + ((size_t)(it.r.begin + row) * QM_GQA_HEADS + head) * (2 * QM_GQA_HD) + QM_GQA_HD + 8 * (ln & 15);
#pragma unroll
            for (int p = 0; p < 2; ++p) gate[p][j] = *reinterpret_cast<const uint4*>(at + 128 * p);
        }
    }
    uint8_t* mine = sh.tile[0] + 16384 * w;
    part += w * 2 * QMK_CHUNK_COLUMN;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int j = 0; j < 16; ++j) *reinterpret_cast<floatx4*>(mine + 512 * col + 16 * ((2 * j + (ln >> 5)) ^ col)) = many_four(st, 16 * p + j) * inv;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (whole) {
            // 16 lanes a row, 8 dims a lane
            const int k = ln & 15, d = 128 * p + 8 * k;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = 4 * j + (ln >> 4), row = i0 + at;
                const floatx4 a = *reinterpret_cast<const floatx4*>(mine + 512 * at + 16 * ((2 * k) ^ at));
                const floatx4 b = *reinterpret_cast<const floatx4*>(mine + 512 * at + 16 * ((2 * k + 1) ^ at));
                if (row < it.r.n)
                    *reinterpret_cast<uint4*>(A.out + ((size_t)(it.r.begin + row) * QM_GQA_HEADS + head) * QM_GQA_HD + d) = chunk_gated8(a, b, gate[p][j]);
            }
        } else {
            // 32 lanes a row, 4 dims a lane
#pragma unroll 4
            for (int j = 0; j < 16; ++j) {
                const int at = 2 * j + (ln >> 5);
                *reinterpret_cast<floatx4*>(part + 256 * at + 128 * p + 4 * col) = *reinterpret_cast<const floatx4*>(mine + 512 * at + 16 * (col ^ at));
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // read, before it is written again
    }
    if (!whole && lane < 32) {
        part[8192 + lane] = st.sum.m;
        part[8224 + lane] = l;
    }
    asm volatile("s_barrier" ::: "memory");                // before the next block's tiles
}

// MANY: rows of more than QMK_CHUNK_FEW tokens are in blocks of many (otherwise
// the call has none of those, or is a short one).
template <int NF, bool MANY>
QM_DEV void chunk_attention(const GqaChunkArgs& A) {
    constexpr int kColumns = MANY ? 2 * CHUNK_WAVES : NF;
    constexpr size_t kBytes = MANY && sizeof(ChunkLds) > sizeof(FewLds<NF>) ? sizeof(ChunkLds) : sizeof(FewLds<NF>);
    __shared__ __attribute__((aligned(1024))) uint8_t sm[kBytes];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kvh = blockIdx.x & 3, index = blockIdx.x >> 2;
    if (CHUNK_SELDOM(blockIdx.x == 0 && w == 0)) {                       // for the merge
        int many = 0, few = 0;
        for (int b = lane; b < A.batch; b += 64) {
            const ChunkRow r = chunk_row(A, b);
            (Deal<NF, MANY>::few(r) ? few : many) += Deal<NF, MANY>::blocks(r);
        }
        many = __builtin_amdgcn_readlane((int)wave_scan((uint32_t)many), 63);
        few = __builtin_amdgcn_readlane((int)wave_scan((uint32_t)few), 63);
        if (lane == 0) *reinterpret_cast<int2*>(A.counts) = make_int2(many, few);
    }
    typename Deal<NF, MANY>::Sums sums{0.0, 0.0};
    typename Deal<NF, MANY>::Place from{0, {0, 0}, 0.0};
    for (double u = -1.0;;) {                              // uniform, as all of it
        // (made anew for each block: little of it takes registers while one is attended)
        const Deal<NF, MANY> deal(A, chunk_lane(lane), u < 0.0 ? nullptr : &sums);
        double end = 0.0;
        if (CHUNK_SELDOM(!deal.pieces)) {
            sums = typename Deal<NF, MANY>::Sums{Deal<NF, MANY>::lane_of(deal.total, 0), Deal<NF, MANY>::lane_of(deal.each, 0)};
            end = deal.begin(index + 1, from);
            if (u < 0.0) u = deal.begin(index, from);
            if (u >= end) return;
        }
        typename Deal<NF, MANY>::Item it;
        int ta, tb, last;                                  // the block's last workgroup
        if (!CHUNK_SELDOM(!deal.pieces)) {
            int n;
            if (!deal.find_piece(index, it, ta, tb, n)) return;
            last = index + n - 1;
            u = -1.0;
        } else {
            it = deal.find(u, true, from);
            const int weight = Deal<NF, MANY>::weight(it.r);
            ta = __builtin_amdgcn_readfirstlane(max(0, (int)((u - it.pages) / weight)));
            tb = __builtin_amdgcn_readfirstlane((int)fmin((double)it.tiles, (end - it.pages) / weight));
            last = tb == it.tiles ? index : (int)((it.pages + (double)it.tiles * weight - 1.0) / deal.each);
            u = Deal<NF, MANY>::lane_of(it.pages + (double)tb * weight, 0);
        }
        const bool more = u >= 0.0 && u < end;
        const bool few = Deal<NF, MANY>::few(it.r);
        // (ranges that overlap can have more row blocks than there are records)
        if (kvh == 0 && threadIdx.x == 0 && ta == 0 && (MANY || few) && it.number < (few ? A.few : A.many))
            A.records[(few ? A.many : 0) + it.number] = ChunkRecord{index, last, it.r.begin, it.r.n, it.block, {0, 0, 0}};
        if (it.r.kind != CHUNK_RUN) {
            const uint32_t fill = it.r.kind == CHUNK_NONE ? 0u : 0x7fc07fc0u;
            uint16_t* out = A.out + (size_t)it.r.begin * QM_GQA_HEADS * QM_GQA_HD + (size_t)4 * kvh * QM_GQA_HD + 4 * lane;
            for (int j = w; j < 4 * it.r.n; j += CHUNK_WAVES)
                *reinterpret_cast<uint2*>(out + ((size_t)(j >> 2) * QM_GQA_HEADS + (j & 3)) * QM_GQA_HD) = make_uint2(fill, fill);
            if (!more) return;
            continue;
        }
        // a workgroup's first block may have begun before it, its last end after it
        float* part = A.partial + (size_t)(2 * blockIdx.x + (ta == 0)) * kColumns * QMK_CHUNK_COLUMN;
        if (MANY && !few) many_item<NF, MANY>(A, *reinterpret_cast<ChunkLds*>(sm), it, ta, tb, kvh, part, w, lane);
        else few_item<NF, MANY>(A, *reinterpret_cast<FewLds<NF>*>(sm), it, ta, tb, kvh, part, w, lane);
        if (!more) return;
    }
}
extern "C" __global__ __launch_bounds__(64 * CHUNK_WAVES, 2) void qm_gqa_chunk_4(GqaChunkArgs A) { chunk_attention<1, false>(A); }
extern "C" __global__ __launch_bounds__(64 * CHUNK_WAVES, 2) void qm_gqa_chunk_32(GqaChunkArgs A) { chunk_attention<2, false>(A); }
extern "C" __global__ __launch_bounds__(64 * CHUNK_WAVES, 2) void qm_gqa_chunk_many(GqaChunkArgs A) { chunk_attention<2, true>(A); }

// The partial sums of a row block that several workgroups share, joined: a
// wave per Q rows of an operand column's 16, or of a wave's 32, 4 dims a lane.
// N partials' loads are in flight at a time.
template <int N, int Q>
QM_DEV void chunk_join(float (&m)[Q], float (&l)[Q], floatx4 (&o)[Q], const float* first, const float* others, int n, size_t stride, int row,
                       int sums, int rows, int lane) {
    for (int s0 = 0; s0 < n; s0 += N) {                    // uniform
        floatx4 a[N][Q];
        float pm[N][Q], pl[N][Q];
#pragma unroll
        for (int k = 0; k < N; ++k) {                      // past the last: the last again, with weight 0
            const int i = min(s0 + k, n - 1);
            const float* part = i == 0 ? first : others + i * stride;
#pragma unroll
            for (int j = 0; j < Q; ++j) {
                a[k][j] = *reinterpret_cast<const floatx4*>(part + 256 * (row + j) + 4 * lane);
                pm[k][j] = part[sums + row + j];
                pl[k][j] = part[sums + rows + row + j];
            }
        }
#pragma unroll
        for (int j = 0; j < Q; ++j) {
            float top = m[j];
#pragma unroll
            for (int k = 0; k < N; ++k) top = fmaxf(top, pm[k][j]);
            const float corr = m[j] == top ? 1.0f : __builtin_amdgcn_exp2f(m[j] - top);
            l[j] *= corr;
            o[j] *= corr;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                // a partial of no weight counts all the same: a NaN in it reaches the output (the last again has no other)
                const float f = s0 + k >= n ? 0.0f : pm[k][j] == top ? 1.0f : __builtin_amdgcn_exp2f(pm[k][j] - top);
                l[j] = fmaf(pl[k][j], f, l[j]);
                o[j] += a[k][j] * f;
            }
            m[j] = top;
        }
    }
}
// FEW: of a block of few tokens, else of many.
template <int NF, bool MANY, bool FEW>
QM_DEV void chunk_merge_one(const GqaChunkArgs& A, int k) {
    constexpr int kColumns = MANY ? 2 * CHUNK_WAVES : NF;  // of a workgroup's partial
    constexpr int kUnits = FEW ? NF : CHUNK_WAVES, kRows = FEW ? 16 : 32, kSums = FEW ? 4096 : 8192, Q = FEW ? 1 : 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = (4 * (k & 3) + wave) * Q, unit = (k >> 2) % kUnits, kvh = (k >> 2) / kUnits & 3, number = k / (16 * kUnits);
    const int count = A.counts[FEW];
    const ChunkRecord rec = A.records[(FEW ? A.many : 0) + number];
    if (number >= count || rec.from == rec.to) return;     // uniform
    // tokens of the block, and heads, of the rows
    const int i = FEW ? 4 * NF * rec.block + 4 * unit + (row >> 2) : QMK_CHUNK_TOKENS * rec.block + 32 * (unit >> 2) + row;
    const int head = 4 * kvh + (FEW ? row & 3 : unit & 3);
    if (i >= rec.n) return;
    uint2 gate[Q];
    uint16_t* out[Q];
#pragma unroll
    for (int j = 0; j < Q; ++j) {
        const size_t at = (size_t)(rec.begin + min(i + j, rec.n - 1)) * QM_GQA_HEADS + head;
        gate[j] = *reinterpret_cast<const uint2*>(A.q_gate + at * (2 * QM_GQA_HD) + QM_GQA_HD + 4 * lane);
        out[j] = A.out + at * QM_GQA_HD + 4 * lane;
    }
    float m[Q], l[Q];
    floatx4 o[Q];
#pragma unroll
    for (int j = 0; j < Q; ++j) {
        m[j] = -INFINITY;
        l[j] = 0.0f;
        o[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // the first workgroup's part ends its run, the others' begin theirs
    const size_t slot = (size_t)kColumns * QMK_CHUNK_COLUMN;
    const float* base = A.partial + (size_t)(2 * (4 * rec.from + kvh)) * slot + (size_t)(FEW ? 1 : 2) * unit * QMK_CHUNK_COLUMN;
    const int n = rec.to - rec.from + 1;
    if (n <= 4) chunk_join<4, Q>(m, l, o, base + slot, base, n, 8 * slot, row, kSums, kRows, lane);
    else chunk_join<8, Q>(m, l, o, base + slot, base, n, 8 * slot, row, kSums, kRows, lane);
#pragma unroll
    for (int j = 0; j < Q; ++j)
        if (i + j < rec.n) *reinterpret_cast<uint2*>(out[j]) = chunk_gated(o[j] * chunk_inverse(l[j]), gate[j]);
}
template <int NF, bool MANY>
QM_DEV void chunk_merge(const GqaChunkArgs& A) {
    const int before = MANY ? A.many * 4 * CHUNK_WAVES * 4 : 0;       // workgroups for blocks of many tokens
    if (MANY && (int)blockIdx.x < before) chunk_merge_one<NF, MANY, false>(A, blockIdx.x);
    else chunk_merge_one<NF, MANY, true>(A, blockIdx.x - before);
}
extern "C" __global__ __launch_bounds__(256) void qm_gqa_chunk_merge_4(GqaChunkArgs A) { chunk_merge<1, false>(A); }
extern "C" __global__ __launch_bounds__(256) void qm_gqa_chunk_merge_32(GqaChunkArgs A) { chunk_merge<2, false>(A); }
extern "C" __global__ __launch_bounds__(256) void qm_gqa_chunk_merge_many(GqaChunkArgs A) { chunk_merge<2, true>(A); }
