// gqa_decode_kv4.hip -- the GQA decode step over the paged 4-bit KV cache
// (qm_kv4.h) for gfx950: the mixer slice of qm_gqa_decode (gemv.rs:927-1011)
// with the cache's rows read as lo + s * code.
//
// Split-K flash decode: workgroup (b, g, split) has `chunk` tokens of kv head
// g and g's four query heads; qm_gqa_kv4_merge joins the splits (a single one
// finishes by itself).  A wave takes half a page (32 tokens) a round.
//
// Mathematics.  With K = lo + s c per group of 64 dims,
//   q . K = sum_groups s (q . c) + lo (sum of q over the group),
//   sum_t p V = sum_groups sum_t (p s) c + (sum_t p lo),
// so both products run on v_mfma_f32_16x16x32_bf16 over the codes themselves,
// and scales and minima enter in f32 on 1/64 of the values.
//   A code c in bits 0..3 (4..7) of a half is the bf16 subnormal c 2^-133
//   (16 c 2^-133): masks alone make operands of a word (5 instructions for 8
//   codes).  The other operand carries 2^90 (2^86 for the elements of bits
//   4..7), so products are in units of 2^-43: p s c of 2^-83 and more is a
//   normal f32, with all three parts from 2^-67 on.  What is lost below is
//   nothing beside K and V, multiples of 2^-24 or 0, and beside a row's largest
//   weight, 1 to 2^8.  q may be up to 2^37.
//   That operand is f32 and enters as three bf16 parts, 24 bits, exactly.
//   QK: A = 16 tokens' codes, B = q (column 4 part + head: 12 of the 16
//   columns that the instruction has anyway).  Lane (g, c) ends with tokens
//   4 g .. + 3 of column c; the parts' scores are summed over columns c & 3 by
//   two DPP adds, so that every lane holds its head's.
//   PV: A = p s (row 4 group + head, so a lane weighs its head's tokens for
//   one group only), B = the codes of 16 dims, an instruction per part; of the
//   result the rows of the dims' own group count.  With the parts as rows each
//   lane would weigh all four groups: a third of the instructions, but 144
//   vector instructions a round to make the operands instead of 52 (19 ragged
//   rows 29.5 us instead of 27.7 when it was changed, 64 x 32769 the same).
//   The minimum terms are the lanes' own: the lane of column 4 j + head adds
//   group j's.
// Softmax in base 2; a running maximum is raised only where a score passes it
// by 2^8, so the accumulators are seldom rescaled.
//
// What bounds it.  64 x 32769 tokens: the HBM stream (2.42 GB; the least of 24
// launches 430 us, 5.6 TB/s, their median 480 to 490; a copy of the kernel that
// only loads takes 419 at least).  Batches of some thousand tokens a row: the
// loads and what comes before the first of them (lengths, the deal, table,
// page), not the arithmetic: 19 ragged rows of up to 7001, 57k tokens, take 19
// us and a copy that only loads 4 less.  While its CUs work there, the vector
// unit is busy half of the time (375 instructions a wave and round; 39% of all
// lie outside the rounds) and the matrix unit a fifth (64).  Few tokens: the
// chain of dependent loads and the launches (1 token 6.4 us; 4097 7.3 and 2.5
// for the merge).
#include "qm_kv4_device.h"
#include "qm_kernel_args.h"

#define KV4_JOIN 32           // splits that the merge loads at a time
#define KV4_PART_STRIDE 260   // acc[256], m, l, pad[2]

// A batch row of the step: its table row and the tokens to read there, the
// last of them new (0: none, the output is zero).  A row that is refused (its
// output is NaN) is longer than max_len, or steps a table row that an earlier
// batch row has; or its last page is not its alone (other rows hold it too, or
// by its count none), which the wave that would write there finds.
struct StepRow {
    int row, len;
    bool refused;
};
// Lane l's batch row b, but for repeats (whose length counts here).
QM_DEV StepRow lane_row(const GqaKv4Args& A, int b) {
    StepRow r{-1, 0, false};
    if (b >= A.batch) return r;
    const int row = A.slots ? A.slots[b] : b;
    if ((uint32_t)row >= (uint32_t)A.c.rows) return r;
    r.row = row;
    const int len = max(A.c.lens[row], 0);
    r.refused = len > A.max_len;
    r.len = r.refused ? 0 : len;
    return r;
}
// Whether a batch row before b has table row `row`.  All lanes call it.
QM_DEV bool repeated(const GqaKv4Args& A, int b, int row, int lane) {
    bool found = false;
    if (A.slots)
        for (int j0 = 0; j0 < b; j0 += 64) {               // uniform
            const int j = j0 + lane;
            if (__ballot(j < b && A.slots[min(j, b - 1)] == row)) found = true;
        }
    return found;
}
// ceil(len / chunk), chunk a multiple of 128: the f32 quotient is off by two at
// most, and put right.
QM_DEV int splits_of(int len, int chunk) {
    const uint32_t all = (uint32_t)len, each = (uint32_t)chunk;
    uint32_t n = (uint32_t)((float)len * __builtin_amdgcn_rcpf((float)chunk));
    n -= n * each >= all && n > 0;
    n -= n * each >= all && n > 0;
    n += n * each < all;
    return (int)(n + (n * each < all));
}

// How the step's tokens are dealt to workgroups: splits of `chunk` tokens of
// each row, the rows one after the other.  The chunk follows from the lengths
// that the rows have now, so that a ragged batch fills the chip as evenly as
// an equal one, and a captured step whose max_len is the capacity as one whose
// max_len is its length.  Every workgroup finds the same chunk: one workgroup
// per CU, or two where that makes the chunk enough shorter, and not a few more
// than that, which would be a round of their own.  Two workgroups on a CU take
// 1.7 times as long as one.  Measured, the step in us, one per CU / two: 1 x
// 32769 tokens 16.7 / 18.3, 8 x 4097 15.8 / 17.9, 16 ragged rows of up to 7001
// 20.6 / 21.1, 64 x 2049 35.1 / 33.3.  One, too, where the merge would have
// more splits of two than it loads at a time (1 x 16000 11.4 / 13.7, 4 rows of
// 20000 and less 17.9 / 19.7).  Where that passes QMK_KV4_MAX_SPLIT tokens, so
// many full rounds of two workgroups a CU that it does not (the longest chunk /
// this: 64 x 10001 166 / 145, 3 x 200001 157 / 139); past QMK_KV4_ROUNDS rounds,
// where a partial one no longer counts, the longest chunk.
struct Deal {
    int chunk;
    int b, first;            // a batch row, and the splits before its own
    StepRow r;
};
QM_DEV int chunk_for(const GqaKv4Args& A, float want, int groups, int len) {
    int chunk = __builtin_amdgcn_readfirstlane(((int)fminf(want, (float)(QMK_KV4_MAX_SPLIT - 1)) + 128) / 128 * 128);   // more than `want`
    if (A.batch <= 64)
        for (int tries = 0; tries < 4 && chunk < QMK_KV4_MAX_SPLIT; ++tries, chunk += 128)
            if (QM_GQA_KV_HEADS * __builtin_amdgcn_readlane((int)wave_scan((uint32_t)splits_of(len, chunk)), 63) <= groups) break;
    return chunk;
}
QM_DEV int deal_chunk(const GqaKv4Args& A, const StepRow& mine, int lane) {
    float total = (float)mine.len, longest = total;        // the first 64 rows stay in the lanes
    for (int b0 = 64; b0 < A.batch; b0 += 64) {
        const float len = (float)lane_row(A, b0 + lane).len;
        total += len;
        longest = fmaxf(longest, len);
    }
    const float want = wave_sum64(total) * QM_GQA_KV_HEADS * __builtin_amdgcn_rcpf((float)A.cus);
    int one = QMK_KV4_MAX_SPLIT;
    if (want < (float)(QMK_KV4_MAX_SPLIT - 1)) one = chunk_for(A, want, A.cus, mine.len);
    if (one == 128) return one;
    // (2^-7: the f32 sum's error must not make a round more than the host counts)
    const float rounds = fmaxf(ceilf(want * (0.5f / QMK_KV4_MAX_SPLIT) - 0x1p-7f), 1.0f);
    if (rounds > (float)QMK_KV4_ROUNDS) return QMK_KV4_MAX_SPLIT;
    const int two = chunk_for(A, want * 0.5f * __builtin_amdgcn_rcpf(rounds), 2 * A.cus * (int)rounds, mine.len);
    const bool many = __builtin_amdgcn_readfirstlane(max_xor32(max_xor16(row_max16(longest))) > (float)(KV4_JOIN * two));
    return (10 * one <= 17 * two || many) && one < QMK_KV4_MAX_SPLIT ? one : two;
}
// The row of split k (all lanes agree), false past the last split; and, where
// `note`, batch row k's splits to the merge: {first, splits}, -1 splits where
// it is refused.
QM_DEV bool deal_split(const GqaKv4Args& A, Deal& d, int k, bool note, int lane) {
    StepRow mine = lane_row(A, lane);
    d.chunk = deal_chunk(A, mine, lane);
    d.first = 0;
    bool found = false;
    int first = 0;
    for (int b0 = 0; b0 < A.batch; b0 += 64) {             // uniform
        if (b0) mine = lane_row(A, b0 + lane);
        const int n = splits_of(mine.len, d.chunk), incl = (int)wave_scan((uint32_t)n), all = __builtin_amdgcn_readlane(incl, 63);
        if (!found && k < first + all) {
            const int at = __popcll(__ballot(first + incl <= k));
            found = true;
            d.b = b0 + at;
            d.first = first + __builtin_amdgcn_readlane(incl - n, at);
            d.r.row = __builtin_amdgcn_readlane(mine.row, at);
            d.r.len = __builtin_amdgcn_readlane(mine.len, at);
            d.r.refused = repeated(A, d.b, d.r.row, lane);
        }
        if (note && k >= b0 && k < b0 + 64) {
            const int row = __builtin_amdgcn_readlane(mine.row, k - b0);
            const bool refused = __builtin_amdgcn_readlane(mine.refused, k - b0) || (row >= 0 && repeated(A, k, row, lane));
            if (lane == k - b0) reinterpret_cast<int2*>(A.splits)[k] = make_int2(first + incl - n, refused ? -1 : n);
        }
        if (found && (!note || k < b0 + 64)) break;
        first += all;
    }
    return found;
}

template <int CTRL>
QM_DEV double dpp_f64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
QM_DEV double readlane_f64(double x, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over the wave in 64 bits.
QM_DEV double wave_sum64_f64(double x) {
    x += dpp_f64<0xB1>(x);
    x += dpp_f64<0x4E>(x);
    x += dpp_f64<0x141>(x);
    x += dpp_f64<0x140>(x);
    return (readlane_f64(x, 0) + readlane_f64(x, 16)) + (readlane_f64(x, 32) + readlane_f64(x, 48));
}

// A head's row, lane l with dims 4 l .. 4 l + 3: RMSNorm (1 + gamma, eps
// 1e-6), and the rotation of dims 0..63 (gemv.rs:586-627).  Apart, so that the
// norm is done by the time the RoPE rows arrive.
QM_DEV void norm_head(float (&x)[4], uint2 gw) {
    const uint16_t g[4] = {(uint16_t)(gw.x & 0xffffu), (uint16_t)(gw.x >> 16), (uint16_t)(gw.y & 0xffffu), (uint16_t)(gw.y >> 16)};
    const float ss = wave_sum64((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]));
    const float inv = 1.0f / sqrtf(ss / (float)QM_GQA_HD + 1e-6f);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = x[i] * inv * (1.0f + f16_to_f32(g[i]));
}
QM_DEV void rotate_head(float (&x)[4], const float (&c)[4], const float (&s)[4], int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p = dpp_f32<0x128>(x[i]);
        x[i] = lane < 8 ? x[i] * c[i] - p * s[i] : lane < 16 ? x[i] * c[i] + p * s[i] : x[i];
    }
}
// The new k row likewise, in 64 bits: a code beside a border must not depend
// on the order of a sum.
QM_DEV void norm_new_k(double (&x)[4], uint2 gw) {
    const uint16_t g[4] = {(uint16_t)(gw.x & 0xffffu), (uint16_t)(gw.x >> 16), (uint16_t)(gw.y & 0xffffu), (uint16_t)(gw.y >> 16)};
    const double mean = wave_sum64_f64((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3])) * (1.0 / QM_GQA_HD) + 1e-6;
    // v_rsq_f64 is good to about 2^-24; each step of Newton's squares the error
    double inv = __builtin_amdgcn_rsq(mean);
#pragma unroll
    for (int i = 0; i < 2; ++i) inv = inv * __builtin_fma(-0.5 * mean * inv, inv, 1.5);
    if (!(mean < __builtin_inf())) inv = mean == mean ? 0.0 : mean;      // rsq's own 0 for an infinity, NaN for NaN
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = x[i] * inv * (1.0 + (double)f16_to_f32(g[i]));
}
// Its rotation, and the roundings to f32 and to the f16 cache's type.
QM_DEV void rotate_new_k(uint16_t (&out)[4], const double (&x)[4], const float (&c)[4], const float (&s)[4], int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double p = dpp_f64<0x128>(x[i]);
        const double turned = lane < 8 ? x[i] * c[i] - p * s[i] : x[i] * c[i] + p * s[i];
        out[i] = f64_to_f16_by_f32(lane < 16 ? turned : x[i]);
    }
}

// Scale, minimum and codes of one head's row, four f16 values a lane (a
// group of 64 dims is a DPP row of 16 lanes).
struct CodedRow {
    uint16_t s, lo;
    uint32_t q[4];
};
QM_DEV CodedRow code_row(const uint16_t (&h)[4]) {
    float x[4];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = f16_to_f32(h[i]);
        bad = bad || (h[i] & 0x7fffu) >= 0x7c00u;
    }
    const float lo = -row_max16(-fminf(fminf(x[0], x[1]), fminf(x[2], x[3])));
    const float hi = row_max16(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    bad = row_max16(bad ? 1.0f : 0.0f) > 0.0f;
    CodedRow c;
    c.s = bad ? (uint16_t)0x7e00u : kv4_scale(lo, hi);
    c.lo = bad ? (uint16_t)0x7e00u : f32_to_f16(lo);
    const float s = f16_to_f32(c.s), inv = __builtin_amdgcn_rcpf(s);
#pragma unroll
    for (int i = 0; i < 4; ++i) c.q[i] = kv4_code(x[i], lo, s, inv);
    return c;
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

#define KV4_WAVES 4
#define KV4_Q_STRIDE (QM_GQA_HD + 8)   // bf16 of a q row in LDS: 16 rows 528 bytes apart fall into different banks

// A wave's half pages come by LDS DMA, as they stand, into one of its two
// buffers, the one after the next in flight; lane (g, c) = (lane >> 4,
// lane & 15) reads its operands from there.
#define KV4_DMA (QMK_KV4_HALF_BYTES / 1024)
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
QM_DEV void lds4(uint32_t* into, const uint8_t* from) {
    const uintx4 v = *reinterpret_cast<const uintx4*>(from);
    into[0] = v[0], into[1] = v[1], into[2] = v[2], into[3] = v[3];
}
QM_DEV void fetch_half(const uint8_t* half, uint32_t buf, int lane) {
#pragma unroll
    for (int i = 0; i < KV4_DMA; ++i) dma16_off(half + 1024 * i, 16 * lane, buf + 1024 * i);
}
// The eight codes of a word as bf16 subnormals, elements 2, 3, 6, 7 times 16.
QM_DEV bf16x8 codes_bf16(uint32_t w) {
    const uint32_t v = w >> 8;
    uint4 m = make_uint4(w & 0x000f000fu, w & 0x00f000f0u, v & 0x000f000fu, v & 0x00f000f0u);
    // opaque to the optimiser, which would otherwise fold each mask into a
    // per-nibble bit-field extract
    asm("" : "+v"(m.x), "+v"(m.y), "+v"(m.z), "+v"(m.w));
    return __builtin_bit_cast(bf16x8, m);
}

// The same with the odd elements' codes from the other end, 15 - c (they are
// the upper halves): one v_bitop3 each instead of the and.
QM_DEV bf16x8 codes_bf16_turned(uint32_t w) {
    const uint32_t v = w >> 8;
    uint4 m = make_uint4((w & 0x000f000fu) ^ 0x000f0000u, (w & 0x00f000f0u) ^ 0x00f00000u, (v & 0x000f000fu) ^ 0x000f0000u,
                         (v & 0x00f000f0u) ^ 0x00f00000u);
    asm("" : "+v"(m.x), "+v"(m.y), "+v"(m.z), "+v"(m.w));
    return __builtin_bit_cast(bf16x8, m);
}

// An f32 with the upper 8 bits of its significand: what a bf16 of its upper
// half holds.
QM_DEV float upper8(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
QM_DEV uint32_t pack_hi(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
QM_DEV half2_t halves(uint32_t u) { return __builtin_bit_cast(half2_t, u); }

// Per-wave softmax state and accumulators.  m: the maximum, in the scores'
// units.  o[m]: dims 16 m + c; in lane group g = m >> 2, whose group of dims
// that is, element e is head e's sum, in units of 2^-43; lo: the lane's share
// of its head's and group's minimum terms, l of its head's sum.
struct WaveKv4 {
    float m, l, lo;
    floatx4 o[16];
};

struct SplitKv4Lds {
    __attribute__((aligned(16))) uint8_t ring[KV4_WAVES][2][QMK_KV4_HALF_BYTES];   // later acc: [wave][head][dim] f32
    __attribute__((aligned(16))) uint16_t q[13][KV4_Q_STRIDE];       // row 4 part + head; row 12 zero
    float qsum[4][4];                                                // [head][group]
    float m[KV4_WAVES][4], l[KV4_WAVES][4];
    // the new token: K words [dims / 128][g], V codes as bytes [c][4 j + m], scales and minima [s, lo of K, of V][group]
    __attribute__((aligned(16))) uint32_t kw[2][4][4];
    __attribute__((aligned(16))) uint8_t vq[16][16];
    uint16_t meta[4][4];
};

// The new token t (0 .. 31 of the half page) into the fetched half page and
// into the cache's.
QM_DEV void put_token(uint8_t* buf, uint8_t* half, const SplitKv4Lds& sh, int t, int lane) {
    if (lane < 8) {
        const uintx4 w = *reinterpret_cast<const uintx4*>(sh.kw[lane >> 2][lane & 3]);
        const int at = 4 * kv4_k_word(t, 128 * (lane >> 2) + 8 * (lane & 3));
        *reinterpret_cast<uintx4*>(buf + at) = w;
        *reinterpret_cast<uintx4*>(half + at) = w;
    }
    const int shift = 4 * kv4_v_nibble(t);
    const int at = 4 * kv4_v_word(t, 64 * (lane >> 4) + (lane & 15));
    const uint32_t q = *reinterpret_cast<const uint32_t*>(&sh.vq[lane & 15][4 * (lane >> 4)]);
    uint32_t w[4];
    lds4(w, buf + at);
#pragma unroll
    for (int m = 0; m < 4; ++m) w[m] = (w[m] & ~(15u << shift)) | ((q >> (8 * m)) & 15u) << shift;
    *reinterpret_cast<uintx4*>(buf + at) = uintx4{w[0], w[1], w[2], w[3]};
    *reinterpret_cast<uintx4*>(half + at) = uintx4{w[0], w[1], w[2], w[3]};
    if (lane < 16) {
        const int which = lane >> 2, group = lane & 3;
        const int m = QMK_KV4_META + 256 * which + 2 * (which & 1 ? kv4_lo_at(t, group) : kv4_s_at(t, group));
        const uint16_t x = sh.meta[which][group];
        *reinterpret_cast<uint16_t*>(buf + m) = x;
        *reinterpret_cast<uint16_t*>(half + m) = x;
    }
}

// Scores of the half page's 32 tokens: x[4 u + i] of token 16 u + 4 g + i and
// head c & 3, in units of 2^-43 ln 2 / 16 (as qsum).
template <int CTRL>
QM_DEV float add_dpp(float x) {      // update_dpp, unlike mov_dpp, is folded into the add
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
QM_DEV void scores(float (&x)[8], const uint8_t* buf, const uint16_t* qsrc, float qsum, int lane) {
    uint32_t w[2][8], s[8][2], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) lds4(&w[i >> 1][4 * (i & 1)], buf + 1024 * i + 16 * lane);
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) lds4(&s[2 * i][0], buf + QMK_KV4_META + 64 * g + 16 * i);
    lds4(lo, buf + QMK_KV4_META + 256 + (4 * (c >> 2) + g) * 16);
    floatx4 acc[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[u][n] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int n = 2 * (i & 3) + (i >> 2);                // both halves of a group four steps apart
        const bf16x8 q = *reinterpret_cast<const bf16x8*>(qsrc + 32 * n);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            acc[u][n >> 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_bf16(w[u][n]), q, acc[u][n >> 1], 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int u = e >> 2, i = e & 3;
        const half2_t s01 = halves(s[e][0]), s23 = halves(s[e][1]);
        float t = fmaf((float)halves(lo[e >> 1])[e & 1], qsum, 0.0f);
        t = fmaf(acc[u][0][i], (float)s01[0], t);
        t = fmaf(acc[u][1][i], (float)s01[1], t);
        t = fmaf(acc[u][2][i], (float)s23[0], t);
        t = fmaf(acc[u][3][i], (float)s23[1], t);
        x[e] = add_dpp<0x124>(add_dpp<0x128>(t));                    // the parts: columns 8 and 4 apart
    }
}

// The softmax weights of a round, and their products with V.
QM_DEV void weigh(WaveKv4& st, float (&x)[8], const uint8_t* buf, int left, float sign, int lane) {
    const int c = lane & 15, g = lane >> 4;
    uint32_t vw[16], lo[4];
    uint16_t sv[8];                                      // scales of the lane's eight tokens, group c >> 2
#pragma unroll
    for (int e = 0; e < 8; ++e) sv[e] = *reinterpret_cast<const uint16_t*>(buf + QMK_KV4_META + 512 + 64 * g + 8 * e + 2 * (c >> 2));
    lds4(lo, buf + QMK_KV4_META + 768 + (4 * (c >> 2) + g) * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) lds4(&vw[4 * j], buf + 4 * QMK_KV4_V_WORDS + 1024 * j + 16 * lane);
    if (left < QMK_KV4_HALF_TOKENS) {                    // uniform: tokens from `left` on are none
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool none = 16 * (e >> 2) + 4 * g + (e & 3) >= left;
            x[e] = none ? -INFINITY : x[e];
            // whatever stands there: a weight of zero times it must be zero
            sv[e] = none ? (uint16_t)0 : sv[e];
            lo[e >> 1] = none ? lo[e >> 1] & (e & 1 ? 0xffffu : 0xffff0000u) : lo[e >> 1];
        }
    }
    float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    mx = max_xor32(max_xor16(mx));
    if (__ballot(mx > st.m + 0x1p-40f)) {                // uniform: 2^8
        const float m = mx > st.m + 0x1p-40f ? mx : st.m, was = st.m;
        st.m = m;
        if (__ballot(was != -INFINITY)) {                // else nothing is summed yet
            const float f = was == m ? 1.0f : __builtin_amdgcn_exp2f((was - m) * 0x1p43f);
            st.l *= f;
            st.lo *= f;
            const float f0 = readlane_f32(f, 0), f1 = readlane_f32(f, 1), f2 = readlane_f32(f, 2), f3 = readlane_f32(f, 3);
#pragma unroll
            for (int m4 = 0; m4 < 16; ++m4) {
                st.o[m4][0] *= f0;
                st.o[m4][1] *= f1;
                st.o[m4][2] *= f2;
                st.o[m4][3] *= f3;
            }
        }
    }
    const float bias = -st.m * 0x1p43f;
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(x[e], 0x1p43f, bias));
    st.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    // Every other token from the other end of its range, lo + s c = (lo + 15 s)
    // - s (15 - c): both sums then hover about the result instead of growing
    // with the tokens and cancelling at the end (at 32769 tokens of like weight
    // that cost a factor 5 of the error).
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float from = (float)halves(lo[e >> 1])[e & 1];
        st.lo = fmaf(p[e], e & 1 ? fmaf((float)__builtin_bit_cast(_Float16, sv[e]), 15.0f, from) : from, st.lo);
    }
    // the three parts of p s: upper 8, middle 8 and lower 8 bits of its significand
    uint32_t part[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a[2], r[2], q[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float w = p[2 * i + h] * ((i & 1 ? 0x1p86f : 0x1p90f) * (h ? -sign : sign));
            a[h] = fmaf(w, (float)__builtin_bit_cast(_Float16, sv[2 * i + h]), 0.0f);
            r[h] = a[h] - upper8(a[h]);
            q[h] = r[h] - upper8(r[h]);
        }
        part[0][i] = pack_hi(__float_as_uint(a[0]), __float_as_uint(a[1]));
        part[1][i] = pack_hi(__float_as_uint(r[0]), __float_as_uint(r[1]));
        part[2][i] = pack_hi(__float_as_uint(q[0]), __float_as_uint(q[1]));
    }
    bf16x8 a[3];
#pragma unroll
    for (int n = 0; n < 3; ++n) a[n] = __builtin_bit_cast(bf16x8, uintx4{part[n][0], part[n][1], part[n][2], part[n][3]});
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        bf16x8 v[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) v[m] = codes_bf16_turned(vw[4 * j + m]);
#pragma unroll
        for (int n = 0; n < 3; ++n)
#pragma unroll
            for (int m = 0; m < 4; ++m) st.o[4 * j + m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[n], v[m], st.o[4 * j + m], 0, 0, 0);
    }
}

// The gated output of head h of g, dims 4 lane .. + 3; l = 0: no tokens.
QM_DEV void kv4_out(const GqaKv4Args& A, int b, int h, int lane, float4 o, float l, float4 gate, bool refused) {
    const float inv = l != 0.0f ? __builtin_amdgcn_rcpf(l) : 0.0f;
    float4 r = make_float4(o.x * inv * sigmoid_fast(gate.x), o.y * inv * sigmoid_fast(gate.y), o.z * inv * sigmoid_fast(gate.z),
                           o.w * inv * sigmoid_fast(gate.w));
    if (refused) r.x = r.y = r.z = r.w = __builtin_nanf("");
    st4(A.out + ((size_t)b * QM_GQA_HEADS + h) * QM_GQA_HD + 4 * lane, r);
}
QM_DEV float4 kv4_gate(const GqaKv4Args& A, int b, int h, int lane) {
    return ld4(A.q_gate + ((size_t)b * QM_GQA_HEADS + h) * (2 * QM_GQA_HD) + QM_GQA_HD + 4 * lane);
}

QM_DEV uint32_t lds_of(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }

extern "C" __global__ __launch_bounds__(64 * KV4_WAVES, 2) void qm_gqa_kv4_split(GqaKv4Args A) {
    __shared__ SplitKv4Lds sh;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x & 3, index = blockIdx.x >> 2;
    if (A.result && A.result[0] != 0 && !A.single) return;
    // A workgroup for each (split, head); with A.single one for each (batch
    // row, head), which then finishes by itself.
    Deal deal;
    if (A.single) {
        deal.chunk = QMK_KV4_MAX_SPLIT;
        deal.b = deal.first = index;
        deal.r = lane_row(A, index);
        deal.r.refused = deal.r.refused || (deal.r.row >= 0 && repeated(A, index, deal.r.row, lane));
        if (A.result && A.result[0] != 0) deal.r = StepRow{-1, 0, false};
    } else if (!deal_split(A, deal, index, kvh == 0 && index < A.batch && w == 0, lane) || deal.r.refused) {
        return;                                            // uniform, as are all values of `deal`
    }
    const int b = __builtin_amdgcn_readfirstlane(deal.b), chunk = deal.chunk;
    StepRow r = deal.r;
    if (r.refused) r.len = 0;
    const int split = index - deal.first, t_begin = split * chunk;

    // The loads that depend on no other: q, the new token's row (wave 0 k, wave
    // 1 v) and the split's page ids, one a lane (a split has at most 64 pages).
    const float4 qx = ld4(A.q_gate + ((size_t)b * QM_GQA_HEADS + 4 * kvh + w) * (2 * QM_GQA_HD) + 4 * lane);
    const uint2 qn = *reinterpret_cast<const uint2*>(A.q_norm + 4 * lane);
    const float4 nx = ld4((w == 0 ? A.k_new : A.v_new) + ((size_t)b * QM_GQA_KV_HEADS + kvh) * QM_GQA_HD + 4 * lane);
    const uint2 kn = *reinterpret_cast<const uint2*>(A.k_norm + 4 * lane);
    float4 gate = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (A.single) gate = kv4_gate(A, b, 4 * kvh + w, lane);
    const int page0 = t_begin / QMK_KV4_PAGE_TOKENS;
    int ids = -1;
    if (lane < chunk / QMK_KV4_PAGE_TOKENS && page0 + lane < A.c.max_pages)
        ids = A.c.table[(size_t)max(r.row, 0) * A.c.max_pages + page0 + lane];

    const int t_end = min(t_begin + chunk, r.len);
    const int h0 = t_begin / QMK_KV4_HALF_TOKENS + w;
    const int h_end = __builtin_amdgcn_readfirstlane((t_end + QMK_KV4_HALF_TOKENS - 1) / QMK_KV4_HALF_TOKENS);
    auto half_of = [&](int h, bool& there) {
        const int id = __builtin_amdgcn_readlane(ids, (h >> 1) - page0);
        there = kv4_is_page(A.c, id);
        return kv4_half(A.c, A.layer, there ? id : 0, kvh, h & 1);
    };
    // The compiler does not count the DMA below: what it loads has to be here
    // before that starts, or its waits would take the DMA's for its own.
    asm volatile("" ::"v"(qx.x), "v"(qn.x), "v"(nx.x), "v"(kn.x), "v"(gate.x), "v"(ids));

    // The RoPE rows of the new position (to LDS, a q row that this wave writes
    // later), then the wave's first two half pages.
    const int pos = max(r.len - 1, 0);
    uint16_t* rope = sh.q[8 + w];
    dma4((lane < 32 ? A.rope_cos : A.rope_sin) + (size_t)pos * (QM_GQA_ROT / 2) + (lane & 31), lds_of(rope));
    bool there[2] = {false, false};
    uint8_t* half[2] = {nullptr, nullptr};
    const uint32_t ring = lds_of(sh.ring[w]);
    int ahead = 0;                                         // DMA instructions after the RoPE rows'
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (h0 + KV4_WAVES * i < h_end) {
            half[i] = half_of(h0 + KV4_WAVES * i, there[i]);
            fetch_half(half[i], ring + QMK_KV4_HALF_BYTES * i, lane);
            ahead += KV4_DMA;
        }
    }
    // the norms meanwhile
    const bool appends = pos >= t_begin && pos < t_end;
    const int new_half = appends ? pos / QMK_KV4_HALF_TOKENS : -1;
    int holders = 0;                                       // of the page to write to
    if (new_half >= h0 && (new_half - h0) % KV4_WAVES == 0) {
        const int id = __builtin_amdgcn_readlane(ids, (new_half >> 1) - page0);
        if (kv4_is_page(A.c, id)) holders = A.c.refs[id];
    }
    float q[4] = {qx.x, qx.y, qx.z, qx.w};
    norm_head(q, qn);
    double k64[4] = {nx.x, nx.y, nx.z, nx.w};
    if (appends && w == 0) norm_new_k(k64, kn);
    if (ahead == 2 * KV4_DMA) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * KV4_DMA) : "memory");
    else if (ahead == KV4_DMA) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(KV4_DMA) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    float rc[4], rs[4];
    lds4(reinterpret_cast<uint32_t*>(rc), reinterpret_cast<const uint8_t*>(rope) + 16 * (lane & 7));
    lds4(reinterpret_cast<uint32_t*>(rs), reinterpret_cast<const uint8_t*>(rope) + 128 + 16 * (lane & 7));

    // q of head 4 kvh + w: RoPE, the softmax's scale, and the parts
    {
        rotate_head(q, rc, rs, lane);
        const float scale = 1.4426950408889634f / 16.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] *= scale;
        const float sum = row_sum16((q[0] + q[1]) + (q[2] + q[3]));
        if (c == 0) sh.qsum[w][g] = sum * 0x1p-43f;
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] *= i < 2 ? 0x1p90f : 0x1p86f;
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            *reinterpret_cast<uint2*>(&sh.q[4 * j + w][4 * lane]) =
                make_uint2(pack_hi(__float_as_uint(q[0]), __float_as_uint(q[1])), pack_hi(__float_as_uint(q[2]), __float_as_uint(q[3])));
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] -= upper8(q[i]);
        }
        if (w == 3) *reinterpret_cast<uint2*>(&sh.q[12][4 * lane]) = make_uint2(0, 0);
    }
    if (appends && w < 2) {                                // uniform per wave
        uint16_t x[4] = {f32_to_f16(nx.x), f32_to_f16(nx.y), f32_to_f16(nx.z), f32_to_f16(nx.w)};
        if (w == 0) rotate_new_k(x, k64, rc, rs, lane);
        const CodedRow q = code_row(x);
        if (w == 0) {
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) word |= q.q[i] << (4 * kv4_nibble(4 * (lane & 1) + i));
            word |= __builtin_amdgcn_mov_dpp((int)word, 0xB1, 0xF, 0xF, false);
            const int d = 4 * lane;
            if ((lane & 1) == 0) sh.kw[d >> 7][(d >> 3) & 3][(d >> 5) & 3] = word;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 4 * lane + i;                // dim 64 j + 16 m + c
                sh.vq[d & 15][d >> 4] = (uint8_t)q.q[i];
            }
        }
        if (c == 0) {
            sh.meta[2 * w][g] = q.s;
            sh.meta[2 * w + 1][g] = q.lo;
        }
    }
    // every wave's q and the new token; the DMA stays in flight
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

    WaveKv4 st;
    st.m = -INFINITY;
    st.l = st.lo = 0.0f;
#pragma unroll
    for (int m = 0; m < 16; ++m) st.o[m] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint16_t* qsrc = &sh.q[min(c, 12)][8 * g];
    const float qsum = sh.qsum[c & 3][c >> 2];
    // Where a product is larger than the accumulator, the matrix instruction cuts
    // the accumulator's last bits off, downwards (measured, 0.46 of the product's
    // unit on average): the same error every round.  Odd waves sum the negatives,
    // and it cancels over the waves (5 rows of up to 27754 tokens: relative error
    // 1.6e-6 - 2.4e-6 without, 6.2e-7 with).
    const float sign = w & 1 ? -1.0f : 1.0f;
    int i = 0;
    for (int h = h0; h < h_end; h += KV4_WAVES, i ^= 1) {
        // this round's half page is here when only the next one's DMA is out
        if (h + KV4_WAVES < h_end) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(KV4_DMA) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        uint8_t* buf = sh.ring[w][i];
        if (there[0]) {
            if (h == new_half) {
                if (holders != 1) st.l = __builtin_nanf("");
                else put_token(buf, half[0], sh, pos & (QMK_KV4_HALF_TOKENS - 1), lane);
            }
            float x[8];
            scores(x, buf, qsrc, qsum, lane);
            weigh(st, x, buf, t_end - h * QMK_KV4_HALF_TOKENS, sign, lane);
        }
        half[0] = half[1];
        there[0] = there[1];
        if (h + 2 * KV4_WAVES < h_end) {
            half[1] = half_of(h + 2 * KV4_WAVES, there[1]);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the buffer's reads are done
            fetch_half(half[1], ring + QMK_KV4_HALF_BYTES * i, lane);
        }
    }

    // Lane group g has group g of the dims, for its four heads.  A head's
    // minimum term of that group stands in the lanes of column 4 g + head.
    {
        const float l = sum_xor32(sum_xor16(st.l)), lo = sum_xor32(sum_xor16(st.lo));
        if (lane < 4) {
            sh.m[w][lane] = st.m;
            sh.l[w][lane] = l;
        }
        float* acc = reinterpret_cast<float*>(sh.ring[w]);          // the wave's own buffers, all read
#pragma unroll
        for (int head = 0; head < 4; ++head) {
            const float base = __shfl(lo, 4 * g + head);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const float a = g & 1 ? st.o[4 + m][head] : st.o[m][head], d = g & 1 ? st.o[12 + m][head] : st.o[8 + m][head];
                acc[head * QM_GQA_HD + 64 * g + 16 * m + c] = fmaf(g & 2 ? d : a, sign * 0x1p43f, base);
            }
        }
    }
    __syncthreads();
    {
        const int h = w;                                    // head 4 kvh + h, dims 4 lane .. + 3
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < KV4_WAVES; ++i) M = fmaxf(M, sh.m[i][h]);
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < KV4_WAVES; ++i) {
            if (sh.l[i][h] == 0.0f) continue;               // uniform: no tokens
            const float f = sh.m[i][h] == M ? 1.0f : __builtin_amdgcn_exp2f((sh.m[i][h] - M) * 0x1p43f);
            l = fmaf(sh.l[i][h], f, l);
            const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sh.ring[i]) + h * QM_GQA_HD + 4 * lane);
            o.x = fmaf(a.x, f, o.x);
            o.y = fmaf(a.y, f, o.y);
            o.z = fmaf(a.z, f, o.z);
            o.w = fmaf(a.w, f, o.w);
        }
        if (A.single) {
            kv4_out(A, b, 4 * kvh + h, lane, o, l, gate, r.refused);
        } else {
            float* P = A.partial + ((size_t)blockIdx.x * 4 + h) * KV4_PART_STRIDE;
            st4(P + 4 * lane, o);
            if (lane == 0) *reinterpret_cast<float2*>(P + 256) = make_float2(M * 0x1p43f, l);
        }
    }
}

// The splits' partials of query head h of batch row b, joined, and the gate:
// one wave per (b, h, 64 dims), N splits' loads in flight at a time.  A split
// whose weight underflows to 0 counts all the same, so that a NaN in it
// reaches the output as it does within a split; a split of no tokens has
// zeros, and past the last one the last is read again with weight 0.
struct Joined {
    float m, l, o;
};
template <int N>
QM_DEV void join(Joined& x, const float* P, int n, int d, int lane) {
    const size_t step = 16 * KV4_PART_STRIDE;
    for (int s0 = 0; s0 < n; s0 += N) {                     // uniform
        float a[N];
#pragma unroll
        for (int j = 0; j < N; ++j) a[j] = P[(size_t)min(s0 + j, n - 1) * step + d];
        const float2 ml = *reinterpret_cast<const float2*>(P + (size_t)min(s0 + lane, n - 1) * step + 256);
        const bool some = lane < N && s0 + lane < n && ml.y != 0.0f;     // a split of tokens
        const float mb = fmaxf(x.m, max_xor32(max_xor16(row_max16(some ? ml.x : -INFINITY))));
        const float c = x.m == mb ? 1.0f : __builtin_amdgcn_exp2f(x.m - mb);
        const float f = !some ? 0.0f : ml.x == mb ? 1.0f : __builtin_amdgcn_exp2f(ml.x - mb);
        x.l = x.l * c + wave_sum64(some ? ml.y * f : 0.0f);
        x.o *= c;
#pragma unroll
        for (int j = 0; j < N; ++j) x.o = fmaf(a[j], readlane_f32(f, j), x.o);
        x.m = mb;
    }
}
extern "C" __global__ __launch_bounds__(64) void qm_gqa_kv4_merge(GqaKv4Args A) {
    const int lane = threadIdx.x, d = 64 * (blockIdx.x & 3) + lane;
    const int h = (blockIdx.x >> 2) % QM_GQA_HEADS, b = blockIdx.x / (4 * QM_GQA_HEADS);
    const float gate = A.q_gate[((size_t)b * QM_GQA_HEADS + h) * (2 * QM_GQA_HD) + QM_GQA_HD + d];
    const bool off = A.result && A.result[0] != 0;          // nobody has dealt
    const int2 mine = off ? make_int2(0, 0) : reinterpret_cast<const int2*>(A.splits)[b];
    // split (first + s) and kv head h >> 2: workgroup 4 (first + s) + (h >> 2)
    const float* P = A.partial + ((size_t)mine.x * 16 + h) * KV4_PART_STRIDE;
    Joined x{-INFINITY, 0.0f, 0.0f};
    // Few splits: few loads, and few past the last one (the step, 8 / 32 loads
    // at a time, us: 900 tokens, 8 splits, 9.05 / 9.33, 4097 tokens, 33 splits,
    // 10.81 / 10.19, 16000 tokens 13.25 / 11.65).
    if (mine.y <= 8) join<8>(x, P, mine.y, d, lane);
    else join<KV4_JOIN>(x, P, mine.y, d, lane);
    float y = x.l != 0.0f ? (x.o * __builtin_amdgcn_rcpf(x.l)) * sigmoid_fast(gate) : 0.0f;
    if (mine.y < 0) y = __builtin_nanf("");
    A.out[((size_t)b * QM_GQA_HEADS + h) * QM_GQA_HD + d] = y;
}
