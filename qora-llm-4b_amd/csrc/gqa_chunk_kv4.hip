// gqa_chunk_kv4.hip -- attention of chunks of new tokens over the paged 4-bit
// KV cache (qm_kv4.h) for gfx950: parts of prompts, drafted tokens, whole
// prompts, of several rows at once.
//
// Mathematics.  Token i of a batch row's n new ones stands at position
// pos = len - n + i.  With q its RMSNorm'd, rotated query (gemv.rs:586-627),
//   out = sigmoid(gate) sum_t p_t V_t / sum_t p_t,  p_t = exp(q . K_t / 16),
// over the cached tokens t <= pos, K and V as the cache keeps them: lo + s c,
// rounded to f16 once.  q, p (relative to a running maximum, in base 2) and
// the operands are f16, all sums f32.
//
// A workgroup (8 waves) owns a row block of 64 new tokens of the four query
// heads of a kv head: wave w has head w & 3 and 32 tokens, two operand columns
// of 16, so that every K and V operand read from LDS feeds two matrix
// instructions.  Both products run transposed, S^T = K Q^T and O^T = V^T P^T,
// so that a lane's scores, its running maximum and its outputs are all of one
// row, and the scores of two runs of 16 tokens are, as they stand, the eight
// keys that a word of V codes holds.  A page of the kv head (64 tokens) is a
// tile: its codes come by LDS DMA, each wave makes f16 operands of an eighth of
// them, and the tile before it is multiplied meanwhile.
//
// The pages of all row blocks of a kv head are dealt to the workgroups in equal
// runs; where a block's pages fall to several, they leave partial sums and
// qm_gqa_chunk_merge joins them.
#include "qm_kv4_device.h"
#include "qm_kernel_args.h"

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

#define CHUNK_WAVES 8
#define CHUNK_COLS 2                   // operand columns (of 16 rows) a wave
#define CHUNK_MIN_TILES 4              // pages of a row block that are worth a workgroup
// A row's reference maximum moves only where a score passes it by this (log2
// units): p <= 2^8 is exact enough in f16, and outputs are seldom rescaled.
#define CHUNK_SLACK 8.0f

// ---- how the work is dealt --------------------------------------------------
// A batch row of the call.  A row that has no tokens to read (its slot is
// outside the table, or empty) or is refused (longer than max_len, more new
// tokens than max_new or than its length) takes one unit a block, in which its
// outputs, 0 or NaN, are written.
enum { CHUNK_RUN = 0, CHUNK_NONE = 1, CHUNK_REFUSED = 2 };
struct ChunkRow {
    int row, len, n, begin, kind;
};
QM_DEV ChunkRow chunk_row(const GqaChunkArgs& A, int b) {
    ChunkRow r{0, 0, 0, 0, CHUNK_NONE};
    if (b >= A.batch) return r;
    const int begin = A.begins[b], end = A.begins[b + 1];
    if (begin < 0 || end < begin || end > A.tokens) return r;
    r.begin = begin;
    r.n = end - begin;
    const int row = A.slots ? A.slots[b] : b;
    if ((A.result && A.result[0] != 0) || (uint32_t)row >= (uint32_t)A.c.rows) return r;
    r.row = row;
    r.len = A.c.lens[row];
    if (r.len <= 0) return r;
    r.kind = r.len > A.max_len || r.n > A.max_new || r.n > r.len ? CHUNK_REFUSED : CHUNK_RUN;
    return r;
}
QM_DEV int chunk_blocks(const ChunkRow& r) { return (r.n + QMK_CHUNK_TOKENS - 1) / QMK_CHUNK_TOKENS; }
// Pages that block j reads, and that the blocks before it do: a block but the
// row's last one ends 64 j + 63 tokens after the row's first new one.
QM_DEV int chunk_tiles(const ChunkRow& r, int j) {
    if (r.kind != CHUNK_RUN) return 1;
    return (r.len - r.n + min(r.n, QMK_CHUNK_TOKENS * (j + 1)) - 1) / QMK_KV4_PAGE_TOKENS + 1;
}
QM_DEV uint64_t chunk_before(const ChunkRow& r, int j) {
    if (r.kind != CHUNK_RUN) return j;
    const uint64_t first = (r.len - r.n + 63) / QMK_KV4_PAGE_TOKENS + 1;
    return j * first + (uint64_t)j * (j - 1) / 2;
}
QM_DEV uint64_t chunk_units(const ChunkRow& r) {
    const int nb = chunk_blocks(r);
    return nb ? chunk_before(r, nb - 1) + chunk_tiles(r, nb - 1) : 0;
}
QM_DEV uint64_t shfl64(uint64_t x, int lane) {
    const uint32_t lo = __shfl((int)(uint32_t)x, lane), hi = __shfl((int)(uint32_t)(x >> 32), lane);
    return (uint64_t)hi << 32 | lo;
}
QM_DEV uint64_t scan64(uint64_t x, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t y = shfl64(x, lane - d);
        x += lane >= d ? y : 0;
    }
    return x;
}
QM_DEV uint64_t uniform64(uint64_t x) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(x >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x);
}
QM_DEV ChunkRow uniform_row(const ChunkRow& r, int lane) {
    return ChunkRow{__builtin_amdgcn_readlane(r.row, lane), __builtin_amdgcn_readlane(r.len, lane),
                    __builtin_amdgcn_readlane(r.n, lane), __builtin_amdgcn_readlane(r.begin, lane),
                    __builtin_amdgcn_readlane(r.kind, lane)};
}

// A row block: its row, number, pages, and the units before it.
struct ChunkItem {
    ChunkRow r;
    int block, tiles;
    uint64_t first;
};
// All units of a kv head, and (all lanes agree) units a workgroup.
QM_DEV uint64_t chunk_total(const GqaChunkArgs& A, int lane) {
    uint64_t all = 0;
    for (int b0 = 0; b0 < A.batch; b0 += 64) all += chunk_units(chunk_row(A, b0 + lane));      // uniform
    return uniform64(shfl64(scan64(all, lane), 63));
}
QM_DEV uint64_t chunk_share(uint64_t total, int groups) {
    const uint64_t each = (total + groups - 1) / groups;
    return each < CHUNK_MIN_TILES ? CHUNK_MIN_TILES : each;
}
// The row block that unit u falls into (u < total), or block number `at` of
// all row blocks where `by_block`; false: there is none.
template <bool BY_BLOCK>
QM_DEV bool chunk_find(const GqaChunkArgs& A, uint64_t u, int lane, ChunkItem& it) {
    uint64_t units = 0, keys = 0;
    for (int b0 = 0; b0 < A.batch; b0 += 64) {             // uniform
        const ChunkRow mine = chunk_row(A, b0 + lane);
        const uint64_t n = chunk_units(mine), incl = scan64(n, lane);
        const uint64_t kn = BY_BLOCK ? (uint64_t)chunk_blocks(mine) : n, kincl = BY_BLOCK ? scan64(kn, lane) : incl;
        const uint64_t all = uniform64(shfl64(kincl, 63));
        if (u < keys + all) {
            const int at = __popcll(__ballot(keys + kincl <= u));
            it.r = uniform_row(mine, at);
            const uint64_t rest = u - keys - uniform64(shfl64(kincl - kn, at));
            int j = (int)rest;
            if (!BY_BLOCK) {                               // the last block that begins at or before `rest`
                int lo = 0, hi = chunk_blocks(it.r) - 1;
                while (lo < hi) {
                    const int mid = lo + (hi - lo + 1) / 2;
                    if (chunk_before(it.r, mid) <= rest) lo = mid;
                    else hi = mid - 1;
                }
                j = lo;
            }
            it.block = j;
            it.tiles = chunk_tiles(it.r, j);
            it.first = units + uniform64(shfl64(incl - n, at)) + chunk_before(it.r, j);
            return true;
        }
        units += uniform64(shfl64(incl, 63));
        keys += all;
    }
    return false;
}

// ---- a tile -------------------------------------------------------------------
// LDS: two buffers of f16 operands, block entry l the 16 bytes that lane
// l = (c, g) = (l & 15, l >> 4) reads for a product:
//   K block (kk, s) at 8 kk + s:      token 16 kk + c, dims 32 s + 8 g .. + 7
//   V block (dt, h) at 32 + 2 dt + h: dim 16 dt + c, tokens 32 h + 16 (e >> 2) + 4 g + (e & 3), e < 8
// and a wave's own part of the next tile's codes, with its half page's scales
// and minima.  Wave w has half page w >> 2 and pieces i = w & 3: K's run i >> 1,
// dims 128 (i & 1) .., and V's group i.
#define CHUNK_TILE 65536
struct ChunkLds {
    __attribute__((aligned(1024))) uint8_t tile[2][CHUNK_TILE];
    __attribute__((aligned(1024))) uint8_t raw[CHUNK_WAVES][3][1024];
    __attribute__((aligned(16))) uint32_t nan[2][2][4];      // [buffer][half][group]: tokens whose V is NaN there
};

QM_DEV uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }

QM_DEV void chunk_fetch(const GqaChunkArgs& A, ChunkLds& sh, int id, int head, int w, int lane) {
    const uint8_t* half = kv4_half(A.c, A.layer, id, head, w >> 2);
    const uint32_t raw = lds_addr(sh.raw[w][0]);
    dma16_off(half + 1024 * (w & 3), 16 * lane, raw);
    dma16_off(half + 4 * QMK_KV4_V_WORDS + 1024 * (w & 3), 16 * lane, raw + 1024);
    dma16_off(half + QMK_KV4_META, 16 * lane, raw + 2048);
}

// Token of score e of run r in lane group g.
QM_DEV int chunk_token(int r, int g, int e) { return 16 * r + 4 * g + e; }

QM_DEV half2_t as_half2(uint32_t u) { return __builtin_bit_cast(half2_t, u); }
// The eight values of a word, s and lo in pairs of elements 2 i, 2 i + 1: a
// code c in the low bits of 1024 (16 c in bits 4..7) is 1024 + c exactly, so
// c is one exact packed step away and the value one rounding more.
QM_DEV half8 chunk_values(uint32_t word, const half2_t (&s)[4], const half2_t (&lo)[4]) {
    const uint32_t v = word >> 8;
    const half2_t k1024 = {(_Float16)1024.0f, (_Float16)1024.0f}, k64 = {(_Float16)64.0f, (_Float16)64.0f},
                  sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    half2_t c[4];
    c[0] = as_half2((word & 0x000f000fu) | 0x64006400u) - k1024;
    c[1] = __builtin_elementwise_fma(as_half2((word & 0x00f000f0u) | 0x64006400u), sixteenth, -k64);
    c[2] = as_half2((v & 0x000f000fu) | 0x64006400u) - k1024;
    c[3] = __builtin_elementwise_fma(as_half2((v & 0x00f000f0u) | 0x64006400u), sixteenth, -k64);
    half8 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2_t x = __builtin_elementwise_fma(c[i], s[i], lo[i]);
        out[2 * i] = x[0];
        out[2 * i + 1] = x[1];
    }
    return out;
}

// The same where a group may be NaN, or its largest values past f16's: those
// are f16's largest, and NaN is `nan`.
QM_DEV half8 chunk_values_odd(uint32_t word, const half2_t (&s)[4], const half2_t (&lo)[4], _Float16 nan) {
    half8 x = chunk_values(word, s, lo);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float y = (float)x[e];
        x[e] = y != y ? nan : (_Float16)fminf(fmaxf(y, -65504.0f), 65504.0f);
    }
    return x;
}
// Whether a group's largest value, lo + 15 s, is finite (lo is where s is).
QM_DEV bool chunk_odd(half2_t s, half2_t lo) {
    const half2_t fifteen = {(_Float16)15.0f, (_Float16)15.0f};
    const uint32_t top = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(fifteen, s, lo));
    return (top & 0x7c00u) == 0x7c00u || (top & 0x7c000000u) == 0x7c000000u;
}

// The wave's part of a tile of which `left` tokens are the row's (64 and more:
// all), from its codes into buffer `buf`.  V of the others is 0, and V that is
// NaN too, which the rows that see it are given beside the product: a weight
// of 0 times it would give it to the others.
QM_DEV void chunk_expand(ChunkLds& sh, int buf, int left, int w, int lane) {
    const uint8_t* raw = sh.raw[w][0];
    const uint8_t* meta = sh.raw[w][2];
    const int half = w >> 2, i = w & 3, c = lane & 15, g = lane >> 4;
    const int run = i >> 1, dims = i & 1;
    {
        const uintx4 k = *reinterpret_cast<const uintx4*>(raw + 16 * lane);
        const half2_t s = as_half2(*reinterpret_cast<const uint32_t*>(meta + 2 * kv4_s_at(16 * run + c, 2 * dims)));
        const half2_t lo = {*reinterpret_cast<const _Float16*>(meta + 256 + 2 * kv4_lo_at(16 * run + c, 2 * dims)),
                            *reinterpret_cast<const _Float16*>(meta + 256 + 2 * kv4_lo_at(16 * run + c, 2 * dims + 1))};
        const bool odd = __any(chunk_odd(s, lo));
        uint8_t* to = sh.tile[buf] + (8 * (2 * half + run) + 4 * dims) * 1024 + 16 * lane;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const half2_t s2 = {s[m >> 1], s[m >> 1]}, l2 = {lo[m >> 1], lo[m >> 1]};
            const half2_t ss[4] = {s2, s2, s2, s2}, ll[4] = {l2, l2, l2, l2};
            half8 x = chunk_values(k[m], ss, ll);
            if (odd) x = chunk_values_odd(k[m], ss, ll, (_Float16)__builtin_nanf(""));
            *reinterpret_cast<half8*>(to + 1024 * m) = x;
        }
    }
    {
        const uintx4 v = *reinterpret_cast<const uintx4*>(raw + 1024 + 16 * lane);
        const uintx4 lo4 = *reinterpret_cast<const uintx4*>(meta + 768 + (4 * i + g) * 16);
        half2_t s[4], lo[4];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            s[e >> 1][e & 1] = *reinterpret_cast<const _Float16*>(meta + 512 + 2 * (g * 32 + (e >> 2) * 16 + (e & 3) * 4 + i));
#pragma unroll
        for (int n = 0; n < 4; ++n) lo[n] = as_half2(lo4[n]);
        if (left < QMK_KV4_PAGE_TOKENS) {                  // uniform
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (32 * half + chunk_token(e >> 2, g, e & 3) >= left) s[e >> 1][e & 1] = lo[e >> 1][e & 1] = (_Float16)0.0f;
        }
        bool odd = false;
#pragma unroll
        for (int n = 0; n < 4; ++n) odd = odd || chunk_odd(s[n], lo[n]);
        odd = __any(odd);
        uint32_t nan = 0;
        if (odd) {                                         // uniform
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint64_t lanes = __ballot(s[e >> 1][e & 1] != s[e >> 1][e & 1]);
#pragma unroll
                for (int q = 0; q < 4; ++q) nan |= (uint32_t)(lanes >> (16 * q) & 1) << chunk_token(e >> 2, q, e & 3);
            }
        }
        if (lane == 0) sh.nan[buf][half][i] = nan;
        uint8_t* to = sh.tile[buf] + 32768 + (8 * i + half) * 1024 + 16 * lane;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            half8 x = chunk_values(v[m], s, lo);
            if (odd) x = chunk_values_odd(v[m], s, lo, (_Float16)0.0f);
            *reinterpret_cast<half8*>(to + 2048 * m) = x;
        }
    }
}

// ---- a wave's rows ---------------------------------------------------------------
// Column f, lane (c, g): row c.  o[f][dt]: dims 16 dt + 4 g + e of it; l: the
// lane's share of its sum.
struct ChunkWave {
    half8 q[CHUNK_COLS][8];            // dims 32 s + 8 g + e
    floatx4 o[CHUNK_COLS][16];
    float m[CHUNK_COLS], l[CHUNK_COLS];
    int pos[CHUNK_COLS];               // -1: no row
};

QM_DEV float4 bf16x4(uint2 u) {
    return make_float4(bf16_to_f32((uint16_t)(u.x & 0xffffu)), bf16_to_f32((uint16_t)(u.x >> 16)),
                       bf16_to_f32((uint16_t)(u.y & 0xffffu)), bf16_to_f32((uint16_t)(u.y >> 16)));
}
QM_DEV void unpack8(uint4 v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[2 * e] = bf16_to_f32((uint16_t)(w[e] & 0xffffu));
        x[2 * e + 1] = bf16_to_f32((uint16_t)(w[e] >> 16));
    }
}

// The rows' queries: RMSNorm (1 + gamma, eps 1e-6) and RoPE straight into the
// operand; a row's sum of squares is over the four lanes c + 16 g, and the
// pairs (i, i + 32) of a rotation are in one lane.
QM_DEV void chunk_query(const GqaChunkArgs& A, ChunkWave& st, const ChunkItem& it, int head, int w, int lane) {
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int f = 0; f < CHUNK_COLS; ++f) {
        const int i = QMK_CHUNK_TOKENS * it.block + 16 * CHUNK_COLS * (w >> 2) + 16 * f + c;
        const int have = min(i, it.r.n - 1);               // rows past the last: any row, never written
        st.pos[f] = i < it.r.n ? it.r.len - it.r.n + i : -1;
        const uint16_t* row = A.q_gate + ((size_t)(it.r.begin + have) * QM_GQA_HEADS + head) * (2 * QM_GQA_HD) + 8 * g;
        const size_t at = (size_t)(it.r.len - it.r.n + have) * (QM_GQA_ROT / 2) + 8 * g;
        uint4 u[8], gq[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) u[s] = *reinterpret_cast<const uint4*>(row + 32 * s);
#pragma unroll
        for (int s = 0; s < 8; ++s) gq[s] = *reinterpret_cast<const uint4*>(A.q_norm + 32 * s + 8 * g);
        const float4 c0 = ld4(A.rope_cos + at), c1 = ld4(A.rope_cos + at + 4), s0 = ld4(A.rope_sin + at), s1 = ld4(A.rope_sin + at + 4);
        float ss = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            float x[8];
            unpack8(u[s], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        }
        ss = sum_xor32(sum_xor16(ss));
        // the softmax's scale in base 2 as well, so that the scores come out of the product in log2 units
        const float inv = (1.4426950408889634f / 16.0f) / sqrtf(ss / (float)QM_GQA_HD + 1e-6f);
        auto normed = [&](int s, float (&x)[8]) {
            unpack8(u[s], x);
            const uint32_t gv[4] = {gq[s].x, gq[s].y, gq[s].z, gq[s].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[2 * e] = x[2 * e] * inv * (1.0f + f16_to_f32((uint16_t)(gv[e] & 0xffffu)));
                x[2 * e + 1] = x[2 * e + 1] * inv * (1.0f + f16_to_f32((uint16_t)(gv[e] >> 16)));
            }
        };
        float x1[8], x2[8];
        normed(0, x1);
        normed(1, x2);
        const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            st.q[f][0][e] = (_Float16)(x1[e] * cs[e] - x2[e] * sn[e]);
            st.q[f][1][e] = (_Float16)(x2[e] * cs[e] + x1[e] * sn[e]);
        }
#pragma unroll
        for (int s = 2; s < 8; ++s) {
            float x[8];
            normed(s, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) st.q[f][s][e] = (_Float16)x[e];
        }
    }
}

// Half a tile (32 tokens from k0 on) at a time, so that outputs, queries and
// operands fit a wave's 256 registers.
QM_DEV void chunk_half(ChunkWave& st, const ChunkLds& sh, int buf, int h, int k0, bool edge, int lane) {
    const uint8_t* K = sh.tile[buf] + 16 * lane + 16384 * h;
    const uint8_t* V = sh.tile[buf] + 16 * lane + 32768 + 1024 * h;
    const int g = lane >> 4;
    floatx4 x[CHUNK_COLS][2];
#pragma unroll
    for (int f = 0; f < CHUNK_COLS; ++f)
#pragma unroll
        for (int r = 0; r < 2; ++r) x[f][r] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const half8 a = *reinterpret_cast<const half8*>(K + (8 * r + s) * 1024);
#pragma unroll
            for (int f = 0; f < CHUNK_COLS; ++f) x[f][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, st.q[f][s], x[f][r], 0, 0, 0);
        }
    half8 p[CHUNK_COLS];
#pragma unroll
    for (int f = 0; f < CHUNK_COLS; ++f) {
        if (edge) {                                        // uniform: some row does not see all of it
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[f][r][e] = k0 + chunk_token(r, g, e) > st.pos[f] ? -INFINITY : x[f][r][e];
        }
        float mx = fmaxf(fmaxf(fmaxf(x[f][0][0], x[f][0][1]), fmaxf(x[f][0][2], x[f][0][3])),
                         fmaxf(fmaxf(x[f][1][0], x[f][1][1]), fmaxf(x[f][1][2], x[f][1][3])));
        mx = max_xor32(max_xor16(mx));
        const float was = st.m[f], m = mx > was + CHUNK_SLACK ? mx : was;      // from -inf: any score
        if (__any(m != was)) {
            // sums beside a maximum of -inf are those of NaN scores
            const float corr = was == m ? 1.0f : __builtin_amdgcn_exp2f(was - m);
            st.m[f] = m;
            st.l[f] *= corr;
#pragma unroll
            for (int dt = 0; dt < 16; ++dt) st.o[f][dt] *= corr;
        }
        const float base = m == -INFINITY ? 0.0f : m;      // a row that sees nothing yet: weights of 0
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const _Float16 w = (_Float16)__builtin_amdgcn_exp2f(x[f][r][e] - base);
                p[f][4 * r + e] = w;
                st.l[f] += (float)w;                       // of what is multiplied
            }
    }
#pragma unroll
    for (int dt = 0; dt < 16; ++dt) {
        const half8 a = *reinterpret_cast<const half8*>(V + 2048 * dt);
#pragma unroll
        for (int f = 0; f < CHUNK_COLS; ++f) st.o[f][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p[f], st.o[f][dt], 0, 0, 0);
    }
    const uintx4 nan = *reinterpret_cast<const uintx4*>(sh.nan[buf][h]);
    if (__builtin_amdgcn_readfirstlane((int)(nan[0] | nan[1] | nan[2] | nan[3]))) {
#pragma unroll
        for (int f = 0; f < CHUNK_COLS; ++f) {
            const int seen = st.pos[f] - k0;               // the last token of the half that the row sees
            const uint32_t mask = seen < 0 ? 0u : seen >= 31 ? ~0u : (2u << seen) - 1;
#pragma unroll
            for (int dt = 0; dt < 16; ++dt)
                if (nan[dt >> 2] & mask) st.o[f][dt] = floatx4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
        }
    }
}
QM_DEV void chunk_tile(ChunkWave& st, const ChunkLds& sh, int buf, int k0, int first_pos, int lane) {
    const bool edge = k0 + QMK_KV4_PAGE_TOKENS - 1 > first_pos;
#pragma unroll
    for (int h = 0; h < 2; ++h) chunk_half(st, sh, buf, h, k0 + QMK_KV4_HALF_TOKENS * h, edge, lane);
}

// Four outputs, gated.
QM_DEV void chunk_out(uint16_t* to, floatx4 o, float inv, uint2 gate) {
    const float4 x = bf16x4(gate);
    uint2 r;
    r.x = pack_bf16x2(o[0] * inv * sigmoid_fast(x.x), o[1] * inv * sigmoid_fast(x.y));
    r.y = pack_bf16x2(o[2] * inv * sigmoid_fast(x.z), o[3] * inv * sigmoid_fast(x.w));
    *reinterpret_cast<uint2*>(to) = r;
}
QM_DEV float chunk_inverse(float l) { return l != 0.0f ? __builtin_amdgcn_rcpf(l) : 0.0f; }      // 0: nothing to see

extern "C" __global__ __launch_bounds__(64 * CHUNK_WAVES, 2) void qm_gqa_chunk_kv4(GqaChunkArgs A) {
    __shared__ ChunkLds sh;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x & 3, index = blockIdx.x >> 2, head = 4 * kvh + (w & 3);
    const uint64_t total = chunk_total(A, lane), each = chunk_share(total, A.groups);
    const uint64_t end = min(total, each * (index + 1));
    for (uint64_t u = each * index; u < end;) {            // uniform, as all of it
        ChunkItem it;
        if (!chunk_find<false>(A, u, lane, it)) return;    // never: u < total
        const int ta = (int)(u - it.first), tb = (int)min((uint64_t)it.tiles, end - it.first);
        u += tb - ta;
        const int i0 = QMK_CHUNK_TOKENS * it.block + 16 * CHUNK_COLS * (w >> 2);      // the wave's first row
        if (it.r.kind != CHUNK_RUN) {
            const uint32_t fill = it.r.kind == CHUNK_NONE ? 0u : 0x7fc07fc0u;
            for (int i = i0; i < min(i0 + 16 * CHUNK_COLS, it.r.n); ++i)
                *reinterpret_cast<uint2*>(A.out + ((size_t)(it.r.begin + i) * QM_GQA_HEADS + head) * QM_GQA_HD + 4 * lane) = make_uint2(fill, fill);
            continue;
        }
        const int32_t* table = A.c.table + (size_t)it.r.row * A.c.max_pages;
        auto page = [&](int t) { return t < tb ? __builtin_amdgcn_readfirstlane(table[t]) : -1; };
        int now = page(ta), next = page(ta + 1), after = page(ta + 2);
        if (kv4_is_page(A.c, now)) chunk_fetch(A, sh, now, kvh, w, lane);
        ChunkWave st;
        chunk_query(A, st, it, head, w, lane);
#pragma unroll
        for (int f = 0; f < CHUNK_COLS; ++f) {
            st.m[f] = -INFINITY;
            st.l[f] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < 16; ++dt) st.o[f][dt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (kv4_is_page(A.c, now)) chunk_expand(sh, ta & 1, it.r.len - QMK_KV4_PAGE_TOKENS * ta, w, lane);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (kv4_is_page(A.c, next)) chunk_fetch(A, sh, next, kvh, w, lane);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int first_pos = it.r.len - it.r.n + i0;
        for (int t = ta; t < tb; ++t) {
            // Half of the waves make the next tile's operands before their
            // products and half after them, so that a SIMD has one of each.
            auto prepare = [&] {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                if (kv4_is_page(A.c, next)) chunk_expand(sh, (t + 1) & 1, it.r.len - QMK_KV4_PAGE_TOKENS * (t + 1), w, lane);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // the codes are read
                if (kv4_is_page(A.c, after)) chunk_fetch(A, sh, after, kvh, w, lane);
            };
            if (w < CHUNK_WAVES / 2) prepare();
            if (kv4_is_page(A.c, now) && i0 < it.r.n) chunk_tile(st, sh, t & 1, QMK_KV4_PAGE_TOKENS * t, first_pos, lane);
            if (w >= CHUNK_WAVES / 2) prepare();
            now = next;
            next = after;
            after = page(t + 3);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        const bool whole = tb - ta == it.tiles;
        float* part = A.partial + (size_t)(2 * blockIdx.x + (ta == 0)) * QMK_CHUNK_PARTIAL + (size_t)w * CHUNK_COLS * (QMK_CHUNK_PARTIAL / 16);
#pragma unroll
        for (int f = 0; f < CHUNK_COLS; ++f) {
            const float l = sum_xor32(sum_xor16(st.l[f]));
            const int i = i0 + 16 * f + c;
            if (whole) {
                const size_t at = (size_t)(it.r.begin + min(i, it.r.n - 1)) * QM_GQA_HEADS + head;
                const uint16_t* gate = A.q_gate + at * (2 * QM_GQA_HD) + QM_GQA_HD + 4 * g;
                uint2 x[16];
#pragma unroll
                for (int dt = 0; dt < 16; ++dt) x[dt] = *reinterpret_cast<const uint2*>(gate + 16 * dt);
                if (i < it.r.n) {
#pragma unroll
                    for (int dt = 0; dt < 16; ++dt) chunk_out(A.out + at * QM_GQA_HD + 16 * dt + 4 * g, st.o[f][dt], chunk_inverse(l), x[dt]);
                }
            } else {
#pragma unroll
                for (int dt = 0; dt < 16; ++dt) *reinterpret_cast<floatx4*>(part + 256 * dt + 4 * lane) = st.o[f][dt];
                if (lane < 16) {
                    part[4096 + lane] = st.m[f];
                    part[4112 + lane] = l;
                }
                part += QMK_CHUNK_PARTIAL / 16;
            }
        }
    }
}

// The partial sums of a row block that several workgroups share, joined: a
// wave per (kv head, operand column of a wave, four of the 16 dim groups).
#define CHUNK_JOIN 8                   // partials loaded at a time
extern "C" __global__ __launch_bounds__(64) void qm_gqa_chunk_merge(GqaChunkArgs A) {
    const int lane = threadIdx.x, c = lane & 15, g = lane >> 4;
    const int dt0 = 4 * (blockIdx.x & 3), col = (blockIdx.x >> 2) & 15, kvh = (blockIdx.x >> 6) & 3;
    ChunkItem it;
    if (!chunk_find<true>(A, blockIdx.x >> 8, lane, it)) return;
    const uint64_t each = chunk_share(chunk_total(A, lane), A.groups);
    const uint64_t from = it.first / each, to = (it.first + it.tiles - 1) / each;
    if (from == to) return;                                // one workgroup had it
    const int w = col / CHUNK_COLS, head = 4 * kvh + (w & 3);
    const int i = QMK_CHUNK_TOKENS * it.block + 16 * CHUNK_COLS * (w >> 2) + 16 * (col % CHUNK_COLS) + c;
    const size_t at = (size_t)(it.r.begin + min(i, it.r.n - 1)) * QM_GQA_HEADS + head;
    const uint16_t* gate = A.q_gate + at * (2 * QM_GQA_HD) + QM_GQA_HD + 16 * dt0 + 4 * g;
    uint2 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const uint2*>(gate + 16 * j);
    float m = -INFINITY, l = 0.0f;
    floatx4 o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint64_t s0 = from; s0 <= to; s0 += CHUNK_JOIN) {
        floatx4 a[CHUNK_JOIN][4];
        float pm[CHUNK_JOIN], pl[CHUNK_JOIN];
#pragma unroll
        for (int k = 0; k < CHUNK_JOIN; ++k) {             // past the last: the last again, with weight 0
            const uint64_t wg = min(s0 + k, to);
            const float* part = A.partial + (size_t)(2 * (4 * wg + kvh) + (each * wg <= it.first)) * QMK_CHUNK_PARTIAL +
                                (size_t)col * (QMK_CHUNK_PARTIAL / 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) a[k][j] = *reinterpret_cast<const floatx4*>(part + 256 * (dt0 + j) + 4 * lane);
            pm[k] = part[4096 + c];
            pl[k] = part[4112 + c];
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < CHUNK_JOIN; ++k) top = fmaxf(top, pm[k]);
        const float corr = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
        l *= corr;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] *= corr;
#pragma unroll
        for (int k = 0; k < CHUNK_JOIN; ++k) {
            if (s0 + k > to) break;                        // uniform
            // a partial of no weight counts all the same: a NaN in it reaches the output
            const float f = pm[k] == top ? 1.0f : __builtin_amdgcn_exp2f(pm[k] - top);
            l = fmaf(pl[k], f, l);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] += a[k][j] * f;
        }
        m = top;
    }
    if (i < it.r.n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) chunk_out(A.out + at * QM_GQA_HD + 16 * (dt0 + j) + 4 * g, o[j], chunk_inverse(l), x[j]);
    }
}
