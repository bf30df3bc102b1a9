// kv4_cache.hip -- the paged 4-bit KV cache (qm_kv4.h) for gfx950: f16 rows
// into the pages and back, and the pages themselves: growing, shrinking and
// freeing rows, forking them, and moving the live pages together.
#include "qm_kv4_device.h"

// ---- f16 rows <-> pages ---------------------------------------------------
// A workgroup takes half a page (32 tokens) of one sequence and head, whose
// 9216 bytes it puts together in LDS.  A token's row is 32 lanes x 8 dims, so
// a group of 64 dims is 8 lanes, and a lane's 8 codes of a token are one K
// word.  A V word holds 8 tokens of one dim: two lanes with 4 tokens each turn
// their 4 x 8 codes in registers and exchange halves (a lane with all 8 was as
// fast on long prompts and took twice the chain on short ones: 45 tokens 10.4 us
// against 7.8).  Long loads are bound by HBM (4 x 32701 tokens, 687 MB: 113 us
// at least, 117 the median), long stores of the same bytes by the vector unit
// (157, 185): 645 instructions a wave keep it busy 85% of the time, 96% of that
// in which the CUs work.  Short ones are bound by the chain of length, table
// entry and page.
#define KV4_ROWS_THREADS 256
#define KV4_STORE_THREADS 512

struct HalfAt {
    int t0;                  // token 0 of the half page
    int lo, hi;              // tokens of the half page taken: [lo, hi)
    int64_t src0;            // row of the f16 side of token 0
};
// false: none taken.
QM_DEV bool half_at(const Kv4RowsArgs& A, int b, int tile, HalfAt& h) {
    const int first = A.first ? A.first[b] : 0;
    const int64_t end = min((int64_t)first + A.n, (int64_t)A.c.lens[A.row + b]);
    const int64_t t0 = ((int64_t)(first >> 5) + tile) << 5;
    if (first < 0 || first >= end || t0 >= end || (t0 >> 6) >= A.c.max_pages) return false;
    h.t0 = (int)t0;
    h.src0 = t0 - first;
    h.lo = (int)max((int64_t)0, -h.src0);
    h.hi = (int)min((int64_t)QMK_KV4_HALF_TOKENS, end - t0);
    return true;
}
// Its table entry, and its place in the pool if that is a page.
QM_DEV int half_id(const Kv4RowsArgs& A, int b, const HalfAt& h) {
    return A.c.table[(size_t)(A.row + b) * A.c.max_pages + (h.t0 >> 6)];
}
QM_DEV uint8_t* half_page(const Kv4RowsArgs& A, int id, int head, const HalfAt& h) {
    return kv4_half(A.c, A.layer, id, head, (h.t0 >> 5) & 1);
}

// Smallest / largest over the 8 lanes of a group.
template <int CTRL>
QM_DEV float dpp_of(float x) {       // update_dpp, unlike mov_dpp, is folded into its user
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
QM_DEV float min_of8(float x) {
    x = fminf(x, dpp_of<0xB1>(x));
    x = fminf(x, dpp_of<0x4E>(x));
    return fminf(x, dpp_of<0x141>(x));
}
QM_DEV float max_of8(float x) {
    x = fmaxf(x, dpp_of<0xB1>(x));
    x = fmaxf(x, dpp_of<0x4E>(x));
    return fmaxf(x, dpp_of<0x141>(x));
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
QM_DEV f16x2 f16_pair(uint32_t w) { return __builtin_bit_cast(f16x2, w); }

// Eight f16 values of a lane -> their codes in a word (element e as in
// kv4_nibble), and the group's scale and minimum.
struct Coded {
    uint32_t word;
    uint16_t s, lo;
};
QM_DEV Coded code8(uint4 raw, int lane) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    const f16x2 least = __builtin_elementwise_min(__builtin_elementwise_min(f16_pair(w[0]), f16_pair(w[1])),
                                                  __builtin_elementwise_min(f16_pair(w[2]), f16_pair(w[3])));
    const f16x2 most = __builtin_elementwise_max(__builtin_elementwise_max(f16_pair(w[0]), f16_pair(w[1])),
                                                 __builtin_elementwise_max(f16_pair(w[2]), f16_pair(w[3])));
    const float lo = min_of8(fminf((float)least[0], (float)least[1])), hi = max_of8(fmaxf((float)most[0], (float)most[1]));
    // an infinity or a NaN in the group's eight lanes
    u16x2 big = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    const uint64_t lanes = __ballot(max(big[0], big[1]) >= 0x7c00u);
    const bool bad = (lanes >> (lane & 56)) & 0xffu;
    Coded c;
    c.s = bad ? (uint16_t)0x7e00u : kv4_scale(lo, hi);
    c.lo = bad ? (uint16_t)0x7e00u : f32_to_f16(lo);
    // In f32, x - lo is off by 2^-20 s at most and the rest by less: a
    // remainder clearly under half a step says that the code is right.  For
    // the others (one value in some 4000 of normal ones: one in 500 of these
    // words, and more than a third of the waves), and where s is subnormal, 0
    // or NaN, kv4_code decides.
    const float s = f16_to_f32(c.s), inv = __builtin_amdgcn_rcpf(s);
    float q[8], worst = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float d = fmaf((float)f16_pair(w[e >> 1])[e & 1], 1.0f, -lo);
        q[e] = rintf(d * inv);
        worst = fmaxf(worst, fabsf(fmaf(-q[e], s, d)));
    }
    // nibbles 0..3 are the even elements, 4..7 the odd ones; 16 bits of codes are whole numbers in f32
    const float even = fmaf(fmaf(fmaf(q[6], 16.0f, q[4]), 16.0f, q[2]), 16.0f, q[0]);
    const float odd = fmaf(fmaf(fmaf(q[7], 16.0f, q[5]), 16.0f, q[3]), 16.0f, q[1]);
    c.word = (uint32_t)even | (uint32_t)odd << 16;
    const float sure = s >= 0x1p-14f ? s * (0.5f - 0x1p-18f) : -1.0f;
    if (!(worst < sure)) {
#pragma clang loop unroll(disable)
        for (int e = 0; e < 8; ++e) {                   // rolled: code to be fetched, and few lanes come here
            const uint32_t we = (e < 4 ? (e < 2 ? w[0] : w[1]) : (e < 6 ? w[2] : w[3])) >> (16 * (e & 1));
            const float x = f16_to_f32((uint16_t)we), d = x - lo;
            const int shift = 4 * kv4_nibble(e);
            if (fabsf(fmaf(-rintf(d * inv), s, d)) < sure) continue;
            c.word = (c.word & ~(15u << shift)) | kv4_code(x, lo, s, inv) << shift;
        }
    }
    return c;
}

// Four rows of eight nibbles, as rows 0, 1, 4, 5 of an 8 x 8 whose others are
// zero, turned: word n has nibble n of them in its nibbles 0, 1, 4, 5.
QM_DEV void turn_nibbles(uint32_t (&out)[8], uint32_t r0, uint32_t r1, uint32_t r4, uint32_t r5) {
    // halves of rows a, a + 4
    const uint32_t h[4] = {__builtin_amdgcn_perm(r4, r0, 0x05040100u), __builtin_amdgcn_perm(r5, r1, 0x05040100u),
                           __builtin_amdgcn_perm(r4, r0, 0x07060302u), __builtin_amdgcn_perm(r5, r1, 0x07060302u)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {                       // words 4 i ..
#pragma unroll
        for (int j = 0; j < 2; ++j) {                   // bytes of rows a, a + 2, then nibbles of rows a, a + 1
            const uint32_t x = (j ? h[2 * i] >> 8 : h[2 * i]) & 0x00ff00ffu, y = (j ? h[2 * i + 1] >> 8 : h[2 * i + 1]) & 0x00ff00ffu;
            out[4 * i + 2 * j] = (x & 0x000f000fu) | (y & 0x000f000fu) << 4;
            out[4 * i + 2 * j + 1] = (x >> 4 & 0x000f000fu) | (y & 0x00f000f0u);
        }
    }
}

extern "C" __global__ __launch_bounds__(KV4_STORE_THREADS) void qm_kv4_store(Kv4RowsArgs A) {
    __shared__ __attribute__((aligned(16))) uint32_t image[QMK_KV4_HALF_BYTES / 4];
    const int tid = threadIdx.x;
    const int tile = blockIdx.x % A.halves, bh = blockIdx.x / A.halves;
    const int head = bh & 3, b = bh >> 2;
    HalfAt h;
    if (!half_at(A, b, tile, h)) return;                // uniform
    const bool whole = h.lo == 0 && h.hi == QMK_KV4_HALF_TOKENS;
    // Waves 0..3 have V, 4..7 K; a lane four tokens 16 u + 4 g + k of dims 8 i ..
    const bool is_v = tid < 256;
    const int i = tid & 31, u = (tid >> 5) & 1, g = (tid >> 6) & 3;
    const size_t base = ((size_t)b * 4 + head) * (size_t)A.cap;
    const uint16_t* from = is_v ? A.v : A.k;
    uint4 raw[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int t = min(max(16 * u + 4 * g + k, h.lo), h.hi - 1);      // any token for those left out
        raw[k] = *reinterpret_cast<const uint4*>(from + (base + (size_t)(h.src0 + t)) * 256 + 8 * i);
    }
    const int id = half_id(A, b, h);
    if (!kv4_is_page(A.c, id)) return;                  // uniform
    const int holders = A.c.refs[id];                   // looked at before the page is written
    uint8_t* page = half_page(A, id, head, h);
    if (!whole) {                                       // uniform: the tokens left out stay
        for (int j = tid; j < QMK_KV4_HALF_BYTES / 16; j += KV4_STORE_THREADS)
            reinterpret_cast<uint4*>(image)[j] = reinterpret_cast<const uint4*>(page)[j];
        __syncthreads();
    }
    uint16_t* meta = reinterpret_cast<uint16_t*>(image) + QMK_KV4_META / 2 + (is_v ? 256 : 0);
    uint32_t word[4], keep = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int t = 16 * u + 4 * g + k;
        const bool in = t >= h.lo && t < h.hi;
        const Coded c = code8(raw[k], tid & 63);
        word[k] = c.word;
        keep |= in ? 0u : 15u << (4 * kv4_nibble(k));
        if (!is_v && in) image[kv4_k_word(t, 8 * i)] = c.word;
        if ((i & 7) == 0 && in) {
            meta[kv4_s_at(t, i >> 3)] = c.s;
            meta[128 + kv4_lo_at(t, i >> 3)] = c.lo;
        }
    }
    if (is_v) {                                         // uniform per wave
        // The run's tokens are elements 4 u + k of the words: nibbles 0, 4, 1, 5,
        // and for u = 1 two further up.  Lane and lane + 32 have the two runs of
        // the same dims; after the exchange the one has elements 0..3 of dims
        // 8 i .. + 3 and the other's there, the other likewise dims 8 i + 4 ..
        uint32_t out[8];                                // word n: dim 8 i + (the element of nibble n)
        turn_nibbles(out, word[0], word[2], word[1], word[3]);
        const auto kept = __builtin_amdgcn_permlane32_swap(keep, keep, false, false);
        const uint32_t stay = kept[0] | kept[1] << 8;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const auto w = __builtin_amdgcn_permlane32_swap(out[kv4_nibble(k)], out[kv4_nibble(k + 4)], false, false);
            const uint32_t both = w[0] | w[1] << 8;
            uint32_t* at = &image[kv4_v_word(4 * g, 8 * i + k + 4 * u)];
            *at = whole ? both : (both & ~stay) | (*at & stay);
        }
    }
    __syncthreads();
    if (holders != 1) return;                           // not the row's alone
    for (int j = tid; j < QMK_KV4_HALF_BYTES / 16; j += KV4_STORE_THREADS)
        reinterpret_cast<uint4*>(page)[j] = reinterpret_cast<const uint4*>(image)[j];
}

// lo + s q of the code in bits `shift` .., rounded to f32 and then to f16.  In
// one step (v_fma_mixlo_f16, which the compiler takes otherwise) it would be
// one rounding, which differs where the f32 sum is halfway between two f16
// values.
QM_DEV uint32_t kv4_read(uint32_t word, int shift, float s, float lo) {
    float x = __builtin_fmaf((float)((word >> shift) & 15u), s, lo);
    asm("" : "+v"(x));
    return f32_to_f16(x);
}

extern "C" __global__ __launch_bounds__(KV4_ROWS_THREADS) void qm_kv4_load(Kv4RowsArgs A) {
    __shared__ __attribute__((aligned(16))) uint32_t w[QMK_KV4_HALF_BYTES / 4];
    const int tid = threadIdx.x;
    const int tile = blockIdx.x % A.halves, bh = blockIdx.x / A.halves;
    const int head = bh & 3, b = bh >> 2;
    HalfAt h;
    if (!half_at(A, b, tile, h)) return;                // uniform
    const int id = half_id(A, b, h);
    if (!kv4_is_page(A.c, id)) return;
    const uint8_t* page = half_page(A, id, head, h);
    for (int j = tid; j < QMK_KV4_HALF_BYTES / 16; j += KV4_ROWS_THREADS)
        reinterpret_cast<uint4*>(w)[j] = reinterpret_cast<const uint4*>(page)[j];
    __syncthreads();
    const uint16_t* meta = reinterpret_cast<const uint16_t*>(&w[QMK_KV4_META / 4]);
    const int i = tid & 31, group = i >> 3;
    const size_t base = ((size_t)b * 4 + head) * (size_t)A.cap;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int t = (tid >> 5) + 8 * r;
        if (t < h.lo || t >= h.hi) continue;
        const int sa = kv4_s_at(t, group), la = kv4_lo_at(t, group);
        const float sk = f16_to_f32(meta[sa]), lk = f16_to_f32(meta[128 + la]);
        const float sv = f16_to_f32(meta[256 + sa]), lv = f16_to_f32(meta[384 + la]);
        const uint32_t kw = w[kv4_k_word(t, 8 * i)];
        const int shift = 4 * kv4_v_nibble(t);
        uint32_t ko[4], vo[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            ko[p] = kv4_read(kw, 4 * kv4_nibble(2 * p), sk, lk) | kv4_read(kw, 4 * kv4_nibble(2 * p + 1), sk, lk) << 16;
            const int d = 8 * i + 2 * p;
            vo[p] = kv4_read(w[kv4_v_word(t, d)], shift, sv, lv) | kv4_read(w[kv4_v_word(t, d + 1)], shift, sv, lv) << 16;
        }
        const size_t at = (base + (size_t)(h.src0 + t)) * 256 + 8 * i;
        *reinterpret_cast<uint4*>(A.k + at) = make_uint4(ko[0], ko[1], ko[2], ko[3]);
        *reinterpret_cast<uint4*>(A.v + at) = make_uint4(vo[0], vo[1], vo[2], vo[3]);
    }
}

// ---- the pages ------------------------------------------------------------
#define KV4_PLAN_THREADS 1024
#define KV4_BLOCK_PAGES (64 * KV4_PLAN_THREADS)     // pages whose state one pass holds: up to 64 a thread
#define KV4_WINDOW 4096                              // free pages handed out at a time

// Exclusive sum over the workgroup's 1024 threads, and the total.  `sums`
// (one word a wave) must not be in use: calls in a row take different ones.
QM_DEV uint32_t plan_scan(uint32_t x, uint32_t* sums, uint32_t& total) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t incl = wave_scan(x);
    if (lane == 63) sums[w] = incl;
    __syncthreads();
    const uint32_t all = wave_scan(lane < KV4_PLAN_THREADS / 64 ? sums[lane] : 0u);
    total = (uint32_t)__builtin_amdgcn_readlane((int)all, 63);
    const uint32_t before = w ? (uint32_t)__builtin_amdgcn_readlane((int)all, __builtin_amdgcn_readfirstlane(w) - 1) : 0u;
    return before + incl - x;
}

// A pass's pages go to the threads 64 at a time, in order, spread over the
// waves: lane l of wave w has the w * each + l-th 64 where l < each.  (With 64 a
// lane from the first wave on, a pool of 4096 was one wave's: 10.1 us to plan a
// compaction, now 5.7; 512 pages 3.8 to resize, now 3.0.)
struct Share {
    int each;
    int64_t page0;           // the lane's first page; past the pool where it has none
};
QM_DEV Share share_of(const Kv4Cache& c, int64_t block) {
    constexpr int WAVES = KV4_PLAN_THREADS / 64;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pages = (int)min(c.num_pages - block, (int64_t)KV4_BLOCK_PAGES);
    Share s;
    s.each = (pages + 64 * WAVES - 1) / (64 * WAVES);
    s.page0 = lane < s.each ? block + 64 * (int64_t)(w * s.each + lane) : (int64_t)c.num_pages;
    return s;
}
// Bit j: page page0 + j is free (reference count 0).  Ids past the pool are
// not free.  N loads in flight, of 64 counts each whether the pool has them or
// not: few where there is little to load, many where the loads take the time
// (4 / 32, us, 16 rows grown and shrunk again: a pool of 512 14.3 / 19.5, 8192
// 15.2 / 19.6, 16384 16.7 / 19.6, 32768 19.6 / 19.7, 262144 57.4 / 54.9,
// 2097152 283 / 226; compacted with nothing to move: 16384 10.2 / 11.4, 32768
// 15.1 / 14.7).
template <int N>
QM_DEV uint64_t free_of(const Kv4Cache& c, int64_t at, int each) {
    const int lane = threadIdx.x & 63;
    uint64_t mine = 0;
    for (int r0 = 0; r0 < each; r0 += N) {
        int v[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int64_t p = at + (r0 + j) * 64 + lane;
            v[j] = c.refs[min(p, (int64_t)c.num_pages - 1)];
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint64_t m = __ballot(v[j] == 0);
            mine = lane == r0 + j ? m : mine;
        }
    }
    return mine;
}
QM_DEV uint64_t free_pages(const Kv4Cache& c, int64_t block, Share& s) {
    s = share_of(c, block);
    const int64_t at = block + 64 * (int64_t)(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * s.each);
    const uint64_t mine = s.each <= 16 ? free_of<4>(c, at, s.each) : free_of<32>(c, at, s.each);
    const int64_t in = c.num_pages - s.page0;           // bits past the pool
    return in >= 64 ? mine : in <= 0 ? 0ull : mine & ((1ull << in) - 1);
}

// 16-byte copy of a third of a page by a workgroup of 256.
#define KV4_COPY_PARTS 3
#define KV4_COPY_THREADS 256
QM_DEV void copy_part(const Kv4Cache& c, int layer, int src, int dst, int part) {
    constexpr int N = QMK_KV4_PAGE_BYTES / 16 / KV4_COPY_PARTS / KV4_COPY_THREADS;
    static_assert(N * 16 * KV4_COPY_PARTS * KV4_COPY_THREADS == QMK_KV4_PAGE_BYTES, "a page in whole vectors");
    const uint4* s = reinterpret_cast<const uint4*>(c.pages + ((size_t)layer * c.num_pages + src) * QMK_KV4_PAGE_BYTES);
    uint4* d = reinterpret_cast<uint4*>(c.pages + ((size_t)layer * c.num_pages + dst) * QMK_KV4_PAGE_BYTES);
    const int at = part * (N * KV4_COPY_THREADS) + threadIdx.x;
    uint4 v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = s[at + j * KV4_COPY_THREADS];
#pragma unroll
    for (int j = 0; j < N; ++j) d[at + j * KV4_COPY_THREADS] = v[j];
}

// Rows take new lengths (one workgroup, thread i has list row i).  A row that
// grows gets pages for the new tokens, and its partly filled last page, if
// other rows hold it too, is replaced by a copy: written pages have one
// holder.  When every holder of such a page grows in this call, the first of
// them keeps it.  Fresh pages are the lowest free ids before the call, in
// list order.  Nothing is changed unless all of it can be.
//
// Bound by its chain of dependent loads (lengths, entry, count) and barriers;
// the pool's counts are loaded first, beside them (1 row, a pool of 512: 3.0 us;
// 64 rows, 32768: 5.6).
extern "C" __global__ __launch_bounds__(KV4_PLAN_THREADS) void qm_kv4_resize(Kv4ResizeArgs A) {
    __shared__ uint32_t sums[2][KV4_PLAN_THREADS / 64];
    __shared__ uint32_t seen[QMK_KV4_MAX_ROWS / 32];
    __shared__ __attribute__((aligned(16))) int last[QMK_KV4_MAX_COUNT];
    __shared__ uint32_t off[QMK_KV4_MAX_COUNT];
    __shared__ int row_of[QMK_KV4_MAX_COUNT], begin_of[QMK_KV4_MAX_COUNT];
    __shared__ int list[KV4_WINDOW];
    __shared__ uint32_t copies;
    __shared__ unsigned long long lacking;
    const int tid = threadIdx.x;
    const Kv4Cache& c = A.c;
    for (int j = tid; j < (c.rows + 31) / 32; j += KV4_PLAN_THREADS) seen[j] = 0;
    if (tid == 0) {
        copies = 0;
        lacking = 0;
    }
    const bool mine = tid < A.count;
    const int row = !mine ? -1 : A.list ? A.list[tid] : tid;
    const bool in = mine && (uint32_t)row < (uint32_t)c.rows;
    const int old = in ? c.lens[row] : 0;
    const int change = mine ? A.lens[tid] : 0;
    Share share;
    uint64_t mask = free_pages(c, 0, share);
    __syncthreads();

    // the list, checked
    int want = 0, page = -1, held = 0;
    bool bad = mine && !in, grow = false;
    if (in) {
        const uint32_t bit = 1u << (row & 31);
        bad = (atomicOr(&seen[row >> 5], bit) & bit) != 0;
        const int64_t to = (int64_t)change + (A.add ? old : 0);
        const int64_t most = (int64_t)c.max_pages * QMK_KV4_PAGE_TOKENS;
        bad = bad || old < 0 || old > most || to < 0 || to > most;
        want = bad ? 0 : (int)to;
        grow = !bad && want > old;
        if (grow && (old & (QMK_KV4_PAGE_TOKENS - 1))) {
            page = c.table[(size_t)row * c.max_pages + old / QMK_KV4_PAGE_TOKENS];
            if (kv4_is_page(c, page)) held = c.refs[page];
            bad = held < 1;
        }
    }
    last[tid] = page;
    row_of[tid] = row;
    if (__syncthreads_or(bad)) {
        if (tid == 0) {
            A.result[0] = -1;
            A.state[0] = 1;
        }
        return;
    }
    bool copy = false;
    if (held > 1) {                                     // a page of one holder is its own
        int growing = 0, before = 0;
        for (int j = 0; j < A.count; j += 4) {          // past the list: -1
            const int4 o = *reinterpret_cast<const int4*>(&last[j]);
            const int n = (o.x == page) + (o.y == page) + (o.z == page) + (o.w == page);
            growing += n;
            before += j + 4 <= tid ? n : (o.x == page && j < tid) + (o.y == page && j + 1 < tid) + (o.z == page && j + 2 < tid);
        }
        copy = !(growing == held && before == 0);
    }
    const int had = kv4_pages_of(old), pages = kv4_pages_of(want);
    const int begin = copy ? old / QMK_KV4_PAGE_TOKENS : had;
    const int mine_need = grow ? pages - begin : 0;
    uint32_t need;
    off[tid] = plan_scan((uint32_t)min(mine_need, QMK_KV4_MAX_PAGES), sums[0], need);
    begin_of[tid] = copy ? ~begin : begin;              // the sign: its first fresh page is a copy

    // enough free pages?
    uint32_t ahead = 0, found = 0;
    int64_t block = 0;
    for (; block < c.num_pages && found < need; block += KV4_BLOCK_PAGES) {
        if (block) {
            __syncthreads();
            mask = free_pages(c, block, share);
        }
        uint32_t total;
        ahead = plan_scan((uint32_t)__popcll(mask), sums[1], total);
        found += total;
    }
    if (found < need) {
        if (mine_need > 0) atomicAdd(&lacking, (unsigned long long)mine_need);
        __syncthreads();
        if (tid == 0) {
            A.result[0] = (int)min(lacking - found, 0x7fffffffull);
            A.state[0] = 1;
        }
        return;
    }

    // hand them out, KV4_WINDOW at a time
    const bool kept = block <= KV4_BLOCK_PAGES;          // the first pass saw them all
    int32_t* job = A.state + 4;
    uint32_t done = 0;
    for (int64_t blk = 0; done < need; blk += KV4_BLOCK_PAGES) {
        uint32_t total = found;
        if (!kept) {
            __syncthreads();
            mask = free_pages(c, blk, share);
            ahead = plan_scan((uint32_t)__popcll(mask), sums[1], total);
        }
        const uint32_t take = min(total, need - done);
        for (uint32_t w0 = 0; w0 < take; w0 += KV4_WINDOW) {
            if (w0) __syncthreads();
            uint32_t k = ahead;
            if (k < w0 + KV4_WINDOW && k < take)
                for (uint64_t m = mask; m && k < min(w0 + KV4_WINDOW, take); m &= m - 1, ++k)
                    if (k >= w0) list[k - w0] = (int)(share.page0 + __builtin_ctzll(m));
            __syncthreads();
            const int n = (int)min((uint32_t)KV4_WINDOW, take - w0);
            for (int j = tid; j < n; j += KV4_PLAN_THREADS) {
                const uint32_t at = done + w0 + j;
                int lo = 0, hi = A.count;               // the last list row that begins at or before `at`
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (off[mid] <= at) lo = mid;
                    else hi = mid;
                }
                const int from = begin_of[lo], index = (from < 0 ? ~from : from) + (int)(at - off[lo]);
                const int id = list[j];
                if (from < 0 && at == off[lo]) {
                    const uint32_t slot = atomicAdd(&copies, 1u);
                    job[2 * slot] = last[lo];
                    job[2 * slot + 1] = id;
                }
                c.table[(size_t)row_of[lo] * c.max_pages + index] = id;
                c.refs[id] = 1;
            }
        }
        done += take;
    }
    if (copy) atomicSub(&c.refs[page], 1);
    if (mine) {
        c.lens[row] = want;
        *reinterpret_cast<int2*>(job + 2 * A.count + 2 * tid) = make_int2(pages, had);
    }
    __syncthreads();
    if (tid == 0) {
        A.state[0] = 0;
        A.state[1] = (int)copies;
        A.result[0] = 0;
    }
}

// The second half of a resize: the pages to copy, in every layer, and the
// references that shrunk rows give up.
extern "C" __global__ __launch_bounds__(KV4_COPY_THREADS) void qm_kv4_resize_pages(Kv4ResizeArgs A) {
    if (A.state[0]) return;
    const Kv4Cache& c = A.c;
    const int32_t* job = A.state + 4;
    for (int i = blockIdx.x; i < A.count; i += gridDim.x) {
        const int2 gone = *reinterpret_cast<const int2*>(job + 2 * A.count + 2 * i);
        const int row = A.list ? A.list[i] : i;
        for (int j = gone.x + threadIdx.x; j < gone.y; j += KV4_COPY_THREADS) {
            const int id = c.table[(size_t)row * c.max_pages + j];
            if (kv4_is_page(c, id)) atomicSub(&c.refs[id], 1);
        }
    }
    const int64_t parts = (int64_t)A.state[1] * c.layers * KV4_COPY_PARTS;
    for (int64_t p = blockIdx.x; p < parts; p += gridDim.x) {
        const int part = (int)(p % KV4_COPY_PARTS);
        const int64_t q = p / KV4_COPY_PARTS;
        const int layer = (int)(q % c.layers), i = (int)(q / c.layers);
        copy_part(c, layer, job[2 * i], job[2 * i + 1], part);
    }
}

// Rows become copies of rows as they were before the call, page by page in
// the table only: references to the new pages are counted and the new entries
// set aside (first half), then the old ones' given up and the entries
// written.  Workgroup i has pair i; each checks the whole list.
extern "C" __global__ __launch_bounds__(256) void qm_kv4_fork(Kv4ForkArgs A) {
    __shared__ uint32_t seen[QMK_KV4_MAX_ROWS / 32];
    const int tid = threadIdx.x, i = blockIdx.x;
    const Kv4Cache& c = A.c;
    for (int j = tid; j < (c.rows + 31) / 32; j += 256) seen[j] = 0;
    __syncthreads();
    bool bad = false;
    for (int j = tid; j < A.count; j += 256) {
        const int src = A.src[j], dst = A.dst[j];
        if ((uint32_t)src >= (uint32_t)c.rows || (uint32_t)dst >= (uint32_t)c.rows) {
            bad = true;
        } else {
            const uint32_t bit = 1u << (dst & 31);
            bad = bad || (atomicOr(&seen[dst >> 5], bit) & bit) != 0;
        }
    }
    bad = __syncthreads_or(bad);
    if (i == 0 && tid == 0) {
        A.state[0] = bad;
        A.result[0] = bad ? -1 : 0;
    }
    if (bad) return;
    const int src = A.src[i], len = c.lens[src];
    const int n = min(max(kv4_pages_of(len), 0), c.max_pages);
    int32_t* aside = A.state + 4 + A.count + (size_t)i * c.max_pages;
    for (int j = tid; j < n; j += 256) {
        const int id = c.table[(size_t)src * c.max_pages + j];
        aside[j] = id;
        if (kv4_is_page(c, id)) atomicAdd(&c.refs[id], 1);
    }
    if (tid == 0) A.state[4 + i] = len;
}

extern "C" __global__ __launch_bounds__(256) void qm_kv4_fork_rows(Kv4ForkArgs A) {
    if (A.state[0]) return;
    const int tid = threadIdx.x, i = blockIdx.x;
    const Kv4Cache& c = A.c;
    const int dst = A.dst[i], len = A.state[4 + i];
    const int n = min(max(kv4_pages_of(len), 0), c.max_pages);
    const int had = min(max(kv4_pages_of(c.lens[dst]), 0), c.max_pages);
    const int32_t* aside = A.state + 4 + A.count + (size_t)i * c.max_pages;
    int32_t* row = c.table + (size_t)dst * c.max_pages;
    for (int j = tid; j < max(n, had); j += 256) {
        if (j < had) {
            const int id = row[j];
            if (kv4_is_page(c, id)) atomicSub(&c.refs[id], 1);
        }
        if (j < n) row[j] = aside[j];
    }
    __syncthreads();
    if (tid == 0) c.lens[dst] = len;
}

// The pages p0 + (a set bit) of lane j, to list from `at` on, in order.
QM_DEV void write_set(int32_t* list, uint64_t bits, uint32_t at, int64_t p0, int j) {
    const int lane = threadIdx.x & 63;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, j);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), j);
    const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)at, j);
    const int page = __builtin_amdgcn_readlane((int)p0, j);
    const uint32_t before = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0u));
    if (((uint64_t)hi << 32 | lo) >> lane & 1) list[first + before] = page + lane;
}

// Live pages move down to [0, live): the k-th live page past that bound goes
// to the k-th free page below it.  First the plan (one workgroup; 5.7 us for a
// pool of 4096), then the moves (8200 pages of 73,728 bytes: 257 us, 4.7 TB/s
// read + written, the rate of a large copy).
extern "C" __global__ __launch_bounds__(KV4_PLAN_THREADS) void qm_kv4_compact(Kv4CompactArgs A) {
    __shared__ uint32_t sums[2][KV4_PLAN_THREADS / 64];
    const int tid = threadIdx.x;
    const Kv4Cache& c = A.c;
    uint32_t free = 0;
    uint64_t mask = 0;
    Share share;
    for (int64_t block = 0; block < c.num_pages; block += KV4_BLOCK_PAGES) {
        if (block) __syncthreads();
        mask = free_pages(c, block, share);
        uint32_t total;
        plan_scan((uint32_t)__popcll(mask), sums[0], total);
        free += total;
    }
    const int64_t live = c.num_pages - (int64_t)free;
    int32_t* movers = A.state + 4;
    int32_t* holes = movers + c.num_pages;
    int32_t* to = holes + c.num_pages;
    uint32_t moves = 0, gaps = 0;
    for (int64_t block = 0; block < c.num_pages; block += KV4_BLOCK_PAGES) {
        if (c.num_pages > KV4_BLOCK_PAGES) {
            __syncthreads();
            mask = free_pages(c, block, share);
        }
        // bits of this thread's pages: in the pool, and below the bound
        const int64_t p0 = share.page0;
        const int in = (int)min(max(c.num_pages - p0, (int64_t)0), (int64_t)64);
        const int low = (int)min(max(live - p0, (int64_t)0), (int64_t)64);
        const uint64_t pool = in == 64 ? ~0ull : (1ull << in) - 1, below = low == 64 ? ~0ull : (1ull << low) - 1;
        const uint64_t hole = mask & below, move = ~mask & pool & ~below;
        uint32_t h_all, m_all;
        const uint32_t h_at = gaps + plan_scan((uint32_t)__popcll(hole), sums[1], h_all);
        const uint32_t m_at = moves + plan_scan((uint32_t)__popcll(move), sums[0], m_all);
        for (int j = 0; j < share.each; ++j) {          // the 64 pages of lane j by the wave
            write_set(holes, hole, h_at, p0, j);
            write_set(movers, move, m_at, p0, j);
        }
        gaps += h_all;
        moves += m_all;
    }
    for (int64_t p = live + tid; p < c.num_pages; p += KV4_PLAN_THREADS) to[p] = (int)p;
    __syncthreads();
    for (uint32_t k = tid; k < moves; k += KV4_PLAN_THREADS) to[movers[k]] = holes[k];
    if (tid == 0) {
        A.state[0] = (int)live;
        A.state[1] = (int)moves;
        A.live[0] = (int)live;
    }
}

extern "C" __global__ __launch_bounds__(KV4_COPY_THREADS) void qm_kv4_compact_pages(Kv4CompactArgs A) {
    const Kv4Cache& c = A.c;
    const int live = A.state[0], moves = A.state[1];
    const int32_t* movers = A.state + 4;
    const int32_t* holes = movers + c.num_pages;
    const int32_t* to = holes + c.num_pages;
    const int tid = threadIdx.x;
    for (int64_t k = (int64_t)blockIdx.x * KV4_COPY_THREADS + tid; k < moves; k += (int64_t)gridDim.x * KV4_COPY_THREADS) {
        c.refs[holes[k]] = c.refs[movers[k]];
        c.refs[movers[k]] = 0;
    }
    for (int r = blockIdx.x; r < c.rows; r += gridDim.x) {
        const int n = min(max(kv4_pages_of(c.lens[r]), 0), c.max_pages);
        int32_t* row = c.table + (size_t)r * c.max_pages;
        for (int j = tid; j < n; j += KV4_COPY_THREADS) {
            const int id = row[j];
            if (kv4_is_page(c, id) && id >= live) row[j] = to[id];
        }
    }
    const int64_t parts = (int64_t)moves * c.layers * KV4_COPY_PARTS;
    for (int64_t p = blockIdx.x; p < parts; p += gridDim.x) {
        const int part = (int)(p % KV4_COPY_PARTS);
        const int64_t q = p / KV4_COPY_PARTS;
        const int layer = (int)(q % c.layers), k = (int)(q / c.layers);
        copy_part(c, layer, movers[k], holes[k], part);
    }
}
