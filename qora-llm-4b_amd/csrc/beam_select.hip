// beam_select.hip -- beam search's selection for gfx950: the best continuations
// of each request's sequences, over sequences and vocabulary.
//
// A sequence's continuation by token t is worth score + x_t - log sum exp x.
// Within a row the logits' order is the values', so the selection needs the
// whole row's largest logits and its sum only:
//   qm_beam_slices  a wave per 1024 logits: their largest, its token, the sum
//                   of exp(x - largest).  The one pass over the logits.
//   qm_beam_draw    a workgroup per request: the rows' log-sums, the `take`
//                   best slices by their largest logits' values, and the best
//                   of those slices' logits.  No other slice can hold a chosen
//                   one: `take` continuations are before all of its.
// The slices are bound by HBM: 87 rows of 248320 logits in 15 us, 5.8 TB/s.  The
// draw is one workgroup's chain of loads and barriers, 11 us for 12 requests of
// 8 rows and 7 for one of 4: log-sums 2, the leaders 3, the rest their logits.
// Values are compared in 64 bits, ties to the lower row and then the lower token.
// The log-sum is off by 22 2^-24 at most: an exponential by 2 (v_exp_f32) and, of
// a logit d below its slice's largest, by d for the difference's rounding, d for
// its product's with log2(e) and d / 4 for that constant's own; weighted as the
// terms are d is ln 1024 at most; and a lane's sum by 4.
#include "qm_device.h"
#include "qm_beam.h"

// Rows that take part and are read: a finite score, not at their end.
QM_DEV bool beam_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
QM_DEV bool beam_live(const BeamArgs& A, int row) { return beam_finite(A.scores[row]) && !(A.done && A.done[row]); }

extern "C" __global__ __launch_bounds__(256) void qm_beam_slices(BeamArgs A) {
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = (int)(at / A.ns), slice = (int)(at - (int64_t)row * A.ns);
    if (row >= A.groups * A.beams || !beam_live(A, row)) return;      // uniform per wave
    const int t0 = slice * QMK_BEAM_SLICE + lane;
    const float* x = A.logits + (size_t)row * A.vocab;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = x[min(t0 + 64 * i, A.vocab - 1)];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (t0 + 64 * i >= A.vocab) v[i] = -INFINITY;
        top = fmaxf(top, v[i]);
    }
    top = max_xor32(max_xor16(row_max16(top)));
    // the lowest token that has it
    int token = A.vocab;
#pragma unroll
    for (int i = 15; i >= 0; --i) {
        const uint64_t have = __ballot(v[i] == top);
        if (have) token = t0 - lane + 64 * i + __builtin_ctzll(have);
    }
    const float base = top == -INFINITY ? 0.0f : top;
    // The sum: NaN where a logit is, or an infinity.  By halves, four roundings of
    // f32 and not 16, and then in 64 bits (the log-sum of many equal logits is off
    // by 3.6 2^-24, in order and in f32 by 14).
    float e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = exp_fast(v[i] - base);
#pragma unroll
    for (int d = 8; d > 0; d /= 2)
#pragma unroll
        for (int i = 0; i < d; ++i) e[i] += e[i + d];
    const double sum = wave_sum64((double)e[0]);
    if (lane == 0) A.slices[at] = BeamSlice{sum, top, token};
}

// ---- the request's choice ------------------------------------------------------
// A continuation's key: larger is better.  value: the f64's bits in order, 0:
// none; index: row of the request * vocab + token.
struct BeamKey {
    uint64_t value;
    uint32_t index;
};
QM_DEV bool before(const BeamKey& a, const BeamKey& b) { return a.value != b.value ? a.value > b.value : a.index < b.index; }
QM_DEV uint64_t ordered(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);          // no -0
    return u >> 63 ? ~u : u | 1ull << 63;
}
QM_DEV double unordered(uint64_t u) { return __builtin_bit_cast(double, u >> 63 ? u & ~(1ull << 63) : ~u); }

#define BEAM_THREADS 1024
#define BEAM_LIST 512              // keys that are sorted by counting
// A slice that is looked through: its row, first token, and the logit below
// which none of its tokens is chosen.
struct BeamLead {
    int32_t row, t0;
    float cut;
    int32_t ended;                 // the row's one continuation
};
struct BeamLds {
    double base[QMK_BEAM_MAX];     // score - log-sum of a row, or an ended one's score; not finite: takes no part
    int32_t ended[QMK_BEAM_MAX];
    int32_t hist[256];
    uint32_t tops[BEAM_THREADS / 16], bound;
    BeamKey list[BEAM_LIST], sorted[QMK_BEAM_MAX];
    BeamKey leaders[QMK_BEAM_MAX];
    BeamLead lead[QMK_BEAM_MAX];
    int32_t n, digit, above;
};

template <int CTRL>
QM_DEV uint64_t max_dpp(uint64_t x) {
    const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)x, CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(x >> 32), CTRL, 0xF, 0xF, false);
    const uint64_t y = (uint64_t)hi << 32 | lo;
    return x > y ? x : y;
}
// Digit d of a key, from the top: eight of the value, then four of the index
// (from the other end: the lower is before).
QM_DEV int key_digit(const BeamKey& k, int d) {
    return d < 8 ? (int)(k.value >> (56 - 8 * d)) & 255 : (int)(~k.index >> (24 - 8 * (d - 8))) & 255;
}
// Whether the digits before d are those of `prefix` (0), or larger (1), or smaller (-1).
QM_DEV int key_against(const BeamKey& k, const BeamKey& prefix, int d) {
    const int vb = min(d, 8) * 8;
    const uint64_t kv = vb ? k.value >> (64 - vb) : 0, pv = vb ? prefix.value >> (64 - vb) : 0;
    if (kv != pv) return kv > pv ? 1 : -1;
    if (d <= 8) return 0;
    const int ib = (d - 8) * 8;
    const uint32_t ki = ~k.index >> (32 - ib), pi = ~prefix.index >> (32 - ib);
    return ki == pi ? 0 : ki > pi ? 1 : -1;
}

QM_DEV void beam_list(BeamLds& sh, const BeamKey& k) {
    const int at = atomicAdd(&sh.n, 1);
    if (at < BEAM_LIST) sh.list[at] = k;
}
// The list's best `take`, in order, into `out`; their number.
QM_DEV int beam_sort(BeamLds& sh, int take, BeamKey* out) {
    const int tid = threadIdx.x, found = min(sh.n, BEAM_LIST);
    if (tid < found) {
        const BeamKey k = sh.list[tid];
        int rank = 0;
        for (int i = 0; i < found; ++i) rank += before(sh.list[i], k);
        if (rank < take) out[rank] = k;
    }
    __syncthreads();
    return min(found, take);
}

// The best `take` of keys key(0 .. n - 1), in order, into `out`; their number.
// 64 groups of threads have a largest key each, and the take-th of those is a
// bound: what is not below is sorted by counting.  Where that is more than
// BEAM_LIST (equal values), a radix select narrows it, from the top digit on
// (keys differ, so in the end there are no more).  A thread keeps its first KEEP
// keys.
template <int KEEP, class F>
QM_DEV int beam_best(BeamLds& sh, int n, int take, BeamKey* out, F key) {
    const int tid = threadIdx.x, lane = tid & 63;
    if (n == 0) return 0;                                  // uniform
    BeamKey kept[KEEP];
#pragma unroll
    for (int r = 0; r < KEEP; ++r) {
        kept[r] = key(min(tid + BEAM_THREADS * r, n - 1));
        if (tid + BEAM_THREADS * r >= n) kept[r].value = 0;
    }
    auto each = [&](auto use) {
#pragma unroll
        for (int r = 0; r < KEEP; ++r) use(kept[r]);
        for (int i = tid + BEAM_THREADS * KEEP; i < n; i += BEAM_THREADS) use(key(i));
    };
    if (tid == 0) sh.n = 0;
    uint64_t top = 0;
    each([&](const BeamKey& k) { top = max(top, k.value); });
    top = max_dpp<0xB1>(top);
    top = max_dpp<0x4E>(top);
    top = max_dpp<0x141>(top);
    top = max_dpp<0x140>(top);
    // (the upper halves, but for six bits that make them differ: a bound all the same)
    if ((lane & 15) == 0) sh.tops[tid >> 4] = ((uint32_t)(top >> 32) & ~63u) | (uint32_t)(63 - (tid >> 4));
    __syncthreads();
    if (tid < 64) {
        const uint32_t mine = sh.tops[lane];
        int rank = 0;
#pragma unroll
        for (int i = 0; i < 64; ++i) rank += (uint32_t)__builtin_amdgcn_readlane((int)mine, i) > mine;
        if (rank == take - 1) sh.bound = mine & ~63u;
    }
    __syncthreads();
    const uint64_t least = max((uint64_t)sh.bound << 32, (uint64_t)1);       // value 0: none
    BeamKey prefix{0, ~0u};
    int digits = 0, above = 0;
    for (;;) {
        // those at or above the prefix
        each([&](const BeamKey& k) {
            if (k.value < least || (digits && key_against(k, prefix, digits) < 0)) return;
            beam_list(sh, k);
        });
        __syncthreads();
        if (sh.n <= BEAM_LIST || digits == 12) break;      // uniform
        if (tid < 256) sh.hist[tid] = 0;
        __syncthreads();
        if (tid == 0) sh.n = 0;                            // all have looked at it
        each([&](const BeamKey& k) {
            if (k.value >= least && key_against(k, prefix, digits) == 0) atomicAdd(&sh.hist[key_digit(k, digits)], 1);
        });
        __syncthreads();
        // the digit at which `take` are reached: a wave, lane l with bins 255 - 4 l ..
        if (tid < 64) {
            int bin[4], mine = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) mine += bin[j] = sh.hist[255 - 4 * tid - j];
            int incl = mine;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int y = __shfl_up(incl, d);
                incl += tid >= d ? y : 0;
            }
            const uint64_t reach = __ballot(above + incl >= take);
            // there are more than BEAM_LIST >= take at or above the prefix
            if (reach && tid == __builtin_ctzll(reach)) {
                int a = above + incl - mine, j = 0;
#pragma unroll
                for (; j < 3; ++j) {
                    if (a + bin[j] >= take) break;
                    a += bin[j];
                }
                sh.digit = 255 - 4 * tid - j;
                sh.above = a;
            }
        }
        __syncthreads();
        above = sh.above;
        if (digits < 8) prefix.value |= (uint64_t)sh.digit << (56 - 8 * digits);
        else prefix.index = ~(~prefix.index | (uint32_t)sh.digit << (24 - 8 * (digits - 8)));
        ++digits;
    }
    return beam_sort(sh, take, out);
}

extern "C" __global__ __launch_bounds__(BEAM_THREADS) void qm_beam_draw(BeamArgs A) {
    __shared__ BeamLds sh;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row0 = blockIdx.x * A.beams;
    for (int b = w; b < A.beams; b += BEAM_THREADS / 64) {             // uniform per wave
        const float score = A.scores[row0 + b];
        const bool ended = A.done && A.done[row0 + b] != 0;
        double base = __builtin_nan("");
        if (beam_finite(score) && ended) {
            base = score;
        } else if (beam_finite(score)) {
            const BeamSlice* s = A.slices + (size_t)(row0 + b) * A.ns;
            BeamSlice x[QMK_BEAM_VOCAB / QMK_BEAM_SLICE / 64];
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < QMK_BEAM_VOCAB / QMK_BEAM_SLICE / 64; ++i) {
                x[i] = s[min(lane + 64 * i, A.ns - 1)];
                top = fmaxf(top, x[i].top);
            }
            top = max_xor32(max_xor16(row_max16(top)));
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < QMK_BEAM_VOCAB / QMK_BEAM_SLICE / 64; ++i)
                if (lane + 64 * i < A.ns && x[i].sum != 0.0) sum += x[i].sum * exp((double)(x[i].top == -INFINITY ? 0.0f : x[i].top) - (double)top);
            sum = wave_sum64(sum);
            base = (double)score - ((double)top + log(sum));           // NaN, infinite: takes no part
        }
        if (lane == 0) {
            sh.base[b] = base;
            sh.ended[b] = ended;
        }
    }
    __syncthreads();
    auto value = [&](int b, float x) {
        const double v = sh.base[b] + (double)x;
        return __builtin_isfinite(v) ? ordered(v) : 0ull;
    };
    // the best slices, by their best tokens; a row at its end has one continuation
    const int leaders = beam_best<2>(sh, A.beams * A.ns, A.take, sh.leaders, [&](int i) {
        const int b = i / A.ns, j = i - b * A.ns;
        if (sh.ended[b]) return BeamKey{j == 0 ? value(b, 0.0f) : 0ull, (uint32_t)(b * A.vocab + A.end_id)};
        if (!__builtin_isfinite(sh.base[b])) return BeamKey{0ull, 0u};
        const BeamSlice s = A.slices[(size_t)(row0 + b) * A.ns + j];
        return BeamKey{value(b, s.top), (uint32_t)(b * A.vocab + s.token)};
    });
    // And the best of those slices' tokens.  Where the slices are `take`, none is
    // worth less than the last one's best: what passes in f32 is compared in f64.
    // Where there are fewer (short vocabularies), the tokens find a bound of their
    // own (7 requests of 2 rows of 1985, take 25: 16.3 / 13.6 us).
    const bool bound = leaders == A.take;
    const uint64_t least = bound ? sh.leaders[leaders - 1].value : 1ull;
    if (tid < leaders) {
        const int index = (int)sh.leaders[tid].index, b = index / A.vocab;
        // less what the sum's rounding to 64 bits, the difference's and the cut's own can be
        const double base = sh.base[b], last = unordered(least);
        const float cut = (float)(last - base - (fabs(base) + fabs(last)) * 0x1p-50);
        sh.lead[tid] = BeamLead{b, (index - b * A.vocab) / QMK_BEAM_SLICE * QMK_BEAM_SLICE, fminf(cut - fabsf(cut) * 0x1p-20f - 0x1p-100f, 0x1.fffffep127f), sh.ended[b]};
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    for (int r0 = 0; bound && r0 < leaders; r0 += 8) {     // uniform
        BeamLead lead[8];
        float x[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            lead[r] = sh.lead[min(r0 + r, leaders - 1)];
            x[r] = A.logits[(size_t)(row0 + lead[r].row) * A.vocab + min(lead[r].t0 + tid, A.vocab - 1)];
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if (r0 + r >= leaders) break;                  // uniform
            if (lead[r].ended) {
                if (tid == 0) beam_list(sh, sh.leaders[r0 + r]);
            } else if (x[r] >= lead[r].cut && lead[r].t0 + tid < A.vocab) {
                const uint64_t v = value(lead[r].row, x[r]);
                if (v >= least) beam_list(sh, BeamKey{v, (uint32_t)(lead[r].row * A.vocab + lead[r].t0 + tid)});
            }
        }
    }
    __syncthreads();
    int found;
    if (bound && sh.n <= BEAM_LIST) {
        found = beam_sort(sh, A.take, sh.sorted);
    } else {
        __syncthreads();                                   // all have looked at it
        found = beam_best<4>(sh, leaders * QMK_BEAM_SLICE, A.take, sh.sorted, [&](int i) {
            const BeamLead lead = sh.lead[i / QMK_BEAM_SLICE];
            const int t = lead.t0 + i % QMK_BEAM_SLICE;
            if (lead.ended) return BeamKey{i % QMK_BEAM_SLICE == 0 ? value(lead.row, 0.0f) : 0ull, (uint32_t)(lead.row * A.vocab + A.end_id)};
            if (t >= A.vocab) return BeamKey{0ull, 0u};
            return BeamKey{value(lead.row, A.logits[(size_t)(row0 + lead.row) * A.vocab + t]), (uint32_t)(lead.row * A.vocab + t)};
        });
    }
    if (tid < A.take) {
        const size_t to = (size_t)blockIdx.x * A.take + tid;
        // A place that no continuation takes: where the places are the request's
        // rows, it stays the row that it is, so that parents is a list for the
        // forks whatever the requests have.
        int parent = A.take == A.beams ? row0 + tid : -1, token = -1, over = 0;
        float score = -INFINITY;
        if (tid < found) {
            const BeamKey k = sh.sorted[tid];
            const int b = k.index / A.vocab;
            parent = row0 + b;
            token = (int)(k.index - b * A.vocab);
            score = (float)unordered(k.value);
            over = sh.ended[b] || token == A.end_id;
        }
        // (its scores and flags may stand where its choice goes: all are read)
        A.parents[to] = parent;
        A.tokens[to] = token;
        A.out_scores[to] = score;
        if (A.out_done) A.out_done[to] = over;
    }
}
