// gqa_decode_kv4.hip -- the GQA decode step over the paged 4-bit KV cache
// (qm_kv4.h) for gfx950: the mixer slice of qm_gqa_decode (gemv.rs:927-1011)
// with the cache's rows read as lo + s * code.
#include "qm_kv4_device.h"
#include "qm_kernel_args.h"
#include "qm_gqa_common.h"

#define KV4_PART_STRIDE 260   // acc[256], m, l, pad[2]

// What a batch row of the step is: a table row of `len` tokens, the last of
// them new; none (len 0: the output is zero); or one that is refused (its
// output is NaN): longer than max_len, or a table row that an earlier batch
// row has.
struct StepRow {
    int row, len;
    bool refused;
};
QM_DEV StepRow step_row(const GqaKv4Args& A, int b) {
    StepRow r{-1, 0, false};
    if (A.result && A.result[0] != 0) return r;
    const int row = A.slots ? A.slots[b] : b;
    if ((uint32_t)row >= (uint32_t)A.c.rows) return r;
    r.row = row;
    r.len = max(A.c.lens[row], 0);
    r.refused = r.len > A.max_len;
    if (A.slots) {
        const int lane = threadIdx.x & 63;
        for (int j0 = 0; j0 < b; j0 += 64) {          // uniform
            const int j = j0 + lane;
            if (__ballot(j < b && A.slots[min(j, b - 1)] == row)) r.refused = true;
        }
    }
    if (r.refused) r.len = 0;
    return r;
}

// Sum over the wave in 64 bits.
QM_DEV double wave_sum64_f64(double x) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) x += __shfl_xor(x, off);
    return x;
}

// The new k row of a head as the f16 cache holds it: per-head RMSNorm
// (1 + gamma, eps 1e-6) and RoPE in 64 bits, rounded to f32 and f16.  64 bits
// because a code beside a border must not depend on the order of a sum.
// Lane l has dims 4 l .. 4 l + 3.
QM_DEV void new_k(const float4 x, uint2 gw, float4 c, float4 s, int lane, uint16_t (&out)[4]) {
    const double v[4] = {x.x, x.y, x.z, x.w};
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
    const uint16_t g[4] = {(uint16_t)(gw.x & 0xffffu), (uint16_t)(gw.x >> 16), (uint16_t)(gw.y & 0xffffu), (uint16_t)(gw.y >> 16)};
    const double sum = wave_sum64_f64((v[0] * v[0] + v[1] * v[1]) + (v[2] * v[2] + v[3] * v[3]));
    const double inv = 1.0 / __builtin_sqrt(sum / QM_GQA_HD + 1e-6);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double y = v[i] * inv * (1.0 + (double)f16_to_f32(g[i]));
        const double partner = __shfl_xor(y, 8);
        const double turned = lane < 8 ? y * cc[i] - partner * ss[i] : y * cc[i] + partner * ss[i];
        out[i] = f64_to_f16_by_f32(lane < 16 ? turned : y);
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
    const float s = f16_to_f32(c.s), inv = s > 0.0f ? 1.0f / s : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) c.q[i] = kv4_code(x[i], lo, s, inv);
    return c;
}

// The new token's K and V rows into the cache: one wave per (batch row, kv
// head).
extern "C" __global__ __launch_bounds__(64) void qm_gqa_kv4_append(GqaKv4Args A) {
    const int lane = threadIdx.x, g = blockIdx.x & 3, b = blockIdx.x >> 2;
    const StepRow r = step_row(A, b);
    if (r.len == 0) return;
    const int pos = r.len - 1, t = pos & 31;
    if ((pos >> 6) >= A.c.max_pages) return;
    const int id = A.c.table[(size_t)r.row * A.c.max_pages + (pos >> 6)];
    if (!kv4_is_page(A.c, id)) return;
    const size_t src = ((size_t)b * QM_GQA_KV_HEADS + g) * QM_GQA_HD + 4 * lane;
    float4 rc, rs;
    rope_row_loads(A.rope_cos + (size_t)pos * (QM_GQA_ROT / 2), A.rope_sin + (size_t)pos * (QM_GQA_ROT / 2), lane, rc, rs);
    uint16_t kh[4];
    new_k(ld4(A.k_new + src), *reinterpret_cast<const uint2*>(A.k_norm + 4 * lane), rc, rs, lane, kh);
    const float4 v = ld4(A.v_new + src);
    const uint16_t vh[4] = {f32_to_f16(v.x), f32_to_f16(v.y), f32_to_f16(v.z), f32_to_f16(v.w)};
    const CodedRow ck = code_row(kh), cv = code_row(vh);
    uint32_t* words = reinterpret_cast<uint32_t*>(kv4_half(A.c, A.layer, id, g, (pos >> 5) & 1));
    uint32_t kw = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) kw |= ck.q[i] << (4 * kv4_nibble(4 * (lane & 1) + i));
    kw |= __shfl_xor(kw, 1);
    if ((lane & 1) == 0) words[kv4_k_word(t, 4 * lane)] = kw;
    const int shift = 4 * kv4_v_nibble(t);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t* w = words + kv4_v_word(t, 4 * lane + i);
        *w = (*w & ~(15u << shift)) | (cv.q[i] << shift);
    }
    if ((lane & 15) == 0) {
        uint16_t* meta = reinterpret_cast<uint16_t*>(words) + QMK_KV4_META / 2;
        const int sa = kv4_s_at(t, lane >> 4), la = kv4_lo_at(t, lane >> 4);
        meta[sa] = ck.s;
        meta[128 + la] = ck.lo;
        meta[256 + sa] = cv.s;
        meta[384 + la] = cv.lo;
    }
}

// Attention of one split: `chunk` tokens of one (batch row, kv head), all
// four query heads, half a page at a time through LDS in f32.
extern "C" __global__ __launch_bounds__(256) void qm_gqa_kv4_split(GqaKv4Args A) {
    __shared__ __attribute__((aligned(16))) uint32_t w[QMK_KV4_HALF_BYTES / 4];
    __shared__ float tile[32][257];
    __shared__ float q[4][256], p[4][32], top[4], total[4], corr[4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int split = blockIdx.x % A.nsplit, bg = blockIdx.x / A.nsplit;
    const int g = bg & 3, b = bg >> 2;
    const StepRow r = step_row(A, b);
    const int t_begin = split * A.chunk, t_end = min(t_begin + A.chunk, r.len);
    float acc[4] = {0, 0, 0, 0};
    {
        const int pos = max(r.len - 1, 0);
        float4 rc, rs;
        rope_row_loads(A.rope_cos + (size_t)pos * (QM_GQA_ROT / 2), A.rope_sin + (size_t)pos * (QM_GQA_ROT / 2), lane, rc, rs);
        const float4 x = norm_rope_head(ld4(A.q_gate + ((size_t)b * QM_GQA_HEADS + 4 * g + wv) * (2 * QM_GQA_HD) + 4 * lane),
                                        *reinterpret_cast<const uint2*>(A.q_norm + 4 * lane), rc, rs, lane);
        *reinterpret_cast<float4*>(&q[wv][4 * lane]) = x;
        if (tid < 4) { top[tid] = -INFINITY; total[tid] = 0.0f; }
    }
    for (int t0 = t_begin; t0 < t_end; t0 += 32) {
        if ((t0 >> 6) >= A.c.max_pages) break;
        const int id = A.c.table[(size_t)r.row * A.c.max_pages + (t0 >> 6)];
        if (!kv4_is_page(A.c, id)) continue;
        const uint4* src = reinterpret_cast<const uint4*>(kv4_half(A.c, A.layer, id, g, (t0 >> 5) & 1));
        __syncthreads();
        for (int j = tid; j < QMK_KV4_HALF_BYTES / 16; j += 256) reinterpret_cast<uint4*>(w)[j] = src[j];
        __syncthreads();
        const uint16_t* meta = reinterpret_cast<const uint16_t*>(&w[QMK_KV4_META / 4]);
        const int d = tid, group = d >> 6;
        for (int t = 0; t < 32; ++t)
            tile[t][d] = fmaf((float)((w[kv4_k_word(t, d)] >> (4 * kv4_k_nibble(d))) & 15u),
                              f16_to_f32(meta[kv4_s_at(t, group)]), f16_to_f32(meta[128 + kv4_lo_at(t, group)]));
        __syncthreads();
        if (tid < 128) {
            const int h = tid >> 5, t = tid & 31;
            float s = 0.0f;
            for (int j = 0; j < 256; ++j) s = fmaf(q[h][j], tile[t][j], s);
            s = t0 + t < t_end ? s * (1.4426950408889634f / 16.0f) : -INFINITY;
            float m = s;
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
            const float mn = fmaxf(top[h], m), co = top[h] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[h] - mn);
            const float e = s == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s - mn);
            float l = e;
            for (int o = 16; o; o >>= 1) l += __shfl_xor(l, o);
            p[h][t] = e;
            if (t == 0) { total[h] = total[h] * co + l; corr[h] = co; top[h] = mn; }
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 4; ++h) acc[h] *= corr[h];
        for (int t = 0; t < 32; ++t) {
            if (t0 + t >= t_end) break;
            const float v = fmaf((float)((w[kv4_v_word(t, d)] >> (4 * kv4_v_nibble(t))) & 15u),
                                 f16_to_f32(meta[256 + kv4_s_at(t, group)]), f16_to_f32(meta[384 + kv4_lo_at(t, group)]));
#pragma unroll
            for (int h = 0; h < 4; ++h) acc[h] = fmaf(p[h][t], v, acc[h]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        float* P = A.partial + ((size_t)(bg * (size_t)A.nsplit + split) * 4 + h) * KV4_PART_STRIDE;
        P[tid] = acc[h];
        if (tid == 0) { P[256] = top[h]; P[257] = total[h]; }
    }
}

// The splits' partials of one query head, joined, and the gate.
extern "C" __global__ __launch_bounds__(256) void qm_gqa_kv4_merge(GqaKv4Args A) {
    const int d = threadIdx.x, h = blockIdx.x % QM_GQA_HEADS, b = blockIdx.x / QM_GQA_HEADS;
    const StepRow r = step_row(A, b);
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int s = 0; s < A.nsplit; ++s) {
        const float* P = A.partial + ((size_t)((b * 4 + (h >> 2)) * (size_t)A.nsplit + s) * 4 + (h & 3)) * KV4_PART_STRIDE;
        const float ms = P[256];
        if (P[257] == 0.0f) continue;                 // no tokens
        const float mn = fmaxf(m, ms), c0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn), c1 = __builtin_amdgcn_exp2f(ms - mn);
        l = l * c0 + P[257] * c1;
        o = o * c0 + P[d] * c1;
        m = mn;
    }
    const float gate = A.q_gate[((size_t)b * QM_GQA_HEADS + h) * (2 * QM_GQA_HD) + QM_GQA_HD + d];
    float y = l != 0.0f ? (o * __builtin_amdgcn_rcpf(l)) * sigmoid_fast(gate) : 0.0f;
    if (r.refused) y = __builtin_nanf("");
    A.out[((size_t)b * QM_GQA_HEADS + h) * QM_GQA_HD + d] = y;
}
