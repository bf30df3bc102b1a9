// qm_kv4_device.h -- device helpers of the paged 4-bit KV cache.
#pragma once
#include "qm_device.h"
#include "qm_kv4.h"

// The head's half page h (0, 1) of page id; the id is the caller's to check.
QM_DEV uint8_t* kv4_half(const Kv4Cache& c, int layer, int id, int head, int h) {
    return c.pages + ((size_t)layer * c.num_pages + id) * QMK_KV4_PAGE_BYTES + head * QMK_KV4_HEAD_BYTES + h * QMK_KV4_HALF_BYTES;
}
QM_DEV bool kv4_is_page(const Kv4Cache& c, int id) { return (uint32_t)id < (uint32_t)c.num_pages; }

// f64 -> f32 -> f16, both to nearest even.  The compiler makes one rounding
// of the two casts, which differs where the f32 value is halfway between two
// f16 values.
QM_DEV uint16_t f64_to_f16_by_f32(double x) {
    float f = (float)x;
    asm("" : "+v"(f));
    return f32_to_f16(f);
}

// 1 / sqrt(x): v_rsq_f64 is good to about 2^-24; each step of Newton's squares
// the error.
QM_DEV double inverse_root_f64(double x) {
    double inv = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; ++i) inv = inv * __builtin_fma(-0.5 * x * inv, inv, 1.5);
    if (!(x < __builtin_inf())) inv = x == x ? 0.0 : x;      // rsq's own 0 for an infinity, NaN for NaN
    return inv;
}

// The scale of a group, f16 bits: the quotient in 64 bits, so that it is the
// same whoever computes it, then f32, then f16.
QM_DEV uint16_t kv4_scale(float lo, float hi) {
    return f64_to_f16_by_f32(((double)hi - (double)lo) * (1.0 / 15.0));
}

// The code of x in a group (lo, s), inv ~ 1 / s: an estimate, then one step
// by the exact remainder (x, lo, s are f16 values, so x - lo - q s is exact
// in 64 bits): a value beside the border of two codes, or on it, gets the
// same one whoever computes it.  Ties go to the even code.
QM_DEV uint32_t kv4_code(float x, float lo, float s, float inv) {
    const float q0 = fminf(fmaxf(rintf((x - lo) * inv), 0.0f), 15.0f);
    const double r = __builtin_fma(-(double)q0, (double)s, (double)x - (double)lo);
    const double h = 0.5 * (double)s;
    int q = (int)q0;
    const bool odd = q & 1;
    if (r > h || (r == h && odd)) ++q;
    else if (r < -h || (r == -h && odd)) --q;
    q = min(max(q, 0), 15);
    return s > 0.0f ? (uint32_t)q : 0u;     // s = 0, NaN
}

// Inclusive sum over the wave's lanes: within the rows of 16, then the last
// lane of a row into the next row, and of the lower half into the upper.
template <int CTRL, int ROWS>
QM_DEV uint32_t scan_step(uint32_t x) { return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false); }
QM_DEV uint32_t wave_scan(uint32_t x) {
    x = scan_step<0x111, 0xF>(x);
    x = scan_step<0x112, 0xF>(x);
    x = scan_step<0x114, 0xF>(x);
    x = scan_step<0x118, 0xF>(x);
    x = scan_step<0x142, 0xA>(x);
    return scan_step<0x143, 0xC>(x);
}
