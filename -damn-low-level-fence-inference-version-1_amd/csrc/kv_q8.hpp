// kv_q8.hpp -- the 8-bit codes of a paged KV cache: rounding to them, reading
// them back, and the checks of a fence_kv_pages.
#pragma once

#include "common.hpp"

namespace fence {

constexpr float kCodeTop[2] = {127.0f, 448.0f};  // the largest code of FENCE_KV_INT8, FENCE_KV_E4M3

inline bool kv_pages_ok(const fence_kv_pages* c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return false;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)) return false;
    if (c->type != FENCE_KV_INT8 && c->type != FENCE_KV_E4M3) return false;
    if (c->n_pages < 1 || c->n_kv_heads < 1 || c->n_kv_heads > 65535) return false;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return false;
    if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16) return false;
    return static_cast<int64_t>(c->n_pages) * c->page_size <= INT32_MAX;
}

// x / s as a float whose last bit says that it is not exact: the quotient
// truncated toward zero with that bit set (rounding to odd).  Rounding that
// once more, to 8 bits or fewer, gives the exact quotient's rounding, ties
// included.  `inv` = 1/s.  t below is within one step of the quotient
// (Markstein's correction of x * inv), and the remainder x - t * s is exact,
// so its sign says on which side t lies.  For |s| >= 2^-80, where nothing of
// the remainder that matters is lost below 2^-149.
__device__ __forceinline__ float quotient_odd(float x, float s, float inv) {
#pragma clang fp contract(off)
    const float t0 = x * inv;
    const float t = __builtin_fmaf(__builtin_fmaf(-t0, s, x), inv, t0);
    const float r = __builtin_fmaf(-t, s, x);
    uint32_t bits = __builtin_bit_cast(uint32_t, t);
    const uint32_t past = (__builtin_bit_cast(uint32_t, r) ^ bits) >> 31;  // |t| is above the quotient's
    if (r != 0.0f) bits = (bits - past) | 1u;
    return __builtin_bit_cast(float, bits);
}

// The same of a 64-bit number that is exact, or off by less than matters.
__device__ __forceinline__ float round_odd(double y) {
    const float f = static_cast<float>(y);
    uint32_t bits = __builtin_bit_cast(uint32_t, f);
    const double d = static_cast<double>(f);
    const uint32_t past = fabs(d) > fabs(y) ? 1u : 0u;
    if (d != y) bits = (bits - past) | 1u;
    return __builtin_bit_cast(float, bits);
}

// Four values, rounded to odd or exact, as codes: nearest, ties to even.
template <int TYPE>
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
    constexpr float top = TYPE == FENCE_KV_INT8 ? 127.0f : 448.0f;
    a = __builtin_amdgcn_fmed3f(a, -top, top);
    b = __builtin_amdgcn_fmed3f(b, -top, top);
    c = __builtin_amdgcn_fmed3f(c, -top, top);
    d = __builtin_amdgcn_fmed3f(d, -top, top);
    if constexpr (TYPE == FENCE_KV_INT8) {
        const uint32_t ia = static_cast<int>(rintf(a)), ib = static_cast<int>(rintf(b));
        const uint32_t ic = static_cast<int>(rintf(c)), id = static_cast<int>(rintf(d));
        return (ia & 0xFF) | (ib & 0xFF) << 8 | (ic & 0xFF) << 16 | id << 24;
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
    }
}

// Code i (0..3) of a word as a float.
template <int TYPE, int I>
__device__ __forceinline__ float code_value(uint32_t w) {
    if constexpr (TYPE == FENCE_KV_INT8) return static_cast<float>(static_cast<int>(w << (24 - 8 * I)) >> 24);
    else return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), I);
}

}  // namespace fence
