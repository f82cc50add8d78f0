// store_q8.hip -- the K and V rows of a batched step into the pages of an
// 8-bit KV cache, on gfx950.
//
// Per page and head, scale = max(old, max|new| / top) and code =
// round(value / scale).  The largest value has to be known before the first
// code, and a scale that grows changes codes already there, so everything
// that falls into one page and head belongs to one workgroup: it reads the
// rows once into registers while it takes their maximum, and writes the codes
// from there.  Rows of one page follow one another, so a workgroup finds its
// work by itself: it owns the rows of a window at which a page's rows begin.
// The stream is bound by the bytes in and out; a code costs about 15 VALU
// operations (an exact rounding of the quotient, kv_q8.hpp), which hides
// behind them.
#include "kv_q8.hpp"

namespace fence {
namespace {

constexpr int kThreads = 256;
constexpr int kHeld = 4;  // groups of 8 values a lane keeps: 64 rows of 128 values a workgroup

struct StoreArgs {
    fence_kv_pages c;
    const void* k;
    const void* v;
    const int32_t* slots;
    int64_t ld, tokens;
    int window, page_shift;
};

// Eight values of a row, in fp32.  VEC: 16-byte aligned.
template <int IN, bool VEC>
__device__ __forceinline__ void load8(const void* base, int64_t at, float* x) {
    if constexpr (IN == FENCE_F32) {
        const float* p = static_cast<const float*>(base) + at;
        if constexpr (VEC) {
            const f4 a = ld4<false>(p), b = ld4<false>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = p[i];
        }
    } else {
        typedef _Float16 h8 __attribute__((ext_vector_type(8)));
        const _Float16* p = static_cast<const _Float16*>(base) + at;
        if constexpr (VEC) {
            const h8 a = *reinterpret_cast<const h8*>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(a[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(p[i]);
        }
    }
}

// The largest magnitude's bits: as whole numbers they order like the values,
// with infinity above every number and NaN above that.
__device__ __forceinline__ uint32_t max_bits(uint32_t m, const float* x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu;
        m = m > b ? m : b;
    }
    return m;
}

template <int TYPE>
__device__ __forceinline__ void put8(uint8_t* to, const float* x, float scale, float inv) {
    float y[8];
    const bool usable = scale > 0.0f && scale < __builtin_inff();
    if (usable && scale >= 0x1p-80f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = quotient_odd(x[i], scale, inv);
    } else {  // codes of 0 where the scale is 0 or not finite; a tiny scale's quotients in 64 bits
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = usable ? round_odd(static_cast<double>(x[i]) / scale) : 0.0f;
    }
    uint2 w;
    w.x = to_codes<TYPE>(y[0], y[1], y[2], y[3]);
    w.y = to_codes<TYPE>(y[4], y[5], y[6], y[7]);
    *reinterpret_cast<uint2*>(to) = w;
}

template <int TYPE, int IN, bool VEC>
__global__ __launch_bounds__(kThreads) void store_q8_kernel(StoreArgs a) {
    __shared__ uint32_t wave_max[2][kThreads / kWave];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const int head = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const void* src = is_v ? a.v : a.k;
    const int hd = a.c.head_dim, page_size = 1 << a.page_shift;
    const int per_row = hd / 8;  // groups of 8 values a row
    const int64_t first = static_cast<int64_t>(blockIdx.x) * a.window;
    const int64_t last = first + a.window < a.tokens ? first + a.window : a.tokens;
    int turn = 0;  // the two halves of wave_max take turns, so one barrier a page is enough
    for (int64_t t = first; t < last; ++t) {
        const int slot = a.slots[t];
        if (slot < 0 || (slot >> a.page_shift) >= a.c.n_pages) continue;
        const int off = slot & (page_size - 1);
        if (off != 0 && t > 0 && a.slots[t - 1] == slot - 1) continue;  // inside a page's rows
        // how many rows of this page follow
        int n = 1;
        const int most = static_cast<int>(a.tokens - t < page_size - off ? a.tokens - t : page_size - off);
        while (n < most) {
            const int i = n + lane;
            const uint64_t differ = __ballot(i >= most || a.slots[t + i] != slot + i);
            const int same = differ ? __builtin_ctzll(differ) : kWave;
            n += same;
            if (same < kWave) break;
        }
        const int groups = n * per_row;
        const int64_t at0 = t * a.ld + static_cast<int64_t>(head) * hd;
        float x[kHeld][8];
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int g = tid + j * kThreads;
            if (g < groups) load8<IN, VEC>(src, at0 + (g / per_row) * a.ld + (g % per_row) * 8, x[j]);
        }
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (tid + j * kThreads < groups) m = max_bits(m, x[j]);
        for (int g = tid + kHeld * kThreads; g < groups; g += kThreads) {  // a page of more than kHeld groups a lane
            float y[8];
            load8<IN, VEC>(src, at0 + (g / per_row) * a.ld + (g % per_row) * 8, y);
            m = max_bits(m, y);
        }
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const uint32_t o = __shfl_xor(m, d);
            m = m > o ? m : o;
        }
        if (lane == 0) wave_max[turn][wave] = m;
        const int64_t page = slot >> a.page_shift;
        float* scale_at = (is_v ? a.c.v_scale : a.c.k_scale) + page * a.c.n_kv_heads + head;
        const float old = off ? *scale_at : 0.0f;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / kWave; ++w) m = m > wave_max[turn][w] ? m : wave_max[turn][w];
        turn ^= 1;
        const float mine = __builtin_bit_cast(float, m) / kCodeTop[TYPE];
        const float scale = old != old || mine != mine ? __builtin_nanf("") : old > mine ? old : mine;
        const float inv = 1.0f / scale;
        uint8_t* codes = static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) +
                         ((page * a.c.n_kv_heads + head) << a.page_shift) * hd;
        if (scale > old && off) {  // what the page held, at the new scale
            const bool finite = scale < __builtin_inff();
            for (int g = tid; g < off * per_row; g += kThreads) {
                uint2* p = reinterpret_cast<uint2*>(codes + g * 8);
                uint2 w = *p;
                // code * old has 31 bits and its quotient by scale no tie that 53 bits could miss
                const auto again = [&](float c) {
                    return finite ? round_odd(static_cast<double>(c) * old / scale) : 0.0f;
                };
                w.x = to_codes<TYPE>(again(code_value<TYPE, 0>(w.x)), again(code_value<TYPE, 1>(w.x)),
                                     again(code_value<TYPE, 2>(w.x)), again(code_value<TYPE, 3>(w.x)));
                w.y = to_codes<TYPE>(again(code_value<TYPE, 0>(w.y)), again(code_value<TYPE, 1>(w.y)),
                                     again(code_value<TYPE, 2>(w.y)), again(code_value<TYPE, 3>(w.y)));
                *p = w;
            }
        }
        codes += static_cast<int64_t>(off) * hd;  // rows of a page are contiguous
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int g = tid + j * kThreads;
            if (g < groups) put8<TYPE>(codes + g * 8, x[j], scale, inv);
        }
        for (int g = tid + kHeld * kThreads; g < groups; g += kThreads) {
            float y[8];
            load8<IN, VEC>(src, at0 + (g / per_row) * a.ld + (g % per_row) * 8, y);
            put8<TYPE>(codes + g * 8, y, scale, inv);
        }
        if (tid == 0) *scale_at = scale;
    }
}

template <int TYPE, int IN>
int store_launch(const StoreArgs& a, bool vec, dim3 grid, hipStream_t s) {
    return vec ? launch(store_q8_kernel<TYPE, IN, true>, grid, dim3(kThreads), 0, s, a)
               : launch(store_q8_kernel<TYPE, IN, false>, grid, dim3(kThreads), 0, s, a);
}

}  // namespace
}  // namespace fence

extern "C" int fence_store_kv_q8(const fence_kv_pages* cache, const void* k, const void* v, int type, int64_t ld,
                                 const int32_t* slots, int64_t tokens, hipStream_t stream) {
    using namespace fence;
    if (!kv_pages_ok(cache) || !k || !v || !slots || tokens < 0 || tokens > INT32_MAX)
        return FENCE_ERROR_INVALID_VALUE;
    if (type != FENCE_F32 && type != FENCE_F16) return FENCE_ERROR_INVALID_VALUE;
    const size_t size = type == FENCE_F32 ? 4 : 2;
    if (!aligned(k, size) || !aligned(v, size) || !aligned(slots, 4)) return FENCE_ERROR_INVALID_VALUE;
    if (ld < static_cast<int64_t>(cache->n_kv_heads) * cache->head_dim || ld > INT64_MAX / 8 / (tokens + 1))
        return FENCE_ERROR_INVALID_VALUE;
    if (tokens == 0) return FENCE_SUCCESS;
    const bool vec = aligned(k, 16) && aligned(v, 16) && ld * size % 16 == 0;
    // Rows a workgroup looks at: one while the grid is small (single tokens, each on a page of its own), more
    // when most rows only continue a page and their workgroups would start for nothing.
    const int64_t all = tokens * cache->n_kv_heads * 2;
    int64_t window = all / 8192;
    window = window < 1 ? 1 : window > cache->page_size ? cache->page_size : window;
    const StoreArgs a{*cache, k, v, slots, ld, tokens, static_cast<int>(window), __builtin_ctz(cache->page_size)};
    const dim3 grid(grid_1d(tokens, window), cache->n_kv_heads, 2);
    if (cache->type == FENCE_KV_INT8)
        return type == FENCE_F32 ? store_launch<FENCE_KV_INT8, FENCE_F32>(a, vec, grid, stream)
                                 : store_launch<FENCE_KV_INT8, FENCE_F16>(a, vec, grid, stream);
    return type == FENCE_F32 ? store_launch<FENCE_KV_E4M3, FENCE_F32>(a, vec, grid, stream)
                             : store_launch<FENCE_KV_E4M3, FENCE_F16>(a, vec, grid, stream);
}
