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
// Where these are several short runs, as with single tokens, a wave each
// takes them: 512 rows of 512 sequences take 8.6 us and 2,048 take 19.4; with
// the workgroup on one after the other they take 15.8 and 53.
//
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
    // At which rows of the window a page's rows begin, and how many follow as far as a wave sees at once.
    const int64_t row = first + lane;
    const int mine = row < a.tokens ? a.slots[row] : -1;
    const int before = row < a.tokens && row > 0 ? a.slots[row - 1] : -1;
    const bool there = mine >= 0 && (mine >> a.page_shift) < a.c.n_pages;
    const bool goes_on = there && (mine & (page_size - 1)) != 0 && before == mine - 1;
    const uint64_t on = __ballot(goes_on);
    const uint64_t begin = __ballot(there && !goes_on && row < last);
    // Rows that follow the one at lane `at`, itself among them, as far as is seen.
    const auto run_of = [&](int at) {
        const uint64_t follow = at == kWave - 1 ? 0 : on >> (at + 1);
        return 1 + __builtin_ctzll(~follow);  // the bits shifted in are 0
    };
    int turn = 0;  // the two halves of wave_max take turns, so one barrier a page is enough

    // The rows of one page from the one at lane `at` on, n of them as far as was seen: by the whole workgroup, or
    // by one wave (SOLO).
    const auto page_rows = [&](int at, int n, auto solo) {
        constexpr bool SOLO = decltype(solo)::value;
        constexpr int T = SOLO ? kWave : kThreads;
        const int me = SOLO ? lane : tid;
        const int64_t t = first + at;
        const int slot = __builtin_amdgcn_readlane(mine, at);
        const int off = slot & (page_size - 1);
        const int most = static_cast<int>(a.tokens - t < page_size - off ? a.tokens - t : page_size - off);
        if (at + n == kWave) {  // to the end of what was seen
            while (n < most) {
                const int i = n + lane;
                const uint64_t differ = __ballot(i >= most || a.slots[t + i] != slot + i);
                const int same = differ ? __builtin_ctzll(differ) : kWave;
                n += same;
                if (same < kWave) break;
            }
        }
        n = n < most ? n : most;
        const int groups = n * per_row;
        const int64_t at0 = t * a.ld + static_cast<int64_t>(head) * hd;
        const int64_t page = slot >> a.page_shift;
        float* scale_at = (is_v ? a.c.v_scale : a.c.k_scale) + page * a.c.n_kv_heads + head;
        const float old = off ? *scale_at : 0.0f;
        float x[kHeld][8];
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int g = me + j * T;
            if (g < groups) load8<IN, VEC>(src, at0 + (g / per_row) * a.ld + (g % per_row) * 8, x[j]);
        }
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (me + j * T < groups) m = max_bits(m, x[j]);
        for (int g = me + kHeld * T; g < groups; g += T) {  // a page of more than kHeld groups a lane
            float y[8];
            load8<IN, VEC>(src, at0 + (g / per_row) * a.ld + (g % per_row) * 8, y);
            m = max_bits(m, y);
        }
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const uint32_t o = __shfl_xor(m, d);
            m = m > o ? m : o;
        }
        if constexpr (!SOLO) {
            if (lane == 0) wave_max[turn][wave] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kThreads / kWave; ++w) m = m > wave_max[turn][w] ? m : wave_max[turn][w];
            turn ^= 1;
        }
        const float now = __builtin_bit_cast(float, m) / kCodeTop[TYPE];
        const float scale = old != old || now != now ? __builtin_nanf("") : old > now ? old : now;
        const float inv = 1.0f / scale;
        uint8_t* codes = static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) +
                         ((page * a.c.n_kv_heads + head) << a.page_shift) * hd;
        if (scale > old && off) {  // what the page held, at the new scale
            const bool finite = scale < __builtin_inff();
            for (int g = me; g < off * per_row; g += T) {
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
            const int g = me + j * T;
            if (g < groups) put8<TYPE>(codes + g * 8, x[j], scale, inv);
        }
        for (int g = me + kHeld * T; g < groups; g += T) {
            float y[8];
            load8<IN, VEC>(src, at0 + (g / per_row) * a.ld + (g % per_row) * 8, y);
            put8<TYPE>(codes + g * 8, y, scale, inv);
        }
        if (me == 0) *scale_at = scale;
    };

    // Several short runs (single tokens, small pages): a wave each.  The choice is the same in every wave.
    const int run = run_of(lane);
    const bool any_long = __any((begin >> lane & 1) && (lane + run == kWave || run * per_row > kHeld * kWave));
    if (__builtin_popcountll(begin) > 1 && !any_long) {
        int k = 0;
        for (uint64_t left = begin; left; left &= left - 1, ++k)
            if (k % (kThreads / kWave) == wave) {
                const int at = __builtin_ctzll(left);
                page_rows(at, run_of(at), std::true_type{});
            }
    } else {
        for (uint64_t left = begin; left; left &= left - 1) {
            const int at = __builtin_ctzll(left);
            page_rows(at, run_of(at), std::false_type{});
        }
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
    // Rows a workgroup looks at, 64 at most, which a wave sees at once: one while the grid is small (single tokens,
    // each on a page of its own), more when most rows only continue a page and their workgroups would start for
    // nothing.  8,001 rows of prompts take 18 us on a grid of 2,048 workgroups, 21 on one of 8,192 and 36 on 32,768.
    const int64_t all = tokens * cache->n_kv_heads * 2;
    int64_t window = all / 2048;
    window = window < 1 ? 1 : window > kWave ? kWave : window;
    const StoreArgs a{*cache, k, v, slots, ld, tokens, static_cast<int>(window), __builtin_ctz(cache->page_size)};
    const dim3 grid(grid_1d(tokens, window), cache->n_kv_heads, 2);
    if (cache->type == FENCE_KV_INT8)
        return type == FENCE_F32 ? store_launch<FENCE_KV_INT8, FENCE_F32>(a, vec, grid, stream)
                                 : store_launch<FENCE_KV_INT8, FENCE_F16>(a, vec, grid, stream);
    return type == FENCE_F32 ? store_launch<FENCE_KV_E4M3, FENCE_F32>(a, vec, grid, stream)
                             : store_launch<FENCE_KV_E4M3, FENCE_F16>(a, vec, grid, stream);
}
