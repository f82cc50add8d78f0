// sample.hip -- sampling with temperature, top-k, top-p and min-p from given
// random numbers, on gfx950.
//
// In the order of falling logits (the lowest index first among equals) every
// filter keeps a beginning, and the draw is the place where a running sum
// passes a target, so all that is ever asked is at which element a running
// count or sum reaches a number.  Weights are exp((x - max) / T) in 64 bits,
// rounded to whole multiples of 2^-shift: their sums are exact in 64-bit
// integers in any order, so histograms by atomics give the same result every
// time, and a sum over a whole vocabulary stays exact enough that tokens next
// to a border fall on the right side.
//
// A call is four launches over workgroups that find out on the device what is
// left to do:
//   1. sample_scan: a thread takes a few dozen logits of a row and leaves their
//      maximum and, where a filter or the draw is about the whole row, the
//      sum of their weights relative to that maximum.
//   2. sample_list, a workgroup a row: the row's maximum; a bound that as many
//      of the threads' maxima reach as top-k asks for (or kTopThreads); the
//      logits above it, out of those threads' alone, sorted and summed; the
//      filters and the draw from the sums.  Peaked rows and any top-k up to
//      kListK end here, having read the row once.
//   3. sample_histogram, for the rows that are left (flat ones): weights and
//      counts by distance from the maximum.
//   4. sample_flat: the bins in which the borders of the filters and the draw
//      can lie; their elements are listed by all of a row's workgroups, and
//      the last to come sorts and answers.  If they are too many for a list,
//      one workgroup takes one question after the other, to one bin and, where
//      that is too many as well, by the digits of its elements' keys.
//
// Bound by the latency of these steps, not by bytes: one row of 151,936 with
// top-k 20 takes 2.9 + 10.4 us (scan, list) and 3 to 6 of the two launches that
// find nothing to do; 32 rows of 128,256 with top-p take 8.8 + 22.7 + 13.4 +
// 32.5 us; 256 rows of 151,936 with mixed filters 35 (4.4 TB/s) + 25.6 + 23 +
// 42.
#include "common.hpp"

namespace fence {
namespace {

constexpr int kThreads = 1024;  // of a workgroup that has a row
constexpr int kWaves = kThreads / kWave;
constexpr int kScanThreads = 256;
constexpr int kListK = 1024;       // largest top-k that the bound from the threads' maxima serves
constexpr int kTopThreads = 320;   // threads whose maxima bound the list without a top-k
constexpr int kList = 4096;        // elements a list holds
constexpr int kBins = 4096;        // of the histogram; the last one takes everything further away
constexpr int kMaxVocab = 1 << 26; // so that a row's threads can be counted in 21 bits
constexpr float kReach = 24.0f;    // how far below the maximum the histogram reaches, in units of T
typedef unsigned long long u64;

struct RowState {  // from sample_list to the launches behind it
    uint32_t top;  // the maximum's key
    uint32_t flat; // whether anything is left to do
    u64 mass;      // the whole row's weight
    uint32_t n, arrived;  // sample_flat: what its workgroups have listed, and how many have
};

struct SampleArgs {
    int32_t* out;
    const float* x;
    int64_t ld;
    int vocab, shift;
    int slots;  // threads of sample_scan a row has
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    // workspace, per row
    double* slot_mass;    // [slots]
    u64* bin_mass;        // [kBins]
    u64* list;            // [kList]
    RowState* state;
    uint32_t* slot_top;   // [slots]
    uint32_t* bin_count;  // [kBins]
};

// Unsigned keys that order like the logits; NaN as -inf, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    x = x != x ? -__builtin_inff() : x + 0.0f;
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kKeyLowest = 0x007FFFFFu;  // of -inf

// 2^y in 64 bits for y <= 0: 2^f for |f| <= 1/2 by the Taylor series of
// e^(f ln 2), whose first term left out is below 2^-50 of it.
__device__ __forceinline__ double exp2_64(double y) {
    y = y > -1100.0 ? y : -1100.0;
    const double n = rint(y);
    const double f = (y - n) * 0.693147180559945309417;
    double p = 1.0 / 39916800.0;
    p = fma(p, f, 1.0 / 3628800.0);
    p = fma(p, f, 1.0 / 362880.0);
    p = fma(p, f, 1.0 / 40320.0);
    p = fma(p, f, 1.0 / 5040.0);
    p = fma(p, f, 1.0 / 720.0);
    p = fma(p, f, 1.0 / 120.0);
    p = fma(p, f, 1.0 / 24.0);
    p = fma(p, f, 1.0 / 6.0);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    return ldexp(p, static_cast<int>(n));
}

// The same to about 3e-10, for the many: 2^y = 2^n 2^(j/64) e^r with |r| <=
// ln 2 / 128, the middle factor from a table in LDS and e^r - 1 in 32 bits,
// where its rounding is 2^-24 of 0.0054.  A third of the other's time.
constexpr int kTable = 64;
__device__ __forceinline__ void fill_table(double* table) {
    if (threadIdx.x < kTable) table[threadIdx.x] = 2.0 * exp2_64(threadIdx.x * (1.0 / kTable) - 1.0);
}
__device__ __forceinline__ double exp2_table(double y, const double* table) {
    y = y > -1000.0 ? y : -1000.0;
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    const double z = fma(y, static_cast<double>(kTable), kRound);
    const int n = static_cast<int>(__builtin_bit_cast(u64, z));
    const float r = static_cast<float>(fma(z - kRound, -1.0 / kTable, y)) * 0.693147182464599609375f;
    const float e = r + r * r * (0.5f + r * (0.16666667f + r * 0.041666668f));
    const double t = table[n & (kTable - 1)];
    return ldexp(fma(t, static_cast<double>(e), t), n >> 6);
}

struct Params {
    int k;        // 0: no top-k
    float top_p;  // at least 1: none
    float least;  // 0: no min-p
    float u;
    float t;
    bool greedy;
    __device__ __forceinline__ Params(const SampleArgs& a, int64_t r) {
        t = a.temperature ? a.temperature[r] : 1.0f;
        greedy = !(t > 0.0f);
        k = a.top_k ? a.top_k[r] : 0;
        if (k <= 0 || k >= a.vocab) k = 0;
        top_p = a.top_p ? a.top_p[r] : 1.0f;
        if (!(top_p < 1.0f)) top_p = 1.0f;
        const float m = a.min_p ? a.min_p[r] : 0.0f;
        least = m > 0.0f ? (m < 1.0f ? m : 1.0f) : 0.0f;
        u = a.u[r];
    }
    __device__ __forceinline__ bool use_p() const { return top_p < 1.0f; }
    // a list of the largest k logits answers everything
    __device__ __forceinline__ bool by_k(const SampleArgs& a) const { return k && k <= kListK && 2 * k <= a.slots; }
};

// ------------------------------------------------------------------ 1. scan

// E float4s a thread: which logits slot `slot` of a row has.
__device__ __forceinline__ int64_t slot_first(int slot, int e, int j) {
    return 4 * ((static_cast<int64_t>(slot / kScanThreads) * e + j) * kScanThreads + slot % kScanThreads);
}

// Four logits from index i on; -inf behind the last.
__device__ __forceinline__ f4 load4(const float* x, int64_t i, int n, bool wide) {
    if (wide && i + 4 <= n) return *reinterpret_cast<const f4*>(x + i);
    f4 v;
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = i + c < n ? x[i + c] : -__builtin_inff();
    return v;
}

template <int E>
__global__ __launch_bounds__(kScanThreads) void sample_scan(SampleArgs a) {
    __shared__ double table[kTable];
    const int64_t r = blockIdx.y;
    const int slot = blockIdx.x * kScanThreads + threadIdx.x;
    const float* x = a.x + r * a.ld;
    const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0;
    f4 v[E];
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = load4(x, slot_first(slot, E, j), a.vocab, wide);
    const Params par(a, r);
    const bool weigh = !par.greedy && !par.by_k(a);
    if (weigh) {
        fill_table(table);
        __syncthreads();
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < E; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t key = key_of(v[j][c]);
            top = key > top ? key : top;
        }
    a.slot_top[r * a.slots + slot] = top;
    if (!weigh) return;
    const double rate = 1.4426950408889634074 / static_cast<double>(par.t);
    const double ref = static_cast<double>(of_key(top));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < E; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            // behind the last logit and NaN: weight 0, unless all is -inf, which weighs nothing in the row
            const float y = v[j][c];
            if (key_of(y) == top) sum += 1.0;
            else if (y > -__builtin_inff()) sum += exp2_table((static_cast<double>(y) - ref) * rate, table);
        }
    a.slot_mass[r * a.slots + slot] = sum;
}

// ------------------------------------------------------------------ what the others share

struct Shared {
    u64 mass[kBins];
    uint32_t count[kBins];
    u64 list[kList];  // key << 32 | ~index: larger comes first
    double table[kTable];
    u64 wave[kWaves], wave2[kWaves];
    u64 found[4];
    int bin[8];  // a place for each of the bins that Borders looks for
    uint32_t n;
};

// A row and its weights.
struct Row {
    const float* x;
    int n;
    bool wide;
    uint32_t top;    // the maximum's key
    float top_value;
    double rate;     // log2(e) / T
    double one;      // 2^shift
    float bins_per;  // histogram bins per unit of logit

    __device__ __forceinline__ Row(const SampleArgs& a, int64_t r, float t, uint32_t top_key) {
        x = a.x + r * a.ld;
        n = a.vocab;
        wide = reinterpret_cast<uintptr_t>(x) % 16 == 0;
        top = top_key;
        top_value = of_key(top);
        rate = 1.4426950408889634074 / static_cast<double>(t);
        one = ldexp(1.0, a.shift);
        const float per = static_cast<float>(kBins) / kReach / t;
        bins_per = per < 3e38f ? per : 3e38f;
    }
    // f(logit, index) for every one, THREADS of a workgroup from float4 `from` to `to`; AHEAD loads a thread in
    // flight, which the compiler would not move over what f does.
    template <int THREADS, class F>
    __device__ __forceinline__ void each(int64_t from, int64_t to, F f) const {
        constexpr int AHEAD = 8;
        for (int64_t i0 = from + threadIdx.x; i0 < to; i0 += AHEAD * THREADS) {
            f4 v[AHEAD];
            if (wide && 4 * (i0 + (AHEAD - 1) * THREADS) + 4 <= n) {
#pragma unroll
                for (int d = 0; d < AHEAD; ++d) v[d] = *reinterpret_cast<const f4*>(x + 4 * (i0 + d * THREADS));
            } else {
#pragma unroll
                for (int d = 0; d < AHEAD; ++d) v[d] = load4(x, 4 * (i0 + d * THREADS), n, wide);
            }
#pragma unroll
            for (int d = 0; d < AHEAD; ++d) {
                const int64_t i = i0 + d * THREADS;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i < to && 4 * i + j < n) f(v[d][j], static_cast<int>(4 * i + j));
            }
        }
    }
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        each<kThreads>(0, (static_cast<int64_t>(n) + 3) / 4, f);
    }
    __device__ __forceinline__ double weight(uint32_t key) const {
        if (key == top) return 1.0;
        return exp2_64((static_cast<double>(of_key(key)) - static_cast<double>(top_value)) * rate);
    }
    __device__ __forceinline__ u64 units(uint32_t key) const { return static_cast<u64>(rint(weight(key) * one)); }
    __device__ __forceinline__ u64 units(uint32_t key, const double* table) const {
        if (key == top) return static_cast<u64>(one);
        return static_cast<u64>(
            rint(exp2_table((static_cast<double>(of_key(key)) - static_cast<double>(top_value)) * rate, table) * one));
    }
    // never falls as the key does: the order of bins is the order of elements
    __device__ __forceinline__ int bin(uint32_t key) const {
        if (key == top) return 0;
        const float d = (top_value - of_key(key)) * bins_per;
        return d < static_cast<float>(kBins - 1) ? static_cast<int>(d) : kBins - 1;
    }
    // Logits that a bin's elements lie between, with room for the rounding of bin(): two comparisons a logit leave
    // few for the exact test.  NaN passes.
    __device__ __forceinline__ void bin_range(int b, float* least, float* most) const {
        const float room = fabsf(top_value) * 0x1p-20f + 2.0f / bins_per;
        *most = top_value - static_cast<float>(b) / bins_per + room;
        *least = b == kBins - 1 ? -__builtin_inff() : top_value - static_cast<float>(b + 1) / bins_per - room;
        if (top_value == __builtin_inff()) *least = -__builtin_inff(), *most = __builtin_inff();
    }
    // a bin that no element weighing w is more than one away from
    __device__ __forceinline__ int bin_of_weight(float w, float t) const {
        const float d = -logf(w) * t * bins_per;
        return d < static_cast<float>(kBins - 1) ? static_cast<int>(d) : kBins - 1;
    }
};

// Inclusive sums of two numbers over the workgroup's threads, and their totals.
__device__ __forceinline__ void block_scan2(Shared& s, u64& v, u64& w, u64* v_total, u64* w_total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const u64 v_up = __shfl_up(v, d), w_up = __shfl_up(w, d);
        if (lane >= d) v += v_up, w += w_up;
    }
    __syncthreads();
    if (lane == kWave - 1) s.wave[wave] = v, s.wave2[wave] = w;
    __syncthreads();
    u64 v_before = 0, w_before = 0;
    *v_total = *w_total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i < wave) v_before += s.wave[i], w_before += s.wave2[i];
        *v_total += s.wave[i];
        *w_total += s.wave2[i];
    }
    v += v_before;
    w += w_before;
}

// Inclusive sum over the workgroup's threads and its total.
__device__ __forceinline__ u64 block_scan(Shared& s, u64 v, u64* total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const u64 up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    __syncthreads();
    if (lane == kWave - 1) s.wave[wave] = v;
    __syncthreads();
    u64 before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += s.wave[w];
        sum += s.wave[w];
    }
    *total = sum;
    return before + v;
}

__device__ __forceinline__ u64 block_max(Shared& s, u64 v) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const u64 o = __shfl_xor(v, d);
        v = v > o ? v : o;
    }
    __syncthreads();
    if (lane == 0) s.wave[wave] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v = v > s.wave[w] ? v : s.wave[w];
    return v;
}

__device__ __forceinline__ void append(Shared& s, uint32_t key, int index) {
    const uint32_t at = atomicAdd(&s.n, 1u);
    if (at < kList) s.list[at] = static_cast<u64>(key) << 32 | static_cast<uint32_t>(~index);
}

// The value of lane ^ J, in the vector ALU: within rows of 16 lanes by DPP,
// across them by the swaps of rows.
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    if constexpr (J == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);       // quad_perm 1,0,3,2
    else if constexpr (J == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);  // quad_perm 2,3,0,1
    else if constexpr (J == 4)  // the mirror of 8 lanes (^7), then of 4 (^3)
        return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true), 0x1B, 0xF, 0xF, true);
    else if constexpr (J == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, true);  // row_ror:8
    else return static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), J));
}
template <int J>
__device__ __forceinline__ u64 lane_xor(u64 v) {
    return static_cast<u64>(lane_xor<J>(static_cast<uint32_t>(v >> 32))) << 32 | lane_xor<J>(static_cast<uint32_t>(v));
}

// One step of a bitonic network among a wave's lanes and those below it: `falls`: the part of the network that this
// place is in puts the larger ones first.
template <int J>
__device__ __forceinline__ void lane_steps(u64& v, int at, bool falls) {
    const u64 o = lane_xor<J>(v);
    v = (o > v) == (((at & J) == 0) == falls) ? o : v;
    if constexpr (J > 1) lane_steps<J / 2>(v, at, falls);
}
template <int K>
__device__ __forceinline__ void sort_lanes(u64& v, int at) {
    if constexpr (K > 2) sort_lanes<K / 2>(v, at);
    lane_steps<K / 2>(v, at, (at & K) == 0);
}

// The first n entries of the list in falling order: a bitonic network over the
// next power of two, filled up with zeros, which come last.  Up to one entry a
// thread the entries stay in registers and only exchanges across waves go
// through LDS and a barrier (10 of 55 steps for 1024 entries).
__device__ __forceinline__ void sort_list(Shared& s, int n) {
    int size = kWave;
    while (size < n) size *= 2;
    const int tid = threadIdx.x;
    if (size <= kThreads) {
        u64 v = tid < n ? s.list[tid] : 0;
        if (tid < size) sort_lanes<kWave>(v, tid);
        for (int k = 2 * kWave; k <= size; k *= 2) {
            const bool falls = (tid & k) == 0;
            for (int j = k / 2; j >= kWave; j /= 2) {
                __syncthreads();
                if (tid < size) s.list[tid] = v;
                __syncthreads();
                const u64 o = tid < size ? s.list[tid ^ j] : 0;
                v = (o > v) == (((tid & j) == 0) == falls) ? o : v;  // this place keeps the larger or the smaller one
            }
            if (tid < size) lane_steps<kWave / 2>(v, tid, falls);
        }
        __syncthreads();
        if (tid < size) s.list[tid] = v;
        __syncthreads();
        return;
    }
    for (int i = n + tid; i < size; i += kThreads) s.list[i] = 0;
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            for (int i = tid; i < size / 2; i += kThreads) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const u64 x = s.list[a], y = s.list[b];
                if ((x < y) == ((a & k) == 0)) s.list[a] = y, s.list[b] = x;
            }
        }
    __syncthreads();
}

// Running sums over the sorted list, `per` consecutive entries a thread.
constexpr int kPer = kList / kThreads;
struct Sums {
    u64 upto[kPer];  // inclusive
    u64 before;      // this thread's first
    int per, n;
    __device__ __forceinline__ Sums(Shared& s, const Row& row, int count) : n(count) {
        per = (n + kThreads - 1) / kThreads;
        u64 mine = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = threadIdx.x * per + j;
            if (j < per && i < n) mine += row.units(static_cast<uint32_t>(s.list[i] >> 32));
            upto[j] = mine;
        }
        u64 total;
        before = block_scan(s, mine, &total) - mine;
#pragma unroll
        for (int j = 0; j < kPer; ++j) upto[j] += before;
    }
    // the sum at place i < n
    __device__ __forceinline__ u64 at(Shared& s, int i) const {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (j < per && static_cast<int>(threadIdx.x) * per + j == i) s.found[1] = upto[j];
        __syncthreads();
        return s.found[1];
    }
    // the first place whose sum reaches goal, or n - 1
    __device__ __forceinline__ int reaches(Shared& s, u64 goal) const {
        __syncthreads();
        if (threadIdx.x == 0) s.found[0] = n - 1;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; ++j) {  // one place at most: sums never fall
            const int i = threadIdx.x * per + j;
            if (j < per && i < n && upto[j] >= goal && (j ? upto[j - 1] : before) < goal) s.found[0] = i;
        }
        __syncthreads();
        return static_cast<int>(s.found[0]);
    }
};

// u times a sum, rounded down: the running sum has to be above it.
__device__ __forceinline__ u64 draw_goal(float u, u64 mass) {
    u = u > 0.0f ? u : 0.0f;
    const u64 goal = static_cast<u64>(static_cast<double>(u) * static_cast<double>(mass)) + 1;
    return goal < mass ? goal : mass > 0 ? mass : 1;  // u = 1 and above: the last one
}

__device__ __forceinline__ u64 top_p_goal(float p, u64 mass) {
    p = p > 0.0f ? p : 0.0f;
    const u64 goal = static_cast<u64>(ceil(static_cast<double>(p) * static_cast<double>(mass)));
    return goal < 1 ? 1 : goal < mass ? goal : mass;
}

// ------------------------------------------------------------------ 2. lists

// The answer from a list of up to 64 logits with the largest k among them: one
// wave, an entry a lane, without a barrier.
__device__ __forceinline__ void short_list(Shared& s, const SampleArgs& a, int64_t r, const Row& row, const Params& par, int n) {
    const int lane = threadIdx.x;
    u64 v = lane < n ? s.list[lane] : 0;
    sort_lanes<kWave>(v, lane);
    const double w = lane < par.k ? row.weight(static_cast<uint32_t>(v >> 32)) : 0.0;
    u64 upto = static_cast<u64>(rint(w * row.one));
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const u64 up = __shfl_up(upto, d);
        if (lane >= d) upto += up;
    }
    int keep = par.k;  // at most n
    if (par.use_p()) {
        const u64 goal = top_p_goal(par.top_p, __shfl(upto, kWave - 1));
        keep = __builtin_ctzll(__ballot(upto >= goal)) + 1;
        if (keep > par.k) keep = par.k;
    }
    if (par.least > 0.0f) {
        const int passing = __builtin_popcountll(__ballot(lane < keep && w >= static_cast<double>(par.least)));
        keep = passing < 1 ? 1 : passing;
    }
    const u64 goal = draw_goal(par.u, __shfl(upto, keep - 1));
    const int at = __builtin_ctzll(__ballot(upto >= goal));
    if (lane == at) a.out[r] = static_cast<int>(~static_cast<uint32_t>(v));
}

template <int E>
__global__ __launch_bounds__(kThreads) void sample_list(SampleArgs a) {
    __shared__ Shared s;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    const Params par(a, r);
    const uint32_t* tops = a.slot_top + r * a.slots;
    // the threads' maxima, the first kKept a thread in registers (a row of up to 320,000 logits)
    constexpr int kKept = 8;
    uint32_t kept_tops[kKept], best = 0;
#pragma unroll
    for (int j = 0; j < kKept; ++j) kept_tops[j] = tid + j * kThreads < a.slots ? tops[tid + j * kThreads] : 0;
    const auto each_top = [&](auto f) {
#pragma unroll
        for (int j = 0; j < kKept; ++j)
            if (j * kThreads < a.slots) f(kept_tops[j], tid + j * kThreads);
        for (int i = tid + kKept * kThreads; __any(i < a.slots); i += kThreads) f(i < a.slots ? tops[i] : 0, i);
    };
    each_top([&](uint32_t t, int) { best = t > best ? t : best; });
    const uint32_t top = static_cast<uint32_t>(block_max(s, best));
    if (tid == 0) a.state[r] = RowState{top, 0, 0, 0, 0};
    if (top <= kKeyLowest) {
        if (tid == 0) a.out[r] = 0;
        return;
    }
    const Row row(a, r, par.greedy ? 1.0f : par.t, top);

    u64 mass = 0;
    if (!par.greedy && !par.by_k(a)) {  // the whole row's weight
        const double* slot_mass = a.slot_mass + r * a.slots;
        u64 v = 0;
        each_top([&](uint32_t t, int i) {
            if (i < a.slots) v += static_cast<u64>(rint(slot_mass[i] * row.weight(t) * row.one));
        });
        block_scan(s, v, &mass);
    }
    // A bound that `want` of the threads' maxima reach, to 16 bits of the key.
    uint32_t bound = 0;
    const bool all = a.vocab <= kList && !par.greedy;
    const int want = par.by_k(a) ? par.k : kTopThreads < a.slots / 2 ? kTopThreads : a.slots / 2;
    if (par.greedy) {
        bound = top;
    } else if (!all) {
        if (2 * want <= (a.slots < kThreads ? a.slots : kThreads)) {
            // Out of each thread's largest alone, a somewhat lower bound for a fraction of the work: by one wave, that
            // keeps all of them in registers and needs no barrier, 2 us where the whole workgroup takes 6.
            uint32_t* bests = reinterpret_cast<uint32_t*>(s.list);
            bests[tid] = best;
            __syncthreads();
            if (tid < kWave) {
                uint32_t t[kWaves];
#pragma unroll
                for (int w = 0; w < kWaves; ++w) t[w] = bests[w * kWave + tid];
                for (int bit = 31; bit >= 16; --bit) {
                    const uint32_t least = bound | 1u << bit;
                    int n = 0;  // the same in every lane
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) n += __builtin_popcountll(__ballot(t[w] >= least));
                    if (n >= want) bound = least;
                }
                if (tid == 0) s.n = bound;
            }
            __syncthreads();
            bound = s.n;
        } else {
            int turn = 0;  // the two halves of s.list take turns, so one barrier a turn is enough
            for (int bit = 30; bit >= 16; bit -= 2) {  // two bits a turn
                uint32_t c[3] = {0, 0, 0};             // the same in every lane
                each_top([&](uint32_t t, int) {
#pragma unroll
                    for (int j = 0; j < 3; ++j)
                        c[j] += __builtin_popcountll(__ballot(t >= (bound | static_cast<uint32_t>(j + 1) << bit)));
                });
                u64* sums = s.list + turn * kWaves;
                if (tid % kWave == 0) sums[tid / kWave] = c[0] | static_cast<u64>(c[1]) << 21 | static_cast<u64>(c[2]) << 42;
                __syncthreads();
                u64 sum = 0;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) sum += sums[w];
                turn ^= 1;
                for (int j = 2; j >= 0; --j)
                    if (static_cast<int>(sum >> (21 * j) & 0x1FFFFF) >= want) {
                        bound |= static_cast<uint32_t>(j + 1) << bit;
                        break;
                    }
            }
        }
    }
    // The logits above it, out of the threads' that have one; s.mass holds those threads' numbers meanwhile.
    uint32_t* slots = reinterpret_cast<uint32_t*>(s.mass);
    constexpr int kSlots = kBins * 2;
    __syncthreads();
    if (tid == 0) s.n = 0, s.found[2] = 0, s.found[3] = ~0ull;
    __syncthreads();
    each_top([&](uint32_t t, int i) {
        if (t >= bound && i < a.slots) {
            const uint32_t at = static_cast<uint32_t>(atomicAdd(&s.found[2], 1ull));
            if (at < kSlots) slots[at] = i;
        }
    });
    __syncthreads();
    const uint32_t named = static_cast<uint32_t>(s.found[2]);
    bool listed = named <= kSlots;
    if (listed || par.greedy) {
        const int64_t work = static_cast<int64_t>(listed ? named : a.slots) * E;
        u64 lowest = ~0ull;
        constexpr int AHEAD = 4;
        for (int64_t w0 = tid; w0 < work; w0 += AHEAD * kThreads) {
            f4 v[AHEAD];
            int64_t at[AHEAD];
#pragma unroll
            for (int d = 0; d < AHEAD; ++d) {
                const int64_t w = w0 + d * kThreads;
                const int slot = w >= work ? 0 : listed ? slots[w / E] : static_cast<int>(w / E);
                at[d] = w < work ? slot_first(slot, E, static_cast<int>(w % E)) : row.n;
                v[d] = load4(row.x, at[d], row.n, row.wide);
            }
#pragma unroll
            for (int d = 0; d < AHEAD; ++d)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t key = key_of(v[d][c]);
                    if (key < bound || at[d] + c >= row.n) continue;
                    if (par.greedy) lowest = lowest < static_cast<u64>(at[d] + c) ? lowest : static_cast<u64>(at[d] + c);
                    else append(s, key, static_cast<int>(at[d] + c));
                }
        }
        if (par.greedy) {
            const u64 first = ~block_max(s, ~lowest);
            if (tid == 0) a.out[r] = static_cast<int>(first);
            return;
        }
        __syncthreads();
        listed = s.n <= kList;
    }
    if (listed) {
        const int n = static_cast<int>(s.n);
        if (n <= kWave && par.by_k(a)) {
            if (tid < kWave) short_list(s, a, r, row, par, n);
            return;
        }
        sort_list(s, n);
        const Sums sums(s, row, n);
        const u64 held = sums.at(s, n - 1);
        const bool complete = n == row.n;
        // The filters, as long as the list holds what they keep.
        bool known = true;
        int keep = n;
        u64 kept = complete ? held : mass;
        if (par.k) {
            known = par.k <= n;
            if (known) keep = par.k, kept = sums.at(s, keep - 1);
        }
        if (known && par.use_p()) {
            const u64 goal = top_p_goal(par.top_p, kept);
            known = goal <= held || complete;
            const int at = sums.reaches(s, goal);
            if (known && at + 1 <= keep) keep = at + 1, kept = sums.at(s, at);
        }
        if (par.least > 0.0f && (known || !par.k || !par.use_p())) {
            // An element past the end of the list weighs no more than its last one.  (With both top-k and top-p
            // the weight that top-p is about has to be known first.)
            int passing = 0;
            for (int i = tid; i < keep; i += kThreads)
                passing += row.weight(static_cast<uint32_t>(s.list[i] >> 32)) >= static_cast<double>(par.least);
            u64 total;
            block_scan(s, static_cast<u64>(passing), &total);
            if (static_cast<int>(total) < n || complete) {
                known = true;
                keep = total < 1 ? 1 : static_cast<int>(total);
                kept = sums.at(s, keep - 1);
            } else {
                known = known && (par.k || par.use_p());
            }
        }
        if (known) {
            const u64 goal = draw_goal(par.u, kept);
            if (goal <= held || complete) {
                const int at = sums.reaches(s, goal);
                if (tid == 0) a.out[r] = static_cast<int>(~static_cast<uint32_t>(s.list[at]));
                return;
            }
        }
    }
    // Not here: a histogram, from zero.
    if (tid == 0) a.state[r] = RowState{top, 1, mass, 0, 0};
    for (int i = tid; i < kBins; i += kThreads) a.bin_mass[r * kBins + i] = 0, a.bin_count[r * kBins + i] = 0;
}

// ------------------------------------------------------------------ 3. histograms

// A thread's share of the last bin, which takes most of a peaked row, stays in
// registers: not through one address.
__global__ __launch_bounds__(kThreads) void sample_histogram(SampleArgs a, int64_t chunk) {
    __shared__ u64 mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ double table[kTable];
    const int64_t r = blockIdx.y;
    const RowState state = a.state[r];
    if (!state.flat) return;
    const Params par(a, r);
    const Row row(a, r, par.t, state.top);
    fill_table(table);
    for (int i = threadIdx.x; i < kBins; i += kThreads) mass[i] = 0, count[i] = 0;
    __syncthreads();
    u64 last_mass = 0;
    uint32_t last_count = 0;
    const int64_t n4 = (static_cast<int64_t>(row.n) + 3) / 4;
    const int64_t from = blockIdx.x * chunk, to = from + chunk < n4 ? from + chunk : n4;
    row.each<kThreads>(from, to, [&](float x, int) {
        const uint32_t key = key_of(x);
        const int b = row.bin(key);
        const u64 w = row.units(key, table);
        if (b == kBins - 1) {
            last_mass += w;
            ++last_count;
        } else {
            atomicAdd(&mass[b], w);
            atomicAdd(&count[b], 1u);
        }
    });
    if (last_count) {
        atomicAdd(&mass[kBins - 1], last_mass);
        atomicAdd(&count[kBins - 1], last_count);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads)
        if (count[i]) {
            atomicAdd(&a.bin_mass[r * kBins + i], mass[i]);
            atomicAdd(&a.bin_count[r * kBins + i], count[i]);
        }
}

// ------------------------------------------------------------------ 4. flat rows

// The running sums over s's bins, and the bin in which they reach a goal.
struct BinSums {
    static constexpr int kEach = kBins / kThreads;
    u64 m[kEach], c[kEach], m0, c0;  // of this thread's bins, and of those before them
    u64 masses, counts;              // of all

    __device__ __forceinline__ explicit BinSums(Shared& s) {
        u64 mm = 0, cc = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            mm += m[j] = s.mass[threadIdx.x * kEach + j];
            cc += c[j] = s.count[threadIdx.x * kEach + j];
        }
        m0 = mm, c0 = cc;
        block_scan2(s, m0, c0, &masses, &counts);
        m0 -= mm, c0 -= cc;
    }
    // The bin in which a running sum reaches a goal, in s.bin[slot] behind the next barrier.
    __device__ __forceinline__ void leave(Shared& s, int slot, bool by_count, u64 goal) const {
        const u64 all = by_count ? counts : masses;
        goal = goal < all ? goal : all;
        u64 before = by_count ? c0 : m0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const u64 here = by_count ? c[j] : m[j];
            if (before < goal && before + here >= goal) s.bin[slot] = threadIdx.x * kEach + j;  // one bin: sums never fall
            before += here;
        }
    }
    // A goal past the last sum counts as the last one.
    __device__ __forceinline__ int find(Shared& s, bool by_count, u64 goal, u64* mass_before, u64* count_before) const {
        const u64 all = by_count ? counts : masses;
        goal = goal < all ? goal : all;
        u64 ms = m0, cs = c0;
        __syncthreads();
        if (threadIdx.x == 0) s.found[0] = s.found[1] = s.found[2] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const u64 before = by_count ? cs : ms, here = by_count ? c[j] : m[j];
            if (before < goal && before + here >= goal) {  // one bin at most: sums never fall
                s.found[0] = threadIdx.x * kEach + j;
                s.found[1] = ms;
                s.found[2] = cs;
            }
            ms += m[j];
            cs += c[j];
        }
        __syncthreads();
        *mass_before = s.found[1];
        *count_before = s.found[2];
        return static_cast<int>(s.found[0]);
    }
};

// The row's histogram by distance into s.
__device__ __forceinline__ void load_bins(Shared& s, const SampleArgs& a, int64_t r) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        s.mass[i] = a.bin_mass[r * kBins + i];
        s.count[i] = a.bin_count[r * kBins + i];
    }
    __syncthreads();
}

// At which element does the row's running sum of weights (or count) reach a
// number?
struct Place {
    int index;
    u64 mass;  // the running sum of weights there, inclusive
};

// For goal >= 1, from the histogram by distance.
__device__ __forceinline__ Place locate(Shared& s, const SampleArgs& a, int64_t r, const Row& row, bool by_count, u64 goal) {
    load_bins(s, a, r);
    u64 mass, count;
    const int b = BinSums(s).find(s, by_count, goal, &mass, &count);
    uint32_t lo = 0, hi = ~0u;  // keys that are left, both inclusive
    int left = static_cast<int>(s.count[b]);
    const auto in = [&](uint32_t k) { return k >= lo && k <= hi && row.bin(k) == b; };
    // too many for a list: their keys by 11 bits at a time, the larger digit first
    for (int bits = 32; left > kList && bits > 0;) {
        const int take = bits < 11 ? bits : 11;
        bits -= take;
        const uint32_t mask = (1u << take) - 1;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0, s.count[i] = 0;
        __syncthreads();
        row.each([&](float x, int) {
            const uint32_t key = key_of(x);
            if (!in(key)) return;
            const uint32_t d = mask - ((key >> bits) & mask);
            atomicAdd(&s.mass[d], row.units(key, s.table));
            atomicAdd(&s.count[d], 1u);
        });
        __syncthreads();
        u64 m, c;
        const u64 before = by_count ? count : mass;
        const int d = BinSums(s).find(s, by_count, goal > before ? goal - before : 1, &m, &c);
        mass += m;
        count += c;
        left = static_cast<int>(s.count[d]);
        lo |= (mask - static_cast<uint32_t>(d)) << bits;
        hi = lo | ((1u << bits) - 1);
    }
    Place p;
    const u64 before = by_count ? count : mass;
    const u64 rest = goal > before ? goal - before : 1;
    if (left <= kList) {
        __syncthreads();
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
        float least, most;
        row.bin_range(b, &least, &most);
        row.each([&](float x, int i) {
            if (x < least || x > most) return;
            const uint32_t key = key_of(x);
            if (in(key)) append(s, key, i);
        });
        __syncthreads();
        sort_list(s, left);
        const Sums sums(s, row, left);
        const int at = by_count ? static_cast<int>(rest < static_cast<u64>(left) ? rest : left) - 1 : sums.reaches(s, rest);
        p.mass = mass + sums.at(s, at);
        p.index = static_cast<int>(~static_cast<uint32_t>(s.list[at]));
    } else {
        // equal logits, more than a list holds: the n-th of them by index
        const u64 w = row.units(lo);
        u64 nth = by_count ? rest : w ? (rest + w - 1) / w : 1;
        if (nth > static_cast<u64>(left)) nth = left;
        const int64_t each = (static_cast<int64_t>(row.n) + kThreads - 1) / kThreads;
        const int64_t i0 = threadIdx.x * each, i1 = i0 + each < row.n ? i0 + each : row.n;
        u64 mine = 0, total;
        for (int64_t i = i0; i < i1; ++i) mine += key_of(row.x[i]) == lo;
        u64 at = block_scan(s, mine, &total) - mine;
        __syncthreads();
        if (at < nth && nth <= at + mine)
            for (int64_t i = i0; i < i1; ++i)
                if (key_of(row.x[i]) == lo && ++at == nth) {
                    s.found[3] = static_cast<u64>(i);
                    break;
                }
        __syncthreads();
        p.index = static_cast<int>(s.found[3]);
        p.mass = mass + nth * w;
    }
    __syncthreads();
    return p;
}

// A row's answer from one list.  The histogram says in which bins every
// border can lie: top-k's in one; top-p's in those that its goal falls into
// for the least and the most weight that top-k may leave; min-p's in three;
// the draw's in those for the least and the most weight that is left then.
// These bins' elements are listed, few as a rule, and with the sums of the
// bins between them every border and the draw come out of one sort.
struct Borders {
    static constexpr int kRanges = 4;
    int from[kRanges], to[kRanges];  // bins, apart from one another and rising; from > to: none
    int min_from, min_to;            // min-p's, none if it cannot matter
    u64 mass;                        // what top-k and the others start from
    bool fits;                       // the list holds all

    // Leaves s.mass and s.count as sums before each bin.
    __device__ __forceinline__ Borders(Shared& s, const SampleArgs& a, int64_t r, const Row& row, const Params& par,
                                       u64 row_mass) {
        load_bins(s, a, r);
        const BinSums bins(s);
        mass = par.by_k(a) ? bins.masses : row_mass;  // sample_scan summed nothing then: its list was too long for ties
        __syncthreads();
        u64 ms = bins.m0, cs = bins.c0;
#pragma unroll
        for (int j = 0; j < BinSums::kEach; ++j) {
            s.mass[threadIdx.x * BinSums::kEach + j] = ms;
            s.count[threadIdx.x * BinSums::kEach + j] = static_cast<uint32_t>(cs);
            ms += bins.m[j];
            cs += bins.c[j];
        }
        __syncthreads();
        const auto end = [&](int b) { return b == kBins - 1 ? bins.masses : s.mass[b + 1]; };
        const auto count_end = [&](int b) { return b == kBins - 1 ? bins.counts : s.count[b + 1]; };
        const u64 slack = (mass >> 28) + 1;  // weights in bins are off by 2^-31 of themselves
        const auto less = [&](u64 v) { return v > slack ? v - slack : 1; };
#pragma unroll
        for (int i = 0; i < kRanges; ++i) from[i] = kBins, to[i] = -1;
        u64 lo = mass, hi = mass;
        if (par.k) {
            bins.leave(s, 0, true, par.k);
            __syncthreads();
            from[0] = to[0] = s.bin[0];
            lo = s.mass[from[0]] + 1, hi = end(to[0]);
        }
        if (par.use_p()) {
            bins.leave(s, 1, false, less(top_p_goal(par.top_p, lo)));
            bins.leave(s, 2, false, top_p_goal(par.top_p, hi) + slack);
            __syncthreads();
            from[1] = s.bin[1], to[1] = s.bin[2];
            const u64 most = end(to[1]);
            lo = s.mass[from[1]] + 1 < lo ? s.mass[from[1]] + 1 : lo;
            hi = most < hi ? most : hi;
        }
        min_from = kBins, min_to = -1;
        if (par.least > 0.0f) {
            const int border = row.bin_of_weight(par.least, par.t);
            const int b0 = border > 0 ? border - 1 : 0, b1 = border < kBins - 1 ? border + 1 : border;
            if (s.mass[b0] < hi + slack) {
                from[2] = min_from = b0, to[2] = min_to = b1;
                const u64 before = s.mass[b0] + 1, most = end(b1);
                lo = before < lo ? before : lo;
                hi = most < hi ? most : hi;
            }
        }
        bins.leave(s, 3, false, less(draw_goal(par.u, lo)));
        bins.leave(s, 4, false, draw_goal(par.u, hi) + slack);
        __syncthreads();
        from[3] = s.bin[3], to[3] = s.bin[4];
        // in order, joined where they touch
#pragma unroll
        for (int i = 1; i < kRanges; ++i)
#pragma unroll
            for (int j = i; j > 0; --j)
                if (from[j] < from[j - 1]) {
                    const int f = from[j], t = to[j];
                    from[j] = from[j - 1], to[j] = to[j - 1];
                    from[j - 1] = f, to[j - 1] = t;
                }
#pragma unroll
        for (int i = 1; i < kRanges; ++i)
            if (to[i] >= 0 && from[i] <= to[i - 1] + 1) {
                from[i] = from[i - 1];
                to[i] = to[i] > to[i - 1] ? to[i] : to[i - 1];
                from[i - 1] = kBins, to[i - 1] = -1;
            }
        u64 n = 0;
#pragma unroll
        for (int i = 0; i < kRanges; ++i)
            if (to[i] >= 0) n += count_end(to[i]) - s.count[from[i]];
        fits = n <= kList;
    }
    __device__ __forceinline__ bool holds(int b) const {
        bool in = false;
#pragma unroll
        for (int i = 0; i < kRanges; ++i) in = in || (b >= from[i] && b <= to[i]);
        return in;
    }
};

// The answer from the listed elements, n of them in s.list.
__device__ __forceinline__ int from_borders(Shared& s, const Row& row, const Params& par, const Borders& borders, int n) {
    sort_list(s, n);
    // Running sums of weights and numbers, the bins between included.
    const int per = (n + kThreads - 1) / kThreads;
    u64 upto[kPer], place[kPer], mine = 0, places = 0, light = 0, total, unused;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = threadIdx.x * per + j;
        if (j < per && i < n) {
            const uint32_t key = static_cast<uint32_t>(s.list[i] >> 32);
            const int b = row.bin(key), last = i ? row.bin(static_cast<uint32_t>(s.list[i - 1] >> 32)) : -1;
            const double w = row.weight(key);
            const u64 units = static_cast<u64>(rint(w * row.one));
            if (b > last + 1) {  // between the bins: from the end of the one to the start of the other
                mine += s.mass[b] - s.mass[last + 1];
                places += s.count[b] - s.count[last + 1];
            }
            mine += units;
            ++places;
            if (b >= borders.min_from && b <= borders.min_to && w >= static_cast<double>(par.least)) light += units;
        }
        upto[j] = mine;
        place[j] = places;
    }
    u64 before = mine, placed = places;
    block_scan2(s, before, placed, &total, &unused);
    before -= mine, placed -= places;
#pragma unroll
    for (int j = 0; j < kPer; ++j) upto[j] += before, place[j] += placed;
    // the first element whose sum (or place) reaches goal, or the last: its index, and *sum
    const auto reaches = [&](const u64* sums, u64 first, u64 goal, u64* sum) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; ++j) {  // one at most reaches it first: sums never fall
            const int i = threadIdx.x * per + j;
            if (j < per && i < n && (j ? sums[j - 1] : first) < goal && (sums[j] >= goal || i == n - 1))
                s.found[0] = i, s.found[1] = upto[j];
        }
        __syncthreads();
        *sum = s.found[1];
        return static_cast<int>(s.found[0]);
    };
    u64 kept = borders.mass;
    if (par.k) reaches(place, placed, par.k, &kept);
    if (par.use_p()) reaches(upto, before, top_p_goal(par.top_p, kept), &kept);
    if (borders.min_to >= 0) {
        block_scan(s, light, &total);
        total += s.mass[borders.min_from];
        kept = total < kept ? total : kept;
    }
    const int at = reaches(upto, before, draw_goal(par.u, kept), &unused);
    return static_cast<int>(~static_cast<uint32_t>(s.list[at]));
}

__global__ __launch_bounds__(kThreads) void sample_flat(SampleArgs a, int64_t chunk) {
    __shared__ Shared s;
    const int64_t r = blockIdx.y;
    const RowState state = a.state[r];
    if (!state.flat) return;
    const Params par(a, r);
    const Row row(a, r, par.t, state.top);
    fill_table(s.table);
    __syncthreads();
    {
        const Borders borders(s, a, r, row, par, state.mass);
        if (borders.fits) {
            // A row's workgroups list their parts of it; the last to come answers.
            if (threadIdx.x == 0) s.n = 0;
            __syncthreads();
            const int64_t n4 = (static_cast<int64_t>(row.n) + 3) / 4;
            const int64_t from = blockIdx.x * chunk, to = from + chunk < n4 ? from + chunk : n4;
            row.each<kThreads>(from, to, [&](float x, int i) {
                const uint32_t key = key_of(x);
                if (borders.holds(row.bin(key))) append(s, key, i);
            });
            __syncthreads();
            int n = s.n < kList ? static_cast<int>(s.n) : kList;  // as the histogram counted them, never more
            if (gridDim.x > 1) {
                if (threadIdx.x == 0 && n)
                    s.found[2] = __hip_atomic_fetch_add(&a.state[r].n, static_cast<uint32_t>(n), __ATOMIC_RELAXED,
                                                        __HIP_MEMORY_SCOPE_AGENT);
                __syncthreads();
                u64* list = a.list + r * kList;
                for (int i = threadIdx.x; i < n; i += kThreads)
                    if (s.found[2] + i < kList)
                        __hip_atomic_store(list + s.found[2] + i, s.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                // every wave's stores have completed before the one arrival
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                if (threadIdx.x == 0) {
                    const uint32_t before = __hip_atomic_fetch_add(&a.state[r].arrived, 1u, __ATOMIC_RELAXED,
                                                                   __HIP_MEMORY_SCOPE_AGENT);
                    s.found[3] = before + 1 == gridDim.x;
                    s.n = __hip_atomic_load(&a.state[r].n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                if (!s.found[3]) return;
                n = s.n < kList ? static_cast<int>(s.n) : kList;
                for (int i = threadIdx.x; i < n; i += kThreads)
                    s.list[i] = __hip_atomic_load(list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __syncthreads();
            }
            const int index = from_borders(s, row, par, borders, n);
            if (threadIdx.x == 0) a.out[r] = index;
            return;
        }
    }
    // Lists too long for that: one question after the other, by one workgroup.
    if (blockIdx.x) return;
    u64 kept = state.mass;
    if (par.by_k(a)) {  // sample_scan summed nothing: its list was too long for ties
        u64 v = 0;
        for (int i = threadIdx.x; i < kBins; i += kThreads) v += a.bin_mass[r * kBins + i];
        block_scan(s, v, &kept);
    }
    if (par.k) kept = locate(s, a, r, row, true, par.k).mass;
    if (par.use_p()) {
        const u64 goal = top_p_goal(par.top_p, kept);
        kept = locate(s, a, r, row, false, goal).mass;
    }
    if (par.least > 0.0f) {
        // whole bins above the border's, and what weighs enough in the three about it
        const int border = row.bin_of_weight(par.least, par.t);
        u64 v = 0, total;
        for (int i = threadIdx.x; i < border - 1; i += kThreads) v += a.bin_mass[r * kBins + i];
        float least, most, unused;
        row.bin_range(border < kBins - 1 ? border + 1 : border, &least, &unused);
        row.bin_range(border > 0 ? border - 1 : 0, &unused, &most);
        row.each([&](float x, int) {
            if (x < least || x > most) return;
            const uint32_t key = key_of(x);
            const int b = row.bin(key);
            if (b >= border - 1 && b <= border + 1 && row.weight(key) >= static_cast<double>(par.least)) v += row.units(key);
        });
        block_scan(s, v, &total);
        kept = total < kept ? total : kept;
    }
    const Place p = locate(s, a, r, row, false, draw_goal(par.u, kept));
    if (threadIdx.x == 0) a.out[r] = p.index;
}

// ------------------------------------------------------------------ host

int shift_for(int vocab) {
    int bits = 1;
    while ((int64_t(1) << bits) < vocab) ++bits;
    return 62 - bits;  // the sum of vocab weights of at most 2^shift stays below 2^63
}

// float4s a thread of sample_scan takes: fewer while the grid would not fill the GPU.
int64_t wide_groups(int vocab) { return (static_cast<int64_t>(vocab) + 40 * kScanThreads - 1) / (40 * kScanThreads); }
int scan_width(int64_t rows, int vocab) { return rows * wide_groups(vocab) < 512 ? 5 : 10; }
int slots_of(int64_t rows, int vocab) {
    const int64_t per = 4ll * scan_width(rows, vocab) * kScanThreads;
    return static_cast<int>((vocab + per - 1) / per) * kScanThreads;
}

int64_t row_bytes(int slots) {
    return slots * static_cast<int64_t>(sizeof(double) + sizeof(uint32_t)) +
           kBins * static_cast<int64_t>(sizeof(u64) + sizeof(uint32_t)) + kList * static_cast<int64_t>(sizeof(u64)) +
           static_cast<int64_t>(sizeof(RowState));
}

}  // namespace
}  // namespace fence

extern "C" int64_t fence_sample_workspace(int64_t rows, int vocab) {
    using namespace fence;
    if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > kMaxVocab) return 0;
    // Rows that are few have twice the slots, so 34 rows of 151,936 need more than 46: what the most such rows need is
    // the least, and a workspace serves every smaller number of rows.
    const int64_t few = 511 / wide_groups(vocab) < rows ? 511 / wide_groups(vocab) : rows;
    const int64_t n = rows * row_bytes(slots_of(rows, vocab)), m = few * row_bytes(slots_of(few, vocab));
    return n > m ? n : m < 16 ? 16 : m;
}

extern "C" int fence_sample(int32_t* out, const float* logits, int64_t rows, int vocab, int64_t ld,
                            const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                            const float* u, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    using namespace fence;
    if (!out || !logits || !u || !workspace || rows < 0 || vocab < 1 || vocab > kMaxVocab || ld < vocab)
        return FENCE_ERROR_INVALID_VALUE;
    if (rows > INT32_MAX || ld > INT64_MAX / 8 / (rows + 1)) return FENCE_ERROR_INVALID_VALUE;
    if (!aligned(out, 4) || !aligned(logits, 4) || !aligned(u, 4) || !aligned(workspace, 16) ||
        (temperature && !aligned(temperature, 4)) || (top_k && !aligned(top_k, 4)) || (top_p && !aligned(top_p, 4)) ||
        (min_p && !aligned(min_p, 4)))
        return FENCE_ERROR_INVALID_VALUE;
    if (workspace_bytes < fence_sample_workspace(rows, vocab)) return FENCE_ERROR_INVALID_VALUE;
    if (rows == 0) return FENCE_SUCCESS;
    const int slots = slots_of(rows, vocab), width = scan_width(rows, vocab);
    SampleArgs a{out, logits, ld, vocab, shift_for(vocab), slots, temperature, top_k, top_p, min_p, u,
                 nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
    a.slot_mass = static_cast<double*>(workspace);
    a.bin_mass = reinterpret_cast<u64*>(a.slot_mass + rows * slots);
    a.list = a.bin_mass + rows * kBins;
    a.state = reinterpret_cast<RowState*>(a.list + rows * kList);
    a.slot_top = reinterpret_cast<uint32_t*>(a.state + rows);
    a.bin_count = a.slot_top + rows * slots;
    const int64_t n4 = (static_cast<int64_t>(vocab) + 3) / 4;
    // Workgroups that share a flat row: one for each CU, but four at least, and none with fewer than 2048 logits.
    // Each adds its bins to the row's by atomics: the histograms of 32 rows of 128,256 take 14 us in 8 workgroups a
    // row, 22 in 16 and 34 in 32; those of 256 rows of 151,936 take 64 us in one a row and 22 in 4.  Listing, they
    // all begin with the whole histogram: 38 us in 8 a row and 62 in 32; 83 us in one a row, 60 in 2 and 47 in 4.
    int64_t parts = (256 + rows - 1) / rows, chunk;
    if (parts < 4) parts = 4;
    if (parts > (n4 + 511) / 512) parts = (n4 + 511) / 512;
    chunk = (n4 + parts - 1) / parts;
    constexpr int64_t kRows = 32768;  // of a launch: grid.y and the lanes of a grid are bounded
    for (int64_t r0 = 0; r0 < rows; r0 += kRows) {
        const unsigned m = static_cast<unsigned>(rows - r0 < kRows ? rows - r0 : kRows);
        SampleArgs p = a;
        p.out += r0;
        p.x += r0 * ld;
        if (p.temperature) p.temperature += r0;
        if (p.top_k) p.top_k += r0;
        if (p.top_p) p.top_p += r0;
        if (p.min_p) p.min_p += r0;
        p.u += r0;
        p.slot_mass += r0 * slots;
        p.bin_mass += r0 * kBins;
        p.list += r0 * kList;
        p.state += r0;
        p.slot_top += r0 * slots;
        p.bin_count += r0 * kBins;
        const dim3 scan(slots / kScanThreads, m);
        int st = width == 5 ? launch(sample_scan<5>, scan, dim3(kScanThreads), 0, stream, p)
                            : launch(sample_scan<10>, scan, dim3(kScanThreads), 0, stream, p);
        if (st) return st;
        st = width == 5 ? launch(sample_list<5>, dim3(m), dim3(kThreads), 0, stream, p)
                        : launch(sample_list<10>, dim3(m), dim3(kThreads), 0, stream, p);
        if (st) return st;
        if ((st = launch(sample_histogram, dim3(static_cast<unsigned>(parts), m), dim3(kThreads), 0, stream, p, chunk)))
            return st;
        if ((st = launch(sample_flat, dim3(static_cast<unsigned>(parts), m), dim3(kThreads), 0, stream, p, chunk))) return st;
    }
    return FENCE_SUCCESS;
}
