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
// One workgroup takes a row.
//   1. One pass finds the maximum and each thread's maximum.  For a top-k up
//      to kListK, the k-th largest of those is a lower bound of the k-th
//      largest logit with few more logits above it than k.
//   2. A second pass collects the logits above that bound in LDS.  Without a
//      small top-k it makes a histogram by distance from the maximum instead,
//      which says how far down the filters and the draw can reach, and a third
//      pass collects what lies above that.
//   3. The list is sorted and summed, and the filters and the draw are read
//      off the sums.
// A list that would not fit (flat rows) is never made: the histogram leads to
// one bin for each question, whose elements are listed, or, if they are too
// many as well, divided by the digits of their keys.
#include "common.hpp"

namespace fence {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kListK = 512;    // largest top-k that the bound from the threads' maxima serves
constexpr int kList = 4096;    // elements a list holds
constexpr int kBins = 2048;    // of the histogram; the last one takes everything further away
constexpr float kReach = 10.0f;  // how far below the maximum the histogram reaches, in units of T
typedef unsigned long long u64;

struct SampleArgs {
    int32_t* out;
    const float* x;
    int64_t ld;
    int vocab, shift;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
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

struct Shared {
    u64 mass[kBins];
    uint32_t count[kBins];
    u64 list[kList];  // key << 32 | ~index: larger comes first
    u64 wave[kWaves];
    u64 found[4];
    uint32_t n;
};

// What a row's passes have in common.
struct Row {
    const float* x;
    int n;
    bool vec;
    uint32_t top;    // the maximum's key
    float top_value;
    double rate;     // log2(e) / T
    double one;      // 2^shift
    float bins_per;  // histogram bins per unit of logit

    template <class F>
    __device__ __forceinline__ void each(F f) const {
        int done = 0;
        if (vec) {
            const int n4 = n / 4;
#pragma unroll 4
            for (int i = threadIdx.x; i < n4; i += kThreads) {
                const f4 v = *reinterpret_cast<const f4*>(x + 4 * static_cast<int64_t>(i));
#pragma unroll
                for (int j = 0; j < 4; ++j) f(v[j], 4 * i + j);
            }
            done = n4 * 4;
        }
        for (int64_t i = done + threadIdx.x; i < n; i += kThreads) f(x[i], static_cast<int>(i));
    }
    __device__ __forceinline__ double weight(uint32_t key) const {
        if (key == top) return 1.0;
        return exp2_64((static_cast<double>(of_key(key)) - static_cast<double>(top_value)) * rate);
    }
    __device__ __forceinline__ u64 units(uint32_t key) const { return static_cast<u64>(rint(weight(key) * one)); }
    // non-increasing in the key: the order of bins is the order of elements
    __device__ __forceinline__ int bin(uint32_t key) const {
        if (key == top) return 0;
        const float d = (top_value - of_key(key)) * bins_per;
        return d < static_cast<float>(kBins - 1) ? static_cast<int>(d) : kBins - 1;
    }
};

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

// The list's elements that pass `in`, in any order; how many there were,
// which may be more than a list holds.
template <class P>
__device__ __forceinline__ uint32_t collect(Shared& s, const Row& row, P in) {
    __syncthreads();
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    row.each([&](float x, int i) {
        const uint32_t key = key_of(x);
        if (in(key)) {
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < kList) s.list[at] = static_cast<u64>(key) << 32 | static_cast<uint32_t>(~i);
        }
    });
    __syncthreads();
    return s.n;
}

// The first n entries of the list in falling order (bitonic, over the next
// power of two, filled up with zeros, which come last).
__device__ __forceinline__ void sort_list(Shared& s, int n) {
    int size = kWave;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += kThreads) s.list[i] = 0;
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += kThreads) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const u64 x = s.list[a], y = s.list[b];
                if ((x < y) == ((a & k) == 0)) s.list[a] = y, s.list[b] = x;
            }
        }
    __syncthreads();
}

// Running sums over the sorted list, kPer consecutive entries a thread.
constexpr int kPer = kList / kThreads;
struct Sums {
    u64 upto[kPer];  // inclusive
};
__device__ __forceinline__ Sums list_sums(Shared& s, const Row& row, int n, int per) {
    Sums r;
    u64 mine = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = threadIdx.x * per + j;
        if (j < per && i < n) mine += row.units(static_cast<uint32_t>(s.list[i] >> 32));
        r.upto[j] = mine;
    }
    u64 total;
    const u64 before = block_scan(s, mine, &total) - mine;
#pragma unroll
    for (int j = 0; j < kPer; ++j) r.upto[j] += before;
    return r;
}

// The first place of the list whose sum passes(), or n - 1, and its sum.
template <class P>
__device__ __forceinline__ int first_place(Shared& s, const Sums& sums, int n, int per, P passes, u64* sum) {
    __syncthreads();
    if (threadIdx.x == 0) s.found[0] = n - 1;
    __syncthreads();
    for (int j = kPer - 1; j >= 0; --j) {
        const int i = threadIdx.x * per + j;
        if (j < per && i < n && passes(sums.upto[j])) atomicMin(&s.found[0], static_cast<u64>(i));
    }
    __syncthreads();
    const int at = static_cast<int>(s.found[0]);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (j < per && static_cast<int>(threadIdx.x) * per + j == at) s.found[1] = sums.upto[j];
    __syncthreads();
    *sum = s.found[1];
    return at;
}

// A question about the whole order: at which element does the running sum of
// weights (or the running count) reach `goal`?
struct Place {
    int index;
    u64 mass;  // the running sum of weights there, inclusive
};

// Divides the elements that pass `in` by `digit` (0 .. kBins - 1, falling along
// the order is 0 first), adding up weights and counts.
template <class P, class D>
__device__ __forceinline__ void histogram(Shared& s, const Row& row, P in, D digit) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0, s.count[i] = 0;
    __syncthreads();
    u64 last_mass = 0;
    uint32_t last_count = 0;
    row.each([&](float x, int) {
        const uint32_t key = key_of(x);
        if (!in(key)) return;
        const int d = digit(key);
        const u64 w = row.units(key);
        if (d == kBins - 1) {  // most of a peaked row: not through one address
            last_mass += w;
            ++last_count;
        } else {
            atomicAdd(&s.mass[d], w);
            atomicAdd(&s.count[d], 1u);
        }
    });
    if (last_count) {
        atomicAdd(&s.mass[kBins - 1], last_mass);
        atomicAdd(&s.count[kBins - 1], last_count);
    }
    __syncthreads();
}

// The bin in which the running sum (count) reaches goal; what came before it.
__device__ __forceinline__ int find_bin(Shared& s, bool by_count, u64 goal, u64* mass_before, u64* count_before) {
    constexpr int kEach = kBins / kThreads;
    u64 m[kEach], c[kEach], mm = 0, cc = 0, total;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        mm += m[j] = s.mass[threadIdx.x * kEach + j];
        cc += c[j] = s.count[threadIdx.x * kEach + j];
    }
    u64 m0 = block_scan(s, mm, &total) - mm;
    u64 c0 = block_scan(s, cc, &total) - cc;
    __syncthreads();
    if (threadIdx.x == 0) s.found[0] = ~0ull;
    __syncthreads();
    u64 ms = m0, cs = c0;
    int at = -1;
    u64 mb = 0, cb = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        if (at < 0 && c[j] && (by_count ? cs + c[j] : ms + m[j]) >= goal) at = threadIdx.x * kEach + j, mb = ms, cb = cs;
        ms += m[j];
        cs += c[j];
    }
    if (at >= 0) atomicMin(&s.found[0], static_cast<u64>(at));
    __syncthreads();
    const u64 first = s.found[0];
    if (at >= 0 && static_cast<u64>(at) == first) s.found[1] = mb, s.found[2] = cb;
    __syncthreads();
    *mass_before = s.found[1];
    *count_before = s.found[2];
    return first == ~0ull ? -1 : static_cast<int>(first);
}

// Where the running sum (or count) over the whole row reaches goal >= 1, from
// the row's histogram by distance, which is in s on entry if `fresh`.
__device__ __forceinline__ Place locate(Shared& s, const Row& row, bool by_count, u64 goal, bool fresh) {
    const auto all = [](uint32_t) { return true; };
    if (!fresh) histogram(s, row, all, [&](uint32_t k) { return row.bin(k); });
    u64 mass, count;
    const int b = find_bin(s, by_count, goal, &mass, &count);
    uint32_t lo = 0, hi = ~0u;  // keys that are left, both inclusive
    int left = static_cast<int>(s.count[b]);
    const auto in = [&](uint32_t k) { return k >= lo && k <= hi && row.bin(k) == b; };
    // too many for a list: their keys by 11 bits at a time
    for (int bits = 32; left > kList && bits > 0;) {
        const int take = bits < 11 ? bits : 11;
        bits -= take;
        const uint32_t mask = (1u << take) - 1;
        histogram(s, row, in, [&](uint32_t k) { return static_cast<int>(mask - ((k >> bits) & mask)); });
        u64 m, c;
        const int d = find_bin(s, by_count, by_count ? goal - count : goal - mass, &m, &c);
        mass += m;
        count += c;
        left = static_cast<int>(s.count[d]);
        const uint32_t digit = mask - static_cast<uint32_t>(d);
        lo |= digit << bits;
        hi = lo | ((1u << bits) - 1);
    }
    Place p;
    if (left <= kList) {
        collect(s, row, in);
        sort_list(s, left);
        const int per = (left + kThreads - 1) / kThreads;
        const Sums sums = list_sums(s, row, left, per);
        u64 sum;
        int at;
        if (by_count) {
            at = static_cast<int>(goal - count) - 1;
            const int want = at;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (j < per && static_cast<int>(threadIdx.x) * per + j == want) s.found[1] = sums.upto[j];
            __syncthreads();
            sum = s.found[1];
        } else {
            const u64 rest = goal - mass;
            at = first_place(s, sums, left, per, [&](u64 v) { return v >= rest; }, &sum);
        }
        p.index = static_cast<int>(~static_cast<uint32_t>(s.list[at]));
        p.mass = mass + sum;
    } else {
        // equal logits, more than a list holds: the n-th of them by index
        const u64 w = row.units(lo);
        u64 nth = by_count ? goal - count : w ? (goal - mass + w - 1) / w : 1;
        if (nth < 1) nth = 1;
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

// u times a sum, rounded down: the running sum has to be above it.
__device__ __forceinline__ u64 draw_goal(float u, u64 mass) {
    u = u > 0.0f ? u : 0.0f;
    double t = static_cast<double>(u) * static_cast<double>(mass);
    const u64 goal = static_cast<u64>(t) + 1;
    return goal < mass ? goal : mass > 0 ? mass : 1;  // u = 1 and above: the last one
}

__device__ __forceinline__ u64 top_p_goal(float p, u64 mass) {
    p = p > 0.0f ? p : 0.0f;
    const u64 goal = static_cast<u64>(ceil(static_cast<double>(p) * static_cast<double>(mass)));
    return goal < 1 ? 1 : goal < mass ? goal : mass;
}

__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int64_t r = blockIdx.x;
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    Row row;
    row.x = a.x + r * a.ld;
    row.n = a.vocab;
    row.vec = reinterpret_cast<uintptr_t>(row.x) % 16 == 0;
    // 1. the maximum, its first index, and this thread's maximum
    u64 best = 0;
    row.each([&](float x, int i) {
        const u64 e = static_cast<u64>(key_of(x)) << 32 | static_cast<uint32_t>(~i);
        best = e > best ? e : best;
    });
    const u64 first = block_max(s, best);
    row.top = static_cast<uint32_t>(first >> 32);
    row.top_value = of_key(row.top);
    if (!(t > 0.0f) || row.top <= kKeyLowest) {
        if (threadIdx.x == 0)
            a.out[r] = row.top <= kKeyLowest ? 0 : static_cast<int>(~static_cast<uint32_t>(first));
        return;
    }
    row.rate = 1.4426950408889634074 / static_cast<double>(t);
    row.one = ldexp(1.0, a.shift);
    const float per = static_cast<float>(kBins) / kReach / t;
    row.bins_per = per < 3e38f ? per : 3e38f;
    int k = a.top_k ? a.top_k[r] : 0;
    if (k <= 0 || k >= row.n) k = 0;
    const float top_p = a.top_p ? a.top_p[r] : 1.0f;
    const bool use_p = top_p < 1.0f;
    const float min_p = a.min_p ? a.min_p[r] : 0.0f;
    const float least = min_p > 0.0f ? (min_p < 1.0f ? min_p : 1.0f) : 0.0f;
    const float u = a.u ? a.u[r] : 0.0f;

    // 2. a list that holds all that the filters keep, if one can
    int n = 0;
    u64 mass = 0;  // of the elements that top-p is about, if the list does not say it
    bool listed = false, fresh = false;
    if (k && k <= kListK) {
        // the largest bound (of 16 bits) that k threads' maxima reach
        uint32_t bound = 0;
        const uint32_t mine = static_cast<uint32_t>(best >> 32);
        for (int bit = 31; bit >= 16; --bit) {
            const uint32_t trial = bound | 1u << bit;
            if (__syncthreads_count(mine >= trial) >= k) bound = trial;
        }
        const uint32_t found = collect(s, row, [&](uint32_t key) { return key >= bound; });
        listed = found <= kList;
        n = static_cast<int>(found);
    }
    if (!listed) {
        histogram(s, row, [](uint32_t) { return true; }, [&](uint32_t key) { return row.bin(key); });
        fresh = true;
        u64 total = 0, part, before, count;
        {
            u64 v = 0;
            for (int i = threadIdx.x; i < kBins; i += kThreads) v += s.mass[i];
            block_scan(s, v, &total);
        }
        mass = total;
        // the last bin that matters
        int reach = kBins - 1;
        if (k) {
            reach = find_bin(s, true, k, &before, &count);
        } else {
            if (use_p) reach = find_bin(s, false, top_p_goal(top_p, total), &before, &count);
            else if (!(least > 0.0f)) reach = find_bin(s, false, draw_goal(u, total), &before, &count);
        }
        if (least > 0.0f && !(k && use_p)) {  // (top-p after top-k needs the weight of all k.)  One bin more than the distance says, for its rounding
            const float d = -logf(least) * t * row.bins_per + 1.0f;
            const int last = d < static_cast<float>(kBins - 1) ? static_cast<int>(d) + 1 : kBins - 1;
            reach = last < reach ? last : reach;
        }
        u64 v = 0;
        for (int i = threadIdx.x; i <= reach; i += kThreads) v += s.count[i];
        block_scan(s, v, &part);
        if (part <= kList) {
            collect(s, row, [&](uint32_t key) { return row.bin(key) <= reach; });
            n = static_cast<int>(part);
            listed = true;
        }
    }

    if (listed) {
        // 3. the filters and the draw on the sorted list
        sort_list(s, n);
        const int per_thread = (n + kThreads - 1) / kThreads;
        const Sums sums = list_sums(s, row, n, per_thread);
        int keep = n;
        u64 kept = mass, sum;
        if (k && k <= n) {
            keep = k;
            // the sum at place k - 1
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (j < per_thread && static_cast<int>(threadIdx.x) * per_thread + j == k - 1) s.found[1] = sums.upto[j];
            __syncthreads();
            kept = s.found[1];
        }
        if (use_p) {
            const u64 goal = top_p_goal(top_p, kept);
            const int at = first_place(s, sums, n, per_thread, [&](u64 v) { return v >= goal; }, &sum);
            if (at + 1 <= keep) keep = at + 1, kept = sum;
        }
        if (least > 0.0f) {
            int passing = 0;
            for (int i = threadIdx.x; i < keep; i += kThreads)
                passing += row.weight(static_cast<uint32_t>(s.list[i] >> 32)) >= static_cast<double>(least);
            u64 total;
            block_scan(s, static_cast<u64>(passing), &total);
            keep = total < 1 ? 1 : static_cast<int>(total);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (j < per_thread && static_cast<int>(threadIdx.x) * per_thread + j == keep - 1) s.found[1] = sums.upto[j];
            __syncthreads();
            kept = s.found[1];
        }
        const u64 goal = draw_goal(u, kept);
        const int at = first_place(s, sums, n, per_thread, [&](u64 v) { return v >= goal; }, &sum);
        if (threadIdx.x == 0) a.out[r] = static_cast<int>(~static_cast<uint32_t>(s.list[at]));
        return;
    }

    // A flat row: one question at a time on the whole of it.
    u64 kept = mass;
    if (k) kept = locate(s, row, true, k, fresh).mass, fresh = false;
    if (use_p) kept = locate(s, row, false, top_p_goal(top_p, kept), fresh).mass, fresh = false;
    if (least > 0.0f) {
        u64 v = 0, total;
        row.each([&](float x, int) {
            const uint32_t key = key_of(x);
            if (row.weight(key) >= static_cast<double>(least)) v += row.units(key);
        });
        block_scan(s, v, &total);
        kept = total < kept ? total : kept;
    }
    const Place p = locate(s, row, false, draw_goal(u, kept), fresh);
    if (threadIdx.x == 0) a.out[r] = p.index;
}

int shift_for(int vocab) {
    int bits = 1;
    while ((int64_t(1) << bits) < vocab) ++bits;
    return 62 - bits;  // the sum of vocab weights of at most 2^shift stays below 2^63
}

}  // namespace
}  // namespace fence

extern "C" int64_t fence_sample_workspace(int64_t rows, int vocab) {
    if (rows < 0 || vocab < 1) return 0;
    return 16;
}

extern "C" int fence_sample(int32_t* out, const float* logits, int64_t rows, int vocab, int64_t ld,
                            const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                            const float* u, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    using namespace fence;
    if (!out || !logits || !u || !workspace || rows < 0 || vocab < 1 || ld < vocab) return FENCE_ERROR_INVALID_VALUE;
    if (rows > INT32_MAX || ld > INT64_MAX / 8 / (rows + 1)) return FENCE_ERROR_INVALID_VALUE;
    if (!aligned(out, 4) || !aligned(logits, 4) || !aligned(u, 4) || !aligned(workspace, 16) ||
        (temperature && !aligned(temperature, 4)) || (top_k && !aligned(top_k, 4)) || (top_p && !aligned(top_p, 4)) ||
        (min_p && !aligned(min_p, 4)))
        return FENCE_ERROR_INVALID_VALUE;
    if (workspace_bytes < fence_sample_workspace(rows, vocab)) return FENCE_ERROR_INVALID_VALUE;
    if (rows == 0) return FENCE_SUCCESS;
    const int64_t most = kMaxLaunchLanes / kThreads;  // rows of a launch
    for (int64_t r0 = 0; r0 < rows; r0 += most) {
        const int64_t m = rows - r0 < most ? rows - r0 : most;
        const SampleArgs part{out + r0, logits + r0 * ld, ld, vocab, shift_for(vocab), temperature ? temperature + r0 : nullptr,
                              top_k ? top_k + r0 : nullptr, top_p ? top_p + r0 : nullptr,
                              min_p ? min_p + r0 : nullptr, u + r0};
        if (const int st = launch(sample_kernel, dim3(static_cast<unsigned>(m)), dim3(kThreads), 0, stream, part))
            return st;
    }
    return FENCE_SUCCESS;
}
