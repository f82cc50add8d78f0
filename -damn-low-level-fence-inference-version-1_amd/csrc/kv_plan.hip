// kv_plan.hip -- the plan of a batched step over a paged KV cache on gfx950:
// pages of ended sequences back on the free stack, pages of new tokens off
// it, and every token's row, position and slot.
//
// All of it is prefix sums over the batch (pages given back, pages needed,
// tokens) and then flat lists: item i of a list belongs to the sequence whose
// range of the prefix sum holds i, which a binary search of the sums in LDS
// finds.  One workgroup walks the batch kBatchChunk sequences at a time with
// the sums so far in registers, so no sequence waits for another's pages and
// no atomics decide an order.  The tokens' rows are filled by the same
// workgroup while they are few (kOneLaunchTokens), else by a second launch
// over many workgroups.
//
// Bound by latency: a scan is two barriers and 64-bit shuffles, a list item
// the ten LDS reads of its search, so the searches of kAhead items run side
// by side, without a branch.  64 single tokens take 8.9 us, 384 prompts of
// 265,152 rows 13.8 us and another 6.8 for the rows.
#include "common.hpp"

#include <climits>

namespace fence {
namespace {

constexpr int kThreads = 1024;
constexpr int kBatchChunk = kThreads;  // one sequence per thread
constexpr int kAhead = 4;              // items whose loads a thread has in flight
constexpr int kFillThreads = 256;
constexpr int kFillTokens = kAhead * kFillThreads;  // tokens a workgroup of the second launch fills
constexpr int kFillLds = 4096;  // row ends the second launch keeps in LDS
// Rows that one workgroup fills.  64 sequences, back to back: 4,096 rows take 10.9 us so and 14.7 with the second
// launch, 8,192 take 13.3 and 15.0, 16,384 take 18.0 and 15.0.
constexpr int64_t kOneLaunchTokens = 8192;

struct PlanArgs {
    int32_t* lens_out;
    const int32_t* lens;
    const int32_t* new_lens;
    int32_t* table;
    int32_t* free_pages;
    int32_t* free_count_out;
    const int32_t* free_count;
    int32_t* q_start;
    int32_t* positions;
    int32_t* slots;
    int32_t* admitted;
    int batch, max_blocks, page_shift, n_pages;
    int max_tokens;
    int fill;  // the rows too, in this launch (batch <= kBatchChunk)
};

// Inclusive prefix sum over the workgroup and its total.  64 bits: lengths
// are the caller's and may add up past 2^31.  `waves` holds 16 sums; callers
// barrier before they reuse it.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* waves, int64_t* total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int64_t up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    if (lane == kWave - 1) waves[wave] = v;
    __syncthreads();
    int64_t sums = waves[lane % (kThreads / kWave)];  // and their sums, in every wave's first lanes
#pragma unroll
    for (int d = 1; d < kThreads / kWave; d *= 2) {
        const int64_t up = __shfl_up(sums, d);
        if (lane >= d) sums += up;
    }
    *total = __shfl(sums, kThreads / kWave - 1);
    const int64_t before = __shfl(sums, wave > 0 ? wave - 1 : 0);
    return wave > 0 ? before + v : v;
}

// The first i with ends[i] > at (ends ascending, at < ends[n - 1]).
__device__ __forceinline__ int holder(const int* ends, int n, int at) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (ends[mid] > at) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// The same among N entries, a power of two, in steps without a branch: several
// searches of a thread run side by side.
template <int N>
__device__ __forceinline__ int holder_of(const int* ends, int at) {
    int i = 0;
#pragma unroll
    for (int step = N / 2; step > 0; step /= 2) i += ends[i + step - 1] <= at ? step : 0;
    return i;
}

__device__ __forceinline__ int sat32(int64_t v) { return v > INT_MAX ? INT_MAX : static_cast<int>(v); }

// Row t: the token at `position` of a sequence with this table row.
__device__ __forceinline__ void put_row(const PlanArgs& a, int t, int position, bool in, const int32_t* row) {
    int slot = -1;
    if (in)  // an admitted sequence's positions lie within max_blocks pages
        slot = (row[position >> a.page_shift] << a.page_shift) + (position & ((1 << a.page_shift) - 1));
    a.positions[t] = position;
    a.slots[t] = slot;
}

__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs a) {
    __shared__ int64_t waves[2][kThreads / kWave];
    __shared__ int ends[kBatchChunk];    // ends of a flat list's ranges
    __shared__ int begins[kBatchChunk];  // what a range's items are counted from
    __shared__ int bases[kBatchChunk];   // cached tokens (-1 - them if not admitted)
    __shared__ int last_taken;           // pages needed up to the last sequence that got one
    const int tid = threadIdx.x;
    const int page = 1 << a.page_shift;
    int64_t count = a.free_count[0];
    count = count < 0 ? 0 : count > a.n_pages ? a.n_pages : count;
    if (tid == 0) last_taken = 0;

    // 1. What ended sequences held, onto the stack.
    for (int b0 = 0; b0 < a.batch; b0 += kBatchChunk) {
        const int b = b0 + tid;
        const int add = b < a.batch ? a.new_lens[b] : 0;
        if (!__syncthreads_or(add < 0)) continue;
        int64_t back = 0;
        if (add < 0) {
            const int len = a.lens[b] > 0 ? a.lens[b] : 0;
            back = (static_cast<int64_t>(len) + page - 1) >> a.page_shift;
            if (back > a.max_blocks) back = a.max_blocks;
        }
        int64_t total;
        const int64_t end = block_scan(back, waves[0], &total);
        if (total > a.n_pages - count) total = a.n_pages - count;  // ids that would not fit are dropped
        ends[tid] = sat32(end);
        begins[tid] = sat32(end - back);
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < total; i += kThreads) {
            const int s = holder_of<kBatchChunk>(ends, i);
            a.free_pages[count + i] = a.table[static_cast<int64_t>(b0 + s) * a.max_blocks + (i - begins[s])];
        }
        count += total;
        __syncthreads();
    }

    // 2. Who is admitted, with which pages.
    int64_t upto = 0, rows = 0, taken = 0;  // pages needed, rows, pages taken by the chunks before
    for (int b0 = 0; b0 < a.batch; b0 += kBatchChunk) {
        const int b = b0 + tid;
        const bool here = b < a.batch;
        const int given = here ? a.new_lens[b] : 0;
        const int len = here && a.lens[b] > 0 ? a.lens[b] : 0;
        const bool ended = given < 0;
        const int64_t add = ended ? 0 : given;
        int64_t new_rows, new_need;
        const int64_t row_end = rows + block_scan(add, waves[0], &new_rows);
        const int64_t held = (static_cast<int64_t>(len) + page - 1) >> a.page_shift;
        const int64_t after = (len + add + page - 1) >> a.page_shift;
        const bool fits = here && !ended && after <= a.max_blocks && row_end <= a.max_tokens;
        const int64_t need = fits ? after - held : 0;
        const int64_t need_end = upto + block_scan(need, waves[1], &new_need);
        const bool in = fits && (need == 0 || need_end <= count);
        // A sequence gets pages only if all that were needed before it were there, so the pages taken are the
        // first ones needed, and the n-th of them is the n-th from the top.
        if (in && need > 0) atomicMax(&last_taken, static_cast<int>(need_end));  // at most n_pages
        __syncthreads();
        const int new_taken = last_taken > upto ? static_cast<int>(last_taken - upto) : 0;
        const int64_t need_here = need_end - upto;
        ends[tid] = need_here < new_taken ? static_cast<int>(need_here) : new_taken;
        begins[tid] = sat32(need_here - need - held);
        if (here) {
            a.lens_out[b] = ended ? 0 : in ? static_cast<int>(len + add) : len;
            a.admitted[b] = in || ended;
            a.q_start[b + 1] = sat32(row_end);
        }
        __syncthreads();
#pragma unroll 1
        for (int i0 = tid; i0 < new_taken; i0 += kAhead * kThreads) {
            int id[kAhead], s[kAhead];
#pragma unroll
            for (int d = 0; d < kAhead; ++d) {
                const int i = i0 + d * kThreads;
                id[d] = i < new_taken ? a.free_pages[count - 1 - taken - i] : 0;
                s[d] = holder_of<kBatchChunk>(ends, i);
            }
#pragma unroll
            for (int d = 0; d < kAhead; ++d) {
                const int i = i0 + d * kThreads;
                if (i < new_taken) a.table[static_cast<int64_t>(b0 + s[d]) * a.max_blocks + (i - begins[s[d]])] = id[d];
            }
        }
        upto += new_need;
        rows += new_rows;
        taken += new_taken;
        __syncthreads();
        if (a.fill) {  // the only chunk: from here on the ranges are those of the rows
            ends[tid] = sat32(row_end);
            begins[tid] = sat32(row_end - add);
            bases[tid] = in ? len : -1 - len;
        }
    }
    if (tid == 0) {
        a.q_start[0] = 0;
        a.free_count_out[0] = static_cast<int>(count - taken);
    }
    if (!a.fill) return;

    // 3. The rows, where they are few.
    __syncthreads();
#pragma unroll 1
    for (int64_t t64 = tid; t64 < a.max_tokens; t64 += kThreads) {
        const int t = static_cast<int>(t64);
        if (t >= rows) {
            a.positions[t] = 0;
            a.slots[t] = -1;
            continue;
        }
        const int s = holder_of<kBatchChunk>(ends, t);
        const bool in = bases[s] >= 0;
        put_row(a, t, (in ? bases[s] : -1 - bases[s]) + (t - begins[s]), in,
                a.table + static_cast<int64_t>(s) * a.max_blocks);
    }
}

// The rows from what the first launch wrote.
__global__ __launch_bounds__(kFillThreads) void plan_fill_kernel(PlanArgs a) {
    __shared__ int lds[kFillLds];
    const bool near = a.batch <= kFillLds;
    if (near) {
        for (int i = threadIdx.x; i < kFillLds; i += kFillThreads) lds[i] = i < a.batch ? a.q_start[i + 1] : INT_MAX;
        __syncthreads();
    }
    const int* ends = near ? lds : a.q_start + 1;
    const int rows = ends[a.batch - 1];
    int t[kAhead], s[kAhead], slot[kAhead], position[kAhead];
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
        const int64_t at = static_cast<int64_t>(blockIdx.x) * kFillTokens + d * kFillThreads + threadIdx.x;
        t[d] = at < a.max_tokens ? static_cast<int>(at) : -1;
        const int within = t[d] >= 0 && t[d] < rows ? t[d] : 0;
        s[d] = rows > 0 ? near ? holder_of<kFillLds>(ends, within) : holder(ends, a.batch, within) : 0;
    }
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
        const int start = s[d] ? ends[s[d] - 1] : 0;
        const bool in = a.admitted[s[d]] != 0;  // a sequence with rows has not ended
        const int len = a.lens_out[s[d]];
        position[d] = (in ? len - (ends[s[d]] - start) : len) + (t[d] - start);
        slot[d] = in && t[d] >= 0 && t[d] < rows
                      ? a.table[static_cast<int64_t>(s[d]) * a.max_blocks + (position[d] >> a.page_shift)]
                      : -1;
    }
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
        if (t[d] < 0) continue;
        const bool row = t[d] < rows;
        const bool in = row && a.admitted[s[d]] != 0;
        a.positions[t[d]] = row ? position[d] : 0;
        a.slots[t[d]] = in ? (slot[d] << a.page_shift) + (position[d] & ((1 << a.page_shift) - 1)) : -1;
    }
}

}  // namespace
}  // namespace fence

extern "C" int fence_kv_plan(int32_t* lens_out, const int32_t* lens, const int32_t* new_lens, int batch,
                             int32_t* block_table, int max_blocks, int page_size, int32_t* free_pages,
                             int32_t* free_count_out, const int32_t* free_count, int n_pages, int32_t* q_start,
                             int32_t* positions, int32_t* slots, int64_t max_tokens, int32_t* admitted,
                             hipStream_t stream) {
    using namespace fence;
    if (batch < 0 || max_blocks < 1 || n_pages < 1 || max_tokens < 0 || max_tokens > INT32_MAX)
        return FENCE_ERROR_INVALID_VALUE;
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1))) return FENCE_ERROR_INVALID_VALUE;
    if (static_cast<int64_t>(n_pages) * page_size > INT32_MAX ||
        static_cast<int64_t>(max_blocks) * page_size > INT32_MAX)
        return FENCE_ERROR_INVALID_VALUE;
    // an array without entries may be NULL
    const void* const always[] = {free_pages, free_count_out, free_count, q_start};
    const void* const per_sequence[] = {lens_out, lens, new_lens, block_table, admitted};
    const void* const per_row[] = {positions, slots};
    for (const void* p : always)
        if (!p || !aligned(p, 4)) return FENCE_ERROR_INVALID_VALUE;
    for (const void* p : per_sequence)
        if ((!p && batch > 0) || !aligned(p, 4)) return FENCE_ERROR_INVALID_VALUE;
    for (const void* p : per_row)
        if ((!p && max_tokens > 0) || !aligned(p, 4)) return FENCE_ERROR_INVALID_VALUE;
    const bool fill = batch == 0 || (batch <= kBatchChunk && max_tokens <= kOneLaunchTokens);
    const PlanArgs a{lens_out, lens, new_lens, block_table, free_pages, free_count_out, free_count, q_start,
                     positions, slots, admitted, batch, max_blocks, __builtin_ctz(page_size), n_pages,
                     static_cast<int>(max_tokens), fill};
    if (const int st = launch(plan_kernel, dim3(1), dim3(kThreads), 0, stream, a)) return st;
    if (fill || max_tokens == 0) return FENCE_SUCCESS;
    return launch(plan_fill_kernel, dim3(grid_1d(max_tokens, kFillTokens)), dim3(kFillThreads), 0, stream, a);
}
