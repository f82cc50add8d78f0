// attention_q8.hip -- attention of a batch over the pages of an 8-bit KV
// cache, on gfx950.
//
//   s_j = (q . k_j) * scale,  p = softmax(s),  out = sum_j p_j v_j,
//   k_j = code * k_scale[page of j][kv head], v_j likewise.
//
// The codes go into the matrix cores as binary16, which holds every int8 and
// every e4m3 value exactly; a page's K scale multiplies its scores, its V
// scale the probabilities.  The query heads of a kv head's group and the rows
// of a sequence are the columns of the products, so a code is read and
// converted once for all of them.
#include "kv_q8.hpp"

#include <cmath>


namespace fence {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
// Columns of the products are the (row, head of the group) pairs of one kv
// head; a sequence's are taken kCols or kPromptCols at a time.
constexpr int kCols = 16;           // few_columns; a sequence with no more of them goes there
constexpr int kUnit = 32 * kWaves;  // positions its workgroup takes at a time
constexpr int kPromptCols = 32 * kWaves;  // many_columns
constexpr int64_t kMaxLd = int64_t(1) << 32;  // elements from row to row: times a row's number they fit 63 bits
constexpr int kBeyond = 1024;  // positions past the last that may be looked up: units loaded turns ahead
// What an item of many columns costs besides its positions, in positions.  With 384, 192 and 128: 24 x 5 drafted rows
// in groups of seven 28.7, 30.1 and 28.5 us, one prompt of 8,192 rows 736, 730 and 734, six prompt chunks of 500 rows
// in fp32 131, 126 and 131, in binary16 151, 147 and 152.
constexpr int kBigItem = 384;
// Workgroups that share the work, two a CU.  With few columns, where more fit (two, four and eight a CU): one token at
// 32,768 positions takes 33, 51 and 80 us, as each part that an item is cut into has to be joined; 64 tokens at up to
// 4,096 60, 66 and 78, and at up to 32,768 302, 305 and 320.  With many columns two fit: a prompt of 8,192 rows takes
// 736 us, with one a CU 1,162.
constexpr int kGrid = 512;
constexpr int kBigGrid = 512;
constexpr int kXcds = 8;

// Where a workgroup begins, as it leaves it for the join.
struct Border {
    int64_t item, cost, total;  // where the item begins in the work, what it costs, and all work
    int seq, tile, head, unit, units;
    int grid;  // workgroups that share the work; 0: nothing to do for this one
};
static_assert(sizeof(Border) == 48);

struct Q8Args {
    void* out;
    const void* q;
    int64_t ldq, ldo;
    const uint8_t* k;
    const uint8_t* v;
    const float* ks;
    const float* vs;
    const int32_t* table;
    const int32_t* kv_lens;
    const int32_t* q_start;
    float* ws;
    Border* borders;  // in the workspace, one for each workgroup
    int n_pages, page_shift, n_kv_heads, head_dim, group;
    int max_blocks, batch, max_q_len;
    int part_cols;  // columns of a part in the workspace
    float scale_log2;
    int wide;  // out and its rows are 16-byte aligned
};

// Read-only data at addresses that are the same in every lane, through the
// scalar cache: it does not queue behind the codes that are being loaded.
template <class T>
__device__ __forceinline__ T uniform_load(const T* p, int64_t i) {
    return reinterpret_cast<const __attribute__((address_space(4))) T*>(reinterpret_cast<uintptr_t>(p))[i];
}

// The two kernels: work is counted in units, COLS columns of one kv head by
// UNIT positions.
struct Few {  // few_columns: each wave all columns, its own positions
    static constexpr bool MANY = false;
    static constexpr int COLS = kCols, UNIT = kUnit;
};
struct Prompt {  // many_columns: each wave its own columns, all positions
    static constexpr bool MANY = true;
    static constexpr int COLS = kPromptCols, UNIT = 64;
};

// A sequence as one of the kernels sees it: rows = 0 if it is the other's.
template <class KIND>
struct Seq {
    static constexpr bool BIG = KIND::MANY;
    static constexpr int COLS = KIND::COLS, UNIT = KIND::UNIT;
    int row0, rows, q_len, kv, cap, group;  // first row, rows computed, rows there are, positions, those the table has room for

    __device__ __forceinline__ Seq(const Q8Args& a, int row, int row_end, int len) : row0(row), group(a.group) {
        q_len = row_end > row ? row_end - row : 0;
        rows = q_len < a.max_q_len ? q_len : a.max_q_len;
        if ((rows * group > kCols) != BIG) rows = 0;
        cap = a.max_blocks << a.page_shift;
        kv = len < 0 ? 0 : len;
    }
    // of the same index in every lane
    static __device__ __forceinline__ Seq uniform(const Q8Args& a, int b) {
        return Seq(a, uniform_load(a.q_start, b), uniform_load(a.q_start, b + 1), uniform_load(a.kv_lens, b));
    }
    __device__ __forceinline__ int tiles() const { return (rows * group + COLS - 1) / COLS; }
    // Positions that row i sees: the last row the last one, whether the table reaches it or not.
    __device__ __forceinline__ int row_sees(int i) const {
        const int64_t n = static_cast<int64_t>(kv) - q_len + i + 1;
        return n < 0 ? 0 : n > cap ? cap : static_cast<int>(n);
    }
    // positions that the last column of a tile sees
    __device__ __forceinline__ int sees(int tile) const {
        const int i = (tile * COLS + COLS - 1) / group;
        return row_sees(i < q_len - 1 ? i : q_len - 1);
    }
    // units of one kv head's tile: one at least, which writes the zeros of rows that see nothing
    __device__ __forceinline__ int units(int tile) const {
        const int n = sees(tile);
        return n > UNIT ? (n + UNIT - 1) / UNIT : 1;
    }
    // What a tile of one kv head costs and what the tiles before it do, for the even split.  Few columns, so one
    // tile: its units.  Many: about the positions that its columns see and kBigItem more for beginning and ending an item,
    // times the group; a linear function of the tile, so that the sum needs no loop over the tiles.
    __device__ __forceinline__ int64_t slope() const {
        const int64_t n = static_cast<int64_t>(kv) - q_len + 1;
        return ((n < 1 ? 1 : n > cap ? cap : n) + kBigItem) * group - 1;
    }
    __device__ __forceinline__ int64_t cost(int tile) const {
        if constexpr (!BIG) return units(tile);
        else return slope() + static_cast<int64_t>(COLS) * (tile + 1);
    }
    __device__ __forceinline__ int64_t before(int tile) const {
        if constexpr (!BIG) {
            return tile ? units(0) : 0;
        } else {
            return slope() * tile + static_cast<int64_t>(COLS) * (static_cast<int64_t>(tile) * (tile + 1) / 2);
        }
    }
    __device__ __forceinline__ int64_t all(const Q8Args& a) const { return before(tiles()) * a.n_kv_heads; }
};

// 64-bit inclusive sum over a wave.
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int64_t up = __shfl_up(v, d);
        if (lane >= d) v += up;
    }
    return v;
}

// A value that is the same in every lane, where the compiler cannot know it.
__device__ __forceinline__ int64_t uniform64(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
    return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// x / y rounded down for numbers below 2^53, where the quotient in 64-bit
// floating point cannot be rounded up to a whole number it does not reach.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
    return static_cast<int64_t>(static_cast<double>(x) / static_cast<double>(y));
}

// The unit of a tile of many columns that a point `off` into its cost lies in.  The product passes 64 bits where a group
// of 256 heads meets 2^31 positions, so it is taken in 64-bit floating point, where it is as exact as the quotient.
__device__ __forceinline__ int unit_at(int64_t off, int units, int64_t cost) {
    return static_cast<int>(static_cast<double>(off) * units / static_cast<double>(cost));
}

// Workgroups that share the work: none without any.
__device__ __forceinline__ int sharers(int64_t total, int grid) {
    return total < grid ? static_cast<int>(total) : grid;
}

// Where workgroup w begins, when `grid` of them share `total`.
__device__ __forceinline__ int64_t cut(int w, int64_t total, int grid) { return quotient(w * total, grid); }

// A place in the work, in the order of sequences, kv heads, tiles and units.
// An item is a sequence's tile of one kv head.
struct Place {
    int seq, tile, head, unit, units;
    int64_t item, cost;  // where the item begins, and what it costs
};

// The place of each of N points at(i, total, grid) < total, by sums over the
// batch, and the total; grid becomes the number of sharers.  Returns false
// if there is no work or at(0, ..) is negative.
template <class KIND, int N, class F>
__device__ __forceinline__ bool find(const Q8Args& a, int* grid, int64_t* total, Place (&p)[N], F at) {
    __shared__ int64_t waves[kWaves];
    __shared__ int64_t found_before[N];
    __shared__ int found[N];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    int64_t point[N], before[N];
    const auto all_of = [&](int b) {
        return b < a.batch ? Seq<KIND>(a, a.q_start[b], a.q_start[b + 1], a.kv_lens[b]).all(a) : 0;
    };
    const auto points = [&]() {
        *total = uniform64(*total);
        *grid = sharers(*total, *grid);
        if (*grid == 0) return false;
#pragma unroll
        for (int i = 0; i < N; ++i) point[i] = uniform64(at(i, *total, *grid));
        return point[0] >= 0;
    };
    if (a.batch == 1) {
        *total = Seq<KIND>::uniform(a, 0).all(a);
        if (!points()) return false;
#pragma unroll
        for (int i = 0; i < N; ++i) p[i].seq = 0, before[i] = 0;
    } else if (a.batch <= kWave) {  // every wave for itself
        const int64_t mine = all_of(lane);
        const int64_t upto = wave_scan(mine);
        *total = __shfl(upto, kWave - 1);
        if (!points()) return false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int l = __builtin_ctzll(__ballot(upto > point[i]));
            p[i].seq = l;
            before[i] = __shfl(upto - mine, l);
        }
    } else {
        int64_t sum = 0;
        for (int pass = 0; pass < 2; ++pass) {
            if (pass) {
                *total = sum;
                if (!points()) return false;
                sum = 0;
            }
            for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
                const int64_t mine = all_of(b0 + tid);
                const int64_t upto = wave_scan(mine);
                __syncthreads();
                if (lane == kWave - 1) waves[wave] = upto;
                __syncthreads();
                int64_t pre = sum;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    if (w < wave) pre += waves[w];
                    sum += waves[w];
                }
                if (pass) {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (pre + upto > point[i] && pre + upto - mine <= point[i])
                            found[i] = b0 + tid, found_before[i] = pre + upto - mine;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) p[i].seq = found[i], before[i] = found_before[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        p[i].seq = __builtin_amdgcn_readfirstlane(p[i].seq);
        const Seq<KIND> s = Seq<KIND>::uniform(a, p[i].seq);
        const int64_t rest = point[i] - uniform64(before[i]);
        const int64_t per_head = s.before(s.tiles());
        p[i].head = __builtin_amdgcn_readfirstlane(static_cast<int>(quotient(rest, per_head)));
        const int64_t in_head = rest - p[i].head * per_head;
        int lo = 0, hi = s.tiles() - 1;  // the last tile that begins at or before it
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (s.before(mid) <= in_head) lo = mid;
            else hi = mid - 1;
        }
        p[i].tile = __builtin_amdgcn_readfirstlane(lo);
        p[i].units = s.units(p[i].tile);
        p[i].cost = s.cost(p[i].tile);
        const int64_t off = in_head - s.before(p[i].tile);
        p[i].item = point[i] - off;
        const int unit = KIND::MANY ? unit_at(off, p[i].units, p[i].cost) : static_cast<int>(off);
        p[i].unit = __builtin_amdgcn_readfirstlane(unit);
    }
    return true;
}

// A workgroup's share: from one place to another.
template <class KIND>
struct Share {
    Place p;
    int end_seq, end_tile, end_head, end_unit;

    // workgroup `me` of `grid`
    __device__ __forceinline__ bool find_mine(const Q8Args& a, int me, int grid) {
        int64_t total;
        Place ends[2];
        // the last place is in front of the next workgroup's first; the last workgroup's is the end of all
        bool to_end = false;
        if (!find<KIND, 2>(a, &grid, &total, ends, [&](int i, int64_t n, int g) -> int64_t {
                if (me >= g) return -1;
                if (i == 0) return cut(me, n, g);
                to_end = me + 1 == g;
                return to_end ? n - 1 : cut(me + 1, n, g);
            })) {
            if (threadIdx.x == 0) a.borders[me].grid = 0;
            return false;
        }
        p = ends[0];
        if (threadIdx.x == 0)
            a.borders[me] = Border{p.item, p.cost, total, p.seq, p.tile, p.head, p.unit, p.units, grid};
        __builtin_amdgcn_sched_barrier(0);  // or its values stay in registers that the products then lack
        end_seq = ends[1].seq;
        end_tile = ends[1].tile;
        end_head = ends[1].head;
        end_unit = to_end ? ends[1].units : ends[1].unit;
        return true;
    }
    // the end of this workgroup's units of the item p is in
    __device__ __forceinline__ bool in_last() const {
        return p.seq == end_seq && p.tile == end_tile && p.head == end_head;
    }
    __device__ __forceinline__ int last() const { return in_last() ? end_unit : p.units; }
    // To the next item; false past the end of the share.
    __device__ __forceinline__ bool next(const Q8Args& a) {
        if (in_last()) return false;
        p.unit = 0;
        Seq<KIND> s = Seq<KIND>::uniform(a, p.seq);
        if (++p.tile == s.tiles()) {
            p.tile = 0;
            if (++p.head == a.n_kv_heads) {
                p.head = 0;
                do s = Seq<KIND>::uniform(a, ++p.seq);
                while (s.rows == 0);  // the end lies in a sequence behind
            }
        }
        p.units = s.units(p.tile);
        return true;
    }
};

// Where a workgroup leaves its part of an item that it shares: the one that
// it ends (or passes through) and the one that it begins.  A part: per column
// the unnormalised output, then per column the running maximum and the sum.
__host__ __device__ __forceinline__ int64_t part_size(int cols, int hd) {
    return (static_cast<int64_t>(cols) * (hd + 2) + 3) / 4 * 4;
}
__device__ __forceinline__ float* part_at(const Q8Args& a, int wg, bool begins, int hd) {
    return a.ws + (wg * 2 + (begins ? 1 : 0)) * part_size(a.part_cols, hd);
}
__device__ __forceinline__ float* part_sums(const Q8Args& a, float* part, int hd) { return part + a.part_cols * hd; }

// The least that a V scale counts as when it becomes the unit of an output: the inverse of a subnormal number may be
// infinite.
constexpr float kLeastUnit = 0x1p-126f;

// y as the sum of two binary16 numbers, 22 bits of it.  The empty asm makes y
// one fp32 value: otherwise the product that it came from may be rounded to
// binary16 a second time, unrounded, and next to a tie that gives another
// first number than the one the second number completes.
__device__ __forceinline__ void split(float y, _Float16* hi, _Float16* lo) {
    asm volatile("" : "+v"(y));
    *hi = static_cast<_Float16>(y);
    *lo = static_cast<_Float16>(y - static_cast<float>(*hi));
}

template <int QT>
__device__ __forceinline__ void put(void* out, int64_t at, float v) {
    if constexpr (QT == FENCE_F32) static_cast<float*>(out)[at] = v;
    else static_cast<uint16_t*>(out)[at] = f32_to_f16_bits(v);
}

// Eight in a row.  a.wide: 16-byte aligned.
template <int QT>
__device__ __forceinline__ void put8(const Q8Args& a, int64_t at, const float* y) {
    if (!a.wide) {
#pragma unroll
        for (int i = 0; i < 8; ++i) put<QT>(a.out, at + i, y[i]);
    } else if constexpr (QT == FENCE_F32) {
        float* p = static_cast<float*>(a.out) + at;
        *reinterpret_cast<f4*>(p) = f4{y[0], y[1], y[2], y[3]};
        *reinterpret_cast<f4*>(p + 4) = f4{y[4], y[5], y[6], y[7]};
    } else {
        h8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = static_cast<_Float16>(y[i]);
        *reinterpret_cast<h8*>(static_cast<_Float16*>(a.out) + at) = h;
    }
}

// Codes to binary16, four bytes to two pairs.  int8: with the sign bit
// flipped, byte u under the exponent byte 0x64 is 1024 + u in binary16;
// 1152 less is the code.
template <int TYPE>
__device__ __forceinline__ void codes_h(uint32_t w, h2* lo, h2* hi) {
    if constexpr (TYPE == FENCE_KV_INT8) {
        const h2 off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
        w ^= 0x80808080u;
        *lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off;
        *hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off;
    } else {
        *lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        *hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    }
}

// The larger of lanes l and l + 32, for both.  The two operands are exchanged
// halfwise, so they have to be two registers; the empty asm keeps them apart.
__device__ __forceinline__ float halves_max(float v) {
    uint32_t x = __builtin_bit_cast(uint32_t, v), y = x;
    asm volatile("" : "+v"(x), "+v"(y));
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    x = r[0];
    y = r[1];
    asm volatile("" : "+v"(x), "+v"(y));
    return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}

__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) {
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Over the four 16-lane rows of a wave, for every lane.
template <class Op>
__device__ __forceinline__ float across_rows(float v, Op op) {
    v = op(v, __shfl_xor(v, 16));
    return op(v, __shfl_xor(v, 32));
}

// Single tokens and drafts.  A wave multiplies 32 positions (two groups of 16,
// each inside one page) by 16 columns at a time:
//   S' [16 positions x 16 columns] = K [16 x HD] Q' [HD x 16]
//   O' [HD x 16 columns] += V' [HD x 32 positions] P [32 x 16]
// The first product leaves lane (column r, row group g) with the positions
// 4 g .. 4 g + 3 of each group of 16, and those eight are what the second
// product takes from it as its k index, so P stays where it is.  A lane's
// dimensions are r * HD / 16 + i for product i, so it reads V with one load a
// position.  The next positions' codes are loaded before these are used.
//
// Bound by HBM where the batch is large: 64 tokens over 1.6 GB of int8 pages
// take 302 us, 5.4 TB/s.  One token at 2,916 positions takes 9 us and the join
// 6: the chain of place, page ids, codes, products and merge.
template <int TYPE, int QT, int HD>
__device__ __forceinline__ void few_columns(const Q8Args& a, float* lds, int me, int grid) {
    constexpr int PIECES = HD / 64;       // 64 dimensions of K: 16 a lane
    constexpr int DT = HD / 16;           // products over V; also dimensions a lane reads of a position
    constexpr int VW = DT / 4;            // words of them
    constexpr bool F32 = QT == FENCE_F32;
    constexpr int PARTS = F32 ? 2 : 1;    // binary16 numbers that hold a q or a p
    const int tid = threadIdx.x, lane = tid % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int r = lane % 16, g = lane / 16;
    const int hd = a.head_dim, page_mask = (1 << a.page_shift) - 1;

    Share<Few> share;
    if (!share.find_mine(a, me, grid)) return;
    do {
        const Seq<Few> s = Seq<Few>::uniform(a, share.p.seq);
        const int tile = share.p.tile, head = share.p.head, first = share.p.unit, units = share.p.units;
        const int last = share.last();
        if (first >= last) continue;  // a share has at least one unit, but its end may be an item's beginning
        const int cols = s.rows * a.group - tile * kCols < kCols ? s.rows * a.group - tile * kCols : kCols;
        // this lane's column
        const int col = tile * kCols + r;
        const int row = col / a.group;
        const bool mine = r < cols;
        const int qhead = head * a.group + col % a.group;
        const int sees = mine ? s.row_sees(row) : 0;
        const int end = s.sees(tile);
        const int least = s.row_sees(tile * kCols / a.group);  // what every column sees

        // The codes of 32 positions; none of those that are not there.
        struct Codes {
            u4 k[2][PIECES];
            uint32_t v[8][VW];
            float ks[2], vs[2];
            bool ok[2];  // the page is there
        };
        const int64_t table = static_cast<int64_t>(share.p.seq) * a.max_blocks;
        const auto page_of = [&](int un, int t) {
            const int pos = un * kUnit + wave * 32 + 16 * t;
            return un < last && pos < end ? uniform_load(a.table, table + (pos >> a.page_shift)) : -1;
        };
        const auto load = [&](Codes& c, int un, const int (&ids)[2]) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int pos = un * kUnit + wave * 32 + 16 * t;
                c.ok[t] = ids[t] >= 0 && ids[t] < a.n_pages;
                const int64_t base = static_cast<int64_t>(c.ok[t] ? ids[t] : 0) * a.n_kv_heads + head;
                c.ks[t] = c.ok[t] ? uniform_load(a.ks, base) : 0.0f;
                c.vs[t] = c.ok[t] ? uniform_load(a.vs, base) : 0.0f;
                const int64_t at = ((base << a.page_shift) + (pos & page_mask)) * hd;
                const uint8_t* k = a.k + at + r * hd;
                const uint8_t* v = a.v + at + g * 4 * hd + r * DT;
#pragma unroll
                for (int p = 0; p < PIECES; ++p) {
                    const int d = p * 64 + g * 16;
                    c.k[t][p] = u4{0, 0, 0, 0};
                    if (c.ok[t] && d < hd) c.k[t][p] = *reinterpret_cast<const u4*>(k + d);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int w = 0; w < VW; ++w) c.v[4 * t + i][w] = 0;
                    if (c.ok[t] && pos + g * 4 + i < end && r * DT < hd) {
#pragma unroll
                        for (int w = 0; w < VW; ++w) c.v[4 * t + i][w] = reinterpret_cast<const uint32_t*>(v + i * hd)[w];
                    }
                }
            }
        };
        int ids[2] = {page_of(first, 0), page_of(first, 1)};
        Codes now, then;
        load(now, first, ids);

        h8 qf[PARTS][PIECES][2];
        float unscale = a.scale_log2;
        {
            const int64_t at = mine ? static_cast<int64_t>(s.row0 + row) * a.ldq + static_cast<int64_t>(qhead) * hd : 0;
            if constexpr (F32) {
                // q times a power of two that brings the row's largest value to 2^14, as the sum of two
                // binary16 numbers: 22 bits of it
                float x[PIECES][16];
                float most = 0.0f;
#pragma unroll
                for (int p = 0; p < PIECES; ++p) {
                    const int d = p * 64 + g * 16;
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[p][i] = 0.0f;
                    if (mine && d < hd) {
                        const float* src = static_cast<const float*>(a.q) + at + d;
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[p][i] = src[i];
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(x[p][i]));
                }
                most = across_rows(most, OpMax{});
                uint32_t e = __builtin_bit_cast(uint32_t, most) >> 23;
                e = e < 15 ? 15 : e > 254 ? 254 : e;
                const float up = __builtin_bit_cast(float, (268 - e) << 23);
                unscale *= __builtin_bit_cast(float, (e - 14) << 23);
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        _Float16 hi, lo;
                        split(x[p][i] * up, &hi, &lo);
                        qf[0][p][i / 8][i % 8] = hi;
                        qf[1][p][i / 8][i % 8] = lo;
                    }
            } else {
#pragma unroll
                for (int p = 0; p < PIECES; ++p) {
                    const int d = p * 64 + g * 16;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        h8 x = {};
                        if (mine && d < hd) {
                            const _Float16* src = static_cast<const _Float16*>(a.q) + at + d + 8 * j;
#pragma unroll
                            for (int i = 0; i < 8; ++i) x[i] = src[i];
                        }
                        qf[0][p][j] = x;
                    }
                }
            }
        }

        f4 o[DT];
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -__builtin_inff(), l = 0.0f;
        float vref = 0.0f;  // the largest V scale so far: o is in units of it times 2^-14

        const auto turn = [&](const Codes& c, int pos0, auto masked) {
            f4 st[2];
            float top = m;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        h2 c0, c1, c2, c3;
                        codes_h<TYPE>(c.k[t][p][2 * j], &c0, &c1);
                        codes_h<TYPE>(c.k[t][p][2 * j + 1], &c2, &c3);
                        const h8 kf = join(c0, c1, c2, c3);
#pragma unroll
                        for (int x = 0; x < PARTS; ++x)
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[x][p][j], acc, 0, 0, 0);
                    }
                const float f = c.ks[t] * unscale;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    st[t][i] = acc[i] * f;
                    if (!c.ok[t] || (masked && pos0 + 16 * t + g * 4 + i >= sees)) st[t][i] = -__builtin_inff();
                    top = fmaxf(top, st[t][i]);
                }
            }
            top = across_rows(top, OpMax{});
            float vtop = vref;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (c.vs[t] > vtop && c.vs[t] < __builtin_inff()) vtop = fmaxf(c.vs[t], kLeastUnit);
            if (__any(top > m) || vtop > vref) {
                const float alpha = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - top);
                const float beta = vtop > 0.0f ? alpha * (vref * __builtin_amdgcn_rcpf(vtop)) : 0.0f;
                m = top;
                vref = vtop;
                l *= alpha;
#pragma unroll
                for (int i = 0; i < DT; ++i) o[i] *= beta;
            }
            const float ref = m == -__builtin_inff() ? 0.0f : m;
            const float to_v = vref > 0.0f ? __builtin_amdgcn_rcpf(vref) : 0.0f;
            h8 pf[PARTS];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const float f = c.vs[t] * to_v * 16384.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(st[t][i] - ref);
                    l += p;
                    float y = p * f;
                    if (masked && p == 0.0f) y = 0.0f;  // behind a scale that is not finite
                    if constexpr (F32) {
                        _Float16 hi, lo;
                        split(y, &hi, &lo);
                        pf[0][4 * t + i] = hi;
                        pf[1][4 * t + i] = lo;
                    } else {
                        pf[0][4 * t + i] = static_cast<_Float16>(y);
                    }
                }
            }
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                h2 x[4][4];  // [pair of positions][dimension of the word]
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t y = c.v[2 * j][w], z = c.v[2 * j + 1][w];
                    codes_h<TYPE>(__builtin_amdgcn_perm(z, y, 0x05010400u), &x[j][0], &x[j][1]);
                    codes_h<TYPE>(__builtin_amdgcn_perm(z, y, 0x07030602u), &x[j][2], &x[j][3]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const h8 vf = join(x[0][i], x[1][i], x[2][i], x[3][i]);
#pragma unroll
                    for (int k = 0; k < PARTS; ++k)
                        o[4 * w + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[k], o[4 * w + i], 0, 0, 0);
                }
            }
        };

        ids[0] = page_of(first + 1, 0);
        ids[1] = page_of(first + 1, 1);
#pragma unroll 1
        for (int un = first; un < last; ++un) {
            const int pos0 = un * kUnit + wave * 32;
            if (pos0 >= end) break;
            load(then, un + 1, ids);
            ids[0] = page_of(un + 2, 0);
            ids[1] = page_of(un + 2, 1);
            if (pos0 + 32 <= least) turn(now, pos0, std::false_type{});
            else turn(now, pos0, std::true_type{});
            now = then;
        }

        // The waves' parts together: lane (r, g) has dimensions (4 g + j) * DT + i of column r in o[i][j].
        l = across_rows(l, OpAdd{});
        const int pc = a.part_cols;
        float* mo = lds;                               // [wave][column][HD]
        float* ml = lds + kWaves * pc * HD;            // [wave][column][2]
        if (mine) {
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    mo[(wave * pc + r) * HD + (4 * g + j) * DT + i] = o[i][j] * 0x1p-14f * vref;
            if (g == 0) {
                ml[(wave * pc + r) * 2] = m;
                ml[(wave * pc + r) * 2 + 1] = l;
            }
        }
        __syncthreads();
        const bool whole = first == 0 && last == units;
        float* part = part_at(a, me, first == 0, HD);
        for (int x = tid; x < cols * HD; x += kThreads) {
            const int c = x / HD, d = x % HD;
            float top = -__builtin_inff();
#pragma unroll
            for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[(w * pc + c) * 2]);
            const float ref = top == -__builtin_inff() ? 0.0f : top;
            float sum = 0.0f, val = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(ml[(w * pc + c) * 2] - ref);
                sum += f * ml[(w * pc + c) * 2 + 1];
                val += f * mo[(w * pc + c) * HD + d];
            }
            if (whole) {
                if (d < hd) {
                    const int cc = tile * kCols + c;
                    const int64_t to = static_cast<int64_t>(s.row0 + cc / a.group) * a.ldo +
                                       static_cast<int64_t>(head * a.group + cc % a.group) * hd + d;
                    put<QT>(a.out, to, sum != 0.0f ? val / sum : 0.0f);
                }
            } else {
                part[c * HD + d] = val;
                if (d == 0) {
                    float* to = part_sums(a, part, HD) + 2 * c;
                    to[0] = top, to[1] = sum;
                }
            }
        }
        __syncthreads();
    } while (share.next(a));
}

// Prompts: a workgroup takes kPromptCols columns, 32 a wave, and 64 positions
// at a time, whose codes it converts once into LDS for all of its columns:
//   S' [32 positions x 32 columns] = K [32 x HD] Q' [HD x 32],  twice
//   O' [HD x 32 columns] += V' [HD x 64 positions] P [64 x 32]
// LDS holds the fragments as the products read them (16 bytes a lane, lanes in
// a row, so reads and writes meet no bank twice).  The first product leaves
// lane (column n, half g) with positions 8 q + 4 g + (0 .. 3) of 32, which
// the second takes as its k index in that order, so P stays in registers; row
// r of V' product t stands for dimension r * HD / 32 + t, so a thread that
// converts 4 dimensions of 8 positions writes whole fragments, and a lane ends
// with runs of 4 * HD / 32 dimensions of its column.
//
// Wave w converts positions 16 w .. 16 w + 15, which lie in one page, so its
// addresses are a scalar and a 32-bit offset a lane.  Codes are loaded two
// turns ahead and converted one turn ahead, into the other half of LDS, with
// one barrier a turn.  The vector pipe is the narrow one (an exponential is
// 16 clocks, a conversion about 6 a code), and it can run behind a product
// that takes 32 clocks, so the conversion stands beside the first products
// and the exponentials of 16 positions beside the second products of the 16
// before; the scheduling groups keep the compiler to that and its LDS reads
// ahead.  (Two column tiles a wave would halve what a column pays for
// conversions and LDS reads, but take all registers of a SIMD for one wave:
// 8,192 rows in 1,130 us where this form, in an earlier state, took 868.)
//
// Two waves share a SIMD, and of two that are ready the older one goes first,
// so one workgroup of a CU would run a quarter faster and leave the other
// alone at the end.  With the second half of a turn at the higher priority
// both keep the same pace and one's products stand beside the other's
// exponentials: 736 us for 8,192 rows against 770, and 742 with the first half
// at the higher one.
//
// binary16 (QT = FENCE_F16): with the page's V scale in the exponent, one
// fused multiply-add and one exponential make the probability that the
// product takes.  The sum takes it before it is rounded, in fp32, and with the
// V scale taken out again: rounded, a page's weight would be lost where its
// V scale is small beside another's.
// The running maximum and the largest V scale are only moved when a value
// would grow past 2^15 (kSlack), so O is rarely rescaled.
//
// 8,192 rows of 32 heads over 8 by 128 dimensions take 736 us in binary16 (716
// to 757 from machine to machine), 747 TFLOP/s, with the MFMA pipes busy for a
// third of it and the vector pipe for most of the rest; 3,000 rows in fp32
// (twice the products) 131 us, 302 TFLOP/s of the result's.
template <int HD>
struct PromptLds {
    // A half in 16-byte pieces: K fragments [2][HD / 16][64 lanes], V fragments [4][HD / 32][64 lanes], per 16
    // positions K scale (-1 if the page is not there), V scale and its log2, and a place for each lane to write what
    // nobody reads.
    static constexpr int V0 = HD / 8 * kWave, S0 = V0 + HD / 8 * kWave, X0 = S0 + 4, HALF = X0 + kWave;
};

template <int TYPE, int QT, int HD>
__device__ __forceinline__ void many_columns(const Q8Args& a, h8* buf, int me, int grid) {
    constexpr bool F32 = QT == FENCE_F32;
    constexpr int PARTS = F32 ? 2 : 1;
    constexpr int KS = HD / 16;   // k steps of the first product
    constexpr int NT = HD / 32;   // products over V
    constexpr int KJ = HD / 64;   // 16-byte pieces of K a lane converts
    constexpr int VJ = HD <= 128 ? 1 : 2;  // 8 positions x 4 dimensions of V a lane converts
    constexpr float kBase = F32 ? 14.0f : 10.0f;  // log2 of what stands for 1 times the largest V scale
    constexpr float kSlack = F32 ? 0.0f : 4.0f;
    constexpr int V0 = PromptLds<HD>::V0, S0 = PromptLds<HD>::S0, X0 = PromptLds<HD>::X0, HALF = PromptLds<HD>::HALF;
    const int tid = threadIdx.x, lane = tid % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int n = lane % 32, g = lane / 32;
    const int hd = a.head_dim, page_mask = (1 << a.page_shift) - 1;

    Share<Prompt> share;
    if (!share.find_mine(a, me, grid)) return;
    // What this lane converts: K position lane % 16, dimensions 16 (lane / 16 + 4 j) on; V positions 4 vg + (0 .. 3)
    // and 8 more, dimensions vd on.  At HD = 64 the upper lanes load the V that the lower ones do.
    const int kr = lane % 16, kc = lane / 16;
    const int vd = HD == 256 ? lane * 4 : lane % (HD / 4) * 4;
    const int vg = HD == 256 ? 0 : lane / (HD / 4) % 2;
    const bool vmine = (HD == 64 ? lane < 32 : true) && vd < hd;
    int kto[KJ], vto[4], sto;  // where to
#pragma unroll
    for (int j = 0; j < KJ; ++j)
        kto[j] = (kc + 4 * j) * 16 < hd ? (wave / 2 * KS + kc + 4 * j) * kWave + (wave % 2) * 16 + kr : X0 + kr;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        vto[i] = vmine ? V0 + (wave * NT + (vd + i) % NT) * kWave + vg * 32 + (vd + i) / NT : -1;
    sto = lane == 0 ? S0 + wave : X0 + lane;
    if (hd < HD) {  // dimensions that are not there stay zero
        const h8 zero = {};
        for (int i = tid; i < 2 * HALF; i += kThreads) buf[i] = zero;
        __syncthreads();
    }
    do {
        const Seq<Prompt> s = Seq<Prompt>::uniform(a, share.p.seq);
        const int tile = share.p.tile, head = share.p.head, first = share.p.unit, units = share.p.units;
        const int last = share.last();
        const int cols = s.rows * a.group - tile * Prompt::COLS;
        const int c = wave * 32 + n;  // this lane's column
        const bool mine = c < cols;
        const int row = (tile * Prompt::COLS + c) / a.group;
        const int qhead = head * a.group + (tile * Prompt::COLS + c) % a.group;
        const int sees = mine ? s.row_sees(row) : 0;
        const int end = s.sees(tile);
        if (first >= last) {
            // Nothing of this item; if others take what is before and after, the join finds an empty part.
            if (first > 0 && mine && g == 0) {
                float* ml = part_sums(a, part_at(a, me, false, HD), HD) + 2 * c;
                ml[0] = -__builtin_inff(), ml[1] = 0.0f;
            }
            continue;
        }
        // what every column of this wave sees
        const int least = s.row_sees((tile * Prompt::COLS + wave * 32) / a.group);
        const int64_t table = static_cast<int64_t>(share.p.seq) * a.max_blocks;

        // The page of this wave's 16 positions of a unit.
        const auto page_of = [&](int un) {
            const int pos = un * Prompt::UNIT + wave * 16;
            const int id = un < last && pos < end ? uniform_load(a.table, table + (pos >> a.page_shift)) : -1;
            return id < a.n_pages ? id : -1;
        };
        u4 kw[KJ];
        uint32_t vw[VJ][8];
        float ks, vs;
        // the codes of a unit, of page 0 if the page is not there
        const auto load = [&](int un, int id) {
            const int64_t base = static_cast<int64_t>(id < 0 ? 0 : id) * a.n_kv_heads + head;
            const int64_t at = ((base << a.page_shift) + ((un * Prompt::UNIT + wave * 16) & page_mask)) * hd;
            const uint8_t* k = a.k + at;
            const uint8_t* v = a.v + at;
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                const uint32_t d = (kc + 4 * j) * 16;
                kw[j] = *reinterpret_cast<const u4*>(k + static_cast<uint32_t>(kr * hd) + (d < static_cast<uint32_t>(hd) ? d : 0));
            }
#pragma unroll
            for (int j = 0; j < VJ; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    vw[j][i] = *reinterpret_cast<const uint32_t*>(
                        v + ((i / 4) * 8 + i % 4) * hd +
                        (static_cast<uint32_t>((vg + j) * 4 * hd) + static_cast<uint32_t>(vd < hd ? vd : 0)));
        };
        const auto scales = [&](int id) {
            const int64_t base = static_cast<int64_t>(id < 0 ? 0 : id) * a.n_kv_heads + head;
            const float x = uniform_load(a.ks, base), y = uniform_load(a.vs, base);
            ks = id < 0 ? -1.0f : x;
            vs = id < 0 ? 0.0f : y;
        };
        // V codes of positions past the end: an e4m3 one may be NaN, which no weight of 0 removes.
        const auto trim = [&](int un) {
            const int pos0 = un * Prompt::UNIT + wave * 16;
            if (TYPE == FENCE_KV_E4M3 && pos0 + 16 > end) {
#pragma unroll
                for (int j = 0; j < VJ; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (pos0 + (vg + j) * 4 + (i / 4) * 8 + i % 4 >= end) vw[j][i] = 0;
            }
        };
        // Into a half of LDS.  V codes of pages that are not there or whose scale is 0 become 0.
        const auto convert = [&](h8* half) {
#pragma unroll
            for (int j = 0; j < KJ; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    h2 c0, c1, c2, c3;
                    codes_h<TYPE>(kw[j][2 * i], &c0, &c1);
                    codes_h<TYPE>(kw[j][2 * i + 1], &c2, &c3);
                    half[kto[j] + i * 32] = join(c0, c1, c2, c3);
                }
            const uint32_t keep = vs == 0.0f ? 0u : ~0u;
#pragma unroll
            for (int j = 0; j < VJ; ++j) {
                h2 x[4][4];
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const uint32_t y = vw[j][2 * p] & keep, z = vw[j][2 * p + 1] & keep;
                    codes_h<TYPE>(__builtin_amdgcn_perm(z, y, 0x05010400u), &x[p][0], &x[p][1]);
                    codes_h<TYPE>(__builtin_amdgcn_perm(z, y, 0x07030602u), &x[p][2], &x[p][3]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    half[vto[i] < 0 ? X0 + lane : vto[i] + j * 32] = join(x[0][i], x[1][i], x[2][i], x[3][i]);
            }
            *reinterpret_cast<f4*>(half + sto) = f4{ks, vs, __builtin_amdgcn_logf(vs), 0.0f};
        };

        int id_next = page_of(first);
        load(first, id_next);
        scales(id_next);
        id_next = page_of(first + 1);

        h8 qf[PARTS][KS];
        float unscale = a.scale_log2;
        {
            const int64_t from = mine ? static_cast<int64_t>(s.row0 + row) * a.ldq + static_cast<int64_t>(qhead) * hd : 0;
            if constexpr (F32) {
                float x[KS][8], biggest = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[k][i] = 0.0f;
                    if (mine && k * 16 < hd) {
                        const float* src = static_cast<const float*>(a.q) + from + k * 16 + g * 8;
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[k][i] = src[i];
                    }
                }
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int i = 0; i < 8; ++i) biggest = fmaxf(biggest, fabsf(x[k][i]));
                biggest = fmaxf(biggest, __shfl_xor(biggest, 32));
                uint32_t e = __builtin_bit_cast(uint32_t, biggest) >> 23;
                e = e < 15 ? 15 : e > 254 ? 254 : e;
                const float up = __builtin_bit_cast(float, (268 - e) << 23);
                unscale *= __builtin_bit_cast(float, (e - 14) << 23);
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        _Float16 hi, lo;
                        split(x[k][i] * up, &hi, &lo);
                        qf[0][k][i] = hi;
                        qf[1][k][i] = lo;
                    }
            } else {
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    h8 y = {};
                    if (mine && k * 16 < hd) {
                        const _Float16* src = static_cast<const _Float16*>(a.q) + from + k * 16 + g * 8;
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[i] = src[i];
                    }
                    qf[0][k] = y;
                }
            }
        }

        f16v o[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
        float m = -__builtin_inff(), l = 0.0f, vref = 0.0f;
        trim(first);
        convert(buf + (first & 1) * HALF);
        load(first + 1, id_next);
        scales(id_next);
        id_next = page_of(first + 2);
        __syncthreads();

        const auto turn = [&](int un, auto masked) {
            __builtin_amdgcn_s_setprio(0);
            const h8* half = buf + (un & 1) * HALF;
            const int pos0 = un * Prompt::UNIT;
            trim(un + 1);
            f16v st[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 16; ++i) st[h][i] = 0.0f;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const h8 kf = half[(h * KS + k) * kWave + lane];
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
                        st[h] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[p][k], st[h], 0, 0, 0);
                }
            f4 sc[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) sc[q] = *reinterpret_cast<const f4*>(half + S0 + q);
            convert(buf + ((un + 1) & 1) * HALF);
            // LDS reads kAhead fragments ahead of the products, and the conversion between them
            constexpr int kAhead = 4, kEach = 128 * HD / 128 / (2 * KS) + 1;
            __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
            for (int i = 0; i < 2 * KS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, PARTS, 0);
                if (i < 2 * KS - kAhead + 4) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, kEach, 0);
                __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            load(un + 2, id_next);
            // Scalar loads here, where no LDS read is waited for: with one in flight such a wait is for all.
            scales(id_next);
            id_next = page_of(un + 3);

            bool in[4];
            float vtop = vref;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                in[q] = !(sc[q][0] < 0.0f);
                if (sc[q][1] > vtop && sc[q][1] < __builtin_inff()) vtop = fmaxf(sc[q][1], kLeastUnit);
            }
            const bool grow_v = vtop > (F32 ? vref : 2.0f * vref);
            const float vnow = grow_v ? vtop : vref;
            const float vone = vnow > 0.0f ? __builtin_amdgcn_rcpf(vnow) : 0.0f;
            const float vlog = vnow > 0.0f ? __builtin_amdgcn_logf(vnow) : 0.0f;
            const int limit = sees - pos0 - g * 4;  // of this lane's positions: those below it are seen
            const auto seen = [&](int h, int i) { return h * 32 + (i / 4) * 8 + i % 4 < limit; };
            if (masked) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!seen(h, i)) st[h][i] = -__builtin_inff();
            }
            // In place of a page that is not there page 0's codes were multiplied: a NaN among them (e4m3), or a q that
            // is not finite, would pass the weight of 0.  The same branch in every lane.
            if (__any(!(in[0] && in[1] && in[2] && in[3]))) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (!in[q]) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) st[q / 2][(q % 2) * 8 + i] = 0.0f;
                    }
            }
            float top = -__builtin_inff();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float t = st[q / 2][(q % 2) * 8];
#pragma unroll
                for (int i = 1; i < 8; ++i) t = fmaxf(t, st[q / 2][(q % 2) * 8 + i]);
                // scales are not negative, so the largest product is the largest score
                t = in[q] && t > -__builtin_inff() ? t * (sc[q][0] * unscale) : -__builtin_inff();
                top = fmaxf(top, t);
            }
            top = halves_max(top);
            if (__any(top > m + kSlack || grow_v)) {
                const float now = fmaxf(m, top);
                const float alpha = now == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - now);
                const float beta = alpha * (vref * vone);
                m = now;
                vref = vnow;
                l *= alpha;
#pragma unroll
                for (int t = 0; t < NT; ++t) o[t] *= beta;
            }
            const float ref = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                h8 pf[PARTS];
                const float fk = sc[q][0] * unscale;
                if constexpr (F32) {
                    const float to_v = sc[q][1] * vone * 16384.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float p = __builtin_amdgcn_exp2f(st[q / 2][(q % 2) * 8 + i] * fk - ref);
                        if (!in[q] || (masked && !seen(q / 2, (q % 2) * 8 + i))) p = 0.0f;
                        l += p;
                        const float y = masked && p == 0.0f ? 0.0f : p * to_v;
                        _Float16 hi, lo;
                        split(y, &hi, &lo);
                        pf[0][i] = hi;
                        pf[PARTS - 1][i] = lo;
                    }
                } else {
                    // The page's V scale in units of the largest, as a power of two.  Below 2^-60 none of it is left in
                    // binary16, but the weight has to stay; V codes under a scale of 0 are zero.  NaN stays NaN.
                    float rel = sc[q][2] - vlog;
                    rel = rel < -60.0f ? -60.0f : rel;
                    const float shift = in[q] ? rel + (kBase - ref) : -__builtin_inff();
                    float p[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[q / 2][(q % 2) * 8 + i], fk, shift));
                        if (masked && !seen(q / 2, (q % 2) * 8 + i)) p[i] = 0.0f;
                        pf[0][i] = static_cast<_Float16>(p[i]);
                    }
                    const float sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                    // no weight under a scale that is NaN: none of the page's positions is seen
                    if (!(masked && sum == 0.0f)) l += sum * __builtin_amdgcn_exp2f(-kBase - rel);
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const h8 vf = half[V0 + (q * NT + t) * kWave + lane];
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
                        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[p], o[t], 0, 0, 0);
                }
            }
            __syncthreads();
        };
        // The waves turn together; each masks from where its first column ends.
        int un = first;
#pragma unroll 1
        for (; un < last && (un + 1) * Prompt::UNIT <= least; ++un) turn(un, std::false_type{});
#pragma unroll 1
        for (; un < last; ++un) turn(un, std::true_type{});

        // o[t][i] is dimension (8 (i / 4) + 4 g + i % 4) * NT + t of this lane's column: runs of 4 NT.
        const float sum = l + __shfl_xor(l, 32);
        if (mine) {
            const bool whole = first == 0 && last == units;
            const float one = F32 ? 0x1p-14f : 0x1p-10f;  // o is in units of vref times this; vref last, it may be tiny
            const float f = whole ? (sum != 0.0f ? one / sum : 0.0f) : one;
            float* part = part_at(a, me, first == 0, HD);
            const int64_t to = static_cast<int64_t>(s.row0 + row) * a.ldo + static_cast<int64_t>(qhead) * hd;
            if (!whole && g == 0) {
                float* ml = part_sums(a, part, HD) + 2 * c;
                ml[0] = m, ml[1] = sum;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int z = 0; z < 4 * NT; z += 8) {
                    const int d = (8 * q + 4 * g) * NT + z;
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int j = (z + i) / NT, t = (z + i) % NT;
                        y[i] = whole && sum == 0.0f ? 0.0f : o[t][4 * q + j] * f * vref;
                    }
                    if (whole) {
                        if (d < hd) put8<QT>(a, to + d, y);
                    } else {
                        float* p = part + c * HD + d;
                        *reinterpret_cast<f4*>(p) = f4{y[0], y[1], y[2], y[3]};
                        *reinterpret_cast<f4*>(p + 4) = f4{y[4], y[5], y[6], y[7]};
                    }
                }
        }
    } while (share.next(a));
}

template <int TYPE, int QT, int HD>
__global__ __launch_bounds__(kThreads, HD == 256 ? 1 : 2) void attention_q8_kernel(Q8Args a) {
    extern __shared__ float lds[];
    few_columns<TYPE, QT, HD>(a, lds, blockIdx.x, gridDim.x);
}

// Both in one launch, for batches that may hold prompts: the workgroups that
// take few columns come behind those of the prompts and fill what these leave.
template <int TYPE, int QT, int HD>
__global__ __launch_bounds__(kThreads, HD == 256 ? 1 : 2) void mixed_q8_kernel(Q8Args many, int many_grid, Q8Args few) {
    __shared__ h8 buf[2 * PromptLds<HD>::HALF];
    static_assert(sizeof(buf) >= kWaves * kCols * (HD + 2) * sizeof(float), "the other kernel's LDS");
    const int wg = blockIdx.x;
    // Workgroups go to the XCDs in turn; shares that follow one another, mostly tiles of one kv head, to one XCD's L2:
    // 736 us for 8,192 rows against 780, 28.7 against 31.5 for 24 x 5 drafted rows; six chunks of 500 rows take 151 both
    // ways in binary16, 131 against 128 in fp32.
    const int each = many_grid / kXcds;
    const int share = each * kXcds == many_grid ? wg % kXcds * each + wg / kXcds : wg;
    if (wg < many_grid) many_columns<TYPE, QT, HD>(many, buf, share, many_grid);
    else few_columns<TYPE, QT, HD>(few, reinterpret_cast<float*>(buf), wg - many_grid, gridDim.x - many_grid);
}

// Workgroups that join an item of many columns.  24 sequences of 35 columns take 9.2 us with 4, 13.6 with 2 and 10.4
// with 8; 3,000 rows in six prompts 18.0, 23.2 and 16.4 us; a prompt of 8,192 rows 19.9, 18.5 and 20.1.
constexpr int kJoinWide = 4;

// Joins the parts of the items that more than one workgroup took, in workgroup
// order.  Workgroup x looks at the border between workgroups x and x + 1 of
// the other kernel: if it is the first border inside an item, the item's
// columns are its to join, together with the other workgroups of the same x,
// a run of 4 dimensions a thread.
template <int QT, int HD, class KIND>
__device__ __forceinline__ void join_at(const Q8Args& a, int w0, int y, int ys) {
    struct Raw {
        u4 w[sizeof(Border) / 16];
    } raw;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(Border) / 16); ++i)
        raw.w[i] = uniform_load(reinterpret_cast<const u4*>(a.borders + w0 + 1), i);
    const Border p = __builtin_bit_cast(Border, raw);
    const int grid = p.grid;
    const int64_t total = p.total;
    if (grid == 0 || p.unit == 0) return;
    const int64_t off0 = cut(w0, total, grid) - p.item;  // the border before
    if (off0 > 0 && (KIND::MANY ? unit_at(off0, p.units, p.cost) : off0) > 0) return;
    // the workgroup whose share holds the item's end
    const int64_t end = p.item + p.cost;
    int w_end = static_cast<int>(quotient(end * grid - 1, total));
    while (w_end + 1 < grid && cut(w_end + 1, total, grid) < end) ++w_end;
    while (w_end > w0 + 1 && cut(w_end, total, grid) >= end) --w_end;
    w_end = __builtin_amdgcn_readfirstlane(w_end);
    const Seq<KIND> s = Seq<KIND>::uniform(a, p.seq);
    const int col0 = p.tile * Seq<KIND>::COLS;
    const int left = s.rows * a.group - col0;
    const int cols = left < Seq<KIND>::COLS ? left : Seq<KIND>::COLS;
    const int hd = a.head_dim;
    const int step = ys * kThreads, all = cols * (HD / 4);
    // RUNS runs of this thread at once and AHEAD parts of each, whose loads are in flight together.
    const auto join = [&](auto runs, auto ahead) {
        constexpr int RUNS = decltype(runs)::value, AHEAD = decltype(ahead)::value;
        for (int x0 = y * kThreads + threadIdx.x; x0 < all; x0 += RUNS * step) {
            float top[RUNS], sum[RUNS];
            f4 val[RUNS];
#pragma unroll
            for (int r = 0; r < RUNS; ++r) top[r] = -__builtin_inff(), sum[r] = 0.0f, val[r] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            for (int w = w0; w <= w_end; w += AHEAD) {
                float m[RUNS][AHEAD], l[RUNS][AHEAD];
                f4 v[RUNS][AHEAD];
#pragma unroll
                for (int r = 0; r < RUNS; ++r) {
                    const int x = x0 + r * step < all ? x0 + r * step : x0;
                    const int c = x / (HD / 4), d = x % (HD / 4) * 4;
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i) {
                        const int ww = w + i <= w_end ? w + i : w_end;
                        float* part = part_at(a, ww, ww == w0, HD);
                        const float* ml = part_sums(a, part, HD) + 2 * c;
                        m[r][i] = ml[0];
                        l[r][i] = ml[1];
                        v[r][i] = *reinterpret_cast<const f4*>(part + c * HD + d);
                    }
                }
#pragma unroll
                for (int r = 0; r < RUNS; ++r) {
                    float most = top[r];
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i) most = fmaxf(most, m[r][i]);
                    const float ref = most == -__builtin_inff() ? 0.0f : most;
                    const float f0 = __builtin_amdgcn_exp2f(top[r] - ref);
                    sum[r] *= f0;
                    val[r] *= f0;
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i) {
                        // a sum of 0: nothing seen, or a share without units, which leaves no output
                        if (w + i <= w_end && l[r][i] != 0.0f) {
                            const float f = __builtin_amdgcn_exp2f(m[r][i] - ref);
                            sum[r] += f * l[r][i];
                            val[r] += v[r][i] * f;
                        }
                    }
                    top[r] = most;
                }
            }
#pragma unroll
            for (int r = 0; r < RUNS; ++r) {
                const int x = x0 + r * step, d = x % (HD / 4) * 4;
                if (x >= all || d >= hd) continue;
                const int cc = col0 + x / (HD / 4);
                const int64_t to = static_cast<int64_t>(s.row0 + cc / a.group) * a.ldo +
                                   static_cast<int64_t>(p.head * a.group + cc % a.group) * hd + d;
#pragma unroll
                for (int i = 0; i < 4; ++i) put<QT>(a.out, to + i, sum[r] != 0.0f ? val[r][i] / sum[r] : 0.0f);
            }
        }
    };
    const int parts = w_end - w0 + 1;
    if (parts <= 2) join(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
    else join(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
}

// The borders of both kernels in one launch: first those of the prompts.
template <int QT, int HD>
__global__ __launch_bounds__(kThreads) void join_q8_kernel(Q8Args many, int many_grid, Q8Args few) {
    const int of_many = many_grid > 1 ? (many_grid - 1) * kJoinWide : 0, x = blockIdx.x;
    if (x < of_many) join_at<QT, HD, Prompt>(many, x / kJoinWide, x % kJoinWide, kJoinWide);
    else join_at<QT, HD, Few>(few, x - of_many, 0, 1);
}

int padded(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

bool big(int max_q_len, int group) { return static_cast<int64_t>(max_q_len) * group > kCols; }

int part_cols(int max_q_len, int group, bool is_big) {
    const int64_t most = is_big ? kPromptCols : kCols, n = static_cast<int64_t>(max_q_len) * group;
    return static_cast<int>(n < most ? n : most);
}

// Floats of the parts that the workgroups of one kernel may leave.
int64_t part_floats(int max_q_len, int group, int head_dim, bool is_big) {
    return static_cast<int64_t>(is_big ? kBigGrid : kGrid) * 2 *
           part_size(part_cols(max_q_len, group, is_big), padded(head_dim));
}

// Workgroups for at most `units` of work.
unsigned grid_for(int64_t tiles, int64_t heads, int64_t positions, int unit, int batch, int most) {
    const int64_t deep = (positions + unit - 1) / unit;
    const int64_t each = tiles * heads > most ? most : tiles * heads * deep;
    return static_cast<unsigned>(each > most / batch ? most : each * batch);
}

template <int TYPE, int QT, int HD>
int attention_launch(const Q8Args& a, hipStream_t s) {
    const int64_t columns = static_cast<int64_t>(a.max_q_len) * a.group;
    const int64_t positions = static_cast<int64_t>(a.max_blocks) << a.page_shift;
    Q8Args many = a, few = a;
    few.borders = reinterpret_cast<Border*>(a.ws);
    many.borders = few.borders + kGrid;
    many.ws = few.ws = reinterpret_cast<float*>(many.borders + kBigGrid);
    few.part_cols = part_cols(a.max_q_len, a.group, false);
    const unsigned few_grid = grid_for(1, a.n_kv_heads, positions, kUnit, a.batch, kGrid);
    unsigned many_grid = 0;
    if (columns > kCols) {
        many.part_cols = part_cols(a.max_q_len, a.group, true);
        few.ws += part_floats(a.max_q_len, a.group, a.head_dim, true);
        many_grid = grid_for((columns + Prompt::COLS - 1) / Prompt::COLS, a.n_kv_heads, positions, Prompt::UNIT, a.batch,
                             kBigGrid);
        if (const int st = launch(mixed_q8_kernel<TYPE, QT, HD>, dim3(many_grid + few_grid), dim3(kThreads), 0, s, many,
                                  static_cast<int>(many_grid), few))
            return st;
    } else {
        const size_t shmem = static_cast<size_t>(kWaves) * few.part_cols * (HD + 2) * sizeof(float);
        if (const int st = launch(attention_q8_kernel<TYPE, QT, HD>, dim3(few_grid), dim3(kThreads), shmem, s, few))
            return st;
    }
    const unsigned borders = (many_grid > 1 ? (many_grid - 1) * kJoinWide : 0) + few_grid - 1;
    if (borders == 0) return FENCE_SUCCESS;
    return launch(join_q8_kernel<QT, HD>, dim3(borders), dim3(kThreads), 0, s, many, static_cast<int>(many_grid), few);
}

template <int TYPE, int QT>
int attention_hd(const Q8Args& a, hipStream_t s) {
    switch (padded(a.head_dim)) {
        case 64: return attention_launch<TYPE, QT, 64>(a, s);
        case 128: return attention_launch<TYPE, QT, 128>(a, s);
        default: return attention_launch<TYPE, QT, 256>(a, s);
    }
}

}  // namespace
}  // namespace fence

extern "C" int64_t fence_gqa_attention_q8_workspace(int batch, int max_q_len, int n_q_heads, int n_kv_heads,
                                                    int head_dim) {
    using namespace fence;
    if (batch < 0 || max_q_len < 0 || n_q_heads < 1 || n_kv_heads < 1 || n_q_heads % n_kv_heads || head_dim < 16 ||
        head_dim > 256 || head_dim % 16)
        return 0;
    const int group = n_q_heads / n_kv_heads;
    int64_t bytes = 4 * part_floats(max_q_len, group, head_dim, false) + (kGrid + kBigGrid) * int64_t(sizeof(Border));
    if (big(max_q_len, group)) bytes += 4 * part_floats(max_q_len, group, head_dim, true);
    return bytes < 16 ? 16 : bytes;
}

extern "C" int fence_gqa_attention_q8(void* out, const void* q, int type, int64_t ldq, int64_t ldo,
                                      const fence_kv_pages* cache, const int32_t* block_table, int max_blocks,
                                      const int32_t* kv_lens, const int32_t* q_start, int batch, int max_q_len,
                                      int n_q_heads, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    using namespace fence;
    if (!kv_pages_ok(cache) || !out || !q || !block_table || !kv_lens || !q_start || !workspace)
        return FENCE_ERROR_INVALID_VALUE;
    if (type != FENCE_F32 && type != FENCE_F16) return FENCE_ERROR_INVALID_VALUE;
    const size_t size = type == FENCE_F32 ? 4 : 2;
    if (!aligned(out, size) || !aligned(q, size) || !aligned(block_table, 4) || !aligned(kv_lens, 4) ||
        !aligned(q_start, 4) || !aligned(workspace, 16))
        return FENCE_ERROR_INVALID_VALUE;
    if (batch < 0 || batch > 65535 || max_q_len < 0 || max_blocks < 1 || n_q_heads < 1 ||
        n_q_heads % cache->n_kv_heads)
        return FENCE_ERROR_INVALID_VALUE;
    if (static_cast<int64_t>(max_blocks) * cache->page_size > INT32_MAX - kBeyond) return FENCE_ERROR_INVALID_VALUE;
    const int64_t width = static_cast<int64_t>(n_q_heads) * cache->head_dim;
    if (ldq < width || ldo < width || ldq > kMaxLd || ldo > kMaxLd)
        return FENCE_ERROR_INVALID_VALUE;
    const int group = n_q_heads / cache->n_kv_heads;
    if (static_cast<int64_t>(max_q_len) * group > INT32_MAX - kBeyond ||
        (static_cast<int64_t>(max_q_len) * group / kCols + 1) * cache->n_kv_heads > INT32_MAX)
        return FENCE_ERROR_INVALID_VALUE;
    if (workspace_bytes < fence_gqa_attention_q8_workspace(batch, max_q_len, n_q_heads, cache->n_kv_heads,
                                                           cache->head_dim))
        return FENCE_ERROR_INVALID_VALUE;
    if (batch == 0 || max_q_len == 0) return FENCE_SUCCESS;
    const float scale = 1.0f / sqrtf(static_cast<float>(cache->head_dim));
    const Q8Args a{out, q, ldq, ldo, static_cast<const uint8_t*>(cache->k), static_cast<const uint8_t*>(cache->v),
                   cache->k_scale, cache->v_scale, block_table, kv_lens, q_start, static_cast<float*>(workspace), nullptr,
                   cache->n_pages, __builtin_ctz(cache->page_size), cache->n_kv_heads, cache->head_dim, group,
                   max_blocks, batch, max_q_len, 0,
                   static_cast<float>(scale * 1.4426950408889634), aligned(out, 16) && ldo * size % 16 == 0};
    if (cache->type == FENCE_KV_INT8)
        return type == FENCE_F32 ? attention_hd<FENCE_KV_INT8, FENCE_F32>(a, stream)
                                 : attention_hd<FENCE_KV_INT8, FENCE_F16>(a, stream);
    return type == FENCE_F32 ? attention_hd<FENCE_KV_E4M3, FENCE_F32>(a, stream)
                             : attention_hd<FENCE_KV_E4M3, FENCE_F16>(a, stream);
}
