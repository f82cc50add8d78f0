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

constexpr int kCols = 16;          // columns of a product: (row, head of the group) pairs
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kUnit = 32 * kWaves; // positions a workgroup takes at a time, 32 a wave
#ifndef FENCE_ATTN_Q8_GRID
#define FENCE_ATTN_Q8_GRID 1024
#endif
constexpr int kMaxGrid = FENCE_ATTN_Q8_GRID;

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
    int n_pages, page_shift, n_kv_heads, head_dim, group;
    int max_blocks, batch, max_q_len;
    int part_cols;  // columns of a partial in the workspace
    float scale_log2;
};

// A sequence as the products see it.
struct Seq {
    int row0, rows, q_len, kv;  // first row, rows computed, rows there are, positions
    __device__ __forceinline__ int tiles(int group) const { return (rows * group + kCols - 1) / kCols; }
    // positions that the last column of a tile sees
    __device__ __forceinline__ int sees(int tile, int group) const {
        int i = (tile * kCols + kCols - 1) / group;
        if (i > q_len - 1) i = q_len - 1;
        const int n = kv - q_len + i + 1;
        return n < 0 ? 0 : n;
    }
    // workgroup units of one kv head's tile: one at least, which writes the zeros of rows that see nothing
    __device__ __forceinline__ int units(int tile, int group) const {
        const int n = (sees(tile, group) + kUnit - 1) / kUnit;
        return n < 1 ? 1 : n;
    }
};

__device__ __forceinline__ Seq sequence(const Q8Args& a, int b) {
    Seq s;
    s.row0 = a.q_start[b];
    const int n = a.q_start[b + 1] - s.row0;
    s.q_len = n < 0 ? 0 : n;
    s.rows = s.q_len < a.max_q_len ? s.q_len : a.max_q_len;
    const int cap = a.max_blocks << a.page_shift;
    const int kv = a.kv_lens[b];
    s.kv = kv < 0 ? 0 : kv > cap ? cap : kv;
    return s;
}

// Units of a whole sequence.
__device__ __forceinline__ int64_t seq_units(const Q8Args& a, int b) {
    const Seq s = sequence(a, b);
    int64_t n = 0;
    for (int t = 0; t < s.tiles(a.group); ++t) n += s.units(t, a.group);
    return n * a.n_kv_heads;
}

// Prefix sums of the sequences' units over the workgroup: the total, and the
// sequence that unit `find(total)` belongs to with the units before it.
template <class F>
__device__ __forceinline__ int64_t locate(const Q8Args& a, F find, int* seq, int64_t* before) {
    __shared__ int64_t waves[kWaves];
    __shared__ int64_t found_before;
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    int64_t total = 0, mine = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int64_t at = 0;
        const int64_t target = pass ? find(total) : -1;
        for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
            if (!pass || a.batch > kThreads) mine = b0 + tid < a.batch ? seq_units(a, b0 + tid) : 0;
            int64_t v = mine;
#pragma unroll
            for (int d = 1; d < kWave; d *= 2) {
                const int64_t up = __shfl_up(v, d);
                if (lane >= d) v += up;
            }
            __syncthreads();
            if (lane == kWave - 1) waves[wave] = v;
            __syncthreads();
            int64_t pre = at;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                if (w < wave) pre += waves[w];
                at += waves[w];
            }
            if (pass && pre + v > target && pre + v - mine <= target) {
                found = b0 + tid;
                found_before = pre + v - mine;
            }
        }
        total = at;
    }
    __syncthreads();
    *seq = __builtin_amdgcn_readfirstlane(found);
    *before = found_before;
    return total;
}

// Workgroups that get units: every one of them at least one, so that each
// workgroup between an item's first and last has a part of it.
__device__ __forceinline__ int sharers(int64_t total, int grid) {
    return total < 1 ? 1 : total < grid ? static_cast<int>(total) : grid;
}

// The workgroup of `grid` that unit u of `total` falls to, when workgroup w
// takes the units from w * total / grid to (w + 1) * total / grid.
__device__ __forceinline__ int owner(int64_t u, int64_t total, int grid) {
    return static_cast<int>(((u + 1) * grid - 1) / total);
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

__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) {
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Over the four 16-lane rows of a wave, for every lane.
template <class Op>
__device__ __forceinline__ float across_rows(float v, Op op) {
    v = op(v, __shfl_xor(v, 16));
    return op(v, __shfl_xor(v, 32));
}

// One workgroup's share of the units.  A wave multiplies 32 positions (two
// groups of 16, each inside one page) by 16 columns at a time:
//   S' [16 positions x 16 columns] = K [16 x HD] Q' [HD x 16]
//   O' [HD x 16 columns] += V' [HD x 32 positions] P [32 x 16]
// The first product leaves lane (column r, row group g) with the positions
// 4 g .. 4 g + 3 of each group of 16, and those eight are what the second
// product takes from it as its k index, so P stays where it is.  A lane's
// dimensions are r * HD / 16 + i for product i, so it reads V with one load a
// position.
template <int TYPE, int QT, int HD>
__global__ __launch_bounds__(kThreads) void attention_q8_kernel(Q8Args a) {
    constexpr int PIECES = HD / 64;       // 64 dimensions of K: 16 a lane
    constexpr int DT = HD / 16;           // products over V; also dimensions a lane reads of a position
    constexpr bool F32 = QT == FENCE_F32;
    constexpr int PARTS = F32 ? 2 : 1;    // binary16 numbers that hold a q or a p
    extern __shared__ float lds[];
    const int tid = threadIdx.x, lane = tid % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int r = lane % 16, g = lane / 16;
    const int hd = a.head_dim, page_mask = (1 << a.page_shift) - 1;

    int b;
    int64_t before;
    const int me = blockIdx.x;
    const int64_t total = locate(a, [&](int64_t n) { return me * n / sharers(n, gridDim.x); }, &b, &before);
    const int grid = sharers(total, gridDim.x);
    if (me >= grid || total == 0) return;
    int64_t u = me * total / grid;
    const int64_t u_end = (me + 1) * total / grid;
    Seq s = sequence(a, b);
    // the tile and head in which u lies, in the order of tiles and then heads
    int tile = 0, units = s.units(0, a.group);
    int64_t rest = u - before;
    while (rest >= static_cast<int64_t>(units) * a.n_kv_heads) {
        rest -= static_cast<int64_t>(units) * a.n_kv_heads;
        units = s.units(++tile, a.group);
    }
    int head = static_cast<int>(rest / units);
    int unit = static_cast<int>(rest % units);

    while (u < u_end) {
        const int first = unit;
        const int last = u_end - u < units - unit ? unit + static_cast<int>(u_end - u) : units;
        const int cols = s.rows * a.group - tile * kCols < kCols ? s.rows * a.group - tile * kCols : kCols;
        // this lane's column
        const int col = tile * kCols + r;
        const int row = col / a.group;
        const bool mine = r < cols;
        const int qhead = head * a.group + col % a.group;
        int sees = mine ? s.kv - s.q_len + row + 1 : 0;  // of its row
        if (sees < 0) sees = 0;
        const int end = s.sees(tile, a.group);

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
                        const float y = x[p][i] * up;
                        const _Float16 hi = static_cast<_Float16>(y);
                        qf[0][p][i / 8][i % 8] = hi;
                        qf[1][p][i / 8][i % 8] = static_cast<_Float16>(y - static_cast<float>(hi));
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

        const int32_t* row_of_table = a.table + static_cast<int64_t>(b) * a.max_blocks;
        for (int un = first; un < last; ++un) {
            const int pos0 = un * kUnit + wave * 32;
            if (pos0 >= end) break;
            f4 st[2];
            uint32_t vw[8][(DT + 3) / 4];
            float vscale[2], kscale[2];
            bool bad[2];
            u4 kw[2][PIECES];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int pos = pos0 + 16 * t;
                const int id = pos < end ? row_of_table[pos >> a.page_shift] : -1;
                bad[t] = id < 0 || id >= a.n_pages;
                const int64_t base = static_cast<int64_t>(bad[t] ? 0 : id) * a.n_kv_heads + head;
                kscale[t] = bad[t] ? 0.0f : a.ks[base];
                vscale[t] = bad[t] ? 0.0f : a.vs[base];
                const int64_t at = ((base << a.page_shift) + (pos & page_mask)) * hd;
#pragma unroll
                for (int p = 0; p < PIECES; ++p) {
                    const int d = p * 64 + g * 16;
                    kw[t][p] = u4{0, 0, 0, 0};
                    if (!bad[t] && d < hd) kw[t][p] = *reinterpret_cast<const u4*>(a.k + at + r * hd + d);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool there = !bad[t] && pos + g * 4 + i < end && r * DT < hd;
                    const uint8_t* src = a.v + at + (g * 4 + i) * hd + r * DT;
#pragma unroll
                    for (int w = 0; w < DT / 4; ++w)
                        vw[4 * t + i][w] = there ? reinterpret_cast<const uint32_t*>(src)[w] : 0;
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        h2 c0, c1, c2, c3;
                        codes_h<TYPE>(kw[t][p][2 * j], &c0, &c1);
                        codes_h<TYPE>(kw[t][p][2 * j + 1], &c2, &c3);
                        const h8 kf = join(c0, c1, c2, c3);
#pragma unroll
                        for (int x = 0; x < PARTS; ++x)
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[x][p][j], acc, 0, 0, 0);
                    }
                const float f = kscale[t] * unscale;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int pos = pos0 + 16 * t + g * 4 + i;
                    st[t][i] = bad[t] || pos >= sees ? -__builtin_inff() : acc[i] * f;
                }
            }
            float top = m;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, st[t][i]);
            top = across_rows(top, OpMax{});
            const float ref = top == -__builtin_inff() ? 0.0f : top;
            float vtop = vref;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (vscale[t] > vtop && vscale[t] < __builtin_inff()) vtop = vscale[t];
            const float alpha = __builtin_amdgcn_exp2f(m - ref);  // m = -inf: 0
            const float beta = vtop > 0.0f ? alpha * (vref / vtop) : 0.0f;
            const float to_v = vtop > 0.0f ? 16384.0f / vtop : 0.0f;
            m = top;
            vref = vtop;
            l *= alpha;
            h8 pf[PARTS];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(st[t][i] - ref);
                    l += p;
                    const float y = st[t][i] == -__builtin_inff() ? 0.0f : p * (vscale[t] * to_v);
                    const _Float16 hi = static_cast<_Float16>(y);
                    pf[0][4 * t + i] = hi;
                    if constexpr (F32) pf[1][4 * t + i] = static_cast<_Float16>(y - static_cast<float>(hi));
                }
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] *= beta;
#pragma unroll
            for (int w = 0; w < DT / 4; ++w) {
                h2 c[4][4];  // [pair of positions][dimension of the word]
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t x = vw[2 * j][w], y = vw[2 * j + 1][w];
                    codes_h<TYPE>(__builtin_amdgcn_perm(y, x, 0x05010400u), &c[j][0], &c[j][1]);
                    codes_h<TYPE>(__builtin_amdgcn_perm(y, x, 0x07030602u), &c[j][2], &c[j][3]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const h8 vf = join(c[0][i], c[1][i], c[2][i], c[3][i]);
#pragma unroll
                    for (int x = 0; x < PARTS; ++x)
                        o[4 * w + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[x], o[4 * w + i], 0, 0, 0);
                }
            }
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
                    mo[(wave * pc + r) * HD + (4 * g + j) * DT + i] = o[i][j] * (vref * 0x1p-14f);
            if (g == 0) {
                ml[(wave * pc + r) * 2] = m;
                ml[(wave * pc + r) * 2 + 1] = l;
            }
        }
        __syncthreads();
        const bool whole = first == 0 && last == units;
        float* part = a.ws + static_cast<int64_t>(me * 2 + (first == 0 ? 1 : 0)) * pc * (HD + 2);
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
                    const float res = sum != 0.0f ? val / sum : 0.0f;
                    if constexpr (F32) static_cast<float*>(a.out)[to] = res;
                    else static_cast<uint16_t*>(a.out)[to] = f32_to_f16_bits(res);
                }
            } else {
                part[c * (HD + 2) + 2 + d] = val;
                if (d == 0) part[c * (HD + 2)] = top, part[c * (HD + 2) + 1] = sum;
            }
        }
        __syncthreads();

        u += last - first;
        unit = 0;
        if (u >= u_end) break;
        if (++head == a.n_kv_heads) {
            head = 0;
            if (++tile == s.tiles(a.group)) {
                tile = 0;
                do {
                    s = sequence(a, ++b);
                } while (s.rows == 0);
            }
            units = s.units(tile, a.group);
        }
    }
}

// The parts of the items (a sequence's tile and kv head) that more than one
// workgroup took, in workgroup order.
template <int QT, int HD>
__global__ __launch_bounds__(kThreads) void attention_q8_merge_kernel(Q8Args a, int grid) {
    const int tile = blockIdx.x / a.n_kv_heads, head = blockIdx.x % a.n_kv_heads;
    int seq = blockIdx.y;
    const Seq s = sequence(a, seq);
    if (tile >= s.tiles(a.group)) return;
    // units before this sequence, and in all
    __shared__ int64_t waves[2][kWaves];
    int64_t pre = 0, all = 0;
    for (int b = threadIdx.x; b < a.batch; b += kThreads) {
        const int64_t n = seq_units(a, b);
        all += n;
        if (b < seq) pre += n;
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        pre += __shfl_xor(pre, d);
        all += __shfl_xor(all, d);
    }
    if (threadIdx.x % kWave == 0) {
        waves[0][threadIdx.x / kWave] = pre;
        waves[1][threadIdx.x / kWave] = all;
    }
    __syncthreads();
    pre = all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) pre += waves[0][w], all += waves[1][w];
    grid = sharers(all, grid);
    for (int t = 0; t < tile; ++t) pre += static_cast<int64_t>(s.units(t, a.group)) * a.n_kv_heads;
    const int units = s.units(tile, a.group);
    pre += static_cast<int64_t>(units) * head;
    const int w0 = owner(pre, all, grid), w1 = owner(pre + units - 1, all, grid);
    if (w0 == w1) return;
    const int cols = s.rows * a.group - tile * kCols < kCols ? s.rows * a.group - tile * kCols : kCols;
    const int pc = a.part_cols, hd = a.head_dim;
    const auto part = [&](int w) {
        return a.ws + static_cast<int64_t>(w * 2 + (w == w0 ? 1 : 0)) * pc * (HD + 2);
    };
    for (int x = threadIdx.x; x < cols * HD; x += kThreads) {
        const int c = x / HD, d = x % HD;
        float top = -__builtin_inff();
        for (int w = w0; w <= w1; ++w) top = fmaxf(top, part(w)[c * (HD + 2)]);
        const float ref = top == -__builtin_inff() ? 0.0f : top;
        float sum = 0.0f, val = 0.0f;
        for (int w = w0; w <= w1; ++w) {
            const float* p = part(w) + c * (HD + 2);
            const float f = __builtin_amdgcn_exp2f(p[0] - ref);
            sum += f * p[1];
            val += f * p[2 + d];
        }
        if (d < hd) {
            const int cc = tile * kCols + c;
            const int64_t to = static_cast<int64_t>(s.row0 + cc / a.group) * a.ldo +
                               static_cast<int64_t>(head * a.group + cc % a.group) * hd + d;
            const float res = sum != 0.0f ? val / sum : 0.0f;
            if constexpr (QT == FENCE_F32) static_cast<float*>(a.out)[to] = res;
            else static_cast<uint16_t*>(a.out)[to] = f32_to_f16_bits(res);
        }
    }
}

int padded(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

int part_cols(int max_q_len, int group) {
    return static_cast<int64_t>(max_q_len) * group < kCols ? max_q_len * group : kCols;
}

template <int TYPE, int QT, int HD>
int attention_launch(const Q8Args& a, hipStream_t s) {
    const int64_t tiles = (static_cast<int64_t>(a.max_q_len) * a.group + kCols - 1) / kCols;
    const int64_t deep = (static_cast<int64_t>(a.max_blocks) << a.page_shift) + kUnit - 1;
    const int64_t most = tiles * a.n_kv_heads * (deep / kUnit);
    const int64_t grid = most > kMaxGrid / a.batch ? kMaxGrid : most * a.batch;
    const size_t shmem = static_cast<size_t>(kWaves) * a.part_cols * (HD + 2) * sizeof(float);
    if (const int st = launch(attention_q8_kernel<TYPE, QT, HD>, dim3(static_cast<unsigned>(grid)), dim3(kThreads),
                              shmem, s, a))
        return st;
    if (deep / kUnit * grid == 0) return FENCE_SUCCESS;
    return launch(attention_q8_merge_kernel<QT, HD>, dim3(static_cast<unsigned>(tiles * a.n_kv_heads), a.batch),
                  dim3(kThreads), 0, s, a, static_cast<int>(grid));
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
    const int64_t bytes = static_cast<int64_t>(kMaxGrid) * 2 * part_cols(max_q_len, n_q_heads / n_kv_heads) *
                          (padded(head_dim) + 2) * 4;
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
    if (static_cast<int64_t>(max_blocks) * cache->page_size > INT32_MAX - kUnit) return FENCE_ERROR_INVALID_VALUE;
    const int64_t width = static_cast<int64_t>(n_q_heads) * cache->head_dim;
    if (ldq < width || ldo < width || ldq > INT64_MAX / (int64_t(1) << 34) || ldo > INT64_MAX / (int64_t(1) << 34))
        return FENCE_ERROR_INVALID_VALUE;
    const int group = n_q_heads / cache->n_kv_heads;
    if (static_cast<int64_t>(max_q_len) * group > INT32_MAX - kCols ||
        (static_cast<int64_t>(max_q_len) * group / kCols + 1) * cache->n_kv_heads > INT32_MAX)
        return FENCE_ERROR_INVALID_VALUE;
    if (workspace_bytes < fence_gqa_attention_q8_workspace(batch, max_q_len, n_q_heads, cache->n_kv_heads,
                                                           cache->head_dim))
        return FENCE_ERROR_INVALID_VALUE;
    if (batch == 0 || max_q_len == 0) return FENCE_SUCCESS;
    const float scale = 1.0f / sqrtf(static_cast<float>(cache->head_dim));
    const Q8Args a{out, q, ldq, ldo, static_cast<const uint8_t*>(cache->k), static_cast<const uint8_t*>(cache->v),
                   cache->k_scale, cache->v_scale, block_table, kv_lens, q_start, static_cast<float*>(workspace),
                   cache->n_pages, __builtin_ctz(cache->page_size), cache->n_kv_heads, cache->head_dim, group,
                   max_blocks, batch, max_q_len, part_cols(max_q_len, group),
                   static_cast<float>(scale * 1.4426950408889634)};
    if (cache->type == FENCE_KV_INT8)
        return type == FENCE_F32 ? attention_hd<FENCE_KV_INT8, FENCE_F32>(a, stream)
                                 : attention_hd<FENCE_KV_INT8, FENCE_F16>(a, stream);
    return type == FENCE_F32 ? attention_hd<FENCE_KV_E4M3, FENCE_F32>(a, stream)
                             : attention_hd<FENCE_KV_E4M3, FENCE_F16>(a, stream);
}
