"""The operators of a batched step over a paged 8-bit cache on the GPU, through the C ABI, against 64-bit numpy
(serving_ref.py).  Plans, codes, scales and tokens have to be equal; attention within a bound derived below."""
import numpy as np
import pytest

import fence_ops as F
import serving_ref as R
from gpu_util import LIVE, dev, host, stream, torch_mod

pytestmark = pytest.mark.gpu


def empty(shape, dtype, fill):
    t = torch_mod().full(shape, fill, dtype=dtype, device="cuda")
    LIVE.append(t)
    return t


# ------------------------------------------------------------------ plan

def run_plan(lens, new, table, page, free, count, max_tokens, in_place=False):
    torch = torch_mod()
    batch = len(lens)
    d_lens, d_new, d_table, d_free = (dev(np.asarray(v, np.int32)) for v in (lens, new, table, free))
    d_count = dev(np.array([count], np.int32))
    lens_out = d_lens if in_place else empty((max(batch, 1),), torch.int32, -7)
    count_out = d_count if in_place else empty((1,), torch.int32, -7)
    q_start, adm = empty((batch + 1,), torch.int32, -7), empty((max(batch, 1),), torch.int32, -7)
    pos, slots = (empty((max_tokens + 3,), torch.int32, -9) for _ in range(2))
    F.kv_plan(lens_out.data_ptr(), d_lens.data_ptr(), d_new.data_ptr(), batch, d_table.data_ptr(), table.shape[1], page,
              d_free.data_ptr(), count_out.data_ptr(), d_count.data_ptr(), len(free), q_start.data_ptr(), pos.data_ptr(),
              slots.data_ptr(), max_tokens, adm.data_ptr(), stream())
    assert (host(pos)[max_tokens:] == -9).all() and (host(slots)[max_tokens:] == -9).all()
    return {"lens": host(lens_out)[:batch], "count": host(count_out)[0], "q_start": host(q_start),
            "positions": host(pos)[:max_tokens], "slots": host(slots)[:max_tokens], "admitted": host(adm)[:batch],
            "table": host(d_table), "free": host(d_free)}


def check_plan(lens, new, table, page, free, count, max_tokens, in_place=False):
    got = run_plan(lens, new, table, page, free, count, max_tokens, in_place)
    table, free = table.copy(), np.array(free, np.int32)
    want = R.plan(lens, new, table, page, free, count, max_tokens)
    for name, v in want.items():
        assert np.array_equal(got[name], np.asarray(v)), name
    assert np.array_equal(got["table"], table)
    assert np.array_equal(got["free"], free)
    return got


def pool(rng, lens, page, blocks, extra):
    """A table whose sequences hold shuffled pages, and a free stack with `extra` pages and as much room."""
    held = [min(-(-n // page), blocks) for n in lens]
    ids = rng.permutation(sum(held) + extra).astype(np.int32)
    table = np.full((len(lens), blocks), -5, np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = ids[at:at + h]
        at += h
    free = np.full(len(ids), -6, np.int32)
    free[:extra] = ids[at:]
    return table, free, extra


@pytest.mark.parametrize("batch,page,most_new,extra,max_tokens", [
    (1, 16, 1, 1, 1), (1, 16, 1, 0, 4), (1, 256, 300, 3, 300), (7, 16, 40, 9, 64), (64, 32, 1, 3, 64), (64, 16, 33, 40, 700),
    (300, 64, 90, 200, 20000), (1024, 16, 3, 500, 4096), (1025, 16, 3, 500, 4096), (2500, 16, 9, 300, 30000),
    (4096, 16, 2, 4000, 8193), (4097, 16, 2, 100, 9000), (5000, 32, 7, 900, 12000)])
def test_plan(batch, page, most_new, extra, max_tokens):
    rng = np.random.default_rng(batch * 7 + page + extra)
    lens = rng.integers(0, 5 * page, batch)
    lens[rng.random(batch) < 0.2] = 0
    lens[rng.random(batch) < 0.2] = page * 2
    new = rng.integers(0, most_new + 1, batch)
    new[rng.random(batch) < 0.15] = -1
    blocks = 6 + most_new // page
    check_plan(lens, new, *pool(rng, lens, page, blocks, extra)[:1], page, *pool(rng, lens, page, blocks, extra)[1:],
               max_tokens)


@pytest.mark.parametrize("in_place", [False, True])
def test_plan_in_place_several_steps(in_place):
    """Steps in a row on the state the last one left: sequences grow, end and start again on what came back."""
    rng = np.random.default_rng(5)
    page, blocks, batch = 16, 5, 33
    lens, table = np.zeros(batch, np.int32), np.full((batch, blocks), -1, np.int32)
    free, count = rng.permutation(80).astype(np.int32), 80
    for step in range(12):
        new = rng.integers(0, 25, batch)
        new[rng.random(batch) < 0.3] = -1
        got = check_plan(lens, new, table, page, free, count, 512, in_place)
        lens, count, table, free = got["lens"], int(got["count"]), got["table"], got["free"]
        used = np.concatenate([table[b, : -(-lens[b] // page)] for b in range(batch)] + [free[:count]])
        assert sorted(used.tolist()) == list(range(80)), "a page lost or given twice"


def test_plan_edges():
    one = np.array([[3, -1]], np.int32)
    # no tokens, no rows; a step that only ends a sequence; a length past the table; a request past the rows
    check_plan([5], [0], one, 16, [0, 1, 2, 9], 3, 0)
    check_plan([32], [-1], np.array([[3, 0]], np.int32), 16, [1, 2, 9, 9], 2, 0)
    check_plan([20], [13], one, 16, [0, 1, 2, 9], 3, 64)
    check_plan([2, 2], [30, 5], np.array([[0, 1, 2], [3, 4, 5]], np.int32), 16, [6, 7, 8, 9, 10, 11], 6, 20)
    # a full stack takes nothing back; a count outside it is bounded; a negative length is none
    check_plan([32], [-1], np.array([[3, 0]], np.int32), 16, [1, 2], 2, 0)
    check_plan([0], [40], np.full((1, 3), -1, np.int32), 16, [4, 5, 6], 9, 64)
    check_plan([-4, 3], [2, 2], np.array([[7], [8]], np.int32), 16, [1, 2, 3], 3, 8)
    got = run_plan([], [], np.zeros((0, 2), np.int32), 16, [1, 2, 3], 2, 5)
    assert got["q_start"].tolist() == [0] and got["count"] == 2 and got["slots"].tolist() == [-1] * 5


# ------------------------------------------------------------------ store

def pages_of(codes, scale, cache):
    _, n, heads, page, d = codes.shape
    return F.kv_pages(codes[0].data_ptr(), codes[1].data_ptr(), scale[0].data_ptr(), scale[1].data_ptr(), n, page, heads, d,
                      cache)


def random_cache(rng, n, heads, page, d, cache):
    x = rng.standard_normal((2, n, heads, page, d)) * (36 if cache == R.INT8 else 128)
    codes = R.encode(np.clip(x, -R.TOP[cache], R.TOP[cache]), cache)
    return codes, rng.uniform(0.002, 0.05, (2, n, heads)).astype(np.float32)


def check_store(codes, scale, x, slots, cache, half, pad=0, shift=0):
    """x (k, v) [tokens][heads][d]; pad, shift: elements behind each row and before the first."""
    dtype = np.float16 if half else np.float32
    tokens, heads, d = x[0].shape
    ld = heads * d + pad
    d_codes, d_scale, d_slots = dev(codes), dev(scale), dev(np.asarray(slots, np.int32))
    ptrs = []
    for v in x:
        rows = np.zeros(shift + tokens * ld, dtype)
        for t in range(tokens):
            rows[shift + t * ld: shift + t * ld + heads * d] = v[t].reshape(-1)
        ptrs.append(dev(rows).data_ptr() + shift * rows.itemsize)
    F.store_kv_q8(pages_of(d_codes, d_scale, cache), ptrs[0], ptrs[1], F.F16 if half else F.F32, ld, d_slots.data_ptr(),
                  tokens, stream())
    codes, scale = codes.copy(), scale.copy()
    for i in range(2):
        R.store(codes[i], scale[i], x[i].astype(dtype), slots, cache)
    assert np.array_equal(host(d_scale), scale, equal_nan=True)
    got = host(d_codes)
    if cache == R.E4M3:  # -0 and 0 are the same value
        got, codes = np.where(got == 128, 0, got), np.where(codes == 128, 0, codes)
    assert np.array_equal(got, codes)
    return host(d_codes), host(d_scale)


@pytest.mark.parametrize("cache", [R.INT8, R.E4M3])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,d,page,runs,pad,shift", [
    (1, 16, 16, [(0, 0, 1)], 0, 0),
    (2, 64, 16, [(0, 15, 1), (1, 0, 16), (2, 3, 5)], 0, 0),
    (8, 128, 32, [(i, (i * 7) % 32, 1) for i in range(40)], 0, 0),
    (2, 96, 64, [(3, 0, 64), (1, 0, 64), (0, 0, 17), (2, 63, 1)], 96, 0),
    (1, 256, 256, [(0, 5, 251), (1, 0, 256), (2, 0, 1)], 0, 0),
    (3, 80, 128, [(0, 100, 28), (2, 0, 77)], 5, 0),
    (2, 48, 16, [(0, 1, 15), (1, 0, 4)], 3, 1)])
def test_store(cache, half, heads, d, page, runs, pad, shift):
    rng = np.random.default_rng(heads * d + page + cache)
    n = max(r[0] for r in runs) + 2
    codes, scale = random_cache(rng, n, heads, page, d, cache)
    slots = np.concatenate([[p * page + off + i for i in range(m)] for p, off, m in runs])
    x = rng.standard_normal((2, len(slots), heads, d)) * rng.uniform(0.05, 8, (2, len(slots), 1, 1))
    x[:, :, :, 3] *= 6
    check_store(codes, scale, x, slots, cache, half, pad, shift)


def test_store_many_rows():
    """More rows than a workgroup each: windows, runs that begin and end inside them, skipped rows between."""
    rng = np.random.default_rng(3)
    heads, d, page, n = 8, 16, 16, 700
    codes, scale = random_cache(rng, n, heads, page, d, R.INT8)
    slots, p = [], 0
    while p < n - 1:
        off = int(rng.integers(0, page))
        m = int(rng.integers(1, page - off + 1))
        slots += [p * page + off + i for i in range(m)]
        if rng.random() < 0.3:
            slots += [-1, n * page + 5, -2 ** 31]
        p += int(rng.integers(1, 3))
    x = rng.standard_normal((2, len(slots), heads, d)) * 3
    check_store(codes, scale, x, slots, R.INT8, False)


@pytest.mark.parametrize("cache", [R.INT8, R.E4M3])
def test_store_rounding(cache):
    """Values on the ties between two codes and one step to either side, scales that double and triple, none at all,
    tiny ones and values that are not finite."""
    page, d = 16, 64
    codes, scale = np.zeros((2, 9, 1, page, d), np.uint8), np.zeros((2, 9, 1), np.float32)
    top, s = R.TOP[cache], np.float32(0.37)
    codes[:, :, 0] = np.arange(page * d, dtype=np.uint32).reshape(page, d) % 127
    scale[:] = s
    ties = (np.arange(d) + 0.5) if cache == R.INT8 else (R.E4M3_VALUES[2:2 + d] + R.E4M3_VALUES[3:3 + d]) / 2
    x = np.zeros((2, 13, 1, d), np.float32)
    base = (ties * np.float64(s)).astype(np.float32)
    x[:, 0, 0], x[:, 1, 0], x[:, 2, 0] = base, np.nextafter(base, np.float32(0)), np.nextafter(base, np.float32(1e9))
    x[:, :3, 0, 0] = np.float32(top) * s
    x[:, 3, 0, 0], x[:, 4, 0, 0], x[:, 5, 0, 0] = top * 2 * s, -top * 3 * s, np.float32(top) * s * 1.7
    x[:, 6] = 0
    x[:, 7] = 1e-30 * (1 + np.arange(d))
    x[:, 8] = 3e-42 * (1 + np.arange(d) % 5)
    x[:, 9, 0, 5], x[:, 10, 0, 5], x[:, 11, 0, 5] = np.inf, np.nan, -np.inf
    x[:, 12, 0] = 3e38
    slots = [0, 1, 2, 16 + 9, 32 + 9, 48 + 9, 64, 80, 96, 6 * 16 + 1, 7 * 16 + 3, 7 * 16 + 4, 8 * 16 + 8]
    slots[8] = 6 * 16  # a subnormal scale, then infinity behind it
    check_store(codes, scale, x, slots, cache, False)
    # exact ties of a page whose scale triples and of one whose scale does not change
    assert check_store(codes, scale, x[:, 4:5], [16 + 5], cache, False)[1][0, 1, 0] == np.float32(
        np.abs(np.float64(np.float32(-top * 3 * s))) / top)


# ------------------------------------------------------------------ attention

# How far fp32 arithmetic of any order may be from 64 bits.  With A the largest sum_i |q_i k_i| * scale of a row and S
# = sum_j p_j |v_j| of an output: a score is a sum of 2 d products (q in two parts), each rounded by half a step of at
# most A, then scaled, and the argument of the exponential rounded (|s| <= A): the roundings are independent, so
# 8 sqrt(2 d) 2^-24 A covers them.  A score off by e turns p by a factor of e^e and the output by at most 2 e S.  Sums
# over n positions add 8 sqrt(n) 2^-24 S, the exponential, the division and q's 22 bits (2^-22 A) a few 2^-23 more.
# binary16: the probabilities and the output are rounded by half a step of 2^-10 each (2^-11 S + 2^-11 |out|).
# Both forms hold p times its page's V scale in binary16, as a share of 2^14 of the largest V scale so far: what lies
# below binary16's smallest step 2^-24 is rounded by up to 2^-25, which is 2^-39 of that scale times a code, so of the
# largest |v|, for each of the n positions.
def bound(out, spread, big, d, n, half, vmax):
    rel = 2 * (8 * np.sqrt(2 * d) * 2.0 ** -24 + 2.0 ** -22) * big + 8 * np.sqrt(max(n, 1)) * 2.0 ** -24 + 2.0 ** -20
    if half:
        rel = rel + 2.0 ** -11
    return spread * rel + n * 2.0 ** -39 * vmax + (2.0 ** -11 * np.abs(out) + 2.0 ** -25 if half else 0) + 1e-30


def run_attention(q, codes, scale, table, kv_lens, q_start, cache, half, max_q, pad=0, extra_rows=0):
    torch = torch_mod()
    rows, heads, d = q.shape
    kvh = codes.shape[2]
    dtype = np.float16 if half else np.float32
    buf = np.full((rows, heads * d + pad), 7.0, dtype)
    buf[:, :heads * d] = q.reshape(rows, -1)
    ldo = heads * d + 2 * pad
    out = empty((rows + extra_rows, ldo), torch.float16 if half else torch.float32, 0.1875)
    size = F.gqa_attention_q8_workspace(len(kv_lens), max_q, heads, kvh, d)
    ws = empty((size + 64,), torch.uint8, 255)
    d_codes, d_scale = dev(codes), dev(scale)
    F.gqa_attention_q8(out.data_ptr(), dev(buf).data_ptr(), F.F16 if half else F.F32, heads * d + pad, ldo,
                       pages_of(d_codes, d_scale, cache), dev(table).data_ptr(), table.shape[1],
                       dev(np.asarray(kv_lens, np.int32)).data_ptr(), dev(np.asarray(q_start, np.int32)).data_ptr(),
                       len(kv_lens), max_q, heads, ws.data_ptr(), size, stream())
    got = host(out).astype(np.float64)
    assert (host(ws)[size:] == 255).all(), "past the workspace"
    assert (got[:, heads * d:] == 0.1875).all() and (got[rows:] == 0.1875).all(), "outside the rows"
    return got[:rows, :heads * d].reshape(rows, heads, d)


def check_attention(rng, heads, kvh, d, page, kv_lens, q_lens, cache, half, q_size=2.0, pad=0, change=None, max_q=None):
    kv_lens, q_lens = list(kv_lens), list(q_lens)
    blocks = max(1, max(-(-max(n, 0) // page) for n in kv_lens))
    total = sum(-(-max(n, 0) // page) for n in kv_lens)
    ids = rng.permutation(max(total, 1) + 3).astype(np.int32)
    table, at = np.full((len(kv_lens), blocks), -1, np.int32), 0
    for b, n in enumerate(kv_lens):
        h = -(-max(n, 0) // page)
        table[b, :h] = ids[at:at + h]
        at += h
    codes, scale = random_cache(rng, len(ids), kvh, page, d, cache)
    if cache == R.E4M3:  # what lies behind a sequence's last position may be anything, a NaN code as well
        for b, n in enumerate(kv_lens):
            if n > 0 and n % page:
                codes[:, table[b, n // page], :, n % page:] = 0x7F
    q_start = np.concatenate([[0], np.cumsum(q_lens)])
    q = rng.standard_normal((int(q_start[-1]) + 2, heads, d)) * q_size
    q = q.astype(np.float16 if half else np.float32)
    if change:
        change(codes, scale, table, q)
    most = max(q_lens) if max_q is None else max_q
    got = run_attention(q, codes, scale, table, kv_lens, q_start, cache, half, most, pad, extra_rows=2)
    want, spread, big = R.attention(q, codes, scale, table, kv_lens, q_start, cache, most)
    left = np.isnan(want).all((1, 2)) & (got == 0.1875).all((1, 2))  # rows of no sequence, as they were
    want[left] = 0.1875
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(np.nan_to_num(got) - np.nan_to_num(want))
    most_off = bound(np.nan_to_num(want), spread, big, d, max(kv_lens), half, R.TOP[cache] * np.max(scale[1], where=np.isfinite(scale[1]), initial=0))
    fine = np.isnan(want) | (off <= most_off)
    assert fine.all(), f"{np.nanmax(off):.3g}, {np.nanmax(off / most_off):.3g} of what it may be"
    return got


HEADS = [(4, 4, 64), (8, 2, 128), (14, 2, 64), (32, 8, 128), (6, 2, 256), (8, 1, 128), (40, 2, 96), (3, 1, 16), (20, 4, 80),
         (33, 1, 48)]


@pytest.mark.parametrize("cache", [R.INT8, R.E4M3])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,kvh,d", HEADS)
def test_attention_single_tokens(heads, kvh, d, half, cache):
    rng = np.random.default_rng(heads * d + half + 2 * cache)
    check_attention(rng, heads, kvh, d, 16, [1, 15, 16, 17, 127, 128, 129, 700], [1] * 8, cache, half, pad=16)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("cache,half", [(R.INT8, False), (R.E4M3, True)])
def test_attention_ragged_rows(page, cache, half):
    """Single tokens, drafted tokens, prompts and idle sequences in one batch; lengths around pages and tiles."""
    rng = np.random.default_rng(page + half)
    kv = [0, 1, 5, 33, 64, 65, 300, 257, 31, 600]
    q = [0, 1, 5, 3, 64, 7, 1, 130, 0, 40]
    check_attention(rng, 8, 2, 64, page, kv, q, cache, half)
    check_attention(rng, 10, 2, 128, page, kv, q, cache, half, pad=8)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,kvh,d", HEADS)
def test_attention_prompts(heads, kvh, d, half):
    rng = np.random.default_rng(heads + d + half)
    check_attention(rng, heads, kvh, d, 32, [150, 200, 77], [150, 70, 33], R.INT8, half)
    check_attention(rng, heads, kvh, d, 16, [97], [97], R.E4M3, half, pad=16)


def test_attention_long_and_split():
    """One long sequence over many workgroups, with short ones beside it; the parts are joined."""
    rng = np.random.default_rng(11)
    check_attention(rng, 4, 2, 128, 64, [20011, 3, 517], [1, 1, 1], R.INT8, False)
    check_attention(rng, 4, 2, 128, 64, [9001, 1300], [4, 9], R.E4M3, True)
    check_attention(rng, 4, 1, 64, 64, [5000, 40], [70, 1], R.INT8, False)


@pytest.mark.parametrize("half", [False, True])
def test_attention_rows_that_see_nothing(half):
    """More rows than positions: the first ones are zeros; max_q_len leaves the rows past it as they were."""
    rng = np.random.default_rng(2)
    got = check_attention(rng, 8, 2, 64, 16, [3, 0, 20, 1], [5, 4, 20, 40], R.INT8, half)
    assert (got[0:2] == 0).all() and (got[5:9] == 0).all()
    got = check_attention(rng, 8, 2, 64, 16, [60, 20, 9], [40, 3, 9], R.E4M3, half, max_q=6)
    assert (got[6:40] == 0.1875).all() and (got[49:52] == 0.1875).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q", [1, 6, 90])
def test_attention_pages_that_are_not_there(q, half):
    rng = np.random.default_rng(4)

    def bad(codes, scale, table, q):
        table[0, 2], table[0, 5], table[1, 0], table[2, :] = -1, 2 ** 31 - 1, codes.shape[1], -2 ** 31

    got = check_attention(rng, 8, 2, 128, 16, [200, 100, 95], [q, q, q], R.INT8, half, change=bad)
    assert (got[2 * q:3 * q] == 0).all()


@pytest.mark.parametrize("q", [1, 6, 90])
def test_attention_scales(q):
    """Scales of very different size from page to page, zero ones, and q rows far from one; a scale that is not
    finite reaches only the rows that see its page."""
    rng = np.random.default_rng(9)

    def spread(codes, scale, table, q):
        scale *= np.float32(2.0) ** rng.integers(-9, 4, scale.shape).astype(np.float32)
        scale[:, table[0, 1]] = 0
        q[0] *= np.float32(1e-12)
        q[-3] *= np.float32(30)

    check_attention(rng, 8, 2, 128, 16, [200, 130], [q, q], R.INT8, False, q_size=0.2, change=spread)

    def broken(codes, scale, table, q):
        scale[0, table[0, 10]] = np.nan
        scale[1, table[1, 7]] = np.inf
        codes[1, table[1, 7]] = 0

    got = check_attention(rng, 8, 2, 128, 16, [200, 130], [q, q], R.INT8, False, change=broken)
    assert np.isnan(got[q - 1]).all() and np.isnan(got[2 * q - 1]).all()
    if q > 40:
        assert np.isfinite(got[:40]).all()


def test_attention_peaked_scores():
    """Large scores: one position takes all the weight, and the running maximum moves."""
    rng = np.random.default_rng(6)
    for half in (False, True):
        check_attention(rng, 8, 2, 128, 32, [900, 400], [1, 50], R.INT8, half, q_size=40.0)


# ------------------------------------------------------------------ sampling

def run_sample(x, temperature=None, top_k=None, top_p=None, min_p=None, u=None, ld=None, shift=0):
    torch = torch_mod()
    rows, vocab = x.shape
    ld = ld or vocab
    buf = np.full(shift + rows * ld + 8, 1e30, np.float32)
    for r in range(rows):
        buf[shift + r * ld: shift + r * ld + vocab] = x[r]
    ptr = lambda v, t: None if v is None else dev(np.broadcast_to(np.asarray(v, t), (rows,)).copy()).data_ptr()  # noqa: E731
    out = empty((rows + 2,), torch.int32, -9)
    size = F.sample_workspace(rows, vocab)
    ws = empty((size + 64,), torch.uint8, 255)
    F.sample(out.data_ptr(), dev(buf).data_ptr() + 4 * shift, rows, vocab, ld, ptr(temperature, np.float32),
             ptr(top_k, np.int32), ptr(top_p, np.float32), ptr(min_p, np.float32), ptr(0.0 if u is None else u, np.float32),
             ws.data_ptr(), size, stream())
    got = host(out)
    assert (got[rows:] == -9).all() and (host(ws)[size:] == 255).all()
    return got[:rows]


def check_sample(x, temperature=None, top_k=None, top_p=None, min_p=None, u=None, **kw):
    got = run_sample(x, temperature, top_k, top_p, min_p, u, **kw)
    rows = x.shape[0]
    at = lambda v, d, r: d if v is None else np.broadcast_to(v, (rows,))[r]  # noqa: E731
    want = [R.sample(x[r], at(temperature, 1.0, r), at(top_k, 0, r), at(top_p, 1.0, r), at(min_p, 0.0, r), at(u, 0.0, r))
            for r in range(rows)]
    assert got.tolist() == want


def logits(rng, rows, vocab, sizes):
    x = rng.standard_normal((rows, vocab)) * np.resize(sizes, rows)[:, None]
    for r in range(rows):
        x[r, rng.integers(0, vocab, 20)] += rng.standard_normal(20) * 4 + 3
    return x.astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 1000, 1025, 4097, 32001, 151936])
@pytest.mark.parametrize("filters", ["none", "k", "large_k", "p", "min_p", "k_p", "large_k_p_min", "p_min", "all"])
def test_sample(vocab, filters):
    rng = np.random.default_rng(vocab + len(filters))
    rows = 24 if vocab < 100000 else 8
    x = logits(rng, rows, vocab, [0.02, 0.5, 1.5, 3.0, 8.0])
    k = rng.integers(1, 60, rows) if filters in ("k", "k_p", "all") else rng.integers(500, 9000, rows) if "large_k" in filters else None
    p = rng.uniform(0.05, 0.999, rows) if "p" in filters.replace("min_p", "").replace("_min", "") or filters == "all" else None
    m = rng.uniform(0.001, 0.3, rows) if "min" in filters or filters == "all" else None
    check_sample(x, rng.uniform(0.3, 2.0, rows), k, p, m, rng.random(rows))
    check_sample(x, None, k, p, m, rng.random(rows), ld=vocab + 3, shift=1)


def test_sample_parameters_at_their_ends():
    rng = np.random.default_rng(1)
    x = logits(rng, 20, 5000, [1.0, 4.0])
    u = rng.random(20)
    for t in (0.0, -1.0, np.nan, 1e-30, 1e-3, 1e30, np.inf):
        check_sample(x, t, None, None, None, u)
    for k in (-3, 0, 1, 2, 4999, 5000, 9000, 2 ** 31 - 1):
        check_sample(x, 1.0, k, None, None, u)
        check_sample(x, 1.0, k, 0.9, None, u)
    for p in (-1.0, 0.0, 1e-9, 1.0 - 2.0 ** -24, 1.0, 2.0, np.nan):
        check_sample(x, 1.0, None, p, None, u)
    for m in (-1.0, 0.0, 1e-30, 1.0, 3.0, np.nan):
        check_sample(x, 1.0, None, None, m, u)
    for v in (0.0, 2.0 ** -24, 1.0 - 2.0 ** -24):
        check_sample(x, 1.0, None, None, None, v)
        check_sample(x, 1.0, 50, 0.9, None, v)


@pytest.mark.parametrize("vocab", [5, 1000, 4096, 4097, 9001, 200003])
def test_sample_equal_logits(vocab):
    """Ties go to the lowest index, also where they are more than a list holds."""
    rows = 9
    u = np.array([0, 0.25, 0.5, 0.75, 0.999, 0.1, 0.3, 0.6, 0.9], np.float32)
    x = np.full((rows, vocab), -3.25, np.float32)
    check_sample(x, 0.7, None, None, None, u)
    check_sample(x, 0.7, 3, None, None, u)
    check_sample(x, 0.7, max(1, vocab // 2), None, None, u)
    check_sample(x, 0.7, None, 0.5, None, u)
    check_sample(x, 0.0)
    x[:, ::3] = -3.0
    x[:, 4] = 0.0
    x[1::2] *= -1
    check_sample(x, 0.7, None, None, None, u)
    check_sample(x, 0.7, 700, 0.8, None, u)
    check_sample(x, 0.7, None, None, 0.9, u)
    zeros = np.zeros((rows, vocab), np.float32)
    zeros[:, 1::2] = -0.0
    check_sample(zeros, 1.0, 2, None, None, u)


def test_sample_values_that_are_not_finite():
    rng = np.random.default_rng(8)
    x = logits(rng, 12, 3001, [2.0])
    u = rng.random(12)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2] = np.nan
    x[3, 100:] = -np.inf
    x[4, [7, 2999]] = np.inf
    x[5, :] = np.inf
    x[6, 5:] = -np.inf
    x[7, 1:] = np.nan
    x[8] = -np.inf
    x[8, 3000] = -1e38
    x[9, 17] = 3e38
    x[10] = np.where(np.arange(3001) % 2 == 0, np.float32(3e38), np.float32(-3e38))
    for k, p, m in ((None, None, None), (40, None, None), (None, 0.9, None), (None, None, 0.05), (2000, 0.99, 0.01)):
        check_sample(x, 1.0, k, p, m, u)
        check_sample(x, 0.01, k, p, m, u)
        check_sample(x, 0.0, k, p, m, u)


def test_sample_distribution():
    """20,000 draws of one row against its probabilities: each count within 5 standard deviations."""
    rng = np.random.default_rng(12)
    x = np.tile(np.array([0.0, 1.0, -1.0, 2.0, 0.5], np.float32), (20000, 1))
    got = np.bincount(run_sample(x, None, None, None, None, rng.random(20000)), minlength=5)
    p = np.exp(x[0].astype(np.float64))
    p /= p.sum()
    assert (np.abs(got - 20000 * p) <= 5 * np.sqrt(20000 * p * (1 - p))).all()


def test_sample_many_flat_rows():
    """Rows that need the whole histogram, more than one workgroup each, beside peaked ones; every filter and none."""
    rng = np.random.default_rng(77)
    rows, vocab = 300, 20011
    x = logits(rng, rows, vocab, [0.3, 1.0, 2.0, 5.0])
    t = rng.uniform(0.5, 2.0, rows).astype(np.float32)
    t[::17] = 0
    k = np.where(rng.random(rows) < 0.4, rng.integers(1, vocab, rows), 0).astype(np.int32)
    p = np.where(rng.random(rows) < 0.6, rng.uniform(0.2, 1.0, rows), 1.0).astype(np.float32)
    m = np.where(rng.random(rows) < 0.4, 10.0 ** rng.uniform(-4, 0, rows), 0.0).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    u[::13], u[5::13] = 0.0, np.float32(1 - 2.0 ** -24)
    check_sample(x, t, k, p, m, u)


def test_sample_more_rows_than_a_launch_takes():
    rng = np.random.default_rng(19)
    rows, vocab = 33001, 70
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    k = rng.integers(0, 12, rows).astype(np.int32)
    p = rng.uniform(0.3, 1.1, rows).astype(np.float32)
    check_sample(x, np.float32(0.9), k, p, None, rng.random(rows).astype(np.float32))
