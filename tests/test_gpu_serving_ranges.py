"""The operators of a batched step over a paged 8-bit cache at the ends of what their header allows, against the 64-bit
forms of serving_ref.py, within test_gpu_serving's bound unless one is derived here."""
import numpy as np
import pytest

import fence_ops as F
import serving_ref as R
from gpu_util import dev, host, stream, torch_mod
from test_gpu_serving import bound, check_attention, empty, logits, random_cache, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q", [1, 6, 90])
def test_pages_that_are_not_there_beside_codes_that_are_no_numbers(q, half):
    """Page 0 belongs to no sequence and holds NaN codes, as memory that nothing was stored to may."""
    rng = np.random.default_rng(14)

    def bad(codes, scale, table, q):
        unused = np.setdiff1d(np.arange(1, codes.shape[1]), table)
        table[table == 0] = unused[0]
        codes[:, 0], scale[:, 0] = 0x7F, np.nan
        table[0, 2], table[0, 5], table[1, 0], table[2, :] = -1, 2 ** 31 - 1, codes.shape[1], -2 ** 31

    got = check_attention(rng, 8, 2, 128, 16, [200, 100, 95], [q, q, q], R.E4M3, half, change=bad)
    assert (got[2 * q:3 * q] == 0).all() and np.isfinite(got[:3 * q]).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("cache", [R.INT8, R.E4M3])
def test_rows_that_are_not_finite_and_see_no_page(cache, half):
    """Zeros, whatever q holds."""
    rng = np.random.default_rng(15)

    def bad(codes, scale, table, q):
        table[0, :] = -1
        q[3], q[40, :, 5], q[89, 2] = np.nan, np.inf, -np.inf

    got = check_attention(rng, 8, 2, 64, 16, [95, 70], [90, 30], cache, half, change=bad)
    assert (got[:90] == 0).all()


# ------------------------------------------------------------------ V scales of any size

# What binary16 prompts add to test_gpu_serving's bound: they hold p times its page's V scale as a share of 2^10 of the
# largest V scale so far, not 2^14, so what lies below binary16's smallest step 2^-24 is rounded by up to 2^-25, 2^-35 of
# the largest |v|, for each of the n positions (the sum of the weights is 1 at least: the largest of them).
def check_scales(rng, kv_lens, q_lens, cache, half, v_scale, q_size=2.0, heads=8, kvh=2, d=128, page=16, tiny=1e-30):
    """v_scale(page's place in its sequence) -> the V scale of it; tiny: in place of the bound's 1e-30."""
    blocks = [-(-n // page) for n in kv_lens]
    ids = rng.permutation(sum(blocks)).astype(np.int32)
    table, at = np.full((len(kv_lens), max(blocks)), -1, np.int32), 0
    codes, scale = random_cache(rng, len(ids), kvh, page, d, cache)
    for b, n in enumerate(blocks):
        table[b, :n] = ids[at:at + n]
        at += n
        scale[1, table[b, :n]] = np.array([v_scale(j) for j in range(n)], np.float32)[:, None]
    q_start = np.concatenate([[0], np.cumsum(q_lens)])
    q = (rng.standard_normal((int(q_start[-1]), heads, d)) * q_size).astype(np.float16 if half else np.float32)
    got = run_attention(q, codes, scale, table, kv_lens, q_start, cache, half, max(q_lens))
    want, spread, big = R.attention(q, codes, scale, table, kv_lens, q_start, cache)
    vmax = R.TOP[cache] * scale[1].astype(np.float64).max()
    most = bound(want, spread, big, d, max(kv_lens), half, vmax) - 1e-30 + tiny + (max(kv_lens) * 2.0 ** -35 * vmax if half else 0)
    off = np.abs(got - want)
    assert (off <= most).all(), f"{np.nanmax(off):.3g}, {np.nanmax(off / most):.3g} of what it may be"
    return got, want


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q", [1, 6, 70])
@pytest.mark.parametrize("down", [6, 10, 17, 24, 30, 36, 45, 61, 100])
def test_attention_weight_under_small_v_scales(down, q, half):
    """Half of the pages have a V scale far below the others': they add nothing to speak of to the output, and all of
    their weight to the sum that divides it.  Flat scores over thousands of positions, and ordinary ones."""
    rng = np.random.default_rng(down * 10 + q)
    small = float(np.float32(1.5 * 2.0 ** -down))
    for q_size in (0.01, 2.0):
        check_scales(rng, [4100, 260], [q, q], R.INT8, half, lambda j: small if j % 2 else 1.0, q_size)
        check_scales(rng, [1500], [q], R.E4M3, half, lambda j: 1.0 if j < 2 else small, q_size)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q", [1, 18])
def test_attention_light_positions_under_small_v_scales(q, half):
    """One heavy position on the page with the large V scale; thousands of light ones, whose weights together are as
    much, under V scales 2^-17 of it.  As many copies of the sequence as let one workgroup meet all of one's positions."""
    rng = np.random.default_rng(q)
    heads, kvh, d, page, n, batch = 8, 8, 64, 64, 8256, 64
    table = rng.permutation(n // page).astype(np.int32)[None]
    codes, scale = random_cache(rng, n // page, kvh, page, d, R.INT8)
    scale[1] = 2.0 ** -17
    scale[1, table[0, 0]] = 1.0
    # K of position 7 is 1 in dimension 0 and every other K is 0: one weight of e^9 among ones.  V of the first page's
    # other positions is 0.
    codes[0], codes[1, table[0, 0]] = 0, 0
    codes[0, table[0, 0], :, 7, 0] = 127
    codes[1, table[0, 0], :, 7] = np.arange(1, d + 1, dtype=np.uint8)
    scale[0] = 1.0 / 127
    rows = np.zeros((q, heads, d), np.float16 if half else np.float32)
    rows[:, :, 0] = 9.0 * np.sqrt(d)
    got = run_attention(np.tile(rows, (batch, 1, 1)), codes, scale, np.tile(table, (batch, 1)), [n] * batch,
                        np.arange(batch + 1) * q, R.INT8, half, q).reshape(batch, q, heads, d)
    want, spread, big = R.attention(rows, codes, scale, table, [n], [0, q], R.INT8)
    assert (np.abs(want[-1, 0] / np.arange(1, d + 1) - 0.5) < 0.05).all()  # half of the weight is the heavy one's
    most = bound(want, spread, big, d, n, half, 127.0) + (n * 2.0 ** -35 * 127 if half else 0)
    assert (np.abs(got - want) <= most).all(), np.abs(got - want).max()


@pytest.mark.parametrize("cache", [R.INT8, R.E4M3])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q", [1, 6, 70])
@pytest.mark.parametrize("first,then", [(1e-40, 0.02), (3e-45, 0.02), (0.02, 1e-40), (1e-40, 1e-40), (3e-45, 1e-40),
                                        (2e-36, 2e-36), (1.2e-38, 2e-37), (1e-40, 20.0)])
def test_attention_subnormal_v_scales(first, then, q, half, cache):
    """V scales that the store makes from tiny values: on a sequence's first pages, behind others, and on all.  Where all
    are tiny, 1e-30 says nothing.  In its place: V scales count as 2^-126 at the least where they are the unit of the
    output, so the share of a position that binary16 does not hold is 2^-39 of that times a code; and each wave of each
    workgroup rounds its part to multiples of 2^-149 once, nine workgroups of four waves here, and the result is too."""
    rng = np.random.default_rng(q)
    for lens in ([300, 40], [1100]):
        lens = [max(n, q) for n in lens]
        check_scales(rng, lens, [q] * len(lens), cache, half, lambda j: first if j < 2 else then,
                     tiny=max(lens) * 2.0 ** -39 * R.TOP[cache] * 2.0 ** -126 + 37 * 2.0 ** -150)


# ------------------------------------------------------------------ lengths past the table

@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q", [1, 6, 90])
def test_attention_lengths_past_the_table(q, half):
    """A row sees the positions below kv_len - q_len + i + 1; those that the table has no room for are not there, and
    leave the others where they are.  The reference gets a table with room for all, whose further pages are not there."""
    rng = np.random.default_rng(q + half)
    heads, kvh, d, page, blocks = 8, 2, 64, 16, 7
    table = rng.permutation(3 * blocks).astype(np.int32).reshape(3, blocks)
    codes, scale = random_cache(rng, 3 * blocks, kvh, page, d, R.INT8)
    rows = (rng.standard_normal((3 * q, heads, d)) * 2).astype(np.float16 if half else np.float32)
    kv_lens, q_start = [blocks * page + 1, blocks * page + q // 2, blocks * page + q + 30], [0, q, 2 * q, 3 * q]
    got = run_attention(rows, codes, scale, table, kv_lens, q_start, R.INT8, half, q)
    room = np.concatenate([table, np.full((3, 20), -1, np.int32)], 1)
    want, spread, big = R.attention(rows, codes, scale, room, kv_lens, q_start, R.INT8)
    off, most = np.abs(got - want), bound(want, spread, big, d, max(kv_lens), half, 127 * scale[1].max())
    assert (off <= most).all(), f"{off.max():.3g}, {(off / most).max():.3g} of what it may be"
    # the largest length there is, with a last row far past the table: every row sees the whole table
    got = run_attention(rows, codes, scale, table, [2 ** 31 - 1] * 3, q_start, R.INT8, half, q)
    want, spread, big = R.attention(rows, codes, scale, room, [blocks * page + q] * 3, q_start, R.INT8)
    most = bound(want, spread, big, d, blocks * page, half, 127 * scale[1].max())
    assert (np.abs(got - want) <= most).all()


# ------------------------------------------------------------------ the longest cache

@pytest.mark.parametrize("half", [False, True])
def test_attention_longest_cache_and_wide_group(half):
    """As many positions as a table may have room for, nearly 2^31, under 256 heads of one kv head: the product of a
    place in the work and a number of units passes 64 bits.  Seven pages again and again, so the reference is a softmax
    over theirs, each as often as it comes.

    Weights and V codes are positive, so a running sum of n numbers is off by n 2^-24 of itself at the most, however they
    come.  256 workgroups share the positions of a tile, and a lane adds up 32 of 64, one after the other: 2^22 sums, 2^-2.
    Its products add 16 positions at a time, 2^19 of them, 2^-5; the join's 256 parts and the probabilities' rounding are
    far below 2^-5 more."""
    rng = np.random.default_rng(5)
    page, d, heads, n_pages = 256, 16, 256, 7
    blocks = (2 ** 31 - 1 - 1024) // page
    table = (np.arange(blocks) % n_pages).astype(np.int32)[None]
    codes, scale = random_cache(rng, n_pages, 1, page, d, R.INT8)
    codes[1] = rng.integers(1, 128, codes[1].shape).astype(np.uint8)
    q = rng.standard_normal((1, heads, d)).astype(np.float16 if half else np.float32)
    n = blocks * page
    got = run_attention(q, codes, scale, table, [n], [0, 1], R.INT8, half, 1)
    times = np.repeat(np.bincount(table[0], minlength=n_pages), page).astype(np.float64)
    k, v = ((R.decode(codes[i, :, 0], R.INT8) * scale[i, :, 0].astype(np.float64)[:, None, None]).reshape(-1, d)
            for i in range(2))
    s = q[0].astype(np.float64) @ k.T / np.sqrt(d)
    w = np.exp(s - s.max(1, keepdims=True)) * times
    want = (w @ v) / w.sum(1, keepdims=True)
    assert (np.abs(got[0] - want) <= (2.0 ** -2 + 2.0 ** -4) * want).all(), np.abs(got[0] / want - 1).max()
    print("relative to the reference:", np.abs(got[0] / want - 1).max())


# ------------------------------------------------------------------ a sampling workspace for the largest batch

def test_sample_batches_in_one_workspace():
    """Batches of every size in the workspace of the largest, as a server holds it; nothing is written behind it."""
    torch = torch_mod()
    rng = np.random.default_rng(17)
    vocab, most = 128256, 42
    x = logits(rng, most, vocab, [0.05, 1.0, 3.0])
    u, p = rng.random(most).astype(np.float32), np.full(most, 0.95, np.float32)
    want = [R.sample(x[r], top_p=0.95, u=u[r]) for r in range(most)]
    size = F.sample_workspace(most, vocab)
    ws, d_x, d_u, d_p = empty((size + 64,), torch.uint8, 255), dev(x), dev(u), dev(p)
    for rows in (1, 2, 5, 30, 37, 38, 39, 40, 41, 42):
        out = empty((most,), torch.int32, -9)
        F.sample(out.data_ptr(), d_x.data_ptr(), rows, vocab, vocab, 0, 0, d_p.data_ptr(), 0, d_u.data_ptr(), ws.data_ptr(), size,
                 stream())
        assert host(out).tolist() == want[:rows] + [-9] * (most - rows)
    assert (host(ws)[size:] == 255).all()


# ------------------------------------------------------------------ full tiles

@pytest.mark.parametrize("cache", [R.INT8, R.E4M3])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,kvh,d,q", [(16, 1, 256, 1), (8, 2, 256, 4), (16, 2, 256, 2), (16, 1, 208, 1), (8, 2, 128, 4),
                                           (4, 1, 256, 4)])
def test_attention_exactly_sixteen_columns(heads, kvh, d, q, half, cache):
    """As many columns as the kernel of few columns takes, at the widest heads as well: 66,048 bytes of LDS."""
    rng = np.random.default_rng(heads + d + q)
    check_attention(rng, heads, kvh, d, 32, [300, 17, 1100, q], [q] * 4, cache, half)


# ------------------------------------------------------------------ scales that are not finite

@pytest.mark.parametrize("cache", [R.INT8, R.E4M3])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q", [1, 6, 90])
def test_attention_scales_that_are_not_finite(q, half, cache):
    """They reach the rows that see their page, and no other."""
    rng = np.random.default_rng(19)

    def broken(codes, scale, table, q):
        scale[0, table[0, 10]] = np.nan
        scale[1, table[1, 7]] = np.inf
        codes[1, table[1, 7]] = 0  # times infinity: NaN, as what it is multiplied with
        scale[1, table[2, 6]] = np.nan

    got = check_attention(rng, 8, 2, 128, 16, [200, 130, 120], [q, q, q], cache, half, change=broken)
    for last in (q - 1, 2 * q - 1, 3 * q - 1):
        assert np.isnan(got[last]).all()
    if q > 40:
        assert np.isfinite(got[:40]).all() and np.isfinite(got[90:160]).all() and np.isfinite(got[180:240]).all()
