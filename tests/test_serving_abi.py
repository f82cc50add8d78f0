"""Refusals of the batched serving operators, and the references their GPU tests use, without a GPU.  The addresses
are never dereferenced: every call is refused on the host or has nothing to do."""
import ctypes

import numpy as np
import pytest

import fence_ops as F
import serving_ref as R

E, OK = F.EINVAL, F.SUCCESS
P = [0x10000 * (i + 1) for i in range(16)]  # aligned, non-null


def kv(**change):
    v = dict(k=P[0], v=P[1], k_scale=P[2], v_scale=P[3], n_pages=8, page_size=16, n_kv_heads=2, head_dim=64, type=F.KV_INT8)
    v.update(change)
    return ctypes.byref(F.kv_pages(**v))


BAD_PAGES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=P[0] + 8), dict(v=P[1] + 1),
             dict(k_scale=P[2] + 2), dict(n_pages=0), dict(page_size=8), dict(page_size=48), dict(page_size=512),
             dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=24), dict(head_dim=272), dict(type=2), dict(type=-1),
             dict(n_pages=2 ** 31 - 1, page_size=16)]


def plan(**change):
    v = dict(lens_out=P[0], lens=P[1], new=P[2], batch=4, table=P[3], max_blocks=8, page=16, free=P[4], count_out=P[5],
             count=P[6], n_pages=32, q_start=P[7], positions=P[8], slots=P[9], max_tokens=0, admitted=P[10])
    v.update(change)
    return F.lib().fence_kv_plan(*v.values(), None)


@pytest.mark.parametrize("change", [
    dict(lens_out=None), dict(lens=None), dict(new=None), dict(table=None), dict(free=None), dict(count_out=None),
    dict(count=None), dict(q_start=None), dict(positions=None, max_tokens=4), dict(slots=None, max_tokens=4),
    dict(admitted=None), dict(batch=-1), dict(max_blocks=0), dict(page=0), dict(page=8), dict(page=24), dict(page=512),
    dict(n_pages=0), dict(max_tokens=-1), dict(max_tokens=2 ** 31), dict(n_pages=2 ** 28), dict(max_blocks=2 ** 27),
    dict(lens=P[1] + 2), dict(slots=P[9] + 1), dict(q_start=P[7] + 2)])
def test_plan_refuses(change):
    assert plan(**change) == E


def store(pages=None, k=P[4], v=P[5], type=F.F32, ld=128, slots=P[6], tokens=0):
    return F.lib().fence_store_kv_q8(pages or kv(), k, v, type, ld, slots, tokens, None)


@pytest.mark.parametrize("change", [
    dict(k=None), dict(v=None), dict(slots=None), dict(type=2), dict(ld=127), dict(tokens=-1), dict(tokens=2 ** 31),
    dict(k=P[4] + 2), dict(v=P[5] + 1, type=F.F16), dict(slots=P[6] + 2), dict(ld=2 ** 62)])
def test_store_refuses(change):
    assert store() == OK and store(type=F.F16, k=P[4] + 2) == OK
    assert store(**change) == E
    assert F.lib().fence_store_kv_q8(None, P[4], P[5], F.F32, 128, P[6], 4, None) == E


def attend(pages=None, out=P[4], q=P[5], type=F.F32, ldq=256, ldo=256, table=P[6], max_blocks=8, kv_lens=P[7], q_start=P[8],
           batch=0, max_q=4, heads=4, ws=P[9], size=1 << 40):
    return F.lib().fence_gqa_attention_q8(out, q, type, ldq, ldo, pages or kv(), table, max_blocks, kv_lens, q_start, batch,
                                          max_q, heads, ws, size, None)


@pytest.mark.parametrize("change", [
    dict(out=None), dict(q=None), dict(table=None), dict(kv_lens=None), dict(q_start=None), dict(ws=None), dict(type=7),
    dict(ldq=255), dict(ldo=255), dict(max_blocks=0), dict(batch=-1), dict(batch=65536), dict(max_q=-1), dict(heads=0),
    dict(heads=5), dict(size=0), dict(ws=P[9] + 8), dict(out=P[4] + 2), dict(q=P[5] + 1, type=F.F16), dict(table=P[6] + 2),
    dict(max_blocks=2 ** 27), dict(ldq=2 ** 40), dict(max_q=2 ** 31 - 1)])
def test_attention_refuses(change):
    assert attend() == OK and attend(max_q=0, batch=3) == OK
    assert attend(**change) == E


@pytest.mark.parametrize("change", BAD_PAGES)
def test_pages_are_checked(change):
    assert store(pages=kv(**change), tokens=1) == E
    assert attend(pages=kv(**change), batch=1) == E


def test_attention_workspace():
    size = F.gqa_attention_q8_workspace(4, 1, 32, 8, 128)
    assert size > 0 and attend(heads=4, max_q=1, size=F.gqa_attention_q8_workspace(0, 1, 4, 2, 64) - 1) == E
    for bad in [(-1, 1, 32, 8, 128), (1, -1, 32, 8, 128), (1, 1, 0, 8, 128), (1, 1, 30, 8, 128), (1, 1, 32, 0, 128),
                (1, 1, 32, 8, 100), (1, 1, 32, 8, 0), (1, 1, 32, 8, 512)]:
        assert F.gqa_attention_q8_workspace(*bad) == 0


def sample(out=P[0], x=P[1], rows=0, vocab=100, ld=100, t=None, k=None, p=None, m=None, u=P[2], ws=P[3], size=1 << 40):
    return F.lib().fence_sample(out, x, rows, vocab, ld, t, k, p, m, u, ws, size, None)


@pytest.mark.parametrize("change", [
    dict(out=None), dict(x=None), dict(u=None), dict(ws=None), dict(rows=-1), dict(vocab=0), dict(ld=99), dict(size=0),
    dict(out=P[0] + 2), dict(x=P[1] + 1), dict(t=P[4] + 2), dict(k=P[4] + 2), dict(p=P[4] + 1), dict(m=P[4] + 3),
    dict(u=P[2] + 2), dict(ws=P[3] + 8), dict(rows=2 ** 31), dict(ld=2 ** 62, rows=4),
    dict(vocab=2 ** 26 + 1, ld=2 ** 27)])
def test_sample_refuses(change):
    assert sample() == OK
    assert sample(**change) == E


def test_sample_workspace():
    assert F.sample_workspace(1, 1) > 0
    assert F.sample_workspace(-1, 5) == 0 and F.sample_workspace(1, 0) == 0 and F.sample_workspace(1, 2 ** 26 + 1) == 0


def test_reference_codes():
    """The reference's codes: every value comes back as itself, ties go to the even code."""
    for cache in (R.INT8, R.E4M3):
        codes = np.array([c for c in range(256) if not (c & 127 == 127 and cache == R.E4M3) and c != 128], np.uint8)
        assert np.array_equal(R.encode(R.decode(codes, cache), cache), codes)
    assert R.decode(np.array([0x7E, 0x38, 0x01, 0xC0], np.uint8), R.E4M3).tolist() == [448.0, 1.0, 2.0 ** -9, -2.0]
    assert R.encode(np.array([0.5, 1.5, -2.5, 126.5, 400.0]), R.INT8).view(np.int8).tolist() == [0, 2, -2, 126, 127]
    assert R.decode(R.encode(np.array([1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 1e9]), R.E4M3), R.E4M3).tolist() == \
        [1.0, 1.25, 0.0, 2.0 ** -8, 448.0]


def test_reference_sample():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3], np.float32))
    assert [R.sample(x, u=u) for u in (0.0, 0.39, 0.41, 0.69, 0.71, 0.89, 0.91, 0.999)] == [1, 1, 3, 3, 2, 2, 0, 0]
    assert {R.sample(x, top_k=2, u=u) for u in (0.1, 0.5, 0.9)} == {1, 3}
    assert {R.sample(x, top_p=0.65, u=u) for u in (0.1, 0.5, 0.9)} == {1, 3}
    assert {R.sample(x, min_p=0.6, u=u) for u in (0.1, 0.5, 0.9)} == {1, 3}


def test_model_sample_refuses():
    import ctypes
    import fence_model as M
    token = ctypes.c_int(-5)
    assert M.lib().fence_model_sample(None, P[0], 1.0, 0, 1.0, 0.0, 0.5, ctypes.byref(token)) == E
    assert token.value == -5
