"""Workspaces that are made once, for the largest batch, and used for every smaller one.  No GPU."""
import pytest

import fence_ops as F


@pytest.mark.parametrize("vocab", [1, 3, 1000, 4096, 10241, 32000, 50257, 128256, 151936, 262144, 2 ** 20, 2 ** 26])
def test_sample_workspace_never_falls_as_rows_rise(vocab):
    sizes = [F.sample_workspace(rows, vocab) for rows in range(600)]
    assert sizes[0] >= 16 and sizes == sorted(sizes)
    assert F.sample_workspace(100000, vocab) >= sizes[-1]


def test_sample_takes_a_larger_batch_workspace():
    """The size of 35 rows serves 26 to 34: no refusal (rows of 0 have nothing to do, so the check alone is seen)."""
    P = [0x10000 * (i + 1) for i in range(4)]
    call = lambda rows, size: F.lib().fence_sample(P[0], P[1], rows, 151936, 151936, None, None, None, None, P[2], P[3],  # noqa: E731
                                                   size, None)
    assert call(0, F.sample_workspace(0, 151936)) == F.SUCCESS
    for rows in range(35):
        assert F.sample_workspace(35, 151936) >= F.sample_workspace(rows, 151936)
    assert call(0, 0) == F.EINVAL


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(32, 8, 128), (14, 2, 64), (8, 8, 256), (64, 1, 48)])
def test_attention_workspace_never_falls(heads, kv_heads, head_dim):
    size = lambda batch, q: F.gqa_attention_q8_workspace(batch, q, heads, kv_heads, head_dim)  # noqa: E731
    for batch in (1, 2, 63, 64, 65, 1000, 65535):
        sizes = [size(batch, q) for q in list(range(200)) + [1000, 10000]]
        assert sizes == sorted(sizes) and sizes[1] >= size(batch - 1, 1)
