"""The 8-bit GQA layer on a B200 at its edges: skipped chunks, tiny and huge queries, lists longer than what is in sight."""
import numpy as np
import pytest
import torch

from gqa_cases import Batch, rounded
from oracle import gqa as G8
from test_gqa_gpu import four, get, near, on_gpu, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 32])
def test_skipped_chunks_where_lookups_meet(hk, cuda, page):
    """A warp takes every fourth 16-token chunk and looks 16 of them up at a time: entries that are refused there (each warp's
    last of a lookup, and the first of the next), and bad pages likewise."""
    n = 600
    b = Batch([1, 1], [n * page - 3, n * page - 9], 4, 1, 128, page, seed=50)
    q, c, bt, cu, pos = on_gpu(b, cuda)
    chunks = page // 16
    at = sorted({(64 * k + d) // chunks for k in range(1, 600 * chunks // 64 + 1) for d in (-4, -3, -2, -1, 0, 3)} & set(range(1, 500)))
    lists = np.arange(500, dtype=np.int32)[None, None].repeat(2, 0) + 50
    bad = lists.copy()
    for i in at:
        bad[:, :, i] = bad[:, :, i - 1]  # does not rise: refused
    good = lists.copy()
    good[:, :, at] = -1
    out, lse = hk.gqa_sparse_fp8(q, *four(c), bt, cu, pos, put(bad, cuda), b.scale)
    with pytest.raises(hk.HKError, match="block list"):
        hk.check_errors()
    near(out, lse, b, blocks=good)
    b.bt[:, at] = b.pages  # dense, with the pages of those blocks outside the pool
    out, lse = hk.gqa_decode_fp8(q, *four(c), put(b.bt, cuda), cu, pos, b.max_rows, b.max_kv, b.scale)
    with pytest.raises(hk.HKError, match="attn page"):
        hk.check_errors()
    near(out, lse, b)


@pytest.mark.parametrize("down", [60, 100, 127])
def test_selection_by_tiny_queries(hk, cuda, down):
    """A power of two on a query changes none of its blocks, down to bf16's subnormals."""
    b = Batch([1, 3], [3000, 1500], 8, 2, 128, 16, seed=51)
    k = np.random.default_rng(52).integers(-64, 65, b.q.shape)
    b.q = (k * 2.0 ** -3).astype(np.float32)
    want = G8.select(b.q, b.cache, b.bt, b.cu, b.pos, 9, 1, 2)
    q, c, bt, cu, pos = on_gpu(b, cuda)
    small = put((k * 2.0 ** (-3 - down)).astype(np.float32), cuda, "bf16")
    assert np.array_equal(get(small).astype(np.float64) * 2.0 ** (3 + down), k)  # nothing is lost in bf16
    for x in (q, small):
        got = hk.gqa_select_blocks(x, c["cen"], c["cs"], bt, cu, pos, 16, b.max_kv, 9, sink=1, local=2)
        hk.check_errors()
        assert np.array_equal(get(got), want)
    b.q = (k * 2.0 ** (-3 - down)).astype(np.float32)
    assert np.array_equal(G8.select(b.q, b.cache, b.bt, b.cu, b.pos, 9, 1, 2), want)
