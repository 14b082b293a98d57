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


@pytest.mark.parametrize("rows,ctx", [([1, 4], [50, 200]), ([1, 40], [50, 20]), ([140], [700])])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("size", [2.0 ** 30, 2.0 ** 97, 2.0 ** 101])
@pytest.mark.parametrize("sign", [-1, 1])
def test_scores_of_any_size(hk, cuda, rows, ctx, page, size, sign):
    """Scores up to 1e34 and down to -1e34 weigh against each other as any others do; a row is empty only when it sees nothing."""
    b = Batch(rows, ctx, 8, 2, 128, page, seed=53)
    rng = np.random.default_rng(54)
    pages = b.bt[b.bt > 0]
    code = b.cache["k"][pages]
    b.cache["k"][pages] = np.where(code == 0x7F, code, np.maximum(code & 0x7F, 0x38))  # keys at least 1 in every dim
    b.cache["ks"][pages] = 1
    b.q = rounded(sign * np.abs(rng.standard_normal(b.q.shape)).astype(np.float32) * np.float32(size), "bf16")
    q, c, bt, cu, pos = on_gpu(b, cuda)
    out, lse = hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, b.max_rows, b.max_kv, b.scale)
    hk.check_errors()
    want, wl, mag, _ = G8.attend(b.q, b.cache, b.bt, b.cu, b.pos, b.scale)
    # A score is off by 2^-20 of its size at most, far more than 1: which of two tokens that near each other has the weight is
    # open, all others have none.  So rows whose two largest scores are further apart are that of one token, the others finite.
    assert np.isfinite(get(out)).all()
    assert (np.abs(get(lse).astype(np.float64) - wl) <= 2.0 ** -18 * np.abs(wl)).all()
    second = second_scores(b)
    clear = wl - second > 2.0 ** -17 * np.abs(wl)
    assert clear.mean() > 0.9
    assert (np.abs(get(out) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * mag)[clear].all()


def second_scores(b):
    """The second largest score of each row and head (-inf: none)."""
    out = np.full((b.T, b.heads), -np.inf)
    for lane in range(len(b.rows)):
        for t in range(b.cu[lane], b.cu[lane + 1]):
            i = np.arange(b.pos[t] + 1)
            k = G8.E4M3[b.cache["k"][b.bt[lane, i // b.page], :, i % b.page]].transpose(1, 0, 2)  # ks is 1
            s = np.einsum("ghd,gnd->ghn", b.q[t].reshape(b.kv, -1, b.dim).astype(np.float64), k).reshape(b.heads, -1) * b.scale
            if len(i) > 1:
                out[t] = np.sort(s, -1)[:, -2]
    return out


@pytest.mark.parametrize("tail", [[5], [-1, 1], [-1, -1, 7], [-2], [1 << 30]])
def test_entries_behind_the_blocks_in_sight_are_reported(hk, cuda, tail):
    """A list as long as what is in sight, or shorter, and behind it entries that no row may read."""
    b = Batch([1, 2], [40, 20], 4, 2, 64, 32, seed=55)  # 2 blocks in sight of the first row, 1 of the others
    q, c, bt, cu, pos = on_gpu(b, cuda)
    lists = np.full((3, 2, 8), -1, np.int32)
    lists[0, :, :2], lists[1:, :, 0] = [0, 1], 0
    out, lse = hk.gqa_sparse_fp8(q, *four(c), bt, cu, pos, put(lists, cuda), b.scale)
    hk.check_errors()
    near(out, lse, b, blocks=lists)
    for t, g in ((0, 1), (2, 0)):
        bad = lists.copy()
        at = 2 if t == 0 else 1
        bad[t, g, at:at + len(tail)] = tail
        again = hk.gqa_sparse_fp8(q, *four(c), bt, cu, pos, put(bad, cuda), b.scale)
        with pytest.raises(hk.HKError, match="block list"):
            hk.check_errors()
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    # the list of a row that sees nothing is not read
    p = b.pos.copy()
    p[0] = -1
    bad = lists.copy()
    bad[0] = 99
    out, lse = hk.gqa_sparse_fp8(q, *four(c), bt, cu, put(p, cuda), put(bad, cuda), b.scale)
    hk.check_errors()
    near(out, lse, b, blocks=lists, pos=p)
