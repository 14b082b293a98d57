"""The 8-bit GQA layer on a B200 against oracle/gqa.py (64 bits).

Tolerances, from the arithmetic:
* an output of 16 bits is rounded once: eps / 2 of its value (and half the least subnormal for fp16).
* norm and rotation: the sum of up to 256 squares and the root are off by less than 2^-18 relative in fp32,
  the rotation by three roundings of its two products: 2^-17 of the pair's length covers both.
* attention: a score is a sum of `dim` exact products in fp32 (2^-24 each, the tensor core's sums are truncated,
  so 2^-20 of sum|q k| covers 256 of them) times three fp32 factors; e^s is off by that much and 2^-21 of its
  own; a weight is rounded to fp16 (2^-11) before it meets V; sums and merges are fp32.  So |o - exact| <= eps/2 |o|
  + (2^-11 + 2^-14 + 2 ds) sum_j p_j |v_j| with ds = 2^-20 * max_j sum_d |q k| scale, and |lse - exact| <= ds + 2^-20 (1 + |lse|).
"""
import numpy as np
import pytest
import torch

from gqa_cases import Batch, rounded
from oracle import gqa as G8

pytestmark = pytest.mark.gpu

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = 2.0 ** -25


def put(x, cuda, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to(cuda)
    return t if dtype is None else t.to(TORCH[dtype])


def get(t):
    return t.float().cpu().numpy() if t.dtype in (torch.bfloat16, torch.float16) else t.cpu().numpy()


def on_gpu(b, cuda):
    """The batch's arrays on the GPU: q, the cache's four arrays, block table, cu_seqlens, positions."""
    c = {n: put(a, cuda) for n, a in b.cache.items()}
    return put(b.q, cuda, b.dtype), c, put(b.bt, cuda), put(b.cu, cuda), put(b.pos, cuda)


def four(c):
    return c["k"], c["v"], c["ks"], c["vs"]


def near(got, lse, b, blocks=None, q=None, pos=None, rows=None):
    want, wl, mag, size = G8.attend(b.q if q is None else q, b.cache, b.bt, b.cu, b.pos if pos is None else pos, b.scale, blocks)
    ds = (2.0 ** -20 * size)[..., None]
    tol = HALF_STEP[b.dtype] * np.abs(want) + (2.0 ** -11 + 2.0 ** -14 + 2 * ds) * mag + TINY
    o, l = get(got).astype(np.float64), get(lse).astype(np.float64)
    if rows is not None:
        o, l, want, wl, tol, ds = o[rows], l[rows], want[rows], wl[rows], tol[rows], ds[rows]
    assert np.isfinite(o).all()
    bad = np.abs(o - want) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.max(np.abs(o - want) / tol):.2f} of the tolerance at {np.argwhere(bad)[:4].tolist()}"
    empty = np.isinf(wl)
    assert np.array_equal(np.isneginf(l), empty)
    lt = ds[..., 0] + 2.0 ** -20 * (1 + np.abs(np.where(empty, 0, wl)))
    assert (np.abs(np.where(empty, 0, l) - np.where(empty, 0, wl)) <= lt).all()


# ------------------------------------------------------------------------------------------
# QK norm and rotation
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T,H,G,D,rot,pairs,dtype,gain", [
    (1, 1, 1, 64, 64, False, "bf16", True), (7, 32, 8, 128, 128, False, "bf16", True), (33, 5, 1, 256, 256, False, "f16", True),
    (5, 12, 4, 64, 32, True, "f16", True), (3, 28, 4, 128, 64, False, "bf16", False), (4, 7, 2, 96, 48, True, "bf16", True),
    (2, 3, 3, 80, 16, False, "f16", True), (6, 4, 2, 8, 0, False, "bf16", True), (9, 0, 3, 128, 128, True, "bf16", True), (9, 17, 0, 192, 192, False, "bf16", True)])
def test_norm_rope(hk, cuda, T, H, G, D, rot, pairs, dtype, gain):
    rng = np.random.default_rng(T * D + H)
    x = rounded(rng.standard_normal((T, (H + 2 * G) * D + 8)) * 2.0 ** rng.integers(-6, 6, (T, 1)), dtype)
    x[0, :D] = 0  # a head of zeros
    qg, kg = (rounded(rng.standard_normal((2, D)), dtype) if gain else (None, None))
    pos = rng.integers(0, 40000, T).astype(np.int32)
    if T > 4:
        pos[2] = -1
    table = np.zeros((40000, rot), np.float32) if rot == 0 else hk.rope_table(40000, rot, 1e4, 0, 1.0, 32.0, 1.0)
    xd = put(x, cuda, dtype)
    q, k = xd[:, :H * D].unflatten(1, (H, D)), xd[:, H * D:(H + G) * D].unflatten(1, (G, D))
    outs = [torch.full((T, n, D), 5.0, dtype=TORCH[dtype], device=cuda) for n in (H, G)]
    hk.qk_norm_rope(q, k, put(pos, cuda), put(table, cuda), None if qg is None else put(qg, cuda, dtype), None if kg is None else put(kg, cuda, dtype),
                    interleaved=pairs, eps=1e-6, q_out=outs[0], k_out=outs[1])
    hk.check_errors()
    for n, at, g, got in ((H, 0, qg, outs[0]), (G, H, kg, outs[1])):
        src = x[:, at * D:(at + n) * D].reshape(T, n, D)
        want = G8.norm_rope(src, g, pos, table, pairs, 1e-6)
        want[pos < 0] = 5.0
        i = np.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + rot // 2)
        size = np.abs(want).copy()
        size[..., a] = size[..., b] = np.hypot(want[..., a], want[..., b])
        assert (np.abs(get(got) - want) <= HALF_STEP[dtype] * np.abs(want) + 2.0 ** -17 * size + TINY).all()
    # in place, inside the fused rows: the same bits, and the rest of the rows untouched
    hk.qk_norm_rope(q, k, put(pos, cuda), put(table, cuda), None if qg is None else put(qg, cuda, dtype), None if kg is None else put(kg, cuda, dtype),
                    interleaved=pairs, eps=1e-6, q_out=q, k_out=k)
    y = get(xd)
    keep = pos >= 0
    assert np.array_equal(y[keep, :H * D], get(outs[0]).reshape(T, -1)[keep]) and np.array_equal(y[keep, H * D:(H + G) * D], get(outs[1]).reshape(T, -1)[keep])
    assert np.array_equal(y[:, (H + G) * D:], x[:, (H + G) * D:]) and np.array_equal(y[~keep], x[~keep])


def test_norm_rope_flags_a_position_past_the_table(hk, cuda):
    q = torch.ones((2, 2, 64), dtype=torch.bfloat16, device=cuda)
    out, _ = hk.qk_norm_rope(q, q, put(np.array([3, 4], np.int32), cuda), torch.ones((4, 64), device=cuda), q_out=torch.full_like(q, 7))
    with pytest.raises(hk.HKError, match="position"):
        hk.check_errors()
    assert (out[1] == 7).all() and not (out[0] == 7).any()


# ------------------------------------------------------------------------------------------
# Append
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,ctx,kv,dim,page,dtype", [
    ([1], [0], 1, 64, 16, "bf16"), ([1, 1, 1, 1, 1], [15, 16, 17, 31, 0], 2, 64, 16, "f16"), ([5, 0, 3, 130, 1], [60, 9, 63, 40, 127], 3, 128, 64, "bf16"),
    ([200, 7], [0, 250], 2, 256, 128, "bf16"), ([40, 1, 300], [3, 47, 48], 1, 128, 48, "f16"), ([300], [5], 2, 64, 256, "bf16")])
def test_append(hk, cuda, rows, ctx, kv, dim, page, dtype):
    b = Batch(rows, ctx, kv, kv, dim, page, dtype, seed=dim + page)
    k, v = b.new_rows()
    want = {n: a.copy() for n, a in b.cache.items()}
    G8.append(k, v, b.slots, want)
    c = {n: put(a, cuda) for n, a in b.cache.items()}
    fused = put(np.concatenate([k.reshape(b.T, -1), v.reshape(b.T, -1)], 1), cuda, dtype)
    kd, vd = fused[:, :kv * dim].unflatten(1, (kv, dim)), fused[:, kv * dim:].unflatten(1, (kv, dim))
    for n in range(2):  # a second call on the grown pages changes nothing
        hk.gqa_append_fp8(kd, vd, put(b.slots, cuda), *four(c), c["cen"], c["cs"])
        hk.check_errors()
        for name in ("ks", "vs", "k", "v", "cen", "cs"):
            assert np.array_equal(get(c[name]), want[name], equal_nan=True), name


def test_append_without_centroids_leaves_them(hk, cuda):
    b = Batch([16], [0], 1, 1, 64, 16)
    c = {n: put(a, cuda) for n, a in b.cache.items()}
    cen = c["cen"].clone()
    hk.gqa_append_fp8(put(b.new_rows()[0], cuda, "bf16"), put(b.new_rows()[1], cuda, "bf16"), put(b.slots, cuda), *four(c))
    hk.check_errors()
    assert torch.equal(cen, c["cen"])


def test_append_skips_padding_and_flags_bad_slots(hk, cuda):
    b = Batch([1], [0], 1, 1, 64, 16, spare=6)
    x = put(rounded(np.random.default_rng(0).standard_normal((8, 1, 64)), "bf16"), cuda, "bf16")
    c = {n: put(np.zeros_like(a), cuda) for n, a in b.cache.items()}
    hk.gqa_append_fp8(x, x, put(np.array([-1, 16, 17, -1, -1, 33, -1, -1], np.int32), cuda), *four(c))
    hk.check_errors()
    used = get(c["k"]).reshape(-1, 64).any(1).nonzero()[0].tolist()
    assert used == [16, 17, 33]
    # the same slot twice, a gap, a slot past the pool: skipped and reported, the others written
    c = {n: put(np.zeros_like(a), cuda) for n, a in b.cache.items()}
    hk.gqa_append_fp8(x, x, put(np.array([16, 16, 48, 50, 51, 32, b.pages * 16, 64], np.int32), cuda), *four(c))
    with pytest.raises(hk.HKError, match="append slot"):
        hk.check_errors()
    assert get(c["k"]).reshape(-1, 64).any(1).nonzero()[0].tolist() == [16, 32, 48, 64]


def test_append_stores_no_nan(hk, cuda):
    x = np.random.default_rng(1).standard_normal((3, 1, 64)).astype(np.float32)
    x[0, 0, 3], x[1, 0, 5], x[2, 0, 7] = np.nan, np.inf, -np.inf
    x = rounded(x, "bf16")
    c = dict(k=np.zeros((2, 1, 16, 64), np.uint8), v=np.zeros((2, 1, 16, 64), np.uint8), ks=np.ones((2, 1), np.float32), vs=np.ones((2, 1), np.float32), cen=None)
    d = {n: put(a, cuda) for n, a in c.items() if a is not None}
    slots = np.arange(16, 19, dtype=np.int32)
    G8.append(x, x, slots, c)
    hk.gqa_append_fp8(put(x, cuda, "bf16"), put(x, cuda, "bf16"), put(slots, cuda), *four(d))
    with pytest.raises(hk.HKError, match="kv input"):
        hk.check_errors()
    got = G8.E4M3[get(d["k"])[1, 0]]
    assert got[0, 3] == 0 and got[1, 5] == 448 and got[2, 7] == -448
    assert np.array_equal(get(d["k"]), c["k"]) and np.array_equal(get(d["ks"]), c["ks"])


# ------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------

ATTEND = {
    "one row, one token": dict(rows=[1], ctx=[0], heads=1, kv=1, dim=64, page=16),
    "decode, lengths around page ends": dict(rows=[1] * 9, ctx=[0, 14, 15, 16, 62, 63, 64, 127, 128], heads=32, kv=8, dim=128, page=64),
    "idle lanes": dict(rows=[0, 1, 0, 0, 3, 0], ctx=[5, 100, 0, 9, 70, 1], heads=4, kv=2, dim=128, page=32),
    "three heads to a group, small pages": dict(rows=[1, 2, 7, 3], ctx=[700, 3, 1200, 0], heads=12, kv=4, dim=64, page=16, dtype="f16"),
    "one KV head for all": dict(rows=[1, 4], ctx=[333, 90], heads=16, kv=1, dim=128, page=64),
    "a head to itself": dict(rows=[1, 5, 1], ctx=[500, 61, 2], heads=6, kv=6, dim=64, page=48, dtype="f16"),
    "wide heads": dict(rows=[1, 3, 9], ctx=[900, 127, 30], heads=8, kv=2, dim=256, page=128),
    "verify blocks": dict(rows=[5, 5, 5], ctx=[2000, 59, 64], heads=32, kv=8, dim=128, page=64),
    "verify blocks of wide groups": dict(rows=[4, 8, 1], ctx=[1000, 120, 40], heads=32, kv=2, dim=128, page=64),
    "a long lane": dict(rows=[2], ctx=[30000], heads=8, kv=2, dim=128, page=64),
    "chunk from the start": dict(rows=[200], ctx=[0], heads=4, kv=1, dim=128, page=64),
    "chunks behind a cache": dict(rows=[130, 65, 1, 300], ctx=[77, 640, 500, 1], heads=8, kv=2, dim=128, page=64),
    "chunks, small heads": dict(rows=[150, 40], ctx=[10, 301], heads=6, kv=2, dim=64, page=32, dtype="f16"),
    "chunks, wide heads": dict(rows=[70, 33], ctx=[200, 0], heads=4, kv=2, dim=256, page=64),
    "chunks, odd pages and group": dict(rows=[129, 17], ctx=[47, 144], heads=15, kv=3, dim=128, page=48),
    "chunks, big pages": dict(rows=[257], ctx=[511], heads=4, kv=2, dim=128, page=256, dtype="f16"),
    "scales that are no powers of two": dict(rows=[1, 3, 140], ctx=[400, 100, 90], heads=8, kv=2, dim=128, page=64, pow2=False),
    "sharp scores": dict(rows=[1, 2, 150], ctx=[800, 300, 100], heads=8, kv=2, dim=128, page=64, sharp=30.0),
}


@pytest.mark.parametrize("name", ATTEND)
def test_attention(hk, cuda, name):
    b = Batch(**ATTEND[name], seed=len(name))
    q, c, bt, cu, pos = on_gpu(b, cuda)
    out, lse = hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, b.max_rows, b.max_kv, b.scale)
    hk.check_errors()
    near(out, lse, b)
    again = hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, b.max_rows, b.max_kv, b.scale)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_attention_bounds_may_be_generous(hk, cuda):
    """max_rows and max_kv_len above what the lanes have change nothing but the grid."""
    b = Batch([1, 3, 2], [100, 64, 9], 8, 2, 128, 64, seed=5)
    q, c, bt, cu, pos = on_gpu(b, cuda)
    for rows, kv in ((b.max_rows, b.max_kv), (500, 1 << 20), (b.max_rows, 0)):
        out, lse = hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, rows, kv, b.scale)
        hk.check_errors()
        near(out, lse, b)


def test_attention_leaves_rows_behind_the_last_lane(hk, cuda):
    for rows in ([1, 2], [90, 40]):
        b = Batch(rows, [50, 70], 4, 2, 128, 64, seed=7)
        q, c, bt, cu, pos = on_gpu(b, cuda)
        pad = 5
        qp = torch.cat([q, torch.full((pad, 4, 128), float("nan"), dtype=q.dtype, device=cuda)])
        posp = torch.cat([pos, torch.full((pad,), 1 << 30, dtype=torch.int32, device=cuda)])
        out = torch.full_like(qp, 3.0)
        lse = torch.full((b.T + pad, 4), 4.0, device=cuda)
        hk.gqa_decode_fp8(qp, *four(c), bt, cu, posp, b.max_rows, b.max_kv, b.scale, out=out, lse=lse)
        hk.check_errors()
        near(out[:b.T], lse[:b.T], b)
        assert (out[b.T:] == 3).all() and (lse[b.T:] == 4).all()


def test_attention_row_that_sees_nothing(hk, cuda):
    b = Batch([1, 1, 1], [40, 7, 100], 4, 2, 128, 64, seed=8)
    q, c, bt, cu, pos = on_gpu(b, cuda)
    p = b.pos.copy()
    p[1] = -1
    out, lse = hk.gqa_decode_fp8(q, *four(c), bt, cu, put(p, cuda), 1, b.max_kv, b.scale)
    hk.check_errors()
    near(out, lse, b, pos=p)
    assert (out[1] == 0).all() and torch.isneginf(lse[1]).all()


def test_attention_extreme_queries(hk, cuda):
    """Rows of zeros, of the type's largest and smallest values, beside ordinary ones."""
    for dtype, big, small in (("bf16", 1e4, 1e-30), ("f16", 3e4, 6e-8)):
        b = Batch([1, 4], [90, 300], 8, 2, 128, 64, dtype=dtype, seed=9)
        b.q[0] = 0
        b.q[1, :2] = rounded(np.float32(b.q[1, :2] * np.float32(big / 8)), dtype)
        b.q[2] = rounded(np.float32(np.sign(b.q[2]) * small), dtype)
        q, c, bt, cu, pos = on_gpu(b, cuda)
        out, lse = hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, b.max_rows, b.max_kv, b.scale)
        hk.check_errors()
        near(out, lse, b)


def test_a_query_row_that_is_not_finite_stays_alone(hk, cuda):
    for rows in ([4], [140]):
        b = Batch(rows, [200], 8, 2, 128, 64, seed=10)
        b.q[1, 3, 5] = np.nan
        q, c, bt, cu, pos = on_gpu(b, cuda)
        out, lse = hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, b.max_rows, b.max_kv, b.scale)
        hk.check_errors()
        assert torch.isnan(out[1, 3]).all() and torch.isnan(lse[1, 3])
        out[1, 3], lse[1, 3] = 0, 0
        good = np.ones(b.T, bool)
        good[1] = False
        b.q[1, 3, 5] = 0
        near(out, lse, b, rows=good)


def test_attention_reports_bad_pages_and_reads_none(hk, cuda):
    for rows in ([1, 1], [100, 1]):
        b = Batch(rows, [200, 100], 4, 2, 128, 64, seed=11)
        for bad in (0, b.pages, -3, 1 << 30):
            b.bt[0, 1] = bad
            q, c, bt, cu, pos = on_gpu(b, cuda)
            out, lse = hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, b.max_rows, b.max_kv, b.scale)
            with pytest.raises(hk.HKError, match="attn page"):
                hk.check_errors()
            near(out, lse, b)


def test_attention_reports_a_lane_past_max_rows(hk, cuda):
    b = Batch([1, 40, 2], [30, 20, 80], 4, 2, 128, 64, seed=12)
    q, c, bt, cu, pos = on_gpu(b, cuda)
    out, lse = torch.full_like(q, 3.0), torch.full((b.T, 4), 4.0, device=cuda)
    hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, 2, b.max_kv, b.scale, out=out, lse=lse)
    with pytest.raises(hk.HKError, match="lane rows"):
        hk.check_errors()
    assert (out[1:41] == 3).all() and (lse[1:41] == 4).all()
    near(out, lse, b, rows=np.r_[0, 41, 42])


def test_attention_reads_strided_queries(hk, cuda):
    b = Batch([2, 1, 120], [100, 7, 30], 4, 2, 128, 64, seed=13)
    q, c, bt, cu, pos = on_gpu(b, cuda)
    wide = torch.full((b.T, 4 * 128 + 40), float("nan"), dtype=q.dtype, device=cuda)
    wide[:, :512] = q.view(b.T, -1)
    out, lse = hk.gqa_decode_fp8(wide[:, :512].unflatten(1, (4, 128)), *four(c), bt, cu, pos, b.max_rows, b.max_kv, b.scale)
    hk.check_errors()
    near(out, lse, b)


def test_attention_far_into_a_large_pool(hk, cuda):
    """Pages whose byte offset passes 32 bits."""
    G, D, page = 8, 128, 64
    pages = (1 << 32) // (G * D * page) + 9
    b = Batch([1, 3], [150, 70], 16, G, D, page, seed=14)
    q, _, _, cu, pos = on_gpu(b, cuda)
    big = dict(k=torch.zeros((pages, G, page, D), dtype=torch.uint8, device=cuda), v=torch.zeros((pages, G, page, D), dtype=torch.uint8, device=cuda),
               ks=torch.zeros((pages, G), device=cuda), vs=torch.zeros((pages, G), device=cuda))
    shift = pages - b.pages
    for n in big:
        big[n][shift + 1:] = put(b.cache[n], cuda)[1:]
    bt = np.where(b.bt > 0, b.bt + shift, 0).astype(np.int32)
    out, lse = hk.gqa_decode_fp8(q, *four(big), put(bt, cuda), cu, pos, b.max_rows, b.max_kv, b.scale)
    hk.check_errors()
    near(out, lse, b)


# ------------------------------------------------------------------------------------------
# Selected blocks
# ------------------------------------------------------------------------------------------

SELECT = {
    "fewer blocks than asked": dict(rows=[1, 3, 0, 2], ctx=[5, 200, 9, 0], heads=4, kv=2, dim=64, page=16, top=20),
    "decode": dict(rows=[1, 1, 1, 1], ctx=[3000, 511, 512, 100], heads=8, kv=2, dim=128, page=16, top=9),
    "verify": dict(rows=[5, 2], ctx=[1500, 700], heads=12, kv=4, dim=64, page=32, top=7, dtype="f16"),
    "wide heads": dict(rows=[1, 2], ctx=[2000, 900], heads=4, kv=2, dim=256, page=64, top=5),
    "many blocks": dict(rows=[2], ctx=[20000], heads=4, kv=1, dim=64, page=16, top=100),
    "only the forced ones": dict(rows=[2, 1], ctx=[400, 900], heads=4, kv=1, dim=128, page=32, top=3),
}


def _select(hk, b, cuda, top, sink=1, local=2, q=None):
    qd, c, bt, cu, pos = on_gpu(b, cuda)
    got = hk.gqa_select_blocks(qd if q is None else q, c["cen"], c["cs"], bt, cu, pos, b.page, b.max_kv, top, sink=sink, local=local)
    return got, (qd, c, bt, cu, pos)


@pytest.mark.parametrize("name", SELECT)
def test_selected_blocks_and_their_attention(hk, cuda, name):
    case = dict(SELECT[name])
    top = case.pop("top")
    b = Batch(**case, seed=len(name))
    got, (q, c, bt, cu, pos) = _select(hk, b, cuda, top)
    hk.check_errors()
    want = G8.select(b.q, b.cache, b.bt, b.cu, b.pos, top, 1, 2)
    assert np.array_equal(get(got), want)
    out, lse = hk.gqa_sparse_fp8(q, *four(c), bt, cu, pos, got, b.scale)
    hk.check_errors()
    near(out, lse, b, blocks=want)


def test_equal_scores_go_to_the_lower_block(hk, cuda):
    b = Batch([1, 1], [1200, 1600], 4, 2, 64, 16, seed=3)
    b.cache["cen"][:] = b.cache["cen"][1]
    b.cache["cs"][:] = 0.25
    got, _ = _select(hk, b, cuda, 10)
    hk.check_errors()
    n = b.pos // 16 + 1
    for t in range(2):
        assert (get(got)[t] == np.r_[np.arange(8), n[t] - 2, n[t] - 1]).all()


def test_selection_of_odd_rows(hk, cuda):
    """Zero queries, queries that are not finite, rows in sight of nothing, rows behind the last lane."""
    b = Batch([4, 1], [900, 300], 4, 2, 64, 16, seed=4)
    b.q[0] = 0
    b.q[1, 0, 0], b.q[2, 1, 3] = np.inf, np.nan
    b.pos[4] = -1
    q, c, bt, cu, pos = on_gpu(b, cuda)
    q = torch.cat([q, q[:2]])
    pos = torch.cat([pos, torch.full((2,), 1 << 30, dtype=torch.int32, device=cuda)])
    blocks = torch.full((7, 2, 12), -7, dtype=torch.int32, device=cuda)
    hk.gqa_select_blocks(q, c["cen"], c["cs"], bt, cu, pos, 16, b.max_kv, 12, sink=2, local=3, blocks=blocks)
    hk.check_errors()
    assert np.array_equal(get(blocks)[:5], G8.select(b.q, b.cache, b.bt, b.cu, b.pos, 12, 2, 3))
    assert (blocks[5:] == -7).all()
    # past max_kv_len: reported, an empty list
    hk.gqa_select_blocks(q[:5], c["cen"], c["cs"], bt, cu, pos[:5], 16, 400, 12, blocks=blocks[:5])
    with pytest.raises(hk.HKError, match="position"):
        hk.check_errors()
    assert (blocks[:4] == -1).all()


def test_select_reports_bad_pages(hk, cuda):
    b = Batch([1], [900], 4, 2, 64, 16, seed=5)
    b.bt[0, 20] = b.pages
    got, _ = _select(hk, b, cuda, 12)
    with pytest.raises(hk.HKError, match="attn page"):
        hk.check_errors()
    assert not (get(got) == 20).any()


def test_sparse_attention_of_odd_lists(hk, cuda):
    """Empty lists, lists that do not rise or pass the row's position: what is listed rightly is read."""
    b = Batch([3, 1], [300, 90], 4, 2, 128, 32, seed=6)
    q, c, bt, cu, pos = on_gpu(b, cuda)
    lists = np.full((4, 2, 6), -1, np.int32)
    lists[0, 0, :3], lists[1, 0, :1], lists[2, 1, :6], lists[3, 1, :2] = [0, 4, 9], [9], [1, 2, 3, 5, 7, 9], [1, 2]
    out, lse = hk.gqa_sparse_fp8(q, *four(c), bt, cu, pos, put(lists, cuda), b.scale)
    hk.check_errors()
    near(out, lse, b, blocks=lists)
    bad = lists.copy()
    bad[0, 0, :6] = [0, 4, 4, 3, 9, 40]
    bad[3, 1, :4] = [1, 2, 3, 1 << 30]
    out, lse = hk.gqa_sparse_fp8(q, *four(c), bt, cu, pos, put(bad, cuda), b.scale)
    with pytest.raises(hk.HKError, match="block list"):
        hk.check_errors()
    near(out, lse, b, blocks=lists)


# ------------------------------------------------------------------------------------------
# Together: a layer's steps in order, captured, on another stream
# ------------------------------------------------------------------------------------------

def _layer(hk, qkv, d, b, table, top, ws):
    H, G, D = b.heads, b.kv, b.dim
    q = qkv[:, :H * D].unflatten(1, (H, D))
    k = qkv[:, H * D:(H + G) * D].unflatten(1, (G, D))
    v = qkv[:, (H + G) * D:].unflatten(1, (G, D))
    c = d["c"]
    q, k = hk.qk_norm_rope(q, k, d["pos"], table, d["qg"], d["kg"])
    hk.gqa_append_fp8(k, v, d["slots"], *four(c), c["cen"], c["cs"])
    dense = hk.gqa_decode_fp8(q, *four(c), d["bt"], d["cu"], d["pos"], b.max_rows, b.max_kv, b.scale, workspace=ws)
    blocks = hk.gqa_select_blocks(q, c["cen"], c["cs"], d["bt"], d["cu"], d["pos"], b.page, b.max_kv, top, sink=1, local=2)
    return (*dense, blocks, *hk.gqa_sparse_fp8(q, *four(c), d["bt"], d["cu"], d["pos"], blocks, b.scale, workspace=ws))


@pytest.mark.parametrize("rows", [[1, 1, 4], [90, 1, 3]])
def test_a_layer_from_pack_to_sparse_attention(hk, orc, cuda, rows):
    b = Batch(rows, [300, 0, 700], 8, 2, 128, 32, seed=20)
    T = b.T
    rng = np.random.default_rng(21)
    qkv = rounded(rng.standard_normal((T, 12 * 128)), "bf16")
    gains = rounded(1 + 0.1 * rng.standard_normal((2, 128)), "bf16")
    table = hk.rope_table(2048, 128, 1e4, 0, 1.0, 32.0, 1.0)
    p = hk.pack(put(np.array(rows, np.int32), cuda), put(np.array(b.ctx, np.int32), cuda), put(b.bt, cuda), 32, b.pages, T)
    assert np.array_equal(get(p["slot_mapping"])[:T], b.slots) and np.array_equal(get(p["positions"])[:T], b.pos)
    d = dict(c={n: put(a, cuda) for n, a in b.cache.items()}, pos=p["positions"], slots=p["slot_mapping"], cu=p["cu_seqlens"], bt=put(b.bt, cuda),
             qg=put(gains[0], cuda, "bf16"), kg=put(gains[1], cuda, "bf16"))
    x, tab = put(qkv, cuda, "bf16"), put(table, cuda)
    ws = torch.empty(hk.gqa_fp8_workspace_size(T, 8, 2, 128), dtype=torch.uint8, device=cuda)
    got = _layer(hk, x, d, b, tab, 8, ws)
    hk.check_errors()
    # the same steps in 64 bits, from the device's own rotated and rounded rows
    qr, kr = hk.qk_norm_rope(x[:, :1024].unflatten(1, (8, 128)), x[:, 1024:1280].unflatten(1, (2, 128)), d["pos"], tab, d["qg"], d["kg"])
    b.q = get(qr)
    G8.append(get(kr), qkv[:, 1280:].reshape(T, 2, 128), b.slots, b.cache)
    for n in ("k", "v", "ks", "vs", "cen", "cs"):
        assert np.array_equal(get(d["c"][n]), b.cache[n], equal_nan=True), n
    near(got[0], got[1], b)
    want = G8.select(b.q, b.cache, b.bt, b.cu, b.pos, 8, 1, 2)
    assert np.array_equal(get(got[2]), want)
    near(got[3], got[4], b, blocks=want)

    # the same layer on a stream of its own, and captured into two graphs that share the workspace
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = _layer(hk, x, d, b, tab, 8, ws)
    s.synchronize()
    assert all(torch.equal(u, w) for u, w in zip(got, other))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_layer(hk, x, d, b, tab, 8, ws))
        graphs.append(g)
    for n in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    hk.check_errors()
    for o in outs:
        assert all(torch.equal(u, w) for u, w in zip(got, o))


def test_wrappers_refuse_another_device_and_type(hk, cuda):
    b = Batch([1], [40], 4, 2, 128, 64)
    q, c, bt, cu, pos = on_gpu(b, cuda)
    with pytest.raises(ValueError, match="current device"):
        hk.gqa_decode_fp8(q, *four(c), bt.cpu(), cu, pos, 1, b.max_kv, b.scale)
    with pytest.raises(TypeError):
        hk.gqa_decode_fp8(q.float(), *four(c), bt, cu, pos, 1, b.max_kv, b.scale)
    with pytest.raises(TypeError):
        hk.gqa_decode_fp8(q, *four(c), bt.long(), cu, pos, 1, b.max_kv, b.scale)
    with pytest.raises(ValueError):
        hk.gqa_decode_fp8(q.transpose(1, 2).contiguous().transpose(1, 2), *four(c), bt, cu, pos, 1, b.max_kv, b.scale)
    with pytest.raises(hk.HKError):
        hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, 1, b.max_kv, b.scale, workspace=torch.empty(16, dtype=torch.uint8, device=cuda))


# ------------------------------------------------------------------------------------------
# Batches wider than a CTA's scan, groups wider than a tile, lists longer than its registers
# ------------------------------------------------------------------------------------------

WIDE = {
    "300 decode lanes": dict(rows=[1] * 300, ctx=[(37 * i) % 211 for i in range(300)], heads=4, kv=2, dim=64, page=32),
    "idle lanes among 700, two chunks": dict(rows=[(0, 1, 0, 2)[i % 4] if i not in (513, 699) else 90 for i in range(700)], ctx=[(13 * i) % 90 for i in range(700)],
                                             heads=2, kv=1, dim=64, page=16),
    "64 heads to a group": dict(rows=[1, 3, 0, 1], ctx=[90, 20, 3, 400], heads=64, kv=1, dim=64, page=32),
    "40 heads to a group, fp16": dict(rows=[2, 1], ctx=[300, 5], heads=80, kv=2, dim=128, page=64, dtype="f16"),
    "20 wide heads to a group": dict(rows=[1, 2], ctx=[200, 40], heads=40, kv=2, dim=256, page=64),
}


@pytest.mark.parametrize("name", WIDE)
def test_wide_batches(hk, cuda, name):
    b = Batch(**WIDE[name], seed=len(name))
    q, c, bt, cu, pos = on_gpu(b, cuda)
    out, lse = hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, b.max_rows, b.max_kv, b.scale)
    hk.check_errors()
    near(out, lse, b)
    got = hk.gqa_select_blocks(q, c["cen"], c["cs"], bt, cu, pos, b.page, b.max_kv, 4, sink=1, local=1)
    want = G8.select(b.q, b.cache, b.bt, b.cu, b.pos, 4, 1, 1)
    assert np.array_equal(get(got), want)
    out, lse = hk.gqa_sparse_fp8(q, *four(c), bt, cu, pos, got, b.scale)
    hk.check_errors()
    near(out, lse, b, blocks=want)


@pytest.mark.parametrize("blocks", [4200, 17000])
def test_long_lists_of_blocks(hk, cuda, blocks):
    """More keys than 256 threads hold, and more than 1024 threads hold; equal scores among them."""
    b = Batch([2], [blocks * 16 - 5], 2, 1, 64, 16, seed=blocks)
    b.cache["cen"][1::7] = b.cache["cen"][1]
    b.cache["cs"][1::7] = b.cache["cs"][1]
    for top in (8, 300):
        got, _ = _select(hk, b, cuda, top)
        hk.check_errors()
        assert np.array_equal(get(got), G8.select(b.q, b.cache, b.bt, b.cu, b.pos, top, 1, 2))


@pytest.mark.parametrize("tokens", [3, 1500])
def test_append_of_many_lanes(hk, cuda, tokens):
    """Rows of many lanes, single ones and runs of all lengths around the limits of the short ones, in one call."""
    rows = [1, 9, 8, 1, 70, 1, 17, 2] * (1 + tokens // 100)
    ctx = [(29 * i) % 33 for i in range(len(rows))]
    b = Batch(rows, ctx, 2, 2, 128, 32, seed=tokens)
    k, v = b.new_rows()
    want = {n: a.copy() for n, a in b.cache.items()}
    G8.append(k, v, b.slots, want)
    c = {n: put(a, cuda) for n, a in b.cache.items()}
    hk.gqa_append_fp8(put(k, cuda, "bf16"), put(v, cuda, "bf16"), put(b.slots, cuda), *four(c), c["cen"], c["cs"])
    hk.check_errors()
    for name in ("ks", "vs", "k", "v", "cen", "cs"):
        assert np.array_equal(get(c[name]), want[name], equal_nan=True), name


def test_calls_on_two_streams_with_their_own_workspaces(hk, cuda):
    """Two attentions at once give what each gives alone."""
    cases = [Batch([1, 70, 3], [700, 90, 40], 8, 2, 128, 64, seed=30 + i) for i in range(2)]
    on = [on_gpu(b, cuda) for b in cases]
    alone = [hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, b.max_rows, b.max_kv, b.scale) for b, (q, c, bt, cu, pos) in zip(cases, on)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[], []]
    for _ in range(5):
        for i, (b, (q, c, bt, cu, pos)) in enumerate(zip(cases, on)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(hk.gqa_decode_fp8(q, *four(c), bt, cu, pos, b.max_rows, b.max_kv, b.scale))
    torch.cuda.synchronize()
    hk.check_errors()
    for i in range(2):
        assert all(torch.equal(o, alone[i][0]) and torch.equal(l, alone[i][1]) for o, l in outs[i])
