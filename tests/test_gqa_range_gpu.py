"""Attention over the 8-bit cache where one token outweighs the rest of a long context: a key many nats above the others whose
V is small or zero, so that the output is what the others leave, and a page whose V scale is far above the others'.

Tolerances are those of test_gqa_gpu.py, 2^-11 + 2^-14 + 2 ds of sum_j p_j |v_j| besides the output's rounding, plus one term.  A weight
is held in fp16 relative to 2^M, so what is below 2^-14 of it keeps an absolute error of 2^-25.  M follows the row's scores down as
well as up: it lies 7 bits below a peak, and 256 tokens after it (16 chunks of 16; 128 in the prompt-chunk kernel) it has come down
to the tokens there.  So a peak costs at most 272 tokens 2^-32 of its own weight each: 2^-32 p_peak times their sum of |v| (times the
ratio of V scales where it is a page's scale that is far above).
"""
import numpy as np
import pytest
import torch

from gqa_cases import Batch, rounded
from oracle import gqa as G8

pytestmark = pytest.mark.gpu
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}


def put(x, cuda):
    return torch.from_numpy(np.ascontiguousarray(x)).to(cuda)


def long_lane(rows, ctx, dim, peaks, dtype="f16", equal=False, sink_v=0.0, heads=8, seed=0):
    """One lane.  The first dim of K is 0 but at `peaks` (token: its score in nats above the mean of the rest), where the other dims are
    0; scores of the rest spread by about 1 (`equal`: not at all), V by 32 around 32; V at the peaks is 64 `sink_v`."""
    b = Batch([rows], [ctx], heads, 1, dim, 64, dtype, seed=seed)
    rng = np.random.default_rng(seed + 1)
    n, f, a = rows + ctx, 2.0 ** -5, 16.0
    k = np.zeros((n, dim))
    if not equal:
        k[:, 1:] = rng.standard_normal((n, dim - 1))
    v = 32 + 32 * rng.standard_normal((n, dim))
    for t, nats in peaks.items():
        k[t] = 0
        k[t, 0] = nats / (a * dim ** -0.5)
        v[t] = 64 * sink_v
    total = np.concatenate([np.zeros((1, dim)), np.abs(v).cumsum(0)])
    b.window = (total[272:] - total[:-272]).max()  # the largest sum of |v| over 272 tokens
    pad = -n % 64
    for name, s, x, g in (("k", "ks", k, f), ("v", "vs", v, 2.0 ** -1)):
        x = np.concatenate([x, np.zeros((pad, dim))]).reshape(-1, 1, 64, dim)
        pages = b.bt[0, :len(x)]
        b.cache[name][pages] = G8.to_e4m3(x / g)
        b.cache[s][pages] = g
    b.cache["k"][b.bt[0, (n - 1) // 64], 0, (n - 1) % 64 + 1:] = 0x7F
    b.cache["v"][b.bt[0, (n - 1) // 64], 0, (n - 1) % 64 + 1:] = 0x7F
    q = rng.standard_normal((rows, heads, dim))
    q[..., 0] = a
    b.q = rounded(q, dtype)
    return b


def check(hk, cuda, b, blocks=None, ratio=1.0, lanes=1, unit=1.0):
    """The lane `lanes` times over, so that a CTA walks whole lanes; outputs in units of `unit`, a power of two."""
    c = {n: put(x, cuda) for n, x in b.cache.items()}
    q = put(b.q, cuda).to(TORCH[b.dtype]).repeat(lanes, 1, 1)
    cu = np.arange(lanes + 1, dtype=np.int32) * b.T
    args = q, c["k"], c["v"], c["ks"], c["vs"], put(b.bt, cuda).repeat(lanes, 1), put(cu, cuda), put(b.pos, cuda).repeat(lanes)
    if blocks is None:
        out, lse = hk.gqa_decode_fp8(*args, b.max_rows, b.max_kv, b.scale)
    else:
        out, lse = hk.gqa_sparse_fp8(*args, put(blocks, cuda), b.scale)
    hk.check_errors()
    want, wl, mag, size = G8.attend(b.q, b.cache, b.bt, b.cu, b.pos, b.scale, blocks)
    ds = (2.0 ** -20 * size)[..., None]
    want, mag = want / unit, mag / unit
    peak = 2.0 ** -32 * b.window * ratio
    tol = HALF_STEP[b.dtype] * np.abs(want) + (2.0 ** -11 + 2.0 ** -14 + 2 * ds) * mag + peak + 2.0 ** -25
    off = np.abs(out.float().cpu().numpy().astype(np.float64).reshape(lanes, *want.shape) / unit - want) / tol
    assert off.max() <= 1, f"{(off > 1).sum()} of {off.size} off, worst {off.max():.2f} of the tolerance (outputs up to {np.abs(want).max():.2e})"
    assert (np.abs(lse.cpu().numpy().reshape(lanes, *wl.shape) - wl) <= ds[..., 0] + 2.0 ** -20 * (1 + np.abs(wl))).all()


PEAKS = {
    "first token, 17.5 nats": {0: 17.5},
    "first token, 24 nats": {0: 24.0},
    "middle of the context": {12345: 18.0},
    "rising": {0: 12.0, 5000: 18.0, 9000: 23.0},
    "falling": {100: 23.0, 9000: 17.0, 20000: 12.0},
    "a hundred in a row": {t: 18.0 for t in range(1000, 1100)},
}


@pytest.mark.parametrize("name", PEAKS)
@pytest.mark.parametrize("rows", [1, 20], ids=["row", "chunk"])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_a_peak_leaves(hk, cuda, name, rows, dim):
    check(hk, cuda, long_lane(rows, 30000, dim, PEAKS[name], seed=len(name)))


@pytest.mark.parametrize("rows", [1, 20], ids=["row", "chunk"])
@pytest.mark.parametrize("nats", [17.2, 18.6, 19.5])
def test_equal_weights_round_alike(hk, cuda, rows, nats):
    """Errors of equal weights do not average out."""
    check(hk, cuda, long_lane(rows, 30000, 128, {0: nats}, equal=True, seed=5))


@pytest.mark.parametrize("dim,rows,lanes", [(128, 1, 500), (64, 1, 700), (256, 1, 300), (128, 4, 300), (128, 5, 200)])
@pytest.mark.parametrize("name", ["first token, 17.5 nats", "first token, 24 nats", "falling"])
def test_many_lanes_behind_a_peak(hk, cuda, dim, rows, lanes, name):
    check(hk, cuda, long_lane(rows, 30000, dim, PEAKS[name], seed=11), lanes=lanes)


def test_wide_heads_and_a_small_value_at_the_peak(hk, cuda):
    check(hk, cuda, long_lane(3, 20000, 256, {7: 18.0}, sink_v=0.02, seed=6))
    check(hk, cuda, long_lane(20, 60000, 128, {7: 18.0}, sink_v=0.02, dtype="bf16", heads=4, seed=7))


def test_selected_blocks_behind_a_peak(hk, cuda):
    b = long_lane(1, 30000, 128, {3: 18.0}, seed=8)
    blocks = np.arange(0, 469, 1, dtype=np.int32)[None, None]
    check(hk, cuda, b, blocks=np.ascontiguousarray(blocks))


@pytest.mark.parametrize("rows", [1, 20], ids=["row", "chunk"])
@pytest.mark.parametrize("up", [10, 20])
def test_a_page_with_a_large_value_scale(hk, cuda, rows, up):
    """A page whose V is zero under a scale 2^up times the others': its tokens' weights stand as much above theirs."""
    b = long_lane(rows, 30000, 128, {}, seed=9)
    b.cache["v"][b.bt[0, 100]] = 0
    b.cache["vs"][b.bt[0, 100]] = 2.0 ** (up - 1)
    # one token's weight here is at most e^6 of the mean of 30,000
    check(hk, cuda, b, ratio=2.0 ** up * np.exp(6) / 30000)


@pytest.mark.parametrize("rows", [1, 20], ids=["row", "chunk"])
@pytest.mark.parametrize("peaks,unit", [({0: 20.0}, 2.0 ** -40), ({0: 20.0}, 2.0 ** 60), ({}, 2.0 ** -98), ({}, 2.0 ** 100)])
def test_value_scales_of_any_size(hk, cuda, rows, peaks, unit):
    b = long_lane(rows, 30000, 128, peaks, dtype="bf16", seed=12)
    b.cache["vs"][:] *= np.float32(unit)
    check(hk, cuda, b, unit=unit)
