"""Refusals of the 8-bit GQA entry points and the oracle's own rounding, without a GPU.  Arguments are
checked before the device is asked for, so a bad call is HK_EINVAL or HK_ESPACE here too, and a good
one is HK_ENODEV."""
import numpy as np
import pytest

from oracle import gqa as G8

FAKE = 1 << 20  # an aligned address that no refused call reads


def _rope(**kw):
    a = dict(q=FAKE, qs=256, k=FAKE, ks=128, qg=None, kg=None, table=FAKE, rows=8, rot=64, pairs=0, pos=FAKE, T=2, H=4, G=2, D=64, eps=1e-6, dt=0,
             qo=FAKE, qos=256, ko=FAKE, kos=128)
    a.update(kw)
    return "hk_qk_norm_rope", [*a.values(), None]


def _append(**kw):
    a = dict(k=FAKE, ks=256, v=FAKE, vs=256, dt=0, slots=FAKE, T=2, G=2, D=128, page=64, pages=4, kc=FAKE, vc=FAKE, ksc=FAKE, vsc=FAKE, cen=FAKE, cs=FAKE)
    a.update(kw)
    return "hk_gqa_append_fp8", [*a.values(), None]


def _decode(**kw):
    a = dict(q=FAKE, qs=512, kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, bt=FAKE, stride=4, cu=FAKE, pos=FAKE, lanes=1, T=2, H=4, G=2, D=128, page=64, pages=4, max_rows=2,
             max_kv=64, scale=0.1, dt=0, out=FAKE, lse=FAKE, ws=FAKE, n=1 << 40)
    a.update(kw)
    return "hk_gqa_decode_fp8", [*a.values(), None]


def _select(**kw):
    a = dict(q=FAKE, qs=512, cen=FAKE, cs=FAKE, bt=FAKE, stride=4, cu=FAKE, pos=FAKE, lanes=1, T=2, H=4, G=2, D=128, page=64, pages=4, max_kv=640, top=4, sink=1,
             local=1, dt=0, blocks=FAKE, ws=FAKE, n=1 << 40)
    a.update(kw)
    return "hk_gqa_select_blocks", [*a.values(), None]


def _sparse(**kw):
    a = dict(q=FAKE, qs=512, kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, bt=FAKE, stride=4, cu=FAKE, pos=FAKE, blocks=FAKE, top=4, lanes=1, T=2, H=4, G=2, D=128, page=64,
             pages=4, scale=0.1, dt=0, out=FAKE, lse=FAKE, ws=FAKE, n=1 << 40)
    a.update(kw)
    return "hk_gqa_sparse_fp8", [*a.values(), None]


BAD = [
    _rope(dt=2), _rope(D=60), _rope(D=264, rot=0), _rope(rot=24), _rope(rot=80), _rope(rot=-16), _rope(qs=255), _rope(qs=192), _rope(kos=64), _rope(eps=-1.0),
    _rope(H=0, G=0), _rope(H=-1), _rope(q=None), _rope(ko=None), _rope(table=None), _rope(pos=None), _rope(q=FAKE + 2), _rope(qg=FAKE + 8), _rope(T=-1), _rope(rows=-1),
    _append(dt=-1), _append(D=96), _append(page=8), _append(page=72), _append(page=512), _append(ks=255), _append(vs=128), _append(G=0), _append(pages=0), _append(T=-1),
    _append(cen=None), _append(cs=None), _append(slots=None), _append(kc=None), _append(vsc=None), _append(k=FAKE + 4), _append(vc=FAKE + 8),
    _decode(dt=3), _decode(D=32), _decode(H=5), _decode(G=0), _decode(page=24), _decode(qs=256), _decode(qs=516), _decode(lanes=0), _decode(T=-1), _decode(stride=0),
    _decode(pages=0), _decode(scale=0.0), _decode(scale=float("nan")), _decode(scale=float("inf")), _decode(max_rows=-1), _decode(max_kv=-1), _decode(q=None),
    _decode(lse=None), _decode(bt=None), _decode(out=FAKE + 8), _decode(ws=FAKE + 128),
    _select(dt=2), _select(D=80), _select(H=6, G=4), _select(page=40), _select(top=0), _select(top=5000), _select(local=0), _select(sink=-1), _select(sink=4), _select(qs=500),
    _select(cen=None), _select(blocks=None), _select(max_kv=-1), _select(cen=FAKE + 1), _select(ws=FAKE + 4),
    _sparse(top=0), _sparse(top=4097), _sparse(blocks=None), _sparse(D=512), _sparse(H=3), _sparse(scale=-1.0), _sparse(kc=None),
]


@pytest.mark.parametrize("name,args", BAD, ids=[f"{n}-{i}" for i, (n, _) in enumerate(BAD)])
def test_bad_calls_are_refused(hk, name, args):
    assert getattr(hk.lib(), name)(*args) == hk.HK_EINVAL
    assert name in hk.last_error()


@pytest.mark.parametrize("name,args", [_decode(n=16), _decode(ws=None), _select(n=16), _select(ws=None), _sparse(n=16), _sparse(ws=None)])
def test_short_workspaces_are_refused(hk, name, args):
    assert getattr(hk.lib(), name)(*args) == hk.HK_ESPACE
    assert "workspace" in hk.last_error()


@pytest.mark.parametrize("name,args", [_rope(T=0, q=None, k=None, qo=None, ko=None, pos=None, table=None), _append(T=0, k=None, v=None, slots=None),
                                       _decode(T=0, q=None, out=None, lse=None, ws=None, n=0), _select(T=0, q=None, blocks=None, ws=None, n=0),
                                       _sparse(T=0, q=None, blocks=None, out=None, lse=None, ws=None, n=0)])
def test_empty_calls_do_nothing(hk, name, args):
    assert getattr(hk.lib(), name)(*args) == hk.HK_OK


@pytest.mark.parametrize("name,args", [_rope(), _append(), _decode(), _select(), _sparse()])
def test_good_calls_need_a_device(hk, name, args):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present: these addresses must not be read")
    assert getattr(hk.lib(), name)(*args) in (hk.HK_ENODEV, hk.HK_ECUDA)


def test_workspaces_hold_what_the_calls_ask_for(hk):
    lib = hk.lib()
    assert lib.hk_gqa_select_workspace_size(5, 8, 64, 1 << 20) >= 5 * 8 * 16384 * 4
    assert lib.hk_gqa_select_workspace_size(0, 8, 64, 0) > 0
    assert lib.hk_gqa_select_workspace_size(4096, 64, 16, (1 << 31) - 1) > 1 << 40  # 64-bit sizes
    assert lib.hk_gqa_fp8_workspace_size(1, 32, 8, 128) > 0


def test_wrappers_refuse_what_does_not_fit(hk):
    import torch

    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    pos, table = torch.zeros(2, dtype=torch.int32), torch.zeros((4, 64))
    for bad in (dict(k=k[:1]), dict(k=k.half()), dict(positions=pos[:1]), dict(q_gain=torch.ones(32, dtype=torch.bfloat16))):
        with pytest.raises((ValueError, TypeError)):
            hk.qk_norm_rope(**{**dict(q=q, k=k, positions=pos, table=table), **bad})
    cache = [torch.zeros((3, 2, 16, 64), dtype=torch.uint8) for _ in range(2)] + [torch.ones((3, 2)) for _ in range(2)]
    with pytest.raises(ValueError):
        hk.gqa_append_fp8(k, k, pos, cache[0], cache[1][:2], *cache[2:])
    with pytest.raises(ValueError):
        hk.gqa_append_fp8(k[:, :1], k, pos, *cache)
    with pytest.raises(ValueError):
        hk.gqa_append_fp8(k, k, pos, *cache, centroids=torch.zeros((3, 2, 64), dtype=torch.int8))
    with pytest.raises(ValueError):
        hk.gqa_sparse_fp8(q, *cache, torch.zeros((1, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32), pos, torch.zeros((2, 3, 4), dtype=torch.int32), 0.1)


# -- the oracle's own pieces ------------------------------------------------------------------------

def test_e4m3_rounding_matches_torch():
    import torch

    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(20000) * 2.0 ** rng.integers(-14, 10, 20000), G8.E4M3[np.isfinite(G8.E4M3)],
                        (np.sort(np.unique(G8.E4M3[:127]))[:-1] + np.sort(np.unique(G8.E4M3[:127]))[1:]) / 2]).astype(np.float32)
    want = torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(G8.to_e4m3(x), want)


@pytest.mark.parametrize("top,want", [(448.0, 1.0), (448.0001, 2.0), (224.0, 0.5), (1.0, 2.0 ** -8), (0.0, 2.0 ** -40), (3.3e38, 2.0 ** 120)])
def test_pow2_scale_is_the_least_that_fits(top, want):
    assert G8.pow2_scale(np.float32(top)) == want
    assert max(top, 2.0 ** -32) <= 448 * want and (top < 2.0 ** -32 or max(top, 2.0 ** -32) > 224 * want)


def test_a_growing_page_keeps_its_values():
    """Requantising by a power of two changes no stored value but those that become subnormal."""
    rng = np.random.default_rng(3)
    c = dict(k=np.zeros((2, 1, 16, 64), np.uint8), v=np.zeros((2, 1, 16, 64), np.uint8), ks=np.ones((2, 1), np.float32), vs=np.ones((2, 1), np.float32), cen=None)
    x = rng.standard_normal((16, 1, 64)).astype(np.float32)
    x[8:] *= 64
    G8.append(x[:8], x[:8], np.arange(16, 24), c)
    first = G8.E4M3[c["k"][1, 0, :8]] * c["ks"][1, 0]
    G8.append(x[8:], x[8:], np.arange(24, 32), c)
    again = G8.E4M3[c["k"][1, 0, :8]] * c["ks"][1, 0]
    assert np.abs(first - again).max() <= 2.0 ** -10 * c["ks"][1, 0]
    big = np.abs(first) >= 2.0 ** -6 * c["ks"][1, 0]
    assert big.any() and np.array_equal(first[big], again[big])
