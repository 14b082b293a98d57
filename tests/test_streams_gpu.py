"""Calls that are given a stream, queued there behind other work while the current stream allocates and writes:
the same bits as alone."""
import numpy as np
import pytest
import torch

from gqa_cases import Batch

pytestmark = pytest.mark.gpu


def put(x, cuda):
    return torch.from_numpy(np.ascontiguousarray(x)).to(cuda)


def queued_behind_other_work(hk, call, scratch):
    """`call(stream)`; `scratch`: bytes of the scratch that it allocates."""
    alone = call(None)
    torch.cuda.synchronize()
    alone = [t.clone() for t in alone]
    sizes = {t.numel() * t.element_size() for t in alone} | {scratch}
    s = torch.cuda.Stream()
    for _ in range(3):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            torch.cuda._sleep(10_000_000)  # some milliseconds
        got = call(s)
        junk = [torch.full((n,), 0x7B, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)]
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(a, b) for a, b in zip(alone, got))
        # Outputs freed while the current stream still reads them; the next call on s takes fresh memory.
        torch.cuda._sleep(10_000_000)
        kept = [t.clone() for t in got]
        del got
        call(s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, kept))
        del junk
    hk.check_errors()


@pytest.mark.parametrize("rows", [[1, 3], [90, 1]])
def test_gqa_calls_on_a_given_stream(hk, cuda, rows):
    b = Batch(rows, [700, 300], 8, 2, 128, 32, seed=40)
    c = {n: put(a, cuda) for n, a in b.cache.items()}
    q, bt, cu, pos = put(b.q, cuda).to(torch.bfloat16), put(b.bt, cuda), put(b.cu, cuda), put(b.pos, cuda)
    four = c["k"], c["v"], c["ks"], c["vs"]
    ws = hk.gqa_fp8_workspace_size(b.T, 8, 2, 128)
    queued_behind_other_work(hk, lambda s: hk.gqa_decode_fp8(q, *four, bt, cu, pos, b.max_rows, b.max_kv, b.scale, stream=s), ws)
    queued_behind_other_work(hk, lambda s: (hk.gqa_select_blocks(q, c["cen"], c["cs"], bt, cu, pos, 32, b.max_kv, 6, stream=s),),
                             hk.lib().hk_gqa_select_workspace_size(b.T, 2, 32, b.max_kv))
    blocks = hk.gqa_select_blocks(q, c["cen"], c["cs"], bt, cu, pos, 32, b.max_kv, 6)
    queued_behind_other_work(hk, lambda s: hk.gqa_sparse_fp8(q, *four, bt, cu, pos, blocks, b.scale, stream=s), ws)


def test_mla_calls_on_a_given_stream(hk, cuda):
    g = torch.Generator().manual_seed(0)
    pages, page, heads, kv = 9, 64, 16, 500
    cache = (torch.randn((pages * page, 576), generator=g) * 0.3).to(torch.bfloat16).to(cuda)
    q = (torch.randn((2, heads, 576), generator=g) * 0.3).to(torch.bfloat16).to(cuda)
    bt = put(np.arange(1, 9, dtype=np.int32)[None], cuda)
    cu, pos = put(np.array([0, 2], np.int32), cuda), put(np.array([kv - 2, kv - 1], np.int32), cuda)
    ws = hk.mla_workspace_size(1, 2, heads, kv)
    queued_behind_other_work(hk, lambda s: hk.mla_decode(q, cache, bt, cu, pos, page, kv, 0.05, stream=s), ws)


def test_a_call_on_a_given_stream_is_captured(hk, cuda):
    b = Batch([1, 3], [700, 300], 8, 2, 128, 32, seed=41)
    c = {n: put(a, cuda) for n, a in b.cache.items()}
    q, bt, cu, pos = put(b.q, cuda).to(torch.bfloat16), put(b.bt, cuda), put(b.cu, cuda), put(b.pos, cuda)
    call = lambda s: hk.gqa_decode_fp8(q, c["k"], c["v"], c["ks"], c["vs"], bt, cu, pos, b.max_rows, b.max_kv, b.scale, stream=s)
    alone = call(None)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        here = torch.cuda.current_stream()
        first = call(here)  # the capture's own stream, and one forked from it
        other.wait_stream(here)
        second = call(other)
        here.wait_stream(other)
        both = [torch.cat([u, w]) for u, w in zip(first, second)]
        del first, second
        third = call(here)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    hk.check_errors()
    for u, w, x in zip(alone, both, third):
        assert torch.equal(torch.cat([u, u]), w) and torch.equal(u, x)
