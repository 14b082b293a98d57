"""Wrappers that are given a stream: what they allocate for the call (outputs, scratch) must belong to that
stream, or the allocator hands it to the current stream's next tensor while the kernels still use it.  Here,
without a GPU, by watching the allocations of each wrapper; nothing is launched."""
import contextlib
import inspect

import pytest
import torch


class FakeStream:
    device = None

    def __init__(self, cuda_stream):
        self.cuda_stream = cuda_stream


HERE = FakeStream(0x11)


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


BF, U8, I8, I32 = torch.bfloat16, torch.uint8, torch.int8, torch.int32
ROW = z(1, 64, 576, dtype=BF)
LANE = (z(1, 2, dtype=I32), z(2, dtype=I32), z(1, dtype=I32))  # block table, cu_seqlens, positions
PAGES = (z(3, 2, 16, 64, dtype=U8), z(3, 2, 16, 64, dtype=U8), z(3, 2), z(3, 2))
Q, K = z(1, 4, 64, dtype=BF), z(1, 2, 64, dtype=BF)

CALLS = {
    "pack": (z(1, dtype=I32), z(1, dtype=I32), LANE[0], 16, 3, 4),
    "kv_dequant_fp8": (z(4, 576, dtype=U8), z(4, 9)),
    "gqa_decode": (z(1, 4, 64), z(4, 2, 64), z(4, 2, 64), *LANE, 2, 16, 0.1),
    "mla_decode": (ROW, z(4, 576, dtype=BF), *LANE, 16, 64, 0.1),
    "mla_decode_fp8": (ROW, z(4, 576, dtype=U8), z(4, 9), *LANE, 16, 64, 0.1),
    "mla_partial_fp8": (ROW, z(4, 576, dtype=U8), z(4, 9), *LANE, z(1, dtype=I32), z(1, dtype=I32), 16, 64, 0.1),
    "mla_partial": (ROW, z(4, 576, dtype=BF), *LANE, z(1, dtype=I32), z(1, dtype=I32), 16, 64, 0.1),
    "qk_norm_rope": (Q, K, LANE[2], z(4, 64)),
    "gqa_decode_fp8": (Q, *PAGES, *LANE, 1, 16, 0.1),
    "gqa_select_blocks": (Q, z(3, 2, 64, dtype=I8), z(3, 2), *LANE, 16, 16, 4),
    "gqa_sparse_fp8": (Q, *PAGES, *LANE, z(1, 2, 4, dtype=I32), 0.1),
    "sample_verify": (z(1, 64), z(2, dtype=I32), z(1, 24, dtype=U8), z(1, dtype=torch.int64), z(1, dtype=I32), 1, 2),
    "lse_merge": (z(2, 3, 8), z(2, 3)),
    "quant_fp8": (z(2, 128, dtype=BF),),
    "gemm_fp8": (z(2, 128, dtype=U8), z(2, 1), z(128, 128, dtype=U8), z(1, 1)),
    "route": (z(2, 8), z(8), 2, 1.0),
    "permute": (z(2, 2, dtype=I32), z(2, 2), 8),
    "moe_grouped": (z(2, 128, dtype=U8), z(2, 1), z(3, dtype=I32), z(2, dtype=I32), 2, 128, 128, *[z(1)] * 4),
    "moe_grouped_noalloc": (z(2, 128, dtype=U8), z(2, 1), z(3, dtype=I32), z(2, dtype=I32), 2, 128, 128, *[z(1)] * 4),
    "gather_rows": (z(4, 16), z(2, dtype=I32)),
    "combine": (z(4, 16, dtype=BF), z(4), z(4, dtype=I32), None, 2, 2),
}
WRITES_INTO_ITS_ARGUMENTS = {"kv_append_bf16", "kv_append_fp8", "kv_dequant_fp8_rows", "kv_append_f32", "gqa_append_fp8", "scatter_rows", "stream_ptr"}


@pytest.fixture
def watched(hk, monkeypatch):
    """(allocations, launches, outputs shared with another stream): allocations with the stream that was current, None for the
    caller's own."""
    current, made, launched, shared = [None], [], [], []

    @contextlib.contextmanager
    def stream(s):
        current.append(s)
        yield
        current.pop()

    empty, empty_like, new_empty = torch.empty, torch.empty_like, torch.Tensor.new_empty
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: HERE)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: shared.append((t.data_ptr(), s)))
    monkeypatch.setattr(torch, "empty", lambda *a, **k: (made.append(current[-1]), empty(*a, **k))[1])
    monkeypatch.setattr(torch, "empty_like", lambda *a, **k: (made.append(current[-1]), empty_like(*a, **k))[1])
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda *a, **k: (made.append(current[-1]), new_empty(*a, **k))[1])
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: HERE.cuda_stream, raising=False)
    monkeypatch.setattr(hk, "ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(hk, "call", lambda name, *a: launched.append((name, a[-1])))
    return made, launched, shared


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("how", ["keyword", "position", "none"])
def test_what_a_call_allocates_belongs_to_its_stream(hk, watched, name, how):
    made, launched, shared = watched
    fn, args = getattr(hk, name), CALLS[name]
    s = FakeStream(0x77)
    if how == "keyword":
        out = fn(*args, stream=s)
    elif how == "position":
        params = list(inspect.signature(fn).parameters.values())
        at = [p.name for p in params].index("stream")
        out = fn(*args, *[p.default for p in params[len(args):at]], s)
    else:
        s = None
        out = fn(*args)
    assert made and all(m is s for m in made), f"{sum(m is not s for m in made)} of {len(made)} allocations are another stream's"
    assert [a for _, a in launched] == [0x77 if s else 0x11]
    outs = list(out.values()) if isinstance(out, dict) else list(out) if isinstance(out, tuple) else [out]
    assert shared == ([(t.data_ptr(), HERE) for t in outs] if s else [])


def test_every_wrapper_with_a_stream_is_looked_at(hk):
    with_stream = {n for n, f in inspect.getmembers(hk, inspect.isfunction) if "stream" in inspect.signature(f).parameters and not n.startswith("_")}
    assert with_stream == set(CALLS) | WRITES_INTO_ITS_ARGUMENTS


def test_the_current_stream_without_torchs_private_name(hk, monkeypatch):
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: HERE)
    assert hk.stream_ptr() == HERE.cuda_stream and hk.stream_ptr(FakeStream(5)) == 5
