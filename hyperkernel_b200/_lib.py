"""ctypes binding of libhk.so (include/hk.h) and thin torch-tensor wrappers.

The library is the product: every call below runs a CUDA kernel of libhk.so on the
caller's stream.  There is no CPU fallback — if libhk.so is missing or the device is not an
sm_100 part, calls raise HKError.  torch is used only for device memory and streams.

With `stream=` a wrapper runs as under `torch.cuda.stream(stream)`: the outputs and scratch it allocates belong
to that stream, so that their memory is not handed to another stream while the call's kernels use it.  As
with every call on another stream, the caller orders the streams and keeps the inputs alive.
"""
from __future__ import annotations

import ctypes as C
import functools
import inspect
import os
import re
from pathlib import Path

import numpy as np
import torch

PKG = Path(__file__).resolve().parent
# HK_LIB_PATH selects another build of the same library (A/B timing of kernel variants).
LIB_PATH = Path(os.environ.get("HK_LIB_PATH", PKG / "libhk.so"))
HEADER = PKG.parent / "include" / "hk.h"

HK_OK, HK_EINVAL, HK_ENODEV, HK_ECUDA, HK_EDEVICE, HK_ESPACE, HK_ESTATE = 0, -1, -2, -3, -4, -5, -6

P, I32, I64, F32, SZ, U64 = C.c_void_p, C.c_int32, C.c_int64, C.c_float, C.c_size_t, C.c_uint64

# Prototypes of every entry point in include/hk.h (kept in header order).
SIGNATURES = {
    "hk_version": (C.c_char_p, []),
    "hk_last_error": (C.c_char_p, []),
    "hk_device_info": (C.c_int, [P, P, P]),
    "hk_kernel_launches": (C.c_uint64, []),
    "hk_check_errors": (C.c_int, []),
    "hk_pack": (C.c_int, [P, P, P, I32, I32, I32, I32, I32, P, P, P, P, P, P, P]),
    "hk_kv_append_bf16": (C.c_int, [P, P, I32, I32, I32, P, I64, P]),
    "hk_kv_append_fp8": (C.c_int, [P, P, I32, I32, P, P, I64, P]),
    "hk_kv_dequant_fp8": (C.c_int, [P, P, I64, I32, I32, P, I64, P, P]),
    "hk_kv_dequant_fp8_rows": (C.c_int, [P, P, I64, I32, I32, P, I64, P, P]),
    "hk_pages_within": (C.c_int, [P, U64, P, P]),
    "hk_plan_pools": (C.c_int, [P, P, P, P, P, P]),
    "hk_kv_append_f32": (C.c_int, [P, P, P, I32, I32, P, P, I64, P]),
    "hk_gqa_decode_f32": (C.c_int, [P, P, P, P, I32, P, P, I32, I32, I32, I32, I32, I32, I64, F32, P, P, P]),
    "hk_mla_workspace_size": (SZ, [I32, I32, I32, I32]),
    "hk_mla_decode": (C.c_int, [P, P, P, I32, P, P, I32, I32, I32, I32, I64, I32, F32, P, P, P, SZ, I32, P]),
    "hk_mla_decode_fp8": (C.c_int, [P, P, P, P, I32, P, P, I32, I32, I32, I32, I64, I32, F32, P, P, P, SZ, P]),
    "hk_mla_partial_fp8": (C.c_int, [P, P, P, P, I32, P, P, P, P, I32, I32, I32, I32, I64, I32, F32, P, P, P, SZ, P]),
    "hk_mla_partial": (C.c_int, [P, P, P, I32, P, P, P, P, I32, I32, I32, I32, I64, I32, F32, P, P, P, SZ, P]),
    "hk_lse_merge": (C.c_int, [P, P, I32, I64, I32, P, P, P]),
    "hk_sample_workspace_size": (SZ, [I32, I32]),
    "hk_sample_verify": (C.c_int, [P, I32, P, I32, I32, I32, P, P, P, I32, P, P, P, SZ, P]),
    "hk_qk_norm_rope": (C.c_int, [P, I64, P, I64, P, P, P, I64, I32, I32, P, I32, I32, I32, I32, F32, I32, P, I64, P, I64, P]),
    "hk_gqa_append_fp8": (C.c_int, [P, I64, P, I64, I32, P, I32, I32, I32, I32, I64, P, P, P, P, P, P, P]),
    "hk_gqa_fp8_workspace_size": (SZ, [I32, I32, I32, I32]),
    "hk_gqa_decode_fp8": (C.c_int, [P, I64, P, P, P, P, P, I32, P, P, I32, I32, I32, I32, I32, I32, I64, I32, I32, F32, I32, P, P, P, SZ, P]),
    "hk_gqa_select_workspace_size": (SZ, [I32, I32, I32, I32]),
    "hk_gqa_select_blocks": (C.c_int, [P, I64, P, P, P, I32, P, P, I32, I32, I32, I32, I32, I32, I64, I32, I32, I32, I32, I32, P, P, SZ, P]),
    "hk_gqa_sparse_fp8": (C.c_int, [P, I64, P, P, P, P, P, I32, P, P, P, I32, I32, I32, I32, I32, I32, I32, I64, F32, I32, P, P, P, SZ, P]),
    "hk_quant_fp8": (C.c_int, [P, I64, I32, P, P, P]),
    "hk_gemm_fp8": (C.c_int, [P, P, P, P, I64, I32, I32, P, P]),
    "hk_route": (C.c_int, [P, P, I32, I32, I32, F32, P, P, P]),
    "hk_permute": (C.c_int, [P, P, I32, I32, I32, P, P, P, P, P]),
    "hk_moe_workspace_size": (SZ, [I64, I32, I32]),
    "hk_moe_grouped": (C.c_int, [P, P, I32, P, P, I64, I32, I32, I32, P, P, P, P, P, P, SZ, P]),
    "hk_moe_grouped_noalloc": (C.c_int, [P, P, I32, P, P, I64, I32, I32, I32, P, P, P, P, P, P]),
    "hk_gather_rows": (C.c_int, [P, I64, P, I64, I32, P, P]),
    "hk_scatter_rows": (C.c_int, [P, I64, P, I64, I32, P, P]),
    "hk_ep_counts": (C.c_int, [P, I32, I32, I32, P, P, C.c_uint32, I32, P, P, P, P]),
    "hk_ep_dispatch": (C.c_int, [P, P, I32, P, P, I32, I32, I32, I32, I32, I32, P, P, P, P, P, C.c_uint32, P]),
    "hk_ep_return": (C.c_int, [P, I32, I32, I32, I32, P, P, P, I32, I32, P, P, P, C.c_uint32, P]),
    "hk_ep_wait": (C.c_int, [P, I32, I32, C.c_uint32, I32, P]),
    "hk_sym_alloc": (C.c_int, [SZ, P, P]),
    "hk_sym_import": (C.c_int, [P, P]),
    "hk_sym_close": (C.c_int, [P]),
    "hk_sym_free": (C.c_int, [P]),
    "hk_cp_merge": (C.c_int, [P, P, P, I32, I32, C.c_uint32, I32, I64, I32, P, P, P]),
    "hk_combine": (C.c_int, [P, I64, P, P, P, I32, I32, I32, P, P]),
    "hk_open": (C.c_int, [P, P]),
    "hk_open_mla": (C.c_int, [P, P, P]),
    "hk_model_tensor": (C.c_int, [P, C.c_uint32, C.c_char_p, P, P]),
    "hk_close": (None, [P]),
    "hk_pools": (C.c_int, [P, P, P]),
    "hk_push": (C.c_int, [P, P]),
    "hk_drain": (C.c_int, [P, P, SZ, P, P, SZ, P]),
    "hk_drain_logprobs": (C.c_int, [P, P, SZ, P, P, SZ, P]),
    "hk_encode_share": (C.c_int, [P, P, P, SZ, P]),
    "hk_kernel_ops_of": (C.c_int, [P, P]),
    "hk_engine_defaults": (None, [P]),
    "hk_engine_create": (C.c_int, [P, P, P]),
    "hk_engine_destroy": (None, [P]),
    "hk_engine_submit": (C.c_int, [P, P, SZ, P, U64, P, SZ, P]),
    "hk_engine_reset": (C.c_int, [P, P]),
    "hk_engine_reset_answer": (C.c_int, [P, U64, I64, P]),
    "hk_engine_close": (C.c_int, [P]),
    "hk_engine_run": (C.c_int, [P]),
    "hk_engine_hangup": (C.c_int, [P, U64]),
    "hk_engine_outputs": (C.c_int, [P, U64, I64, P, SZ, P, P, SZ]),
    "hk_engine_outputs_lp": (C.c_int, [P, U64, I64, P, SZ, P, P, SZ, P, SZ, P]),
    "hk_engine_metrics": (C.c_int, [P, P, P, SZ, P, P, SZ, P]),
    "hk_rope_table": (C.c_int, [I64, I32, F32, I32, F32, F32, F32, P]),
}


class HKError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"hk error {code}: {msg}")
        self.code = code


_lib = None


def lib() -> C.CDLL:
    """Loads libhk.so (raises if it was not built: there is no fallback)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise HKError(HK_ENODEV, f"{LIB_PATH} is not built; run python -m hyperkernel_b200.build")
        L = C.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
    return _lib


def header_functions() -> list[str]:
    """Names of the functions declared in include/hk.h."""
    text = HEADER.read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return re.findall(r"^\s*(?:const\s+)?[a-z_0-9]+\s*\*?\s*(hk_[a-z_0-9]+)\s*\(", text, flags=re.M)


def last_error() -> str:
    return lib().hk_last_error().decode()


def check(rc: int) -> None:
    if rc != HK_OK:
        raise HKError(rc, last_error())


def ptr(t):
    """Device address of a tensor (None -> NULL)."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    assert t.is_cuda and t.is_contiguous(), "tensors passed to libhk must be contiguous CUDA tensors"
    return t.data_ptr()


def stream_ptr(stream=None):
    if stream is not None:
        return stream.cuda_stream
    try:
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())  # the current stream, without its Python object
    except AttributeError:  # not a public name of torch
        return torch.cuda.current_stream().cuda_stream


def _on_stream(fn):
    """Runs a wrapper under the stream that it is given.  Its new outputs are the caller's current stream's to
    read too: when they are freed, their memory waits for that stream as well."""
    at = list(inspect.signature(fn).parameters).index("stream")

    @functools.wraps(fn)
    def on(*args, **kw):
        stream = args[at] if len(args) > at else kw.get("stream")
        if stream is None:
            return fn(*args, **kw)
        here = torch.cuda.current_stream(stream.device)
        with torch.cuda.stream(stream):
            out = fn(*args, **kw)
        for t in out.values() if isinstance(out, dict) else out if isinstance(out, tuple) else (out,):
            if t is not None:
                t.record_stream(here)
        return out
    return on


def call(name: str, *args) -> None:
    check(getattr(lib(), name)(*args))


def check_errors() -> None:
    """Raises if any kernel recorded bad input on the current device (synchronises)."""
    check(lib().hk_check_errors())


def device_info():
    sm, ma, mi = C.c_int(), C.c_int(), C.c_int()
    check(lib().hk_device_info(C.byref(sm), C.byref(ma), C.byref(mi)))
    return sm.value, ma.value, mi.value


def kernel_launches() -> int:
    """Kernels libhk.so has launched in this process."""
    return lib().hk_kernel_launches()


def version() -> str:
    return lib().hk_version().decode()


def _u16(t):
    """bf16 tensor viewed as its bit pattern (no copy)."""
    return t.view(torch.int16) if t.dtype == torch.bfloat16 else t


# ------------------------------------------------------------------------------------------
# Kernel wrappers (all tensors on the current CUDA device, contiguous)
# ------------------------------------------------------------------------------------------

@_on_stream
def pack(lane_tokens, lane_pos, block_table, page_size, num_pages, max_tokens, stream=None):
    dev = lane_tokens.device
    L = lane_tokens.shape[0]
    o = dict(
        cu_seqlens=torch.empty(L + 1, dtype=torch.int32, device=dev),
        seq_lens=torch.empty(L, dtype=torch.int32, device=dev),
        positions=torch.empty(max(max_tokens, 1), dtype=torch.int32, device=dev),
        slot_mapping=torch.empty(max(max_tokens, 1), dtype=torch.int32, device=dev),
        token_lane=torch.empty(max(max_tokens, 1), dtype=torch.int32, device=dev),
        active=torch.empty(L + 1, dtype=torch.int32, device=dev))
    call("hk_pack", ptr(lane_tokens), ptr(lane_pos), ptr(block_table), block_table.shape[1], L,
         page_size, num_pages, max_tokens, ptr(o["cu_seqlens"]), ptr(o["seq_lens"]),
         ptr(o["positions"]), ptr(o["slot_mapping"]), ptr(o["token_lane"]), ptr(o["active"]),
         stream_ptr(stream))
    return o


def kv_append_bf16(kv_new, slot_mapping, kv_cache, num_tokens=None, page_rows=64, stream=None):
    """Appends rows into the page-blocked latent cache (page_rows=0: a row-major cache)."""
    n = kv_new.shape[0] if num_tokens is None else num_tokens
    call("hk_kv_append_bf16", ptr(kv_new), ptr(slot_mapping), n, kv_new.shape[-1], page_rows,
         ptr(kv_cache), kv_cache.shape[0], stream_ptr(stream))


def kv_append_fp8(kv_new, slot_mapping, kv_cache, kv_scale, num_tokens=None, stream=None):
    n = kv_new.shape[0] if num_tokens is None else num_tokens
    call("hk_kv_append_fp8", ptr(kv_new), ptr(slot_mapping), n, kv_new.shape[-1], ptr(kv_cache),
         ptr(kv_scale), kv_cache.shape[0], stream_ptr(stream))


def kv_dequant_fp8_rows(kv_cache, kv_scale, slots, out, page_rows=64, stream=None):
    """Refreshes the rows `slots` (int32 device tensor) of the bf16 mirror `out`."""
    slots_n, row = kv_cache.shape
    call("hk_kv_dequant_fp8_rows", ptr(kv_cache), ptr(kv_scale), slots_n, row, page_rows, ptr(slots),
         slots.shape[0], ptr(_u16(out)), stream_ptr(stream))
    return out


@_on_stream
def kv_dequant_fp8(kv_cache, kv_scale, page_rows=64, out=None, pages=None, stream=None):
    """The FP8 cache [slots][576] as the page-blocked bf16 cache of hk_mla_decode (only the
    pages listed in `pages`, an int32 device tensor, when given)."""
    slots, row = kv_cache.shape
    if out is None:
        out = torch.empty((slots, row), dtype=torch.bfloat16, device=kv_cache.device)
    n = 0 if pages is None else pages.shape[0]
    call("hk_kv_dequant_fp8", ptr(kv_cache), ptr(kv_scale), slots, row, page_rows, ptr(pages), n,
         ptr(_u16(out)), stream_ptr(stream))
    return out


def kv_append_f32(k_new, v_new, slot_mapping, k_cache, v_cache, stream=None):
    row = k_new[0].numel() if k_new.shape[0] else 4
    call("hk_kv_append_f32", ptr(k_new), ptr(v_new), ptr(slot_mapping), k_new.shape[0], row,
         ptr(k_cache), ptr(v_cache), k_cache.shape[0], stream_ptr(stream))


@_on_stream
def gqa_decode(q, k_cache, v_cache, block_table, cu_seqlens, positions, kv_heads, page_size,
               scale, stream=None):
    T, qh, D = q.shape
    out = torch.empty_like(q)
    lse = torch.empty((T, qh), dtype=torch.float32, device=q.device)
    call("hk_gqa_decode_f32", ptr(q), ptr(k_cache), ptr(v_cache), ptr(block_table),
         block_table.shape[1], ptr(cu_seqlens), ptr(positions), cu_seqlens.shape[0] - 1, T, qh,
         kv_heads, D, page_size, k_cache.shape[0], scale, ptr(out), ptr(lse), stream_ptr(stream))
    return out, lse


def mla_workspace_size(num_lanes, num_tokens, heads, max_kv_len) -> int:
    return lib().hk_mla_workspace_size(num_lanes, num_tokens, heads, max_kv_len)


@_on_stream
def mla_decode(q, kv_cache, block_table, cu_seqlens, positions, page_size, max_kv_len, scale,
               out=None, lse=None, workspace=None, impl=0, stream=None):
    T, H, _ = q.shape
    dev = q.device
    if out is None:
        out = torch.empty((T, H, 512), dtype=torch.bfloat16, device=dev)
    if lse is None:
        lse = torch.empty((T, H), dtype=torch.float32, device=dev)
    L = cu_seqlens.shape[0] - 1
    if workspace is None:
        ws = mla_workspace_size(L, T, H, max_kv_len)
        workspace = torch.empty(max(ws, 16), dtype=torch.uint8, device=dev)
    call("hk_mla_decode", ptr(q), ptr(kv_cache), ptr(block_table), block_table.shape[1],
         ptr(cu_seqlens), ptr(positions), L, T, H, page_size, kv_cache.shape[0], max_kv_len, scale,
         ptr(out), ptr(lse), ptr(workspace), workspace.numel(), impl, stream_ptr(stream))
    return out, lse


@_on_stream
def mla_decode_fp8(q, kv_cache, kv_scale, block_table, cu_seqlens, positions, page_size,
                   max_kv_len, scale, stream=None):
    T, H, _ = q.shape
    dev = q.device
    out = torch.empty((T, H, 512), dtype=torch.bfloat16, device=dev)
    lse = torch.empty((T, H), dtype=torch.float32, device=dev)
    L = cu_seqlens.shape[0] - 1
    ws = mla_workspace_size(L, T, H, max_kv_len)
    workspace = torch.empty(max(ws, 16), dtype=torch.uint8, device=dev)
    call("hk_mla_decode_fp8", ptr(q), ptr(kv_cache), ptr(kv_scale), ptr(block_table),
         block_table.shape[1], ptr(cu_seqlens), ptr(positions), L, T, H, page_size,
         kv_cache.shape[0], max_kv_len, scale, ptr(out), ptr(lse), ptr(workspace),
         workspace.numel(), stream_ptr(stream))
    return out, lse


@_on_stream
def mla_partial_fp8(q, kv_cache, kv_scale, block_table, cu_seqlens, positions, kv_begin, kv_end,
                    page_size, max_kv_len, scale, stream=None):
    T, H, _ = q.shape
    dev = q.device
    o = torch.empty((T, H, 512), dtype=torch.float32, device=dev)
    lse = torch.empty((T, H), dtype=torch.float32, device=dev)
    L = cu_seqlens.shape[0] - 1
    ws = mla_workspace_size(L, T, H, max_kv_len)
    workspace = torch.empty(max(ws, 16), dtype=torch.uint8, device=dev)
    call("hk_mla_partial_fp8", ptr(q), ptr(kv_cache), ptr(kv_scale), ptr(block_table),
         block_table.shape[1], ptr(cu_seqlens), ptr(positions), ptr(kv_begin), ptr(kv_end), L, T,
         H, page_size, kv_cache.shape[0], max_kv_len, scale, ptr(o), ptr(lse), ptr(workspace),
         workspace.numel(), stream_ptr(stream))
    return o, lse


@_on_stream
def mla_partial(q, kv_cache, block_table, cu_seqlens, positions, kv_begin, kv_end, page_size, max_kv_len,
                scale, stream=None, out=None, lse=None):
    """Partial attention of KV ranges on the tcgen05 kernel over the page-blocked bf16 cache:
    fp32 o [T, H, 512] normalised within the range, lse [T, H] (-inf where it is empty), into
    `out` / `lse` when given (e.g. a context-parallel exchange buffer)."""
    T, H, _ = q.shape
    dev = q.device
    o = out if out is not None else torch.empty((T, H, 512), dtype=torch.float32, device=dev)
    lse = lse if lse is not None else torch.empty((T, H), dtype=torch.float32, device=dev)
    L = cu_seqlens.shape[0] - 1
    ws = mla_workspace_size(L, T, H, max_kv_len)
    workspace = torch.empty(max(ws, 16), dtype=torch.uint8, device=dev)
    call("hk_mla_partial", ptr(q), ptr(_u16(kv_cache)), ptr(block_table), block_table.shape[1],
         ptr(cu_seqlens), ptr(positions), ptr(kv_begin), ptr(kv_end), L, T, H, page_size,
         kv_cache.shape[0], max_kv_len, scale, ptr(o), ptr(lse), ptr(workspace), workspace.numel(),
         stream_ptr(stream))
    return o, lse


# ---- GQA over the block-scaled 8-bit cache -----------------------------------------------

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}  # HK_BF16, HK_F16
_I32, _F32, _U8, _I8 = torch.int32, torch.float32, torch.uint8, torch.int8


def _rows(t):
    """(address, row stride in elements) of a [rows, heads, dim] tensor whose rows may be slices of
    wider ones."""
    T, h, d = t.shape
    s0, s1, s2 = t.stride()
    if h > 0 and (s2 != 1 or (s1 != d and h > 1)):
        raise ValueError("the heads of a row must lie side by side")
    return t.data_ptr(), s0 if T > 1 and h > 0 else h * d


def _code(t):
    """The HK_BF16 / HK_F16 code of a tensor."""
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"expected bfloat16 or float16, got {t.dtype}") from None


def _here(*tensors):
    """The current device, after checking that every tensor is on it."""
    dev = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensor on {t.device}, but the current device is cuda:{dev}")
    return dev


def _typed(t, dtype, name):
    if t is None:
        return None
    if t.dtype != dtype or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous {dtype} tensor")
    return t.data_ptr()


def _output(out, like, shape):
    """(tensor, address, row stride) of an output of `like`'s type: a new one unless given."""
    if out is None:
        out = like.new_empty(shape)
        return out, out.data_ptr(), shape[1] * shape[2]
    if out.shape != shape or out.dtype != like.dtype:
        raise ValueError(f"expected a {like.dtype} output of shape {tuple(shape)}")
    return (out, *_rows(out))


@_on_stream
def qk_norm_rope(q, k, positions, table, q_gain=None, k_gain=None, interleaved=False, eps=1e-6,
                 q_out=None, k_out=None, stream=None):
    """RMS norm of each query and key head, then the rotation by table[positions] (fp32, the layout
    of `rope_table`; its width is the number of rotated dims).  q [T, heads, dim] and k may be
    slices of a fused projection; outputs are new contiguous tensors unless given (q_out=q works
    in place).  Returns (q_out, k_out)."""
    T, H, D = q.shape
    G = k.shape[1]
    if k.shape != (T, G, D) or k.dtype != q.dtype or positions.shape[0] < T or table.dim() != 2:
        raise ValueError("q, k, positions and table do not fit together")
    if (q_gain is not None and q_gain.shape != (D,)) or (k_gain is not None and k_gain.shape != (D,)):
        raise ValueError(f"a gain has {D} elements")
    _here(q, k, positions, table, q_gain, k_gain, q_out, k_out)
    dt = q.dtype
    q_out, yp, ys = _output(q_out, q, (T, H, D))
    k_out, zp, zs = _output(k_out, k, (T, G, D))
    qp, qs = _rows(q)
    kp, ks = _rows(k)
    call("hk_qk_norm_rope", qp, qs, kp, ks, _typed(q_gain, dt, "q_gain"), _typed(k_gain, dt, "k_gain"),
         _typed(table, _F32, "table"), table.shape[0], table.shape[1], int(interleaved),
         _typed(positions, _I32, "positions"), T, H, G, D, eps, _code(q), yp, ys, zp, zs, stream_ptr(stream))
    return q_out, k_out


def _gqa_cache(k_cache, v_cache, k_scale, v_scale):
    """(pages, KV heads, page rows, dim) and the addresses of a cache, after checking its four arrays."""
    shape = N, G, R, D = k_cache.shape
    if v_cache.shape != shape or k_scale.shape != (N, G) or v_scale.shape != (N, G):
        raise ValueError("k_cache, v_cache [pages, kv_heads, page, dim] and their scales [pages, kv_heads] do not fit together")
    return N, G, R, D, (_typed(k_cache, _U8, "k_cache"), _typed(v_cache, _U8, "v_cache"),
                        _typed(k_scale, _F32, "k_scale"), _typed(v_scale, _F32, "v_scale"))


def gqa_append_fp8(k_new, v_new, slot_mapping, k_cache, v_cache, k_scale, v_scale, centroids=None,
                   centroid_scale=None, stream=None):
    """Appends rows to the block-scaled e4m3 cache (uint8 [pages, kv_heads, page, dim], fp32 scales
    [pages, kv_heads]) and, when given, the int8 centroids of the pages that become full."""
    N, G, R, D, cache = _gqa_cache(k_cache, v_cache, k_scale, v_scale)
    T = k_new.shape[0]
    if k_new.shape != (T, G, D) or v_new.shape != (T, G, D) or v_new.dtype != k_new.dtype or slot_mapping.shape[0] < T:
        raise ValueError("k_new, v_new [rows, kv_heads, dim] and slot_mapping do not fit the cache")
    if (centroids is None) != (centroid_scale is None) or (
            centroids is not None and (centroids.shape != (N, G, D) or centroid_scale.shape != (N, G))):
        raise ValueError("centroids [pages, kv_heads, dim] need centroid_scale [pages, kv_heads]")
    _here(k_new, v_new, slot_mapping, k_cache, v_cache, k_scale, v_scale, centroids, centroid_scale)
    kp, ks = _rows(k_new)
    vp, vs = _rows(v_new)
    call("hk_gqa_append_fp8", kp, ks, vp, vs, _code(k_new), _typed(slot_mapping, _I32, "slot_mapping"), T, G, D, R, N,
         *cache, _typed(centroids, _I8, "centroids"), _typed(centroid_scale, _F32, "centroid_scale"), stream_ptr(stream))


def gqa_fp8_workspace_size(num_tokens, q_heads, kv_heads, head_dim) -> int:
    return lib().hk_gqa_fp8_workspace_size(num_tokens, q_heads, kv_heads, head_dim)


@functools.lru_cache(maxsize=256)
def _gqa_scratch(device, *sizes):
    return gqa_fp8_workspace_size(*sizes)  # of the sizes and the device's SMs alone


def _gqa_io(q, G, D, out, lse, workspace, dev):
    T, H, d = q.shape
    if d != D:
        raise ValueError(f"q has heads of {d} dims, the cache of {D}")
    if out is None:
        out = q.new_empty((T, H, D))
    elif out.shape != (T, H, D):
        raise ValueError("out does not fit q")
    if lse is None:
        lse = q.new_empty((T, H), dtype=_F32)
    elif lse.shape != (T, H):
        raise ValueError("lse does not fit q")
    if workspace is None:
        workspace = q.new_empty(_gqa_scratch(dev, T, H, G, D), dtype=_U8)
    return out, lse, workspace, (_typed(out, q.dtype, "out"), _typed(lse, _F32, "lse"), _typed(workspace, _U8, "workspace"), workspace.shape[0])


def _lanes(block_table, cu_seqlens, positions, T):
    if block_table.dim() != 2 or cu_seqlens.shape[0] != block_table.shape[0] + 1 or positions.shape[0] < T:
        raise ValueError("block_table [lanes, pages], cu_seqlens [lanes + 1] and positions do not fit together")
    return (_typed(block_table, _I32, "block_table"), block_table.shape[1], _typed(cu_seqlens, _I32, "cu_seqlens"),
            _typed(positions, _I32, "positions"))


@_on_stream
def gqa_decode_fp8(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens, positions, max_rows,
                   max_kv_len, scale, out=None, lse=None, workspace=None, stream=None):
    """Ragged paged attention over the block-scaled cache of `gqa_append_fp8`: every lane's rows
    (at most max_rows) attend the lane's KV rows up to their positions.  Returns (out, lse)."""
    N, G, R, D, cache = _gqa_cache(k_cache, v_cache, k_scale, v_scale)
    T, H, _ = q.shape
    lanes = _lanes(block_table, cu_seqlens, positions, T)
    dev = _here(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens, positions, out, lse, workspace)
    dt = _code(q)
    out, lse, workspace, io = _gqa_io(q, G, D, out, lse, workspace, dev)
    call("hk_gqa_decode_fp8", *_rows(q), *cache, *lanes, block_table.shape[0], T, H, G, D, R, N, max_rows, max_kv_len,
         scale, dt, *io, stream_ptr(stream))
    return out, lse


@_on_stream
def gqa_select_blocks(q, centroids, centroid_scale, block_table, cu_seqlens, positions, page_size, max_kv_len,
                      top_blocks, sink=1, local=1, blocks=None, workspace=None, stream=None):
    """The blocks each row and KV head reads, by its int8 score against the pages' centroids:
    int32 [T, kv_heads, top_blocks], rising, -1 behind the last."""
    N, G, D = centroids.shape
    T, H, d = q.shape
    if d != D or centroid_scale.shape != (N, G):
        raise ValueError("q, centroids and centroid_scale do not fit together")
    lanes = _lanes(block_table, cu_seqlens, positions, T)
    _here(q, centroids, centroid_scale, block_table, cu_seqlens, positions, blocks, workspace)
    if blocks is None:
        blocks = q.new_empty((T, G, top_blocks), dtype=_I32)
    elif blocks.shape != (T, G, top_blocks):
        raise ValueError("blocks must be [T, kv_heads, top_blocks]")
    if workspace is None:
        workspace = q.new_empty(lib().hk_gqa_select_workspace_size(T, G, page_size, max_kv_len), dtype=_U8)
    call("hk_gqa_select_blocks", *_rows(q), _typed(centroids, _I8, "centroids"),
         _typed(centroid_scale, _F32, "centroid_scale"), *lanes, block_table.shape[0], T, H, G, D, page_size, N,
         max_kv_len, top_blocks, sink, local, _code(q), _typed(blocks, _I32, "blocks"),
         _typed(workspace, _U8, "workspace"), workspace.shape[0], stream_ptr(stream))
    return blocks


@_on_stream
def gqa_sparse_fp8(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens, positions, blocks, scale,
                   out=None, lse=None, workspace=None, stream=None):
    """`gqa_decode_fp8` over the listed blocks of each row and KV head.  Returns (out, lse)."""
    N, G, R, D, cache = _gqa_cache(k_cache, v_cache, k_scale, v_scale)
    T, H, _ = q.shape
    if blocks.dim() != 3 or blocks.shape[:2] != (T, G):
        raise ValueError("blocks must be [T, kv_heads, top_blocks]")
    lanes = _lanes(block_table, cu_seqlens, positions, T)
    dev = _here(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens, positions, blocks, out, lse, workspace)
    dt = _code(q)
    out, lse, workspace, io = _gqa_io(q, G, D, out, lse, workspace, dev)
    call("hk_gqa_sparse_fp8", *_rows(q), *cache, *lanes, _typed(blocks, _I32, "blocks"), blocks.shape[2],
         block_table.shape[0], T, H, G, D, R, N, scale, dt, *io, stream_ptr(stream))
    return out, lse


SAMPLING_DTYPE = np.dtype([("temperature", "<f4"), ("top_p", "<f4"), ("top_k", "<u4"),
                           ("logprobs", "<u4"), ("seed", "<u8")])


def sampling_array(samplings, device):
    """hk_sampling[] on the device from dicts with temperature, top_p, top_k (logprobs, seed)."""
    a = np.zeros(len(samplings), SAMPLING_DTYPE)
    for i, sm in enumerate(samplings):
        a[i] = (sm["temperature"], sm["top_p"], sm["top_k"], sm.get("logprobs", 0), sm.get("seed", 0))
    return torch.from_numpy(a.view(np.uint8).copy()).to(device)


@_on_stream
def sample_verify(logits, cu_rows, sampling, state, drafts, block, n_logprobs, stream=None):
    """Draws and verifies every lane's rows: returns (ids [lanes, block], lp [lanes, block,
    2n+1]); `state` (uint64 stored as int64, one per lane) advances in place."""
    rows, vocab = logits.shape
    lanes = cu_rows.shape[0] - 1
    dev = logits.device
    ids = torch.empty((lanes, block), dtype=torch.int32, device=dev)
    lp = torch.empty((lanes, block, 2 * n_logprobs + 1), dtype=torch.float32, device=dev)
    ws = lib().hk_sample_workspace_size(rows, vocab)
    workspace = torch.empty(ws, dtype=torch.uint8, device=dev)
    call("hk_sample_verify", ptr(logits), vocab, ptr(cu_rows), lanes, rows, block, ptr(sampling), ptr(state),
         ptr(drafts), n_logprobs, ptr(ids), ptr(lp) if n_logprobs > 0 else None, ptr(workspace),
         workspace.numel(), stream_ptr(stream))
    return ids, lp


@_on_stream
def lse_merge(o_parts, lse_parts, stream=None):
    n, rows, dv = o_parts.shape
    out = torch.empty((rows, dv), dtype=torch.bfloat16, device=o_parts.device)
    lse = torch.empty(rows, dtype=torch.float32, device=o_parts.device)
    call("hk_lse_merge", ptr(o_parts), ptr(lse_parts), n, rows, dv, ptr(out), ptr(lse),
         stream_ptr(stream))
    return out, lse


@_on_stream
def quant_fp8(x, stream=None):
    rows, k = x.shape
    xq = torch.empty((rows, k), dtype=torch.uint8, device=x.device)
    sx = torch.empty((rows, k // 128), dtype=torch.float32, device=x.device)
    call("hk_quant_fp8", ptr(x), rows, k, ptr(xq), ptr(sx), stream_ptr(stream))
    return xq, sx


@_on_stream
def gemm_fp8(xq, sx, wq, sw, out=None, stream=None):
    m, k = xq.shape
    n = wq.shape[0]
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=xq.device)
    call("hk_gemm_fp8", ptr(xq), ptr(sx), ptr(wq), ptr(sw), m, n, k, ptr(out), stream_ptr(stream))
    return out


@_on_stream
def route(logits, bias, top_k, route_scale, stream=None):
    T, E = logits.shape
    ids = torch.empty((T, top_k), dtype=torch.int32, device=logits.device)
    w = torch.empty((T, top_k), dtype=torch.float32, device=logits.device)
    call("hk_route", ptr(logits), ptr(bias), T, E, top_k, route_scale, ptr(ids), ptr(w),
         stream_ptr(stream))
    return ids, w


@_on_stream
def permute(ids, weights, num_experts, stream=None, offsets=None, perm_token=None):
    """`offsets` / `perm_token` may be given as contiguous views of larger buffers (the first
    num_experts + 1 and T * K entries are written)."""
    T, K = ids.shape
    dev = ids.device
    if offsets is None:
        offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    if perm_token is None:
        perm_token = torch.empty(max(T * K, 1), dtype=torch.int32, device=dev)
    if offsets.numel() < num_experts + 1 or perm_token.numel() < T * K:
        raise ValueError("permute: output buffers too small")
    perm_weight = torch.empty(max(T * K, 1), dtype=torch.float32, device=dev)
    inv = torch.empty(max(T * K, 1), dtype=torch.int32, device=dev)
    call("hk_permute", ptr(ids), ptr(weights), T, K, num_experts, ptr(offsets), ptr(perm_token),
         ptr(perm_weight), ptr(inv), stream_ptr(stream))
    return offsets, perm_token, perm_weight, inv


def moe_workspace_size(rows, hidden, inter) -> int:
    return lib().hk_moe_workspace_size(rows, hidden, inter)


@_on_stream
def moe_grouped(xq, sx, offsets, perm_token, rows, hidden, inter, w13, s13, w2, s2, out=None,
                workspace=None, stream=None):
    E = offsets.shape[0] - 1
    dev = xq.device
    if out is None:
        out = torch.empty((max(rows, 1), hidden), dtype=torch.bfloat16, device=dev)
    if workspace is None:
        workspace = torch.empty(moe_workspace_size(max(rows, 1), hidden, inter), dtype=torch.uint8, device=dev)
    call("hk_moe_grouped", ptr(xq), ptr(sx), xq.shape[0], ptr(offsets), ptr(perm_token), rows, E,
         hidden, inter, ptr(w13), ptr(s13), ptr(w2), ptr(s2), ptr(out), ptr(workspace),
         workspace.numel(), stream_ptr(stream))
    return out


@_on_stream
def moe_grouped_noalloc(xq, sx, offsets, perm_token, rows, hidden, inter, w13, s13, w2, s2,
                        out=None, stream=None):
    """hk_moe_grouped with the library's fixed scratch array (no workspace argument)."""
    E = offsets.shape[0] - 1
    if out is None:
        out = torch.empty((max(rows, 1), hidden), dtype=torch.bfloat16, device=xq.device)
    call("hk_moe_grouped_noalloc", ptr(xq), ptr(sx), xq.shape[0], ptr(offsets), ptr(perm_token),
         rows, E, hidden, inter, ptr(w13), ptr(s13), ptr(w2), ptr(s2), ptr(out),
         stream_ptr(stream))
    return out


@_on_stream
def gather_rows(src, idx, out=None, stream=None):
    """out[i] = src[idx[i]] (rows of src as bytes; 16-byte multiples)."""
    rows = idx.shape[0]
    if out is None:
        out = torch.empty((rows,) + tuple(src.shape[1:]), dtype=src.dtype, device=src.device)
    row_bytes = src[0].numel() * src.element_size() if src.shape[0] else out[0].numel() * out.element_size()
    call("hk_gather_rows", ptr(src), src.shape[0], ptr(idx), rows, row_bytes, ptr(out), stream_ptr(stream))
    return out


def scatter_rows(src, idx, out, stream=None):
    """out[idx[i]] = src[i]."""
    rows = idx.shape[0]
    row_bytes = out[0].numel() * out.element_size()
    call("hk_scatter_rows", ptr(src), rows, ptr(idx), out.shape[0], row_bytes, ptr(out), stream_ptr(stream))
    return out


@_on_stream
def combine(y, perm_weight, inv, shared, tokens, top_k, out=None, stream=None):
    hidden = y.shape[1]
    if out is None:
        out = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=y.device)
    call("hk_combine", ptr(y), y.shape[0], ptr(perm_weight), ptr(inv), ptr(shared), tokens, top_k,
         hidden, ptr(out), stream_ptr(stream))
    return out


def rope_table(rows, dim, base, original_seq_len, factor, beta_fast, beta_slow):
    """Host-side table (numpy float32 [rows][dim]); needs no GPU."""
    import numpy as np

    t = np.zeros((rows, dim), np.float32)
    check(lib().hk_rope_table(rows, dim, base, original_seq_len, factor, beta_fast, beta_slow,
                              t.ctypes.data_as(C.c_void_p)))
    return t


# ---- pool sizing (host arithmetic; hk_plan_pools reads cudaMemGetInfo when free == 0) ----

UNIT_PAGE, UNIT_WINDOW = 0, 1


class PoolStateC(C.Structure):
    _fields_ = [("home", C.c_uint32), ("unit", C.c_uint32), ("bytes", C.c_uint64)]


class PoolSizingC(C.Structure):
    _fields_ = [("pages", C.c_uint64), ("window_pages", C.c_uint64), ("entries", C.c_uint64),
                ("slots", C.c_uint64), ("states", C.POINTER(PoolStateC)), ("n_states", C.c_size_t)]


class PoolBudgetC(C.Structure):
    _fields_ = [("free", C.c_uint64), ("other", C.c_uint64), ("slack", C.c_uint64),
                ("lanes", C.c_uint32), ("context", C.c_uint32), ("device", C.c_int32),
                ("reserved", C.c_uint32)]


def _pool_c(pages, window_pages, entries, slots, states):
    arr = (PoolStateC * max(len(states), 1))(*[PoolStateC(h, u, b) for h, u, b in states])
    return PoolSizingC(pages, window_pages, entries, slots, arr, len(states)), arr


def pages_within(pages, window_pages, entries, states, nbytes, slots=0):
    """(pages, window_pages) for a pool of `states` [(home, unit, bytes per unit)] within
    `nbytes`, or None when the bytes hold no sequence (src/gpu/load.rs:903-908)."""
    pool, _keep = _pool_c(pages, window_pages, entries, slots, states)
    n, w = C.c_size_t(), C.c_size_t()
    rc = lib().hk_pages_within(C.byref(pool), nbytes, C.byref(n), C.byref(w))
    if rc == HK_ESPACE:
        return None
    check(rc)
    return n.value, w.value


def plan_pools(pages, window_pages, entries, slots, states, *, lanes, context, other=0, slack=0,
               free=0, device=0):
    """(pages, window_pages, slots, used bytes) of the loader's pool plan; free = 0 reads the
    device's free memory.  Raises HKError with the reference's wording."""
    pool, _keep = _pool_c(pages, window_pages, entries, slots, states)
    b = PoolBudgetC(free, other, slack, lanes, context, device, 0)
    n, w, sl, used = C.c_size_t(), C.c_size_t(), C.c_size_t(), C.c_uint64()
    check(lib().hk_plan_pools(C.byref(pool), C.byref(b), C.byref(n), C.byref(w), C.byref(sl),
                              C.byref(used)))
    return n.value, w.value, sl.value, used.value
