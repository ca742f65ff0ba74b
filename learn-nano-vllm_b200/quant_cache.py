"""4-bit paged KV cache: write, read back, and decode / verify attention over it.

A quantised layer cache is uint8 [num_blocks, num_kv_heads, block_size, 80]
(`q4_cache_shape`), one tensor for the keys and one for the values: 80 bytes per
(token, kv head) instead of the 256 of a 16-bit cache of head size 128.  Each
record holds 128 codes of 4 bits and, for every group of 32 head dimensions, a
scale s and a minimum m in the model's type (bf16 or fp16):

    m = min x,  s = (max x - m) / 15 rounded to the model's type (0 below 2^-100),
    code = min(15, rint((x - m) / s)),  value = s * code + m.

A group whose max - min is not finite (an infinity or a NaN among its values)
reads back as NaN.  A cache is read in the type it was written in.

The ops stand beside `store_kvcache`, `flash_attn_with_kvcache` (and, through
`gather_kvcache_q4`, `flash_attn_varlen_func`) of `ops.py` and follow their
contracts (nanovllm/layers/attention.py:33-40, :64-74): they check their tensors, launch on the
current stream of the tensors' device and never synchronise the host (except
`gather_kvcache_q4` without `total_tokens`).
"""
import ctypes
import threading

import torch

from ._native import check, lib
from .ops import _DTYPES

HEAD_DIM = 128
RECORD_BYTES = 80
_CONTROL_BYTES = 16384  # covers the control words and counters at the start of an attention workspace
_U8, _I32 = torch.uint8, torch.int32
# A torch without CUDA has neither; no call gets as far without a CUDA tensor.
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the handle that torch.cuda.current_stream wraps


def q4_cache_shape(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int = HEAD_DIM) -> tuple:
    """Shape of one 4-bit cache tensor (uint8) of a layer's keys or values."""
    if head_dim != HEAD_DIM:
        raise NotImplementedError(f"4-bit KV cache: head_dim {head_dim} (only {HEAD_DIM})")
    return (num_blocks, num_kv_heads, block_size, RECORD_BYTES)


# The checks.  A decode step makes two of these calls per layer, and for small batches the host is what
# bounds them: each op asks once whether everything holds and only looks for the reason if it does not.
def _cache_ok(k_cache, v_cache, shape):
    return (len(shape) == 4 and shape[3] == RECORD_BYTES and k_cache.dtype is _U8 and v_cache.dtype is _U8
            and v_cache.shape == shape and k_cache.is_contiguous() and v_cache.is_contiguous())


def _rows_ok(key, value, shape, ks, vs):
    return (len(shape) == 3 and shape[2] == HEAD_DIM and value.shape == shape and key.dtype in _DTYPES
            and value.dtype is key.dtype and ks[2] == 1 and vs[2] == 1
            and (shape[1] == 1 or (ks[1] == HEAD_DIM and vs[1] == HEAD_DIM)))


def _refuse_type(dtype, head_dim):
    if head_dim != HEAD_DIM:
        raise NotImplementedError(f"4-bit KV cache: head_dim {head_dim} (only {HEAD_DIM})")
    if dtype not in _DTYPES:
        raise NotImplementedError(f"4-bit KV cache: dtype {dtype} (bf16 or fp16 only)")


def _explain_cache(k_cache, v_cache, num_kv_heads):
    assert k_cache.dtype == v_cache.dtype == torch.uint8, "4-bit KV caches are uint8 tensors"
    assert k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.size(3) == RECORD_BYTES, \
        "4-bit KV caches are [num_blocks, num_kv_heads, block_size, 80]"
    assert k_cache.is_contiguous() and v_cache.is_contiguous(), "KV caches must be contiguous"
    assert k_cache.size(1) == num_kv_heads, f"cache of {k_cache.size(1)} kv heads, rows of {num_kv_heads}"


def _explain_rows(key, value):
    assert key.dim() == 3 and value.shape == key.shape, "key and value must be [N, Hkv, 128] of one shape"
    _refuse_type(key.dtype, key.size(2))
    assert value.dtype == key.dtype, "key/value dtypes differ"
    raise AssertionError("rows must hold their heads contiguously")


def _explain_ints(what, t):
    raise AssertionError(f"{what} must be int32 and contiguous, of the call's size, not {t.dtype} {tuple(t.shape)}")


def _explain_devices(*tensors):
    raise AssertionError(f"4-bit KV cache ops take CUDA tensors of one device, not {[str(t.device) for t in tensors]}")


def _call(name, index, fn, *args):
    """fn(*args, stream) with device `index` current and its current stream; raises for a status."""
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        check(rc, name)


def store_kvcache_q4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     slot_mapping: torch.Tensor) -> None:
    """Quantise key[t] and value[t] ([N, Hkv, 128]) into the records of slot_mapping[t].

    Slots of -1 (padding) or outside the cache are skipped; the others must be
    unique within one call (as for `store_kvcache`).
    """
    shape, ks, vs, cs = key.shape, key.stride(), value.stride(), k_cache.shape
    if not _rows_ok(key, value, shape, ks, vs):
        _explain_rows(key, value)
    N, H, _ = shape
    if not (_cache_ok(k_cache, v_cache, cs) and cs[1] == H):
        _explain_cache(k_cache, v_cache, H)
    if slot_mapping.dtype is not _I32 or slot_mapping.numel() != N or N >= 2 ** 31 or not slot_mapping.is_contiguous():
        _explain_ints("slot_mapping", slot_mapping)
    dev = key.get_device()
    if not (dev >= 0 and value.get_device() == dev and k_cache.get_device() == dev and v_cache.get_device() == dev
            and slot_mapping.get_device() == dev):
        _explain_devices(key, value, k_cache, v_cache, slot_mapping)
    row = H * HEAD_DIM  # a single row may carry any stride
    _call("store_kvcache_q4", dev, lib().b200_store_kvcache_q4, key.data_ptr(), ks[0] if N > 1 else row,
          value.data_ptr(), vs[0] if N > 1 else row, k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(),
          N, H, HEAD_DIM, cs[0], cs[2], _DTYPES[key.dtype])


def _out_rows(out, n, k_cache, cs, dtype):
    """The (key, value) rows a reader writes, and their token strides."""
    H = cs[1]
    row = H * HEAD_DIM
    if out is None:
        key = k_cache.new_empty((n, H, HEAD_DIM), dtype=dtype)
        return key, torch.empty_like(key), row, row
    key, value = out
    shape, ks, vs = key.shape, key.stride(), value.stride()
    if not _rows_ok(key, value, shape, ks, vs):
        _explain_rows(key, value)
    assert shape[0] == n and shape[1] == H and key.dtype is dtype, \
        "out rows do not match the tokens, kv heads and dtype asked for"
    if not key.get_device() == value.get_device() == k_cache.get_device():
        _explain_devices(k_cache, key, value)
    return key, value, ks[0] if n > 1 else row, vs[0] if n > 1 else row


def load_kvcache_q4(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, dtype: torch.dtype,
                    out=None):
    """Read the records of slot_mapping [N] back: (key, value) rows [N, Hkv, 128] in `dtype`, the type
    the cache was written in.  Slots of -1 or outside the cache read as zeros.  `out` is an optional
    (key, value) pair to write to."""
    cs = k_cache.shape
    if dtype not in _DTYPES:
        _refuse_type(dtype, HEAD_DIM)
    if not _cache_ok(k_cache, v_cache, cs):
        _explain_cache(k_cache, v_cache, cs[1] if len(cs) == 4 else 0)
    N = slot_mapping.numel()
    if slot_mapping.dtype is not _I32 or N >= 2 ** 31 or not slot_mapping.is_contiguous():
        _explain_ints("slot_mapping", slot_mapping)
    dev = k_cache.get_device()
    if not (dev >= 0 and v_cache.get_device() == dev and slot_mapping.get_device() == dev):
        _explain_devices(k_cache, v_cache, slot_mapping)
    key, value, k_row, v_row = _out_rows(out, N, k_cache, cs, dtype)
    _call("load_kvcache_q4", dev, lib().b200_load_kvcache_q4, key.data_ptr(), k_row, value.data_ptr(), v_row,
          k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), N, cs[1], HEAD_DIM, cs[0], cs[2],
          _DTYPES[dtype])
    return key, value


def gather_kvcache_q4(k_cache: torch.Tensor, v_cache: torch.Tensor, cu_seqlens: torch.Tensor,
                      block_table: torch.Tensor, total_tokens: int | None = None, dtype: torch.dtype = torch.bfloat16,
                      out=None):
    """Read whole sequences back through their pages as packed rows.

    Row cu_seqlens[i] + p of the result is token p of sequence i, whose pages are
    block_table[i]; returns (key, value) [total_tokens, Hkv, 128] in `dtype`, what
    `flash_attn_varlen_func` takes.  total_tokens is cu_seqlens[-1] or any bound on it (rows
    behind the last sequence are left as they were); None reads cu_seqlens[-1] on the host,
    which synchronises.  Tokens of a page outside the cache read as zeros.
    """
    cs = k_cache.shape
    if dtype not in _DTYPES:
        _refuse_type(dtype, HEAD_DIM)
    if not _cache_ok(k_cache, v_cache, cs):
        _explain_cache(k_cache, v_cache, cs[1] if len(cs) == 4 else 0)
    S = cu_seqlens.numel() - 1
    if cu_seqlens.dtype is not _I32 or S < 0 or not cu_seqlens.is_contiguous():
        _explain_ints("cu_seqlens", cu_seqlens)
    bt = block_table.shape
    if block_table.dtype is not _I32 or len(bt) != 2 or bt[0] < S or block_table.stride(1) != 1:
        _explain_ints("block_table (a row per sequence)", block_table)
    dev = k_cache.get_device()
    if not (dev >= 0 and v_cache.get_device() == dev and cu_seqlens.get_device() == dev
            and block_table.get_device() == dev):
        _explain_devices(k_cache, v_cache, cu_seqlens, block_table)
    n = int(cu_seqlens[-1]) if total_tokens is None else int(total_tokens)
    assert 0 <= n < 2 ** 31, f"total_tokens {n}"
    key, value, k_row, v_row = _out_rows(out, n, k_cache, cs, dtype)
    _call("gather_kvcache_q4", dev, lib().b200_gather_kvcache_q4, key.data_ptr(), k_row, value.data_ptr(), v_row,
          k_cache.data_ptr(), v_cache.data_ptr(), cu_seqlens.data_ptr(), block_table.data_ptr(), block_table.stride(0),
          bt[1], S, n, cs[1], HEAD_DIM, cs[0], cs[2], _DTYPES[dtype])
    return key, value


# ------------------------------------------------------------------ attention
_ws_lock = threading.Lock()
_workspaces: dict[tuple, torch.Tensor] = {}
_captures: dict[tuple, tuple] = {}


def q4_workspace_size(query_len: int, group: int) -> int:
    """Bytes of a workspace of `flash_attn_with_kvcache_q4` for query_len * group query rows per kv head
    (of the current device; it does not depend on the batch)."""
    return int(lib().b200_paged_attention_q4_workspace_size(query_len, group))


def q4_workspace(device: torch.device, query_len: int, group: int) -> torch.Tensor:
    """The split-K workspace of a call on the current stream, its control words and counters zero.

    Eager calls keep one per (device, stream), for up to 16 query rows: calls of one stream run one
    after another and leave it re-armed.  The calls captured on one stream into one graph share one from
    the graph's memory pool, zeroed once by the graph itself, so that graphs replayed at the same time share
    nothing."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    with torch.cuda.device(index):
        assert q4_workspace_size(query_len, group) > 0, f"{query_len} queries of {group} heads: 1 to 16 rows per kv head"
        return _workspace(index)


def _workspace(index):
    key = (index, _raw_stream(index))
    if torch.cuda.is_current_stream_capturing():
        capture = ctypes.c_uint64()
        check(lib().b200_stream_capture_id(key[1], ctypes.addressof(capture)), "stream_capture_id")
        held = _captures.get(key)
        if held is None or held[0] != capture.value:
            # Held until the stream's next capture: the graph's pool must not hand it out again meanwhile.
            ws = torch.empty(q4_workspace_size(16, 1), dtype=torch.uint8, device=torch.device("cuda", index))
            ws[:_CONTROL_BYTES].zero_()
            held = _captures[key] = capture.value, ws
        return held[1]
    ws = _workspaces.get(key)
    if ws is None:
        with _ws_lock:
            ws = _workspaces.get(key)
            if ws is None:
                ws = torch.zeros(q4_workspace_size(16, 1), dtype=torch.uint8, device=torch.device("cuda", index))
                _workspaces[key] = ws
    return ws


def _explain_attention(q, k_cache, v_cache, cache_seqlens, block_table, causal, out):
    B, Lq, Hq, D = q.shape
    _refuse_type(q.dtype, D)
    Hkv = k_cache.size(1)
    _explain_cache(k_cache, v_cache, Hkv)
    assert Hkv > 0 and Hq % Hkv == 0, f"num_heads {Hq} not a multiple of num_kv_heads {Hkv}"
    assert q.stride(-1) == 1 and (Hq == 1 or q.stride(-2) == D), "q heads must be contiguous"
    assert Lq == 1 or B <= 1 or q.stride(0) == Lq * q.stride(1), "q rows of one sequence must be evenly strided"
    assert cache_seqlens.dtype == torch.int32 and cache_seqlens.is_contiguous() and cache_seqlens.numel() == B, \
        "cache_seqlens must be contiguous int32, one per sequence"
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.stride(1) == 1, \
        "block_table must be int32 [B, W] with contiguous rows"
    assert block_table.size(0) >= B, "block_table has fewer rows than q"
    assert out.shape == q.shape and out.is_contiguous() and out.dtype == q.dtype, "out must be contiguous and like q"
    _explain_devices(q, k_cache, v_cache, cache_seqlens, block_table, out)


def flash_attn_with_kvcache_q4(q, k_cache, v_cache, cache_seqlens=None, block_table=None, softmax_scale=None,
                               causal=True, out=None, workspace=None):
    """`flash_attn_with_kvcache` over a 4-bit cache: causal (bottom-right) attention of
    q [B, Lq, Hq, 128], Lq * Hq / Hkv <= 16, over the pages block_table [B, W] of caches
    [num_blocks, Hkv, block_size, 80] (block_size a multiple of 128).

    cache_seqlens int32 [B] counts the cached tokens of each row including its Lq queries; rows
    with cache_seqlens <= 0 return zeros.  Tokens whose page lies outside the cache count as zeros.
    workspace: a caller-owned one of q4_workspace_size(Lq, Hq // Hkv) bytes, zero-filled
    once; calls that share it must not overlap (default: one per stream, or per captured graph and stream).
    """
    assert cache_seqlens is not None and block_table is not None, "the B200 path reads a paged cache"
    shape, qs, cs, bt = q.shape, q.stride(), k_cache.shape, block_table.shape
    B, Lq, Hq, D = shape
    if not causal and Lq > 1:
        raise NotImplementedError("non-causal multi-query paged attention")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    dev = q.get_device()
    if not (D == HEAD_DIM and q.dtype in _DTYPES and _cache_ok(k_cache, v_cache, cs) and cs[1] > 0 and Hq % cs[1] == 0
            and qs[3] == 1 and (Hq == 1 or qs[2] == D) and (Lq == 1 or B <= 1 or qs[0] == Lq * qs[1])
            and cache_seqlens.dtype is _I32 and cache_seqlens.numel() == B and cache_seqlens.is_contiguous()
            and block_table.dtype is _I32 and len(bt) == 2 and bt[0] >= B and block_table.stride(1) == 1
            and out.shape == shape and out.dtype is q.dtype and out.is_contiguous()
            and dev >= 0 and k_cache.get_device() == dev and v_cache.get_device() == dev
            and cache_seqlens.get_device() == dev and block_table.get_device() == dev and out.get_device() == dev):
        _explain_attention(q, k_cache, v_cache, cache_seqlens, block_table, causal, out)
    Hkv = cs[1]
    if workspace is None:
        if _current_device() == dev:
            workspace = _workspace(dev)
        else:
            with torch.cuda.device(dev):
                workspace = _workspace(dev)
    else:
        assert workspace.dtype is _U8 and workspace.get_device() == dev and workspace.is_contiguous(), \
            "the workspace must be contiguous uint8 on q's device"
    _call("flash_attn_with_kvcache_q4", dev, lib().b200_paged_attention_q4, out.data_ptr(), q.data_ptr(),
          (qs[0] if B > 1 else Hq * D) if Lq == 1 else qs[1], k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[2],
          block_table.data_ptr(), block_table.stride(0), bt[1], cache_seqlens.data_ptr(), B, Lq, Hq, Hkv, D,
          D ** -0.5 if softmax_scale is None else float(softmax_scale), _DTYPES[q.dtype], workspace.data_ptr(),
          workspace.numel())
    return out
