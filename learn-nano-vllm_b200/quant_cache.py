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
import threading

import torch

from ._native import check, lib
from .ops import _DTYPES, _require_cuda, _stream

HEAD_DIM = 128
RECORD_BYTES = 80
_CONTROL_BYTES = 16384  # covers the control words and counters at the start of an attention workspace


def q4_cache_shape(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int = HEAD_DIM) -> tuple:
    """Shape of one 4-bit cache tensor (uint8) of a layer's keys or values."""
    if head_dim != HEAD_DIM:
        raise NotImplementedError(f"4-bit KV cache: head_dim {head_dim} (only {HEAD_DIM})")
    return (num_blocks, num_kv_heads, block_size, RECORD_BYTES)


def _check_caches(k_cache, v_cache, num_kv_heads):
    assert k_cache.dtype == v_cache.dtype == torch.uint8, "4-bit KV caches are uint8 tensors"
    assert k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.size(3) == RECORD_BYTES, \
        "4-bit KV caches are [num_blocks, num_kv_heads, block_size, 80]"
    assert k_cache.is_contiguous() and v_cache.is_contiguous(), "KV caches must be contiguous"
    assert k_cache.size(1) == num_kv_heads, f"cache of {k_cache.size(1)} kv heads, rows of {num_kv_heads}"


def _check_slots(slot_mapping, n):
    assert slot_mapping.dtype == torch.int32 and slot_mapping.is_contiguous(), "slot_mapping must be contiguous int32"
    assert slot_mapping.numel() == n


def _check_rows(key, value):
    N, H, D = key.shape
    assert value.shape == key.shape, "key and value shapes differ"
    if D != HEAD_DIM:
        raise NotImplementedError(f"4-bit KV cache: head_dim {D} (only {HEAD_DIM})")
    assert key.dtype == value.dtype, "key/value dtypes differ"
    if key.dtype not in _DTYPES:
        raise NotImplementedError(f"4-bit KV cache: dtype {key.dtype} (bf16 or fp16 only)")
    for t in (key, value):
        assert t.stride(-1) == 1 and (H == 1 or t.stride(1) == D), "rows must hold their heads contiguously"
    return N, H


def _token_stride(t):
    """Token stride of [N, H, D] rows; a single row may carry any stride on its size-1 dim."""
    return t.stride(0) if t.size(0) > 1 else t.size(1) * t.size(2)


def store_kvcache_q4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     slot_mapping: torch.Tensor) -> None:
    """Quantise key[t] and value[t] ([N, Hkv, 128]) into the records of slot_mapping[t].

    Slots of -1 (padding) or outside the cache are skipped; the others must be
    unique within one call (as for `store_kvcache`).
    """
    N, H = _check_rows(key, value)
    _check_caches(k_cache, v_cache, H)
    _check_slots(slot_mapping, N)
    _require_cuda(key, value, k_cache, v_cache, slot_mapping)
    with torch.cuda.device(key.device):
        rc = lib().b200_store_kvcache_q4(key.data_ptr(), _token_stride(key), value.data_ptr(), _token_stride(value),
                                         k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), N, H,
                                         HEAD_DIM, k_cache.size(0), k_cache.size(2), _DTYPES[key.dtype], _stream(key))
    check(rc, "store_kvcache_q4")


def _out_rows(out, n, k_cache, dtype):
    if dtype not in _DTYPES:
        raise NotImplementedError(f"4-bit KV cache: dtype {dtype} (bf16 or fp16 only)")
    if out is None:
        shape = (n, k_cache.size(1), HEAD_DIM)
        return (torch.empty(shape, dtype=dtype, device=k_cache.device),
                torch.empty(shape, dtype=dtype, device=k_cache.device))
    key, value = out
    _check_rows(key, value)
    assert key.size(0) == n and key.dtype == dtype, "out rows do not match the tokens and dtype asked for"
    return key, value


def load_kvcache_q4(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, dtype: torch.dtype,
                    out=None):
    """Read the records of slot_mapping [N] back: (key, value) rows [N, Hkv, 128] in `dtype`, the type
    the cache was written in.  Slots of -1 or outside the cache read as zeros.  `out` is an optional
    (key, value) pair to write to."""
    _check_caches(k_cache, v_cache, k_cache.size(1))
    N = slot_mapping.numel()
    _check_slots(slot_mapping, N)
    key, value = _out_rows(out, N, k_cache, dtype)
    assert key.size(1) == k_cache.size(1), "out rows and cache differ in kv heads"
    _require_cuda(k_cache, v_cache, slot_mapping, key, value)
    with torch.cuda.device(k_cache.device):
        rc = lib().b200_load_kvcache_q4(key.data_ptr(), _token_stride(key), value.data_ptr(), _token_stride(value),
                                        k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), N,
                                        k_cache.size(1), HEAD_DIM, k_cache.size(0), k_cache.size(2), _DTYPES[dtype],
                                        _stream(k_cache))
    check(rc, "load_kvcache_q4")
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
    _check_caches(k_cache, v_cache, k_cache.size(1))
    assert cu_seqlens.dtype == torch.int32 and cu_seqlens.is_contiguous() and cu_seqlens.numel() >= 1
    S = cu_seqlens.numel() - 1
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.stride(1) == 1
    assert block_table.size(0) >= S, "block_table has fewer rows than sequences"
    n = int(cu_seqlens[-1]) if total_tokens is None else int(total_tokens)
    assert n >= 0, f"total_tokens {n} < 0"
    key, value = _out_rows(out, n, k_cache, dtype)
    assert key.size(1) == k_cache.size(1), "out rows and cache differ in kv heads"
    _require_cuda(k_cache, v_cache, cu_seqlens, block_table, key, value)
    with torch.cuda.device(k_cache.device):
        rc = lib().b200_gather_kvcache_q4(key.data_ptr(), _token_stride(key), value.data_ptr(), _token_stride(value),
                                          k_cache.data_ptr(), v_cache.data_ptr(), cu_seqlens.data_ptr(),
                                          block_table.data_ptr(), block_table.stride(0), block_table.size(1), S, n,
                                          k_cache.size(1), HEAD_DIM, k_cache.size(0), k_cache.size(2), _DTYPES[dtype],
                                          _stream(k_cache))
    check(rc, "gather_kvcache_q4")
    return key, value


# ------------------------------------------------------------------ attention
_ws_lock = threading.Lock()
_workspaces: dict[tuple, torch.Tensor] = {}


def q4_workspace_size(query_len: int, group: int) -> int:
    """Bytes of a workspace of `flash_attn_with_kvcache_q4` for query_len * group query rows per kv head
    (of the current device; it does not depend on the batch)."""
    return int(lib().b200_paged_attention_q4_workspace_size(query_len, group))


def q4_workspace(device: torch.device, query_len: int, group: int) -> torch.Tensor:
    """The split-K workspace of a call on the current stream, its control words and counters zero.

    Eager calls keep one per (device, stream), grown on demand: calls of one stream run one after
    another and leave it re-armed.  A call that is being captured gets its own from the graph's
    memory pool, zeroed by the graph itself, so that graphs replayed at the same time share nothing."""
    need = q4_workspace_size(query_len, group)
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        ws[:_CONTROL_BYTES].zero_()
        return ws
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    with _ws_lock:
        ws = _workspaces.get(key)
        if ws is None or ws.numel() < need:
            ws = _workspaces[key] = torch.zeros(need, dtype=torch.uint8, device=device)
    return ws


def flash_attn_with_kvcache_q4(q, k_cache, v_cache, cache_seqlens=None, block_table=None, softmax_scale=None,
                               causal=True, out=None, workspace=None):
    """`flash_attn_with_kvcache` over a 4-bit cache: causal (bottom-right) attention of
    q [B, Lq, Hq, 128], Lq * Hq / Hkv <= 16, over the pages block_table [B, W] of caches
    [num_blocks, Hkv, block_size, 80] (block_size a multiple of 128).

    cache_seqlens int32 [B] counts the cached tokens of each row including its Lq queries; rows
    with cache_seqlens <= 0 return zeros.  Tokens whose page lies outside the cache count as zeros.
    workspace: a caller-owned one of q4_workspace_size(Lq, Hq // Hkv) bytes, zero-filled
    once; calls that share it must not overlap (default: one per stream, or per captured call).
    """
    assert cache_seqlens is not None and block_table is not None, "the B200 path reads a paged cache"
    B, Lq, Hq, D = q.shape
    if not causal and Lq > 1:
        raise NotImplementedError("non-causal multi-query paged attention")
    if D != HEAD_DIM:
        raise NotImplementedError(f"4-bit KV cache: head_dim {D} (only {HEAD_DIM})")
    if q.dtype not in _DTYPES:
        raise NotImplementedError(f"4-bit KV cache: dtype {q.dtype} (bf16 or fp16 only)")
    Hkv = k_cache.size(1)
    _check_caches(k_cache, v_cache, Hkv)
    assert Hkv > 0 and Hq % Hkv == 0, f"num_heads {Hq} not a multiple of num_kv_heads {Hkv}"
    assert q.stride(-1) == 1 and (Hq == 1 or q.stride(-2) == D), "q heads must be contiguous"
    if Lq == 1:
        q_tok = q.stride(0) if B > 1 else Hq * D
    else:
        assert B <= 1 or q.stride(0) == Lq * q.stride(1), "q rows of one sequence must be evenly strided"
        q_tok = q.stride(1)
    assert cache_seqlens.dtype == torch.int32 and cache_seqlens.is_contiguous() and cache_seqlens.numel() == B
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.stride(1) == 1
    assert block_table.size(0) >= B, "block_table has fewer rows than q"
    if out is None:
        out = torch.empty((B, Lq, Hq, D), dtype=q.dtype, device=q.device)
    else:
        assert out.shape == (B, Lq, Hq, D) and out.is_contiguous() and out.dtype == q.dtype
    _require_cuda(q, k_cache, v_cache, cache_seqlens, block_table, out)
    scale = D ** -0.5 if softmax_scale is None else softmax_scale
    with torch.cuda.device(q.device):
        ws = q4_workspace(q.device, Lq, Hq // Hkv) if workspace is None else workspace
        rc = lib().b200_paged_attention_q4(out.data_ptr(), q.data_ptr(), q_tok, k_cache.data_ptr(), v_cache.data_ptr(),
                                           k_cache.size(0), k_cache.size(2), block_table.data_ptr(),
                                           block_table.stride(0), block_table.size(1), cache_seqlens.data_ptr(), B, Lq, Hq, Hkv, D,
                                           float(scale), _DTYPES[q.dtype], ws.data_ptr(), ws.numel(), _stream(q))
    check(rc, "flash_attn_with_kvcache_q4")
    return out
