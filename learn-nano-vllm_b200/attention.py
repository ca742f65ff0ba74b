"""Drop-in `Attention` module for nano-vLLM on B200.

Keeps the reference module's contract (nanovllm/layers/attention.py:43-75):
the constructor takes (num_heads, head_dim, scale, num_kv_heads); `k_cache`
and `v_cache` start empty and are assigned by ModelRunner.allocate_kv_cache
(model_runner.py:116-120); `forward(q, k, v)` reads the side-channel
context, stores the new keys/values into the paged cache when the cache is
bound, then runs causal varlen prefill (over the cache when the context
carries block tables, i.e. a prefix-cache hit or a chunked-prefill
continuation) or paged decode.  Output shapes match the reference:
[T, Hq, D] for prefill, [B, 1, Hq, D] for decode.

Caches of dtype uint8 are 4-bit caches (quant_cache.py; install(kv_cache_bits=4) binds
them): keys and values are quantised as they are stored, decode attends to the records,
and a prefill that continues a cached prefix reads its sequences back first.
"""
import torch
from torch import nn

from . import context as _ctx
from .ops import flash_attn_varlen_func, flash_attn_with_kvcache, qk_norm_rope_store, store_kvcache
from .quant_cache import flash_attn_with_kvcache_q4, gather_kvcache_q4, store_kvcache_q4

# Where forward() reads the metadata from; integrate.install() rebinds it to
# the reference's nanovllm.utils.context.get_context.
_get_context = _ctx.get_context


def set_context_source(fn):
    global _get_context
    _get_context = fn


# Rows of packed keys and values that a prefill holds at a time (a row is Hkv * 512 bytes: 537 MB of 8 heads;
# one longer sequence still makes a group of its own).  install(kv_cache_bits=4) leaves room for them.
_PREFIX_ROWS = 1 << 17
# A bound on the rows read back serves as their number up to here.
_MAX_BOUND = 1 << 16

# The last step that read its offsets: its context, the tensor and its version, the values, the layers served.
_step = None


def _offsets(ctx, layer):
    """cu_seqlens_k on the host: one synchronising read per step, shared by the step's layers through its context.
    A layer that comes by again is in another step (its lengths may have been written in place)."""
    global _step
    cu = ctx.cu_seqlens_k
    version = None if cu.is_inference() else cu._version
    step = _step
    if step is None or step[0] is not ctx or step[1] is not cu or step[2] != version or id(layer) in step[4]:
        step = _step = ctx, cu, version, cu.tolist(), set()
    step[4].add(id(layer))
    return step[3]


def prefix_bytes(max_model_len, num_kv_heads):
    """Device memory that reading prefixes back may take beside a cache (head size 128, 16-bit rows)."""
    return max(_PREFIX_ROWS, max_model_len) * num_kv_heads * 128 * 2 * 2


def _groups(ctx, layer):
    """Runs of the step's sequences that are read back together: (first, last + 1, rows, longest), at most
    _PREFIX_ROWS rows each, a bound in place of their number while it is small."""
    n = ctx.cu_seqlens_k.numel() - 1
    bound = n * int(ctx.max_seqlen_k)
    if bound <= min(_MAX_BOUND, _PREFIX_ROWS):
        return [(0, n, bound, ctx.max_seqlen_k)]
    cu = _offsets(ctx, layer)
    runs, first, longest = [], 0, 0
    for i in range(n):
        if i > first and cu[i + 1] - cu[first] > _PREFIX_ROWS:
            runs.append((first, i, cu[i] - cu[first], longest))
            first, longest = i, 0
        longest = max(longest, cu[i + 1] - cu[i])
    return runs + [(first, n, cu[n] - cu[first], longest)]


class Attention(nn.Module):

    def __init__(self, num_heads, head_dim, scale, num_kv_heads):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.k_cache = self.v_cache = torch.tensor([])

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        ctx = _get_context()
        cache_bound = self.k_cache.numel() > 0 and self.v_cache.numel() > 0
        if cache_bound:
            store = store_kvcache_q4 if self._quantised() else store_kvcache
            store(k, v, self.k_cache, self.v_cache, ctx.slot_mapping)
        return self._attend(ctx, q, k, v)

    def _quantised(self) -> bool:
        return self.k_cache.dtype == torch.uint8

    def forward_fused(self, qkv: torch.Tensor, positions: torch.Tensor, q_norm, k_norm,
                      rotary_emb) -> torch.Tensor:
        """q/k RMSNorm, RoPE and the cache store in one kernel, then attention.

        Same result as Qwen3Attention.forward's q_norm / k_norm / rotary_emb
        (nanovllm/models/qwen3.py:82-85) followed by forward(q, k, v); qkv is the
        fused projection output [T, (Hq + 2 Hkv) * D].
        """
        ctx = _get_context()
        cache_bound = self.k_cache.numel() > 0 and self.v_cache.numel() > 0
        if cache_bound and self._quantised():  # the store quantises rows of the norm and the rotation
            q, k, v = qk_norm_rope_store(qkv, positions, self.num_heads, self.num_kv_heads, q_norm.weight,
                                         k_norm.weight, q_norm.eps, rotary_emb.cos_sin_cache)
            store_kvcache_q4(k, v, self.k_cache, self.v_cache, ctx.slot_mapping)
            return self._attend(ctx, q, k, v)
        need_k = ctx.is_prefill and (ctx.block_tables is None or not cache_bound)
        q, k, v = qk_norm_rope_store(qkv, positions, self.num_heads, self.num_kv_heads, q_norm.weight,
                                     k_norm.weight, q_norm.eps, rotary_emb.cos_sin_cache,
                                     self.k_cache if cache_bound else None, self.v_cache if cache_bound else None,
                                     ctx.slot_mapping if cache_bound else None, return_k=need_k)
        return self._attend(ctx, q, k, v)

    def _attend(self, ctx, q, k, v):
        if self._quantised():
            if not ctx.is_prefill:
                return flash_attn_with_kvcache_q4(q.unsqueeze(1), self.k_cache, self.v_cache,
                                                  cache_seqlens=ctx.context_lens, block_table=ctx.block_tables,
                                                  softmax_scale=self.scale, causal=True)
            if ctx.block_tables is not None:
                return self._attend_prefixes(ctx, q)
            return flash_attn_varlen_func(q, k, v, cu_seqlens_q=ctx.cu_seqlens_q, cu_seqlens_k=ctx.cu_seqlens_k,
                                          max_seqlen_q=ctx.max_seqlen_q, max_seqlen_k=ctx.max_seqlen_k,
                                          softmax_scale=self.scale, causal=True)
        if not ctx.is_prefill:
            return flash_attn_with_kvcache(q.unsqueeze(1), self.k_cache, self.v_cache,
                                           cache_seqlens=ctx.context_lens, block_table=ctx.block_tables,
                                           softmax_scale=self.scale, causal=True)
        paged = ctx.block_tables is not None
        return flash_attn_varlen_func(q, self.k_cache if paged else k, self.v_cache if paged else v,
                                      cu_seqlens_q=ctx.cu_seqlens_q, cu_seqlens_k=ctx.cu_seqlens_k,
                                      max_seqlen_q=ctx.max_seqlen_q, max_seqlen_k=ctx.max_seqlen_k,
                                      softmax_scale=self.scale, causal=True, block_table=ctx.block_tables)

    def _attend_prefixes(self, ctx, q):
        """Varlen prefill over a 4-bit cache: the sequences read back as packed rows, a group at a time."""
        groups = _groups(ctx, self)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        for first, last, rows, longest in groups:
            cu_q, cu_k, tables = ctx.cu_seqlens_q, ctx.cu_seqlens_k, ctx.block_tables
            if len(groups) > 1:  # query offsets stay those of the whole batch, key rows start at 0
                cu_q, cu_k, tables = cu_q[first:last + 1], cu_k[first:last + 1], tables[first:last]
                cu_k = cu_k - cu_k[0]
            k, v = gather_kvcache_q4(self.k_cache, self.v_cache, cu_k, tables, rows, q.dtype)
            flash_attn_varlen_func(q, k, v, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, max_seqlen_q=ctx.max_seqlen_q,
                                   max_seqlen_k=longest, softmax_scale=self.scale, causal=True, out=out)
            del k, v  # before the next group's are made
        return out
