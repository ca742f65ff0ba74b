"""Prefills over 4-bit caches read back in groups of sequences: the same result, in bounded memory."""
import numpy as np
import pytest
import torch

from tests.test_q4_attention_gpu import BS, HKV, HQ, attn, i32, rows, slots_of  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_groups_give_the_same_rows(pkg, attn, monkeypatch, dtype):  # noqa: F811
    """Second chunks of six sequences, some sharing pages, one beyond the limit: bit for bit the one-group result."""
    import learn_nano_vllm_b200.attention as mod
    lens_k, lens_q = [300, 513, 1, 1500, 256, 40], [20, 100, 1, 513, 3, 40]
    tables = [[0, 1, -1, -1, -1, -1], [0, 2, 3, -1, -1, -1], [4, -1, -1, -1, -1, -1], [5, 6, 7, 8, 9, 10], [0, -1, -1, -1, -1, -1],
              [11, -1, -1, -1, -1, -1]]
    for p in range(12):  # whole pages, then the chunk's own rows
        n = rows(BS, HKV, p, dtype), rows(BS, HKV, 50 + p, dtype)
        pkg.store_kvcache_q4(n[0], n[1], attn.k_cache, attn.v_cache, torch.arange(p * BS, (p + 1) * BS, dtype=torch.int32, device="cuda"))
    cu = lambda x: i32(np.concatenate([[0], np.cumsum(x)]))
    q, k, v = (rows(sum(lens_q), h, 100 + h, dtype) for h in (HQ, HKV, HKV))
    slots = torch.full((sum(lens_q),), -1, dtype=torch.int32, device="cuda")
    pkg.context.set_context(True, cu(lens_q), cu(lens_k), max(lens_q), max(lens_k), slots, None, i32(tables))
    want = attn(q, k, v)
    monkeypatch.setattr(mod, "_MAX_BOUND", 100)
    for limit in (1 << 17, 1000, 600, 1):
        monkeypatch.setattr(mod, "_PREFIX_ROWS", limit)
        assert torch.equal(attn(q, k, v), want), limit


def test_memory_of_long_prefixes_is_bounded(pkg, attn, monkeypatch):  # noqa: F811
    """64 sequences that share 11 pages: the rows read back take the limit's memory, not the batch's."""
    import learn_nano_vllm_b200.attention as mod
    S, n = 64, 11 * BS + 7
    tables = [list(range(12))] * S
    q, k, v = (rows(S, h, h) for h in (HQ, HKV, HKV))
    pkg.context.set_context(True, i32(np.arange(S + 1)), i32(np.arange(S + 1) * n), 1, n,
                            i32(sum((slots_of(tables[0], n - 1, n) for _ in range(1)), []) + [-1] * (S - 1)), None, i32(tables))
    monkeypatch.setattr(mod, "_PREFIX_ROWS", 4 * n, raising=False)
    attn(q, k, v)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    attn(q, k, v)
    # four sequences' rows (two calls' worth may be live while the next is made), and the outputs
    assert torch.cuda.max_memory_allocated() - before <= 2 * 4 * n * HKV * 512 + 4 * S * HQ * 128 * 2 + (1 << 20)
