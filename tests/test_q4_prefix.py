"""How a prefill over a 4-bit cache reads its prefixes back (CPU, the kernels replaced by recorders)."""
import pytest
import torch

import __graft_entry__

__graft_entry__.load_package()
import learn_nano_vllm_b200.attention as mod  # noqa: E402
from learn_nano_vllm_b200 import context  # noqa: E402


@pytest.fixture
def calls(pkg, monkeypatch):
    """Recorded calls: ("read", total_tokens, offsets), ("attend", cu_q, cu_k, max_k), and host reads of offsets."""
    log = []
    pkg.integrate.uninstall()

    def gather(k_cache, v_cache, cu, bt, total, dtype):
        n = int(cu[-1]) if total is None else total
        log.append(("read", total, cu.tolist(), bt[:, 0].tolist()))
        return torch.zeros(n, 2, 128, dtype=dtype), torch.zeros(n, 2, 128, dtype=dtype)

    def attend(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, out=None, **kw):
        log.append(("attend", cu_seqlens_q.tolist(), cu_seqlens_k.tolist(), max_seqlen_k))
        return torch.empty_like(q) if out is None else out
    monkeypatch.setattr(mod, "gather_kvcache_q4", gather)
    monkeypatch.setattr(mod, "flash_attn_varlen_func", attend)
    monkeypatch.setattr(mod, "store_kvcache_q4", lambda *a: None)
    yield log
    context.reset_context()


def layers(n):
    out = [mod.Attention(4, 128, 1.0, 2) for _ in range(n)]
    for a in out:
        a.k_cache = a.v_cache = torch.zeros(8, 2, 128, 80, dtype=torch.uint8)
    return out


def step(lens_q, lens_k):
    cu = lambda x: torch.tensor([0] + list(torch.tensor(x).cumsum(0)), dtype=torch.int32)
    context.set_context(True, cu(lens_q), cu(lens_k), max(lens_q), max(lens_k), torch.zeros(sum(lens_q), dtype=torch.int32),
                        None, torch.arange(len(lens_k), dtype=torch.int32)[:, None])
    rows = [torch.zeros(sum(lens_q), h, 128, dtype=torch.bfloat16) for h in (4, 2, 2)]
    return rows


def test_total_is_read_once_per_step(calls, monkeypatch):
    """Above the bound, the layers of a step share one read of the offsets: none asks the operator to synchronise,
    and the next step reads its own."""
    reads = []
    real = torch.Tensor.tolist
    ls = layers(3)
    for lens in ([1072] * 64, [1000] * 70):
        rows = step([5] * len(lens), lens)
        with monkeypatch.context() as m:
            m.setattr(torch.Tensor, "tolist", lambda t: reads.append(t) or real(t) if t is context.get_context().cu_seqlens_k
                      else real(t))
            m.setattr(mod, "gather_kvcache_q4", lambda *a: calls.append(a[4]) or (torch.zeros(a[4] or 0, 2, 128),) * 2)
            m.setattr(mod, "flash_attn_varlen_func", lambda q, *a, **k: q)
            for a in ls:
                a(*rows)
        assert calls == [sum(lens)] * 3
        calls.clear()
    assert len(reads) == 2


def test_small_steps_read_nothing(calls):
    """Up to the limit a bound on the rows serves, and nothing is read on the host."""
    rows = step([3, 4], [700, 32])
    layers(1)[0](*rows)
    assert calls[0][1] == 1400 and calls[1] == ("attend", [0, 3, 7], [0, 700, 732], 700)


def test_offsets_changed_in_place(calls):
    """A context whose offsets are written to between two layers is read again."""
    rows = step([1] * 70, [1000] * 70)
    a = layers(1)[0]
    a(*rows)
    context.get_context().cu_seqlens_k[1:] -= 1
    a(*rows)
    assert [c[1] for c in calls if c[0] == "read"] == [70000, 69999]


def test_rows_read_back_at_a_time_are_bounded(calls, monkeypatch):
    """A batch of long prefixes is read back in groups of consecutive sequences; queries keep their places and
    each group's key rows start at 0.  A sequence beyond the limit makes a group of its own."""
    monkeypatch.setattr(mod, "_PREFIX_ROWS", 1000)
    monkeypatch.setattr(mod, "_MAX_BOUND", 500)
    lens_q, lens_k = [5, 7, 1, 2, 9, 3], [400, 600, 1, 2500, 300, 700]
    rows = step(lens_q, lens_k)
    layers(1)[0](*rows)
    assert calls == [
        ("read", 1000, [0, 400, 1000], [0, 1]), ("attend", [0, 5, 12], [0, 400, 1000], 600),
        ("read", 1, [0, 1], [2]), ("attend", [12, 13], [0, 1], 1),
        ("read", 2500, [0, 2500], [3]), ("attend", [13, 15], [0, 2500], 2500),
        ("read", 1000, [0, 300, 1000], [4, 5]), ("attend", [15, 24, 27], [0, 300, 1000], 700)]


def test_allocation_leaves_room(pkg, monkeypatch):
    """The cache's share of the memory excludes the rows read back."""
    import types
    from learn_nano_vllm_b200 import integrate
    block = 2 * 1 * 4 * 256 * 80
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda: (90000 * block, 100000 * block))
    monkeypatch.setattr(torch.cuda, "memory_stats", lambda: {"allocated_bytes.all.peak": 7 * block, "allocated_bytes.all.current": 0})
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    real = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, dtype, device: real(2, 1, *a[2:3], 1, 1, 1, dtype=dtype))
    hf = types.SimpleNamespace(num_key_value_heads=4, num_attention_heads=8, hidden_size=1024, head_dim=128)
    for longest in (4096, 1 << 18):
        cfg = types.SimpleNamespace(gpu_memory_utilization=1.0, num_kvcache_blocks=-1, max_model_len=longest, hf_config=hf)
        run = types.SimpleNamespace(config=cfg, world_size=1, block_size=256, model=torch.nn.ModuleList([mod.Attention(8, 128, 1.0, 4)]))
        integrate._q4_allocate_kv_cache(run)
        assert cfg.num_kvcache_blocks * block <= (90000 - 7) * block - max(1 << 17, longest) * 4 * 512
        assert cfg.num_kvcache_blocks > 85000


def test_a_context_used_for_several_steps(calls):
    """Lengths written in place under one context, in inference mode (no version counts there): each step reads its own."""
    with torch.inference_mode():
        rows = step([1] * 70, [1000] * 70)
        ls = layers(2)
        for taken in (0, 1, 5):
            context.get_context().cu_seqlens_k[1:] -= taken
            for a in ls:
                a(*rows)
    assert [c[1] for c in calls if c[0] == "read"] == [70000] * 2 + [69999] * 2 + [69994] * 2
