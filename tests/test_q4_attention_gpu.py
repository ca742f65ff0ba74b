"""The Attention module on 4-bit caches: a chunked prefill, a prefix hit and decode steps as the engine
makes them, against the oracles on the values the cache holds."""
import types

import numpy as np
import pytest
import torch

from oracle import attention as oatt
from oracle import kv_q4
from tests.helpers import assert_attn_close, host

pytestmark = pytest.mark.gpu

HQ, HKV, BS = 16, 8, 256


@pytest.fixture
def attn(pkg):
    pkg.integrate.uninstall()  # the package's own context
    m = pkg.Attention(HQ, 128, 128 ** -0.5, HKV)
    m.k_cache = torch.zeros(pkg.q4_cache_shape(12, BS, HKV), dtype=torch.uint8, device="cuda")
    m.v_cache = torch.zeros_like(m.k_cache)
    yield m
    pkg.context.reset_context()


def rows(n, h, seed, dtype=torch.bfloat16, scale=128 ** -0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, h, 128, generator=g, device="cuda") * scale).to(dtype)


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def held(cache, table, n):
    """What the first n tokens of a sequence stand for, rounded to bf16 (numpy [n, Hkv, 128])."""
    c = cache.cpu().numpy()
    rec = np.stack([c[table[p // BS], :, p % BS] for p in range(n)])
    return torch.from_numpy(kv_q4.values(rec, True).astype(np.float32)).to(torch.bfloat16).float().numpy()


def causal(q, k, v, lq, lk):
    return oatt._attend(host(q), k, v, 128 ** -0.5, lq, lk)


def slots_of(table, a, b):
    return [table[p // BS] * BS + p % BS for p in range(a, b)]


def test_prefill_chunk_decode(pkg, attn):
    """Two sequences: prefill without a cache read, a second chunk that reads the first back, then decode
    steps captured in a graph with padding rows."""
    tables = [[3, 7], [0, 5]]
    first, second = [200, 33], [300, 40]
    # first chunk: attends to its own unquantised keys
    T = sum(first)
    q, k, v = rows(T, HQ, 1), rows(T, HKV, 2), rows(T, HKV, 3)
    cu = np.concatenate([[0], np.cumsum(first)])
    pkg.context.set_context(True, i32(cu), i32(cu), max(first), max(first),
                            i32(sum((slots_of(t, 0, n) for t, n in zip(tables, first)), [])))
    out = attn(q, k, v)
    for i, n in enumerate(first):
        s = slice(cu[i], cu[i + 1])
        assert_attn_close(host(out[s]), causal(q[s], host(k[s]), host(v[s]), n, n), f"first chunk {i}")
    # second chunk: block tables, the cache read back
    T = sum(second)
    q, k, v = rows(T, HQ, 4), rows(T, HKV, 5), rows(T, HKV, 6)
    total = [a + b for a, b in zip(first, second)]
    cuq, cuk = np.concatenate([[0], np.cumsum(second)]), np.concatenate([[0], np.cumsum(total)])
    pkg.context.set_context(True, i32(cuq), i32(cuk), max(second), max(total),
                            i32(sum((slots_of(t, a, b) for t, a, b in zip(tables, first, total)), [])), None, i32(tables))
    out = attn(q, k, v)
    for i, n in enumerate(second):
        s = slice(cuq[i], cuq[i + 1])
        want = causal(q[s], held(attn.k_cache, tables[i], total[i]), held(attn.v_cache, tables[i], total[i]), n, total[i])
        assert_attn_close(host(out[s]), want, f"second chunk {i}")
    # decode, captured with two padding rows
    B = 4
    q, k, v = (torch.zeros(B, h, 128, dtype=torch.bfloat16, device="cuda") for h in (HQ, HKV, HKV))
    slots, lens = torch.full((B,), -1, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    bt = torch.zeros(B, 2, dtype=torch.int32, device="cuda")
    bt[:2] = i32(tables)
    pkg.context.set_context(False, slot_mapping=slots, context_lens=lens, block_tables=bt)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        attn(q, k, v)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = attn(q, k, v)
    torch.cuda.current_stream().wait_stream(stream)
    assert out.shape == (B, 1, HQ, 128)
    for step in range(3):
        for t, x in enumerate((q, k, v)):
            x.copy_(rows(B, x.shape[1], 10 * step + t))
        n = [a + step + 1 for a in total]
        lens[:2] = i32(n)
        slots[:2] = i32([slots_of(t, m - 1, m)[0] for t, m in zip(tables, n)])
        graph.replay()
        kc, vc = attn.k_cache.cpu().numpy(), attn.v_cache.cpu().numpy()
        want, bound = kv_q4.attention(q[:2, None].double().cpu().numpy(), kc, vc, np.asarray(tables), np.asarray(n),
                                      128 ** -0.5, True)
        err = np.abs(out[:2].double().cpu().numpy() - want)
        assert (err <= kv_q4.tolerance(want, bound, True)).all(), f"decode step {step}"
        assert (out[2:] == 0).all()
    del graph


def test_many_sequences_read_the_total_on_the_host(pkg, attn):
    """A bound on the packed rows beyond its limit is replaced by the number itself: same result."""
    import learn_nano_vllm_b200.attention as mod
    lens = [300, 513, 1]
    tables = [[0, 1, -1], [2, 3, 4], [5, -1, -1]]
    cu = np.concatenate([[0], np.cumsum(lens)])
    q, k, v = rows(sum(lens), HQ, 1), rows(sum(lens), HKV, 2), rows(sum(lens), HKV, 3)
    pkg.context.set_context(True, i32(cu), i32(cu), max(lens), max(lens),
                            i32(sum((slots_of(t, 0, n) for t, n in zip(tables, lens)), [])), None, i32(tables))
    a = attn(q, k, v)
    old, mod._MAX_BOUND = mod._MAX_BOUND, 10
    try:
        assert torch.equal(a, attn(q, k, v))
    finally:
        mod._MAX_BOUND = old


def test_fused_epilogue(pkg, attn):
    """forward_fused: norm and rotation in one kernel, then the quantising store: the same cache and output as
    the separate steps."""
    n = 37
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(n, (HQ + 2 * HKV) * 128, generator=g, device="cuda").to(torch.bfloat16)
    norm = lambda s: types.SimpleNamespace(weight=(1 + 0.1 * torch.randn(128, generator=g, device="cuda")).to(torch.bfloat16), eps=1e-6)
    qn, kn = norm(0), norm(1)
    ang = torch.arange(512, device="cuda")[:, None] * (1e4 ** (-torch.arange(64, device="cuda") / 64))[None]
    rope = types.SimpleNamespace(cos_sin_cache=torch.cat([ang.cos(), ang.sin()], -1)[:, None].contiguous())
    pos = torch.arange(n, device="cuda")
    cu = i32([0, n])
    pkg.context.set_context(True, cu, cu, n, n, i32(slots_of([2], 0, n)))
    out = attn.forward_fused(qkv, pos, qn, kn, rope)
    kc, vc = attn.k_cache.clone(), attn.v_cache.clone()
    assert int(kc.sum()) and int(vc.sum())
    q, k, v = pkg.qk_norm_rope_store(qkv, pos, HQ, HKV, qn.weight, kn.weight, 1e-6, rope.cos_sin_cache)
    attn.k_cache.zero_(), attn.v_cache.zero_()
    assert torch.equal(out, attn(q, k, v))
    assert torch.equal(kc, attn.k_cache) and torch.equal(vc, attn.v_cache)


def test_allocate_kv_cache(pkg):
    """The engine's share of the memory in 4-bit blocks, bound to every attention layer."""
    from learn_nano_vllm_b200.integrate import _q4_allocate_kv_cache
    layers = torch.nn.ModuleList([pkg.Attention(HQ, 128, 1.0, HKV) for _ in range(3)])
    free, total = torch.cuda.mem_get_info()
    run = types.SimpleNamespace(
        config=types.SimpleNamespace(gpu_memory_utilization=(total - free) / total + 0.02, num_kvcache_blocks=-1,
                                     hf_config=types.SimpleNamespace(num_key_value_heads=HKV, num_attention_heads=HQ,
                                                                     hidden_size=2048, head_dim=128)),
        world_size=1, block_size=BS, model=layers)
    torch.cuda.reset_peak_memory_stats()
    _q4_allocate_kv_cache(run)
    n = run.config.num_kvcache_blocks
    block = 2 * 3 * HKV * BS * 80
    # 2 % of the card, less what the caching allocator holds without using it
    assert 0 < n <= 0.02 * total / block + 1
    for i, a in enumerate(layers):
        assert a.k_cache.shape == a.v_cache.shape == (n, HKV, BS, 80) and a.k_cache.dtype == torch.uint8
        assert a.k_cache.is_cuda and a.k_cache.data_ptr() == run.kv_cache[0, i].data_ptr()
        assert a.v_cache.data_ptr() == run.kv_cache[1, i].data_ptr()
    run.block_size = 64
    with pytest.raises(NotImplementedError):
        _q4_allocate_kv_cache(run)
