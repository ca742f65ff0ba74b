"""The 4-bit cache's block count over tensor-parallel ranks (2 gloo ranks, CPU): every rank holds the blocks
that rank 0 schedules, whatever memory it has left."""
import os
import socket
import sys
import types

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BLOCK = 2 * 1 * 4 * 256 * 80  # keys and values of one layer, 4 heads a rank


def _worker(rank, world, port, free_blocks, ret):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        sys.path.insert(0, ROOT)
        import __graft_entry__
        pkg = __graft_entry__.load_package()
        # a device of 1000 blocks, of which this rank finds free_blocks[rank] free; too small to read prefixes back
        pkg.attention.prefix_bytes = lambda *a: 0
        real = torch.zeros
        torch.cuda.mem_get_info = lambda: (free_blocks[rank] * BLOCK, 1000 * BLOCK)
        torch.cuda.memory_stats = lambda: {"allocated_bytes.all.peak": 0, "allocated_bytes.all.current": 0}
        torch.cuda.current_device = lambda: 0
        torch.zeros = lambda *a, **k: real(*a, dtype=k["dtype"])
        hf = types.SimpleNamespace(num_key_value_heads=8, num_attention_heads=16, hidden_size=2048, head_dim=128)
        run = types.SimpleNamespace(
            config=types.SimpleNamespace(gpu_memory_utilization=1.0, num_kvcache_blocks=-1, max_model_len=4096, hf_config=hf),
            world_size=world, block_size=256, model=torch.nn.ModuleList([pkg.Attention(8, 128, 1.0, 4)]))
        try:
            pkg.integrate._q4_allocate_kv_cache(run)
            ret[rank] = run.config.num_kvcache_blocks, tuple(run.model[0].k_cache.shape)
        except AssertionError as e:
            ret[rank] = str(e)
    finally:
        dist.destroy_process_group()


def allocate(free_blocks):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ret = mp.get_context("spawn").Manager().dict()
    mp.spawn(_worker, args=(2, port, free_blocks, ret), nprocs=2)
    return ret[0], ret[1]


@pytest.mark.parametrize("free_blocks", [(900, 700), (650, 800)])
def test_ranks_agree_on_the_blocks(free_blocks):
    a, b = allocate(free_blocks)
    assert a == b and 0 < a[0] <= min(free_blocks) and a[1] == (a[0], 4, 256, 80)


def test_no_memory_on_one_rank_stops_both():
    a, b = allocate((900, 0))
    assert a == b == "no memory left for the KV cache"
