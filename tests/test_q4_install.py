"""install(kv_cache_bits=...) on stand-ins for the engine's modules (CPU)."""
import sys
import types

import pytest


def stub_engine(monkeypatch):
    def original(self):
        return "reference allocation"
    mods = {}
    for name in ("nanovllm", "nanovllm.utils", "nanovllm.utils.context", "nanovllm.layers", "nanovllm.layers.attention",
                 "nanovllm.layers.sampler", "nanovllm.layers.linear", "nanovllm.models", "nanovllm.models.qwen3",
                 "nanovllm.engine", "nanovllm.engine.llm_engine", "nanovllm.engine.model_runner"):
        mods[name] = types.ModuleType(name)
        monkeypatch.setitem(sys.modules, name, mods[name])
    mods["nanovllm.utils.context"].get_context = lambda: None
    mods["nanovllm.layers.sampler"].Sampler = type("Sampler", (), {"forward": lambda self: 0})
    mods["nanovllm.layers.linear"].RowParallelLinear = type("RowParallelLinear", (), {"forward": lambda self: 0})
    mods["nanovllm.models.qwen3"].Qwen3Attention = type("Qwen3Attention", (), {"forward": lambda self: 0})
    runner = type("ModelRunner", (), {"prepare_decode": lambda self: 0, "prepare_sample": lambda self: 0,
                                      "allocate_kv_cache": original})
    mods["nanovllm.engine.model_runner"].ModelRunner = runner
    return mods, runner, original


def test_kv_cache_bits(pkg, monkeypatch):
    import learn_nano_vllm_b200.integrate as integ
    for name in ("_ORIGINAL_FORWARD", "_ORIGINAL_SAMPLER", "_ORIGINAL_PREPARE", "_ORIGINAL_ROW", "_ORIGINAL_ALLOCATE"):
        monkeypatch.setattr(integ, name, [])
    mods, runner, original = stub_engine(monkeypatch)
    try:
        pkg.install(kv_cache_bits=4)
        assert runner.allocate_kv_cache is integ._q4_allocate_kv_cache
        pkg.install(kv_cache_bits=4, workers=True)
        opts = mods["nanovllm.engine.llm_engine"].ModelRunner.keywords["options"]
        assert opts["install"]["kv_cache_bits"] == 4
        pkg.install()
        assert runner.allocate_kv_cache is original
        with pytest.raises(NotImplementedError):
            pkg.install(kv_cache_bits=8)
    finally:
        integ.uninstall()


def test_kv_cache_bits_reach_every_rank(pkg, monkeypatch):
    """A 4-bit cache is bound in the spawned ranks too: a rank left with a 16-bit cache has fewer blocks than
    rank 0 schedules, and its stock store writes past them."""
    import learn_nano_vllm_b200.integrate as integ
    for name in ("_ORIGINAL_FORWARD", "_ORIGINAL_SAMPLER", "_ORIGINAL_PREPARE", "_ORIGINAL_ROW", "_ORIGINAL_ALLOCATE"):
        monkeypatch.setattr(integ, name, [])
    mods, runner, original = stub_engine(monkeypatch)
    engine = mods["nanovllm.engine.llm_engine"]
    try:
        pkg.install(kv_cache_bits=4)
        assert engine.ModelRunner.func.__name__ == "nanovllm_worker"
        assert engine.ModelRunner.keywords["options"]["install"]["kv_cache_bits"] == 4
        pkg.install()
        assert engine.ModelRunner is runner
    finally:
        integ.uninstall()
