"""The 4-bit cache oracle against what the format promises (CPU), and the ops' host-side refusals."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import kv_q4

BF16, F16 = torch.bfloat16, torch.float16


def rows(shape, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("scale", [1e-3, 1.0, 300.0])
def test_values_lie_within_half_a_level(dtype, scale):
    x = rows((40, 3, 128), dtype, 1, scale)
    bf = dtype == BF16
    codes, s, m = kv_q4.quantise(x.double().numpy(), bf)
    rec = kv_q4.pack(codes, s, m)
    assert rec.shape == (40, 3, 80)
    c2, s2, m2 = kv_q4.unpack(rec, bf)
    assert np.array_equal(c2, codes) and np.array_equal(s2, kv_q4.bits_float(s, bf))
    assert np.array_equal(m2, kv_q4.bits_float(m, bf))
    got = kv_q4.values(rec, bf).reshape(40, 3, 4, 32)
    want = x.double().numpy().reshape(40, 3, 4, 32)
    step = s2[..., None]
    # half a level, plus what rounding s to its type leaves of the largest code: 15 s times half a step
    # (fp16 scales may be subnormal: half of 2^-24 instead)
    slack = 15 * np.maximum(step * (2.0 ** -8 if bf else 2.0 ** -11), 0 if bf else 2.0 ** -25)
    assert (np.abs(got - want) <= step / 2 * (1 + 2.0 ** -20) + slack).all()
    assert np.array_equal(got.min(-1), want.min(-1))


def test_constant_and_non_finite_groups():
    x = torch.ones(1, 1, 128, dtype=BF16) * 3
    x[0, 0, 32] = float("inf")
    x[0, 0, 64] = float("nan")
    x[0, 0, 96], x[0, 0, 97] = 3.3e38, -3.3e38
    rec = kv_q4.pack(*kv_q4.quantise(x.double().numpy(), True))
    v = kv_q4.values(rec, True)[0, 0]
    assert (v[:32] == 3).all() and np.isnan(v[32:]).all()


def test_records_match_plain_words():
    """A word's shifted mask leaves neighbouring even / odd dimensions in its halves."""
    codes = np.arange(128).reshape(1, 4, 32).astype(np.uint8) % 16
    rec = kv_q4.pack(codes, np.zeros((1, 4), np.uint16), np.zeros((1, 4), np.uint16))
    words = rec[0, :64].copy().view(np.uint32)
    flat = codes.reshape(128)
    for w in range(16):
        for i in range(4):
            pair = (int(words[w]) >> (4 * i)) & 0x000f000f
            assert pair & 0xffff == flat[8 * w + 2 * i] and pair >> 16 == flat[8 * w + 2 * i + 1]


def test_attention_oracle_against_torch():
    """float64 torch softmax over the dequantised rows, one query token and a causal pair."""
    rng = np.random.default_rng(3)
    hkv, g, bs, nb = 2, 2, 128, 3
    k = kv_q4.pack(*kv_q4.quantise(rows((nb, hkv, bs, 128), F16, 4).double().numpy(), False))
    v = kv_q4.pack(*kv_q4.quantise(rows((nb, hkv, bs, 128), F16, 5).double().numpy(), False))
    bt = np.array([[2, 0, 1], [1, -1, -1]], np.int32)
    ctx = np.array([300, 0], np.int32)
    q = rng.standard_normal((2, 2, hkv * g, 128))
    out, bound = kv_q4.attention(q, k, v, bt, ctx, 0.09, False)
    K = torch.from_numpy(kv_q4.values(k[bt[0]], False)).transpose(0, 1).reshape(hkv, -1, 128)[:, :300]
    V = torch.from_numpy(kv_q4.values(v[bt[0]], False)).transpose(0, 1).reshape(hkv, -1, 128)[:, :300]
    for i, n in ((0, 299), (1, 300)):
        for h in range(hkv * g):
            p = torch.softmax(K[h // g, :n] @ torch.from_numpy(q[0, i, h]) * 0.09, 0)
            assert np.allclose(out[0, i, h], (p @ V[h // g, :n]).numpy(), rtol=1e-12, atol=1e-13)
    assert (out[1] == 0).all() and (bound[0] > 0).all()


# ------------------------------------------------------------------ refusals
def cache(nb=2, h=2, bs=128):
    return torch.zeros(nb, h, bs, 80, dtype=torch.uint8)


def test_store_refusals(pkg):
    k = rows((3, 2, 128), BF16)
    slots = torch.zeros(3, dtype=torch.int32)
    bad = [
        (AssertionError, (k, k, cache(), cache(), slots)),                               # not CUDA
        (AssertionError, (k, k.half(), cache(), cache(), slots)),                        # types differ
        (AssertionError, (k, k[:2], cache(), cache(), slots)),                           # shapes differ
        (NotImplementedError, (k.float(), k.float(), cache(), cache(), slots)),
        (NotImplementedError, (k[..., :64], k[..., :64], cache(), cache(), slots)),
        (AssertionError, (k, k, cache().int(), cache().int(), slots)),
        (AssertionError, (k, k, cache(h=3), cache(h=3), slots)),
        (AssertionError, (k, k, cache(), cache(nb=3), slots)),
        (AssertionError, (k, k, cache(), cache(), slots.long())),
        (AssertionError, (k, k, cache(), cache(), slots[:2])),
        (AssertionError, (k, k, cache().transpose(1, 2), cache().transpose(1, 2), slots)),
        (AssertionError, (k.transpose(0, 1), k.transpose(0, 1), cache(h=3), cache(h=3), slots[:2])),
    ]
    for exc, args in bad:
        with pytest.raises(exc):
            pkg.store_kvcache_q4(*args)


def test_read_refusals(pkg):
    slots = torch.zeros(3, dtype=torch.int32)
    cu = torch.tensor([0, 3], dtype=torch.int32)
    bt = torch.zeros(1, 1, dtype=torch.int32)
    for exc, args in [(AssertionError, (cache(), cache(), slots, BF16)), (NotImplementedError, (cache(), cache(), slots, torch.float32)),
                      (AssertionError, (cache(), cache(), slots.long(), BF16)), (AssertionError, (cache(), cache(bs=64), slots, BF16))]:
        with pytest.raises(exc):
            pkg.load_kvcache_q4(*args)
    k = rows((3, 2, 128), BF16)
    with pytest.raises(AssertionError):
        pkg.load_kvcache_q4(cache(), cache(), slots, F16, out=(k, k))
    for exc, args in [(AssertionError, (cache(), cache(), cu, bt, 3)), (AssertionError, (cache(), cache(), cu.long(), bt, 3)),
                      (AssertionError, (cache(), cache(), cu, bt.long(), 3)), (AssertionError, (cache(), cache(), cu, bt, -1)),
                      (AssertionError, (cache(), cache(), torch.zeros(4, dtype=torch.int32), bt, 3))]:
        with pytest.raises(exc):
            pkg.gather_kvcache_q4(*args)


def test_attention_refusals(pkg):
    q = rows((2, 1, 4, 128), BF16)
    cl = torch.ones(2, dtype=torch.int32)
    bt = torch.zeros(2, 1, dtype=torch.int32)
    f = pkg.flash_attn_with_kvcache_q4
    bad = [
        (AssertionError, dict(q=q, cache_seqlens=cl, block_table=bt)),                   # not CUDA
        (AssertionError, dict(q=q, cache_seqlens=None, block_table=bt)),
        (AssertionError, dict(q=q, cache_seqlens=cl.long(), block_table=bt)),
        (AssertionError, dict(q=q, cache_seqlens=cl, block_table=bt[:1])),
        (AssertionError, dict(q=q[:, :, :3], cache_seqlens=cl, block_table=bt)),         # 3 heads over 2
        (NotImplementedError, dict(q=q.float(), cache_seqlens=cl, block_table=bt)),
        (NotImplementedError, dict(q=q[..., :64], cache_seqlens=cl, block_table=bt)),
        (NotImplementedError, dict(q=q.expand(2, 2, 4, 128), cache_seqlens=cl, block_table=bt, causal=False)),
    ]
    for exc, kw in bad:
        with pytest.raises(exc):
            f(kw.pop("q"), cache(), cache(), **kw)
    with pytest.raises(NotImplementedError):
        pkg.q4_cache_shape(1, 256, 8, 64)
    assert pkg.q4_cache_shape(5, 256, 8) == (5, 8, 256, 80)


def test_c_abi_refusals(pkg):
    """Every check fires before anything is launched (no GPU here)."""
    lib = pkg.lib()
    buf = ctypes.create_string_buffer(4096)
    a = (ctypes.addressof(buf) + 255) & ~255
    ARG, UNS, WS = 1, 2, 3
    st = dict(key=a, ks=256, v=a, vs=256, kc=a, vc=a, slots=a, n=1, h=2, d=128, nb=1, bs=128, dt=1, s=None)

    def store(fn, **kw):
        x = {**st, **kw}
        return fn(*x.values())
    for fn in (lib.b200_store_kvcache_q4, lib.b200_load_kvcache_q4):
        for kw, rc in [(dict(n=0), 0), (dict(n=-1), ARG), (dict(key=None), ARG), (dict(slots=None), ARG), (dict(d=64), UNS),
                       (dict(dt=2), UNS), (dict(h=0), ARG), (dict(nb=0), ARG), (dict(bs=0), ARG), (dict(nb=1 << 24), ARG),
                       (dict(n=2, ks=255), ARG), (dict(kc=a + 8), ARG), (dict(key=a + 1), ARG),
                       (dict(nb=1 << 20, bs=1024, h=4, ks=512, vs=512), UNS), (dict(h=65536), ARG)]:  # 2^32 records
            assert store(fn, **kw) == rc, (kw, lib.b200_last_error())
    ga = dict(key=a, ks=256, v=a, vs=256, kc=a, vc=a, cu=a, bt=a, bts=1, btw=1, s=1, n=1, h=2, d=128, nb=1, bs=128, dt=1,
              st=None)
    for kw, rc in [(dict(n=0), 0), (dict(s=0), 0), (dict(n=-1), ARG), (dict(s=-1), ARG), (dict(cu=None), ARG),
                   (dict(btw=0), ARG), (dict(bts=-1), ARG), (dict(d=96), UNS), (dict(dt=7), UNS)]:
        assert lib.b200_gather_kvcache_q4(*{**ga, **kw}.values()) == rc, kw
    assert lib.b200_stream_capture_id(None, None) == ARG
    pa = dict(out=a, q=a, qs=512, kc=a, vc=a, nb=1, bs=128, bt=a, bts=1, btw=1, cl=a, b=1, lq=1, hq=4, hkv=2, d=128,
              sc=0.1, dt=1, ws=a, wb=1 << 24, st=None)
    for kw, rc in [(dict(b=0), 0), (dict(b=-1), ARG), (dict(q=None), ARG), (dict(hq=3), ARG), (dict(hkv=0), ARG),
                   (dict(lq=0), ARG), (dict(lq=9), UNS), (dict(lq=1 << 30), UNS), (dict(d=64), UNS), (dict(dt=2), UNS),
                   (dict(sc=0.0), ARG), (dict(sc=float("nan")), ARG), (dict(sc=float("inf")), ARG), (dict(b=2049), UNS),
                   (dict(bs=64), ARG), (dict(bs=192), ARG), (dict(nb=0), ARG), (dict(btw=0), ARG), (dict(bts=-1), ARG),
                   (dict(btw=1 << 25), ARG), (dict(qs=511), ARG), (dict(qs=516), ARG), (dict(q=a + 8), ARG),
                   (dict(kc=a + 4), ARG), (dict(ws=None), WS), (dict(ws=a + 16), WS), (dict(wb=1024), WS),
                   (dict(wb=8192), WS), (dict(b=2048, btw=1 << 22), UNS)]:
        assert lib.b200_paged_attention_q4(*{**pa, **kw}.values()) == rc, (kw, lib.b200_last_error())


def test_idle_cta_hook_refusals(pkg):
    lib = pkg.lib()
    for args in ((1, -1, 2_000_000), (1, 1 << 20, 2_000_000), (-1, 0, 2_000_000), (1, 0, 10), (1, 0, 2_000_000_000)):
        assert lib.b200_testing_idle_cta(*args) == 1, args
    assert lib.b200_testing_idle_cta(0, 3, 2_000_000) == 0


def test_import_without_a_cuda_build_of_torch():
    """The package imports where torch has no CUDA bindings; CUDA tensors, which the ops ask for, do not exist there."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_get')]: delattr(torch._C, n)\n"
            "import __graft_entry__\n"
            "pkg = __graft_entry__.load_package()\n"
            "k, c = torch.zeros(1, 1, 128, dtype=torch.bfloat16), torch.zeros(1, 1, 128, 80, dtype=torch.uint8)\n"
            "try: pkg.store_kvcache_q4(k, k, c, c, torch.zeros(1, dtype=torch.int32))\n"
            "except AssertionError as e: print('refused', e)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "refused 4-bit KV cache ops take CUDA tensors" in r.stdout, r.stderr
