"""4-bit KV cache on the GPU: records and rows bit for bit against the oracle, attention against
the oracle's 64-bit result within its derived bound."""
import numpy as np
import pytest
import torch

from oracle import kv_q4

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def rows(shape, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def empty_cache(nb, h, bs, fill=0):
    return torch.full((nb, h, bs, 80), fill, dtype=torch.uint8, device="cuda")


def oracle_records(x):
    """uint8 [N, H, 80] of rows [N, H, 128]."""
    return kv_q4.pack(*kv_q4.quantise(x.double().cpu().numpy(), x.dtype == BF16))


def oracle_store(cache, x, slots):
    """cache [NB, H, bs, 80] (numpy) after storing x."""
    rec = oracle_records(x)
    nb, h, bs, _ = cache.shape
    for t, s in enumerate(slots):
        if 0 <= s < nb * bs:
            cache[s // bs, :, s % bs] = rec[t]
    return cache


def oracle_rows(rec, dtype):
    """Rows in the model's type: the 64-bit values, rounded once."""
    bf = dtype == BF16
    v = kv_q4.bits_float(kv_q4.float_bits(kv_q4.values(rec, bf), bf), bf)
    return torch.from_numpy(v).to(dtype)


def same(a, b):
    """Equal values; NaN equals NaN (their bits are not part of the format's values)."""
    a, b = a.float().cpu(), b.float().cpu()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


# ------------------------------------------------------------ write and read back
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,h,nb,bs", [(1, 1, 1, 128), (7, 2, 3, 128), (33, 8, 2, 256), (64, 3, 5, 48), (700, 4, 4, 256),
                                       (5000, 1, 20, 256), (2, 16, 1, 1)])
def test_store_and_load(pkg, dtype, n, h, nb, bs):
    k = rows((n, h, 128), dtype, n)
    qkv = rows((n, (2 + 2 * h) * 128), dtype, n + 1, 3.0)
    v = qkv[:, -h * 128:].view(n, h, 128)  # a view of the fused projection
    g = torch.Generator().manual_seed(n)
    if n > nb * bs:
        slots = torch.full((n,), -1, dtype=torch.int32)
        slots[:nb * bs] = torch.randperm(nb * bs, generator=g).int()
    else:
        slots = torch.randperm(nb * bs, generator=g)[:n].int()
    if n > 5:
        slots[::5] = -1
        slots[1] = nb * bs          # outside the cache
        slots[2] = 2 ** 31 - 1
        slots[3] = -2 ** 31
    kc, vc = empty_cache(nb, h, bs, 7), empty_cache(nb, h, bs, 9)
    pkg.store_kvcache_q4(k, v, kc, vc, slots.cuda())
    kw = oracle_store(np.full((nb, h, bs, 80), 7, np.uint8), k, slots.tolist())
    vw = oracle_store(np.full((nb, h, bs, 80), 9, np.uint8), v, slots.tolist())
    assert np.array_equal(kc.cpu().numpy(), kw) and np.array_equal(vc.cpu().numpy(), vw)
    ko, vo = pkg.load_kvcache_q4(kc, vc, slots.cuda(), dtype)
    live = (slots >= 0) & (slots < nb * bs)
    assert same(ko[live], oracle_rows(oracle_records(k[live]), dtype))
    assert same(vo[live], oracle_rows(oracle_records(v[live]), dtype))
    assert (ko[~live] == 0).all() and (vo[~live] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_quantise_borders(pkg, dtype):
    """Ties, constants, zeros, subnormals, the type's extremes, infinities and NaN; a non-finite value
    poisons its own group of 32 only."""
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    x = torch.zeros(16, 1, 128, dtype=torch.float64)
    x[0] = 5.0
    x[1, 0, ::2] = 15.0
    x[1, 0, 1::2] = torch.arange(64) % 16 * 1.0
    x[2] = torch.arange(128) % 31 / 2.0              # steps of 1, values on the half: ties to even
    x[3, 0, :32] = tiny * torch.arange(32)
    x[3, 0, 32:64] = 2.0 ** -24 * torch.arange(32)
    x[4] = torch.randn(128, generator=torch.Generator().manual_seed(1)) * big / 8
    x[5, 0, 0], x[5, 0, 1] = big, -big
    x[6, 0, 40] = float("inf")
    x[7, 0, 70] = float("nan")
    x[8, 0, 100] = -float("inf")
    x[9] = -0.0
    x[10] = -3.0
    x[10, 0, ::3] = 2.0 ** -20                       # far below the minimum's last bit
    x[11] = torch.randn(128, generator=torch.Generator().manual_seed(2)) * 1e-4
    x[12] = 1000 + torch.randn(128, generator=torch.Generator().manual_seed(3))
    x[13] = torch.randn(128, generator=torch.Generator().manual_seed(4)) * 1e-30
    x[14] = torch.randn(128, generator=torch.Generator().manual_seed(5)) * 1e-36
    x[15] = torch.arange(128) % 2 * big
    x = x.to(dtype).cuda()
    kc, vc = empty_cache(1, 1, 128), empty_cache(1, 1, 128)
    slots = torch.arange(16, dtype=torch.int32, device="cuda")
    pkg.store_kvcache_q4(x, x, kc, vc, slots)
    want = oracle_records(x)
    got = kc[0, 0, :16].cpu().numpy()[:, None]
    # -0 and +0 are the same minimum: compare the parameters as numbers, the codes as they are
    assert np.array_equal(got[..., :64], want[..., :64])
    for a, b in zip(kv_q4.unpack(got, dtype == BF16)[1:], kv_q4.unpack(want, dtype == BF16)[1:]):
        assert np.array_equal(a, b, equal_nan=True)
    ko, vo = pkg.load_kvcache_q4(kc, vc, slots, dtype)
    assert same(ko, oracle_rows(want, dtype)) and same(vo, ko)
    assert torch.isnan(ko[6, 0, 32:64]).all() and torch.isfinite(ko[6, 0, :32]).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_are_rounded_once(pkg, dtype):
    """A code times its scale half way between two 16-bit numbers, and a minimum far below the last bit of
    the product: 3 s = 3 + 4.5 units lies above the middle by the minimum, which fp32 would drop."""
    unit = 2.0 ** -7 if dtype == BF16 else 2.0 ** -10
    tiny = 2.0 ** -40 if dtype == BF16 else 2.0 ** -24
    s = 1 + 3 * unit
    x = torch.full((1, 1, 128), tiny, dtype=torch.float64)
    x[..., 1::32], x[..., 2::32] = 15 * s, 3 * s
    x = x.to(dtype).cuda()
    kc, vc = empty_cache(1, 1, 128), empty_cache(1, 1, 128)
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    pkg.store_kvcache_q4(x, x, kc, vc, slot)
    rec = oracle_records(x)
    codes, scales, _ = kv_q4.unpack(rec, dtype == BF16)
    assert (scales == s).all() and (codes[..., 2] == 3).all() and (codes[..., 1] == 15).all()
    ko, _ = pkg.load_kvcache_q4(kc, vc, slot, dtype)
    assert (ko[..., 2::32].double() == 3 + 10 * unit).all() and same(ko, oracle_rows(rec, dtype))


def test_rows_of_any_alignment(pkg):
    """Rows off the 16-byte grid (a view that starts one element on, an odd token stride)."""
    n, h = 19, 2
    buf = rows((n * (h * 128 + 3) + 1,), BF16, 3)
    k = buf[1:].as_strided((n, h, 128), (h * 128 + 3, 128, 1))
    v = rows((n, h, 128), BF16, 4)
    slots = torch.randperm(256, generator=torch.Generator().manual_seed(0))[:n].int()
    kc, vc = empty_cache(2, h, 128), empty_cache(2, h, 128)
    pkg.store_kvcache_q4(k, v, kc, vc, slots.cuda())
    assert np.array_equal(kc.cpu().numpy(), oracle_store(np.zeros((2, h, 128, 80), np.uint8), k, slots.tolist()))
    obuf = torch.zeros(n * (h * 128 + 5) + 1, dtype=BF16, device="cuda")
    ko = obuf[1:].as_strided((n, h, 128), (h * 128 + 5, 128, 1))
    vo = torch.empty(n, h, 128, dtype=BF16, device="cuda")
    pkg.load_kvcache_q4(kc, vc, slots.cuda(), BF16, out=(ko, vo))
    k2, v2 = pkg.load_kvcache_q4(kc, vc, slots.cuda(), BF16)
    assert torch.equal(ko, k2) and torch.equal(vo, v2)
    untouched = torch.ones_like(obuf, dtype=torch.bool)
    untouched[1:].as_strided((n, h, 128), (h * 128 + 5, 128, 1)).fill_(False)
    assert (obuf[untouched] == 0).all()


def test_broadcast_head_rows(pkg):
    """One row for every token (stride 0) and empty calls."""
    k = rows((1, 2, 128), BF16, 5)
    kc, vc = empty_cache(1, 2, 128), empty_cache(1, 2, 128)
    with pytest.raises(AssertionError):
        pkg.store_kvcache_q4(k.expand(4, 2, 128), k.expand(4, 2, 128), kc, vc, torch.arange(4, dtype=torch.int32, device="cuda"))
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    pkg.store_kvcache_q4(k[:0], k[:0], kc, vc, none)
    ko, vo = pkg.load_kvcache_q4(kc, vc, none, BF16)
    assert ko.shape == vo.shape == (0, 2, 128) and int(kc.sum()) == 0


@pytest.mark.parametrize("dtype,h,bs,lens", [(BF16, 8, 256, [700]), (F16, 3, 128, [1, 0, 129, 128, 300, 0]),
                                             (BF16, 1, 48, [47, 48, 49, 500, 5]), (F16, 16, 256, [0, 0, 2])])
def test_gather(pkg, dtype, h, bs, lens):
    nb = sum(-(-n // bs) for n in lens) + 3
    rng = np.random.default_rng(sum(lens))
    kc = torch.from_numpy(rng.integers(0, 256, (nb, h, bs, 80), dtype=np.uint8))
    kc[..., 64:] = torch.from_numpy(oracle_records(rows((nb, h * bs, 128), dtype, 9)).reshape(nb, h, bs, 80)[..., 64:])
    vc = kc.flip(2).contiguous()
    perm = rng.permutation(nb)
    W = max(max(-(-n // bs) for n in lens), 1) + 1
    bt = np.full((len(lens), W), -1, np.int32)
    used = 0
    for b, n in enumerate(lens):
        m = -(-n // bs)
        bt[b, :m] = perm[used:used + m]
        used += m
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    total = int(cu[-1])
    cud, btd = torch.from_numpy(cu).cuda(), torch.from_numpy(bt).cuda()
    want = []
    for c in (kc.numpy(), vc.numpy()):
        r = [c[bt[b, p // bs], :, p % bs] for b, n in enumerate(lens) for p in range(n)]
        want.append(oracle_rows(np.stack(r), dtype))
    for tot in (total, None):
        ko, vo = pkg.gather_kvcache_q4(kc.cuda(), vc.cuda(), cud, btd, tot, dtype)
        assert ko.shape == (total, h, 128) and same(ko, want[0]) and same(vo, want[1])
    # a bound on the total: rows behind the last sequence stay as they were
    out = tuple(torch.full((total + 37, h, 128), 5.0, dtype=dtype, device="cuda") for _ in range(2))
    pkg.gather_kvcache_q4(kc.cuda(), vc.cuda(), cud, btd, total + 37, dtype, out=out)
    assert same(out[0][:total], want[0]) and same(out[1][:total], want[1])
    assert (out[0][total:] == 5).all() and (out[1][total:] == 5).all()
    # a bound that is too small stops there
    if total > 2:
        ko, vo = pkg.gather_kvcache_q4(kc.cuda(), vc.cuda(), cud, btd, total - 2, dtype)
        assert same(ko, want[0][:total - 2])


def test_gather_bad_pages(pkg):
    """Block ids outside the cache and tokens past the table read as zeros; a table may be a view or shared."""
    kc = torch.from_numpy(oracle_records(rows((4, 2 * 128, 128), BF16, 1)).reshape(4, 2, 128, 80)).cuda()
    cu = torch.tensor([0, 300, 600], dtype=torch.int32, device="cuda")
    full = torch.tensor([[9, 0, -1, 1, 9], [9, 4, 2, 2 ** 31 - 1, 9]], dtype=torch.int32, device="cuda")
    bt = full[:, 1:4]
    ko, _ = pkg.gather_kvcache_q4(kc, kc, cu, bt, 600, BF16)
    ref, _ = pkg.load_kvcache_q4(kc, kc, torch.arange(512, dtype=torch.int32, device="cuda"), BF16)
    zero = torch.zeros(128, 2, 128, dtype=BF16, device="cuda")
    assert torch.equal(ko[:300], torch.cat([ref[:128], zero, ref[128:172]]))
    assert torch.equal(ko[300:600], torch.cat([zero, ref[256:384], zero[:44]]))
    ko, _ = pkg.gather_kvcache_q4(kc, kc, cu, bt[:, :1], 600, BF16)   # a table one page wide
    assert torch.equal(ko[:300], torch.cat([ref[:128], zero, zero[:44]])) and (ko[300:] == 0).all()
    ko, _ = pkg.gather_kvcache_q4(kc, kc, cu, bt[:1].expand(2, 3), 600, BF16)
    assert torch.equal(ko[:300], ko[300:])


# ------------------------------------------------------------------- attention
def make(ctx, hq, hkv, lq=1, bs=256, dtype=BF16, seed=0, kscale=1.0, vscale=1.0, qscale=1.0, extra=2):
    """A cache of quantised rows with shuffled pages; returns (q, kc, vc, ctx, bt)."""
    rng = np.random.default_rng(seed)
    need = [max(1, -(-max(int(c), 0) // bs)) for c in ctx]
    nb = sum(need) + extra
    g = torch.Generator(device="cuda").manual_seed(seed)

    def cache(scale):
        x = (torch.randn(nb, hkv * bs, 128, generator=g, device="cuda") * scale
             * torch.exp(0.4 * torch.randn(1, 1, 128, generator=g, device="cuda"))).to(dtype)
        return torch.from_numpy(oracle_records(x).reshape(nb, hkv, bs, 80)).cuda()
    perm = rng.permutation(nb)
    bt = np.full((len(ctx), max(need)), -1, np.int32)
    used = 0
    for b, m in enumerate(need):
        bt[b, :m] = perm[used:used + m]
        used += m
    q = (torch.randn(len(ctx), lq, hq, 128, generator=g, device="cuda") * qscale).to(dtype)
    return q, cache(kscale), cache(vscale), torch.tensor(list(ctx), dtype=torch.int32, device="cuda"), torch.from_numpy(bt).cuda()


def check(pkg, q, kc, vc, cl, bt, scale=128 ** -0.5, what="", **kw):
    out = pkg.flash_attn_with_kvcache_q4(q, kc, vc, cache_seqlens=cl, block_table=bt, softmax_scale=scale, **kw)
    bf = q.dtype == BF16
    want, bound = kv_q4.attention(q.double().cpu().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), bt.cpu().numpy(),
                                  cl.cpu().numpy(), scale, bf)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all(), what
    err, tol = np.abs(got - want), kv_q4.tolerance(want, bound, bf)
    worst = np.unravel_index((err - tol).argmax(), err.shape)
    assert (err <= tol).all(), f"{what}: at {worst} got {got[worst]} want {want[worst]} tol {tol[worst]:.3e}"
    return out


@pytest.mark.parametrize("ctx", [1, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 1024, 4096])
@pytest.mark.parametrize("hq,hkv", [(16, 16), (16, 8), (16, 4)])
def test_context_lengths(pkg, ctx, hq, hkv):
    check(pkg, *make([ctx, max(1, ctx // 3), ctx + 1 if ctx < 4096 else 4000], hq, hkv, seed=ctx + hq), what=f"{ctx} {hq}/{hkv}")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 1), (64, 8), (16, 1), (1, 1), (3, 3)])
def test_group_sizes_and_types(pkg, dtype, hq, hkv):
    check(pkg, *make([700, 65, 3001], hq, hkv, dtype=dtype, seed=hq), what=f"{dtype} {hq}/{hkv}")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lq,hq,hkv", [(5, 16, 8), (2, 16, 2), (4, 16, 4), (3, 8, 8), (16, 4, 4), (9, 1, 1), (8, 2, 2)])
def test_several_queries(pkg, dtype, lq, hq, hkv):
    """Bottom-right causal queries; sequences shorter than the queries leave rows without a key."""
    check(pkg, *make([512, 2100, 7, 1300, 2, 1, 128], hq, hkv, lq=lq, dtype=dtype, seed=lq * 10 + hkv), what=f"lq={lq} {hq}/{hkv}")


@pytest.mark.parametrize("lq,hq,hkv", [(1, 12, 4), (3, 12, 4), (5, 12, 4), (3, 5, 1), (1, 7, 1), (2, 14, 2), (1, 13, 1), (1, 11, 1)])
def test_odd_groups(pkg, lq, hq, hkv):
    """Groups that are no power of two, up to 15 rows of a kv head."""
    check(pkg, *make([260, 5, 1111], hq, hkv, lq=lq, seed=hq), what=f"{lq} {hq}/{hkv}")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_offsets_beyond_the_spread(pkg, dtype):
    """Groups whose minimum is far larger than their range, and groups that are constant (scale 0)."""
    q, kc, vc, cl, bt = make([700, 19], 16, 8, dtype=dtype, seed=40)
    nb = kc.shape[0]
    g = torch.Generator(device="cuda").manual_seed(41)

    def cache(base, spread):
        x = torch.randn(nb, 8 * 256, 128, generator=g, device="cuda") * spread
        x[..., 32:64] = 0                                                 # a constant group
        x[..., 64:96] += base * torch.randn(1, 1, 32, generator=g, device="cuda")
        return torch.from_numpy(oracle_records(x.to(dtype)).reshape(nb, 8, 256, 80)).cuda()
    check(pkg, q, cache(20.0, 0.2), cache(300.0, 0.5), cl, bt, what="offsets")
    check(pkg, q, cache(0.0, 0.0), cache(0.0, 0.0), cl, bt, what="zeros")


def test_many_one_tile_sequences(pkg):
    """Hundreds of short sequences (one to 130 tokens), most items one tile, some batch rows empty."""
    n = np.random.default_rng(0).integers(0, 131, 700)
    check(pkg, *make(n, 4, 2, bs=128, seed=42), what="700 short")


@pytest.mark.parametrize("bs", [128, 256, 384, 512])
def test_block_sizes(pkg, bs):
    check(pkg, *make([1000, 385, 128, 513], 16, 8, bs=bs, seed=bs), what=f"block {bs}")


@pytest.mark.parametrize("kscale,vscale,qscale", [(8.0, 1.0, 2.0), (1.0, 1e-4, 1.0), (1.0, 1e3, 1.0), (1e-3, 1e-5, 1e3), (30.0, 30.0, 1e-2)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_ranges(pkg, kscale, vscale, qscale, dtype):
    """Peaked and flat softmaxes, small and large values."""
    check(pkg, *make([900, 130, 3], 16, 8, dtype=dtype, kscale=kscale, vscale=vscale, qscale=qscale, seed=3), what="ranges")


def test_value_scales_that_grow_along_the_context(pkg):
    """Value scales from 2^-14 to 2^14 within one sequence, rising, falling and alternating."""
    for order in ("up", "down", "mixed"):
        q, kc, vc, cl, bt = make([2000], 8, 8, bs=256, seed=11)
        n = 8
        e = np.linspace(-14, 14, n)
        e = {"up": e, "down": e[::-1], "mixed": np.random.default_rng(0).permutation(e)}[order]
        x = rows((vc.shape[0], 8 * 256, 128), BF16, 12)
        rec = x.clone()
        for page in range(n):
            rec[int(bt[0, page])] = x[int(bt[0, page])] * float(2.0 ** np.round(e[page]))
        vc = torch.from_numpy(oracle_records(rec).reshape(vc.shape)).cuda()
        check(pkg, q, kc, vc, cl, bt, what=order)


def test_padding_rows(pkg):
    """Rows of length 0 (or below) return zeros whatever their table holds, and an output that was full is overwritten."""
    q, kc, vc, cl, bt = make([300, 1, 1, 70], 16, 8, seed=5)
    cl[1], cl[2] = 0, -5
    bt[1:3] = 123456789
    out = torch.full_like(q, 3.0)
    got = check(pkg, q, kc, vc, cl, bt, what="padding", out=out)
    assert got is out and (out[1:3] == 0).all()
    check(pkg, *make([0, 0], 16, 8, seed=6), what="all padding")


def test_records_past_the_context_are_ignored(pkg):
    q, kc, vc, cl, bt = make([5, 300, 129], 16, 8, lq=2, seed=6)
    want = check(pkg, q, kc, vc, cl, bt, what="clean")
    for c in (kc, vc):
        for b in range(3):
            n = int(cl[b])
            for page in range(bt.shape[1]):
                blk = int(bt[b, page])
                if blk >= 0:
                    c[blk, :, max(0, min(256, n - page * 256)):] = 0xff  # NaN scales and minima
    got = pkg.flash_attn_with_kvcache_q4(q, kc, vc, cache_seqlens=cl, block_table=bt)
    assert torch.equal(got, want)


def test_pages_outside_the_cache_count_as_zeros(pkg):
    q, kc, vc, cl, bt = make([1000, 300], 16, 8, bs=128, seed=7)
    bt[0, 2], bt[0, 5], bt[1, 0] = -1, kc.shape[0], 2 ** 31 - 1
    check(pkg, q, kc, vc, cl, bt, what="bad pages")


def test_lengths_past_the_table(pkg):
    """A length beyond the table's pages is cut to them; a table may be a view of a wider one, or one shared row."""
    q, kc, vc, cl, bt = make([512, 512], 16, 8, bs=128, seed=8)
    wide = torch.full((2, 9), 77, dtype=torch.int32, device="cuda")
    wide[:, 3:7] = bt
    cl[:] = 100000
    a = check(pkg, q, kc, vc, cl, wide[:, 3:7], what="cut")
    cl[:] = 512
    assert torch.equal(a, check(pkg, q, kc, vc, cl, bt, what="full"))
    q[1] = q[0]
    shared = check(pkg, q, kc, vc, cl, bt[:1].expand(2, 4), what="shared table")
    assert torch.equal(shared[0], shared[1])


def test_non_finite_values(pkg):
    """A poisoned key makes the rows that see it NaN; a poisoned value its own 32 dimensions of them;
    rows that do not see the token, and the other kv heads, are as without it."""
    q, kc, vc, cl, bt = make([200], 4, 2, lq=3, bs=128, seed=9)
    clean = check(pkg, q, kc, vc, cl, bt, what="clean")
    v2 = vc.clone()
    v2[int(bt[0, 1]), 0, 198 - 128, 64 + 4 * 2:64 + 4 * 3] = 0xff    # token 198, head 0, group 2: seen by queries 1 and 2
    got = pkg.flash_attn_with_kvcache_q4(q, kc, v2, cache_seqlens=cl, block_table=bt)
    mask = torch.zeros_like(got, dtype=torch.bool)
    mask[0, 1:, :2, 64:96] = True
    assert torch.isnan(got[mask]).all() and torch.equal(got[~mask], clean[~mask])
    v2 = vc.clone()
    v2[int(bt[0, 0]), 1, 5, 64:68] = 0xff                             # an early token: seen by every query
    got = pkg.flash_attn_with_kvcache_q4(q, kc, v2, cache_seqlens=cl, block_table=bt)
    mask = torch.zeros_like(got, dtype=torch.bool)
    mask[0, :, 2:, :32] = True
    assert torch.isnan(got[mask]).all() and torch.equal(got[~mask], clean[~mask])
    k2 = kc.clone()
    k2[int(bt[0, 1]), 0, 199 - 128, 64:68] = 0xff                     # the last token: seen by query 2 only
    got = pkg.flash_attn_with_kvcache_q4(q, k2, vc, cache_seqlens=cl, block_table=bt)
    mask = torch.zeros_like(got, dtype=torch.bool)
    mask[0, 2, :2] = True
    assert torch.isnan(got[mask]).all() and torch.equal(got[~mask], clean[~mask])
    q2 = q.clone()
    q2[0, 0, 3, 17] = float("nan")
    got = pkg.flash_attn_with_kvcache_q4(q2, kc, vc, cache_seqlens=cl, block_table=bt)
    mask = torch.zeros_like(got, dtype=torch.bool)
    mask[0, 0, 3] = True
    assert torch.isnan(got[mask]).all() and torch.equal(got[~mask], clean[~mask])


def test_non_finite_across_chunks(pkg):
    """The same through the merge of a split sequence."""
    q, kc, vc, cl, bt = make([20000], 4, 1, bs=256, seed=10)
    k2 = kc.clone()
    k2[int(bt[0, 3]), 0, 9, 64:68] = 0xff
    assert torch.isnan(pkg.flash_attn_with_kvcache_q4(q, k2, vc, cache_seqlens=cl, block_table=bt)).all()
    q[0, 0, 2] = float("nan")
    got = pkg.flash_attn_with_kvcache_q4(q, kc, vc, cache_seqlens=cl, block_table=bt)
    assert torch.isnan(got[0, 0, 2]).all() and torch.isfinite(got[0, 0, [0, 1, 3]]).all()


@pytest.mark.parametrize("lq,hq,hkv", [(1, 8, 2), (5, 4, 2)])
def test_long_context_is_split_and_repeatable(pkg, lq, hq, hkv):
    args = make([40000, 17], hq, hkv, lq=lq, seed=12)
    a = check(pkg, *args, what="long")
    q, kc, vc, cl, bt = args
    for _ in range(5):
        assert torch.equal(a, pkg.flash_attn_with_kvcache_q4(q, kc, vc, cache_seqlens=cl, block_table=bt, softmax_scale=128 ** -0.5))


def test_strided_queries(pkg):
    """q as a view of the fused projection."""
    q, kc, vc, cl, bt = make([300, 41], 16, 8, seed=13)
    qkv = torch.zeros(2, (16 + 16) * 128, dtype=BF16, device="cuda")
    qkv[:, :16 * 128] = q.view(2, -1)
    a = check(pkg, qkv[:, :16 * 128].view(2, 1, 16, 128), kc, vc, cl, bt, what="view")
    assert torch.equal(a, check(pkg, q, kc, vc, cl, bt, what="contiguous"))
    with pytest.raises(AssertionError):  # off the 16-byte grid
        flat = torch.zeros(2 * 16 * 128 + 1, dtype=BF16, device="cuda")
        pkg.flash_attn_with_kvcache_q4(flat[1:].view(2, 1, 16, 128), kc, vc, cache_seqlens=cl, block_table=bt)


def test_slots_past_32_bits_of_bytes(pkg):
    """Records beyond 2^31 and 2^32 bytes of a cache (6.9 GB each): written, read back and attended to."""
    hkv, bs = 8, 256
    nb = 42000
    kc = torch.zeros(nb, hkv, bs, 80, dtype=torch.uint8, device="cuda")
    vc = torch.zeros(nb, hkv, bs, 80, dtype=torch.uint8, device="cuda")
    pages = [nb - 1, 13200, 26500]
    n = 3 * bs - 7
    k, v = rows((n, hkv, 128), BF16, 1), rows((n, hkv, 128), BF16, 2)
    t = torch.arange(n)
    slots = (torch.tensor(pages)[t // bs] * bs + t % bs).int().cuda()
    pkg.store_kvcache_q4(k, v, kc, vc, slots)
    ko, vo = pkg.load_kvcache_q4(kc, vc, slots, BF16)
    assert same(ko, oracle_rows(oracle_records(k), BF16)) and same(vo, oracle_rows(oracle_records(v), BF16))
    bt = torch.tensor([pages], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    kg, vg = pkg.gather_kvcache_q4(kc, vc, cu, bt, n, BF16)
    assert torch.equal(kg, ko) and torch.equal(vg, vo)
    q = rows((1, 1, 16, 128), BF16, 3)
    cl = torch.tensor([n], dtype=torch.int32, device="cuda")
    out = pkg.flash_attn_with_kvcache_q4(q, kc, vc, cache_seqlens=cl, block_table=bt)
    small_k, small_v = kc[pages].contiguous(), vc[pages].contiguous()
    small = check(pkg, q, small_k, small_v, cl, torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"), what="small")
    assert torch.equal(out, small)


# --------------------------------------------------- streams, graphs, workspaces
def test_two_streams_at_once(pkg):
    """Split calls in flight on two streams do not share a workspace."""
    a = make([30000, 9000], 8, 2, seed=20)
    b = make([25000, 100], 8, 2, lq=2, seed=21)
    f = lambda x: pkg.flash_attn_with_kvcache_q4(x[0], x[1], x[2], cache_seqlens=x[3], block_table=x[4])
    wa, wb = f(a), f(b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            outs.append((f(a), wa))
        with torch.cuda.stream(s2):
            outs.append((f(b), wb))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in outs)


def test_two_graphs_replayed_at_once(pkg):
    """Graphs captured one after the other on one stream, replayed on two, with new inputs."""
    cases = [make([30000, 9000], 8, 2, seed=22), make([20000, 5], 8, 2, seed=23)]
    s = torch.cuda.Stream()
    graphs, outs = [], []
    f = lambda x, out: pkg.flash_attn_with_kvcache_q4(x[0], x[1], x[2], cache_seqlens=x[3], block_table=x[4], out=out)
    for x in cases:
        out = torch.empty_like(x[0])
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            f(x, out)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                f(x, out)
                f(x, out)  # two layers of one graph
        graphs.append(g)
        outs.append(out)
    torch.cuda.synchronize()
    for x in cases:
        x[0].mul_(0.5)
        x[3][1] += 1 if int(x[3][1]) < 9000 else -700
    want = [f(x, torch.empty_like(x[0])) for x in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for o in outs:
            o.fill_(7)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    del graphs


def test_calls_of_one_graph_share_a_workspace(pkg):
    """Decode and verify calls of one capture take turns on one workspace; another capture, another stream of
    the same capture and the eager calls have their own."""
    a, b = make([9000, 300], 8, 2, seed=24), make([8000, 700], 8, 2, lq=3, seed=25)
    f = lambda x, out: pkg.flash_attn_with_kvcache_q4(x[0], x[1], x[2], cache_seqlens=x[3], block_table=x[4], out=out)
    want = [f(x, None) for x in (a, b)]
    s, side = torch.cuda.Stream(), torch.cuda.Stream()
    held, graphs, results = [], [], []
    for _ in range(2):
        outs = [torch.zeros_like(w) for w in want * 2]
        forked = torch.zeros_like(want[0])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ws = pkg.q4_workspace(torch.device("cuda"), 1, 4)
            side.wait_stream(s)
            with torch.cuda.stream(side):
                f(a, forked)
                other = pkg.q4_workspace(torch.device("cuda"), 1, 4)
            for x, o in zip((a, b) * 2, outs):
                f(x, o)
            assert pkg.q4_workspace(torch.device("cuda"), 3, 4).data_ptr() == ws.data_ptr()
            s.wait_stream(side)
        held += [ws, other]
        graphs.append(g)
        results.append(outs + [forked])
    with torch.cuda.stream(s):
        held.append(pkg.q4_workspace(torch.device("cuda"), 1, 4))
    assert len({w.data_ptr() for w in held}) == 5
    for _ in range(3):
        for outs in results:
            for o in outs:
                o.fill_(7)
        torch.cuda.synchronize()
        for g, st in zip(graphs, (s, side)):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for outs in results:
            assert all(torch.equal(o, w) for o, w in zip(outs, want * 2 + want[:1]))
    del graphs


def test_captured_decode_step(pkg):
    """store + attention of a padded batch, captured once and replayed with new tokens, lengths and tables."""
    B, hq, hkv, bs, nb = 8, 16, 8, 128, 40
    kc, vc = empty_cache(nb, hkv, bs), empty_cache(nb, hkv, bs)
    q, k, v = (torch.zeros(B, h, 128, dtype=BF16, device="cuda") for h in (hq, hkv, hkv))
    slots = torch.full((B,), -1, dtype=torch.int32, device="cuda")
    cl = torch.zeros(B, dtype=torch.int32, device="cuda")
    bt = torch.zeros(B, 4, dtype=torch.int32, device="cuda")
    out = torch.empty(B, 1, hq, 128, dtype=BF16, device="cuda")

    def step():
        pkg.store_kvcache_q4(k, v, kc, vc, slots)
        pkg.flash_attn_with_kvcache_q4(q.unsqueeze(1), kc, vc, cache_seqlens=cl, block_table=bt, out=out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
    torch.cuda.current_stream().wait_stream(s)
    tables = np.random.default_rng(0).permutation(nb)[:B * 4].reshape(B, 4).astype(np.int32)
    bt.copy_(torch.from_numpy(tables))
    kw, vw = np.zeros(kc.shape, np.uint8), np.zeros(vc.shape, np.uint8)
    for it in range(4):
        live = [3, 8, 1, 6][it]
        for t, x in enumerate((q, k, v)):
            x.copy_(rows(x.shape, BF16, 100 * it + t))
        n = np.zeros(B, np.int32)
        n[:live] = it + 1
        sl = np.full(B, -1, np.int32)
        sl[:live] = tables[:live, 0] * bs + it
        cl.copy_(torch.from_numpy(n))
        slots.copy_(torch.from_numpy(sl))
        g.replay()
        torch.cuda.synchronize()
        oracle_store(kw, k, sl.tolist())
        oracle_store(vw, v, sl.tolist())
        assert np.array_equal(kc.cpu().numpy(), kw) and np.array_equal(vc.cpu().numpy(), vw)
        want, bound = kv_q4.attention(q.double().cpu().numpy()[:, None], kw, vw, tables, n, 128 ** -0.5, True)
        err = np.abs(out.double().cpu().numpy() - want)
        assert (err <= kv_q4.tolerance(want, bound, True)).all() and (out[live:] == 0).all()
    del g


def test_caller_owned_workspace(pkg):
    """A workspace is re-armed after each call; one that is too small is refused."""
    args = make([9000, 300, 5000], 8, 2, seed=30)
    need = pkg.q4_workspace_size(1, 4)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    a = check(pkg, *args, what="own workspace", workspace=ws)
    assert int(ws[:8192].view(torch.int32).abs().sum()) == 0 and pkg.workspace_error(ws) == 0
    assert torch.equal(a, check(pkg, *args, what="again", workspace=ws))
    with pytest.raises(pkg.B200Error):
        pkg.flash_attn_with_kvcache_q4(args[0], args[1], args[2], cache_seqlens=args[3], block_table=args[4],
                                       workspace=torch.zeros(need - 4096, dtype=torch.uint8, device="cuda"))
    for bad in (torch.zeros(need, dtype=torch.uint8), ws.view(torch.int32), torch.zeros(2 * need, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(AssertionError):  # on the host, of another type, with gaps
            pkg.flash_attn_with_kvcache_q4(args[0], args[1], args[2], cache_seqlens=args[3], block_table=args[4], workspace=bad)


@pytest.mark.parametrize("ctx,hq,hkv,lq,dtype", [([57000], 4, 1, 1, BF16), ([57000], 16, 1, 1, F16), ([33000, 100, 9000], 4, 2, 5, BF16),
                                                 ([28000, 28000], 2, 2, 1, F16), ([9000, 1, 16500], 8, 1, 1, BF16)])
def test_many_chunks(pkg, ctx, hq, hkv, lq, dtype):
    """Sequences over so many CTAs that their partial results are merged in groups first: right, the same
    each time, and on a workspace that is left re-armed."""
    args = make(ctx, hq, hkv, lq=lq, dtype=dtype, seed=sum(ctx))
    ws = torch.zeros(pkg.q4_workspace_size(lq, hq // hkv), dtype=torch.uint8, device="cuda")
    a = check(pkg, *args, what=f"{ctx} {hq}/{hkv}", workspace=ws)
    assert int(ws[:7424].view(torch.int32).abs().sum()) == 0
    for _ in range(3):
        assert torch.equal(a, pkg.flash_attn_with_kvcache_q4(args[0], args[1], args[2], cache_seqlens=args[3],
                                                             block_table=args[4], out=torch.zeros_like(a), workspace=ws))


def test_poison_survives_grouped_merges(pkg):
    """A NaN value among 57,000 makes its group of 32 dimensions NaN for the rows that see it, and nothing else."""
    q, kc, vc, cl, bt = make([57000], 2, 1, lq=3, seed=42)
    want = pkg.flash_attn_with_kvcache_q4(q, kc, vc, cache_seqlens=cl, block_table=bt, softmax_scale=0.09)
    for token, rows_hit in ((20001, 3), (56998, 2), (56999, 1)):
        bad = vc.clone()
        bad[int(bt[0, token // 256]), 0, token % 256, 64 + 4 * 2:64 + 4 * 3] = 0xff  # group 2: s = m = NaN
        got = pkg.flash_attn_with_kvcache_q4(q, kc, bad, cache_seqlens=cl, block_table=bt, softmax_scale=0.09)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[:, 3 - rows_hit:, :, 64:96] = True
        assert torch.equal(torch.isnan(got), hit)
        assert (got[~hit].float() - want[~hit].float()).abs().max() <= 2 ** -7 * want.float().abs().max()


def test_workspace_serves_every_number_of_rows(pkg):
    """Decode and verify calls in turn on one workspace (the stream's, and a caller's own): the counters of one
    do not lie where another keeps its partial results."""
    decode = make([9000, 500, 4000], 32, 8, seed=40)
    verify = make([8000, 300, 5000], 16, 8, lq=5, seed=41)
    ws = torch.zeros(max(pkg.q4_workspace_size(1, 4), pkg.q4_workspace_size(5, 2)), dtype=torch.uint8, device="cuda")
    first = check(pkg, *decode, what="decode"), check(pkg, *verify, what="verify")
    for kw in (dict(), dict(workspace=ws)):
        for _ in range(2):
            for args, want in zip((decode, verify), first):
                got = pkg.flash_attn_with_kvcache_q4(args[0], args[1], args[2], cache_seqlens=args[3], block_table=args[4],
                                                     out=torch.full_like(args[0], 7.0), **kw)
                assert torch.equal(got, want)
    assert pkg.workspace_error(ws) == 0


def test_wait_that_runs_out_is_reported(pkg):
    """The producer issues nothing (test hook): the call returns with error bit 1, the next one is normal."""
    args = make([300, 1100], 16, 8, seed=31)
    ws = torch.zeros(pkg.q4_workspace_size(1, 2), dtype=torch.uint8, device="cuda")
    assert pkg.lib().b200_testing_idle_producer(1, 2_000_000) == 0
    pkg.flash_attn_with_kvcache_q4(args[0], args[1], args[2], cache_seqlens=args[3], block_table=args[4], workspace=ws)
    assert pkg.workspace_error(ws) & 1
    ws.zero_()
    check(pkg, *args, what="after the stalled call", workspace=ws)
    assert pkg.workspace_error(ws) == 0


def test_gpu_refusals(pkg):
    q, kc, vc, cl, bt = make([10], 16, 8, seed=1)
    f = pkg.flash_attn_with_kvcache_q4
    with pytest.raises(NotImplementedError):
        f(q.expand(1, 9, 16, 128).contiguous(), kc, vc, cache_seqlens=cl, block_table=bt)   # 18 rows of a kv head
    with pytest.raises(AssertionError):
        f(q, kc, vc, cache_seqlens=cl, block_table=bt, softmax_scale=0.0)
    with pytest.raises(AssertionError):
        f(q, kc.cpu(), vc, cache_seqlens=cl, block_table=bt)
    with pytest.raises(AssertionError):
        f(q, kc[:, :, :64].contiguous(), vc[:, :, :64].contiguous(), cache_seqlens=cl, block_table=bt)
    with pytest.raises(AssertionError):
        f(q.transpose(2, 3).contiguous().transpose(2, 3), kc, vc, cache_seqlens=cl, block_table=bt)


@pytest.mark.parametrize("ctx,hq,hkv,lq,cta", [([20000, 300], 8, 2, 1, 3), ([57000], 4, 1, 1, 40), ([57000], 4, 1, 1, 0), ([9000, 1, 16500], 8, 1, 1, 7),
                                               ([33000, 100, 9000], 4, 2, 5, 20), ([2000] * 150, 16, 8, 1, 5)])
def test_a_stalled_cta_leaves_its_workspace_usable(pkg, ctx, hq, hkv, lq, cta):
    """One CTA's producer issues nothing (test hook): the call reports it, what the CTA shares with others comes out as
    NaN, the counters are zero again, and the next call on the workspace, of other queries, is right."""
    q, kc, vc, cl, bt = make(ctx, hq, hkv, lq=lq, seed=sum(ctx) + cta)
    ws = torch.zeros(pkg.q4_workspace_size(lq, hq // hkv), dtype=torch.uint8, device="cuda")
    f = lambda x: pkg.flash_attn_with_kvcache_q4(x, kc, vc, cache_seqlens=cl, block_table=bt, workspace=ws, out=torch.zeros_like(x))
    want = f(q)
    assert pkg.workspace_error(ws) == 0 and torch.isfinite(want).all()
    assert pkg.lib().b200_testing_idle_cta(1, cta, 2_000_000) == 0
    stalled = f(q)
    assert pkg.workspace_error(ws) & 1
    assert int(ws[256:7424].view(torch.int32).abs().sum()) == 0
    hit = torch.isnan(stalled)
    assert hit.any() and not hit.all() or len(ctx) == 1
    same = ~hit & (stalled != 0)   # what no stalled CTA touched
    assert torch.equal(stalled[same], want[same])
    got = f(-q)
    ws.zero_()
    assert torch.equal(got, f(-q)) and pkg.workspace_error(ws) == 0
