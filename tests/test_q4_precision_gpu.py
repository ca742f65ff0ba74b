"""Attention over 4-bit caches against each element's own error bound."""
import numpy as np
import pytest
import torch

from oracle import kv_q4
from tests.test_q4_gpu import BF16, F16, make, oracle_records

pytestmark = pytest.mark.gpu


def close(pkg, q, kc, vc, cl, bt, scale=128 ** -0.5, what="", rows=slice(None)):
    """The call within its bound at the batch rows `rows`."""
    out = pkg.flash_attn_with_kvcache_q4(q, kc, vc, cache_seqlens=cl, block_table=bt, softmax_scale=scale)
    bf = q.dtype == BF16
    rows = torch.arange(len(q), device="cuda")[rows] if isinstance(rows, slice) else torch.tensor(rows, device="cuda")
    q, cl, bt, out = q[rows], cl[rows], bt[rows], out[rows]
    want, bound = kv_q4.attention_bound(q.double().cpu().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), bt.cpu().numpy(),
                                        cl.cpu().numpy(), scale, bf)
    err, tol = np.abs(out.double().cpu().numpy() - want), kv_q4.tolerance(want, bound, bf)
    worst = np.unravel_index(np.nan_to_num(err / tol, nan=np.inf).argmax(), err.shape)
    assert (err <= tol).all(), f"{what}: at {worst} {err[worst] / tol[worst]:.2f} of the bound, want {want[worst]}"


def cache_of(x):
    """A cache [nb, h, bs, 80] of rows [nb, h, bs, 128]."""
    return torch.from_numpy(oracle_records(x.reshape(x.shape[0], -1, 128)).reshape(*x.shape[:3], 80)).cuda()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lq,hq,hkv", [(1, 16, 8), (1, 8, 1), (5, 16, 8), (1, 1, 1)])
def test_ordinary_rows(pkg, dtype, lq, hq, hkv):
    close(pkg, *make([700, 65, 3001, 5], hq, hkv, lq=lq, dtype=dtype, seed=hq + lq), what="ordinary")
    close(pkg, *make([20000, 129], hq, hkv, lq=lq, dtype=dtype, kscale=3.0, vscale=50.0, seed=hq + lq), what="peaked, split")


@pytest.mark.parametrize("dtype,lq,hq,spread", [(BF16, 1, 4, 14), (BF16, 5, 4, 14), (BF16, 1, 4, 40), (F16, 1, 4, 11), (F16, 3, 8, 11)])
def test_small_groups_beside_large_ones(pkg, dtype, lq, hq, spread):
    """Groups of value dimensions 2^spread below and above their neighbours keep their own precision."""
    q, kc, vc, cl, bt = make([900, 300], hq, 2, lq=lq, bs=128, dtype=dtype, kscale=2.0, seed=50)
    g = torch.Generator(device="cuda").manual_seed(51)
    x = torch.randn(vc.shape[0], 2, 128, 128, generator=g, device="cuda") + 0.2
    for j, e in enumerate((0, -spread, spread // 2, -spread // 2)):
        x[..., 32 * j:32 * j + 32] *= 2.0 ** e
    close(pkg, q, kc, cache_of(x.to(dtype)), cl, bt, what=f"groups 2^{spread} apart")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_small_tokens_beside_large_ones(pkg, dtype):
    """Pages whose values differ by 2^12, heads that attend to one page each."""
    nb, bs, lows = 4, 128, (0, -12, -6, -9)
    g = torch.Generator(device="cuda").manual_seed(52)
    rows = lambda s: torch.randn(nb, 1, bs, 128, generator=g, device="cuda") * s
    k, v = rows(0.3), rows(1.0) + 0.1
    q = torch.zeros(1, 1, 4, 128, device="cuda")
    for p, e in enumerate(lows):
        k[p, ..., 32 * p:32 * p + 32] += 4.0
        q[0, 0, p, 32 * p:32 * p + 32] = 1.0
        v[p] *= 2.0 ** e
    bt = torch.arange(nb, dtype=torch.int32, device="cuda")[None]
    cl = torch.tensor([nb * bs - 3], dtype=torch.int32, device="cuda")
    close(pkg, q.to(dtype), cache_of(k.to(dtype)), cache_of(v.to(dtype)), cl, bt, scale=0.25, what="pages apart")


@pytest.mark.parametrize("dtype,n,lq,nats", [(BF16, 4000, 1, 17.5), (BF16, 4000, 1, 16.0), (BF16, 2000, 4, 17.0), (F16, 4000, 1, 17.0),
                                             (F16, 3000, 3, 16.0)])
def test_tail_behind_one_token(pkg, dtype, n, lq, nats):
    """A first token far above all others in score and with values of zero: what is left of the output is the
    tail, thousands of tokens with probabilities around 2^-24.  Enough sequences (of the same pages) that
    none is split, so that the warp that meets the first token meets a quarter of its sequence's tail."""
    bs, hkv, g, B = 256, 8, 4, 80
    nb = -(-n // bs)
    gen = torch.Generator(device="cuda").manual_seed(n)
    scale = 128 ** -0.5
    base = torch.randn(hkv, 1, 1, 128, generator=gen, device="cuda")
    q = base.view(hkv, 1, 128) + 0.05 * torch.randn(B, lq, hkv, g, 128, generator=gen, device="cuda")
    k = 0.05 * torch.randn(nb, hkv, bs, 128, generator=gen, device="cuda")
    v = torch.randn(nb, hkv, bs, 128, generator=gen, device="cuda") * 0.3 + 1
    k[0, :, 0] = (base * (nats / scale) / (base * base).sum(-1, keepdim=True))[:, 0, 0]
    v[0, :, 0] = 0
    q = q.to(dtype).view(B, lq, hkv * g, 128)
    kc, vc = cache_of(k.to(dtype)), cache_of(v.to(dtype))
    bt = torch.arange(nb, dtype=torch.int32, device="cuda").expand(B, nb)
    cl = torch.full((B,), n, dtype=torch.int32, device="cuda")
    close(pkg, q, kc, vc, cl, bt, what=f"tail of {n}", rows=(0, 1, 37, B - 1))


@pytest.mark.parametrize("lq", [1, 9])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_offsets_that_carry_the_scores(pkg, dtype, lq):
    """Queries of one sign and two keys that share the weight, one an offset of the first group of dimensions
    and one of the second (and, to even the scores, the third): minima times sums of queries are all
    that decides, at scores of 300."""
    B, H, bs, scale = 16, 8, 128, 0.3
    g = torch.Generator(device="cuda").manual_seed(61)
    q = (torch.randn(B, 1, H, 128, generator=g, device="cuda") * 1.5).exp()   # of magnitudes whose sums take many bits
    q = q.to(dtype).expand(B, lq, H, 128).contiguous()
    sums = q[:, 0].double().unflatten(-1, (4, 32)).sum(-1)                                 # [B, H, 4]
    k = torch.zeros(B, H, bs, 4, dtype=torch.float64, device="cuda")
    k[:, :, 0, 0] = (300 / scale / sums[..., 0]).to(dtype).double()
    k[:, :, 1, 1] = (300 / scale / sums[..., 1]).to(dtype).double()
    gap = k[:, :, 0, 0] * sums[..., 0] - k[:, :, 1, 1] * sums[..., 1]
    k[:, :, 1, 2] = gap / sums[..., 2]
    v = torch.zeros(B, H, bs, 128, device="cuda")
    v[:, :, 0], v[:, :, 1] = 1, -1
    cl = torch.full((B,), 100, dtype=torch.int32, device="cuda")
    bt = torch.arange(B, dtype=torch.int32, device="cuda")[:, None]
    close(pkg, q, cache_of(k.repeat_interleave(32, -1).to(dtype)), cache_of(v.to(dtype)), cl, bt, scale=scale, what="offsets")
