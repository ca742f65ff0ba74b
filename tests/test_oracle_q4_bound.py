"""The per-element error bound of the 4-bit attention oracle (CPU): it is the same attention, and small
groups, early tokens and long tails cannot go missing within it."""
import numpy as np
import pytest
import torch

from oracle import kv_q4

BF16, F16 = torch.bfloat16, torch.float16


def records(x, dtype):
    """[nb, h, bs, 80] of rows [nb, h, bs, 128]."""
    x = torch.from_numpy(x).to(dtype).double().numpy()
    return kv_q4.pack(*kv_q4.quantise(x, dtype == BF16))


def setup(dtype, value_of, lq=1, n=700, h=2, hq=4, bs=128, seed=0):
    rng = np.random.default_rng(seed)
    nb = -(-n // bs)
    q = torch.from_numpy(rng.standard_normal((1, lq, hq, 128))).to(dtype).double().numpy()
    k = records(rng.standard_normal((nb, h, bs, 128)), dtype)
    v = value_of(rng, rng.standard_normal((nb, h, bs, 128)))
    return q, k, records(v, dtype), np.arange(nb, dtype=np.int32)[None], np.array([n], np.int32), 128 ** -0.5, dtype == BF16


def tol_of(args):
    want, bound = kv_q4.attention_bound(*args)
    return want, kv_q4.tolerance(want, bound, args[-1])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lq", [1, 3])
def test_same_attention(dtype, lq):
    q, k, v, bt, cl, scale, bf = setup(dtype, lambda rng, x: x, lq)
    bt = np.concatenate([bt, bt, bt])
    bt[1, 2] = 99                                     # a page outside the cache
    q, cl = np.concatenate([q, q, q]), np.array([700, 500, 0], np.int32)
    a, loose = kv_q4.attention(q, k, v, bt, cl, scale, bf)
    b, tight = kv_q4.attention_bound(q, k, v, bt, cl, scale, bf)
    assert np.allclose(a, b, rtol=1e-12, atol=1e-13) and (b[2] == 0).all() and (tight[2] == 0).all()
    assert (tight[:2] > 0).all() and (tight[:2] < loose[:2]).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_lost_group_is_seen(dtype):
    """Groups with a spread of 0.5 beside one with offsets of hundreds, and a constant one."""
    def values(rng, x):
        x = x * 0.5
        x[..., 32:64] = 0.25
        x[..., 64:96] += 300 * rng.standard_normal(32)
        return x
    args = setup(dtype, values)
    want, tol = tol_of(args)
    for j in range(4):
        got = want.copy()
        got[..., 32 * j:32 * j + 32] = 0
        lost = (np.abs(got - want) > tol).reshape(-1, 4, 32)
        assert lost[:, j].mean() > 0.9 and not np.delete(lost, j, 1).any()
        got = want.copy()
        got[..., 32 * j:32 * j + 32] *= 1 + 2 ** -3
        assert (np.abs(got - want) > tol).reshape(-1, 4, 32)[:, j].mean() > 0.5


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_lost_tokens_are_seen(dtype):
    """Pages whose values differ by 2^12, one query head per page: a page of zeros shows at its head."""
    nb, bs = 4, 128
    rng = np.random.default_rng(1)
    k, v = 0.3 * rng.standard_normal((nb, 1, bs, 128)), rng.standard_normal((nb, 1, bs, 128)) + 0.5
    q = np.zeros((1, 1, 4, 128))
    for p in range(nb):
        k[p, ..., 32 * p:32 * p + 32] += 4
        q[0, 0, p, 32 * p:32 * p + 32] = 1
        v[p] *= 2.0 ** (-4 * p)
    k, v = records(k, dtype), records(v, dtype)
    rest = (np.arange(nb, dtype=np.int32)[None], np.array([nb * bs], np.int32), 0.25, dtype == BF16)
    want, tol = tol_of((q, k, v, *rest))
    for p in range(nb):
        gone = v.copy()
        gone[p] = 0
        got, _ = kv_q4.attention_bound(q, k, gone, *rest)
        assert (np.abs(got - want) > tol)[0, 0, p].mean() > 0.9


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_lost_tail_is_seen(dtype):
    """One token with nearly all of the weight and values of zero: a tail of zeros, or one off by 5 %, shows."""
    n = 4000
    rng = np.random.default_rng(2)
    base = rng.standard_normal(128)
    k, v = 0.05 * rng.standard_normal((1, 1, n, 128)), 1 + 0.3 * rng.standard_normal((1, 1, n, 128))
    k[0, 0, 0], v[0, 0, 0] = base * (17 * 128 ** 0.5 / (base @ base)), 0
    q = torch.from_numpy(base).to(dtype).double().numpy().reshape(1, 1, 1, 128)
    args = (q, records(k, dtype), records(v, dtype), np.zeros((1, 1), np.int32), np.array([n], np.int32), 128 ** -0.5, dtype == BF16)
    want, tol = tol_of(args)
    assert (np.abs(want) < 1e-3).all() and (np.abs(want) > tol).all() and (0.05 * np.abs(want) > tol).all()
