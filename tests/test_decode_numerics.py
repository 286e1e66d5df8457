"""Decoding where a query gives a large value no weight, and at the ends of the types' ranges, in 64 bits.

Tolerance: as in test_cache_attention.py, but for the last term.  P = p s 2^b is rounded to half, below its normal range
to multiples of 2^-24, and 2^b takes the largest product of a weight and a scale to 2^7 at least.  So a key's P is off by at most
2^-32 of that largest product, its value by 8 times it (av = 16 s):
  n 2^-32 max_j (w_j av_j), each value with its weight;
and exp2 gives 0 for weights below 2^-126 of the largest: 2^-126 max_j av_j (n of them at most).
"""
import pytest
import torch

from tests.test_cache import Guarded, ints, table, tokens
from tests.test_cache_attention import DTYPES, bound
from torch_blocksparse_b200 import SparseSelfAttention, layouts


def reference(q, k, v, lengths, scale):
    """(o, tolerance) of dense rows in 64 bits; k, v [Z, Hk, L, D] the cache's values."""
    half = 2.0 ** -11 if q.dtype == torch.bfloat16 else 2.0 ** -20
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    Z, Hq, T, D = q.shape
    G = Hq // k.size(1)
    o, tol = torch.zeros_like(q), torch.zeros_like(q)
    ak, av = bound(k), bound(v)
    for z in range(Z):
        for t in range(T):
            n = int(lengths[z]) - T + t + 1
            for h in range(Hq):
                s = (k[z, h // G, :n] @ q[z, h, t]) * scale
                w = torch.softmax(s, 0)
                a = av[z, h // G, :n]
                e = abs(scale) * (ak[z, h // G, :n] @ q[z, h, t].abs()) * 2.0 ** -21 + 2.0 ** -20
                o[z, h, t] = w @ v[z, h // G, :n]
                tol[z, h, t] = ((w * (e + half + 2.0 ** -20)) @ a + (w * (e + 2.0 ** -20)).sum() * (w @ a)
                                + n * 2.0 ** -32 * (w[:, None] * a).amax(0) + n * 2.0 ** -126 * a.amax(0))
    return o, tol


def assert_near(got, q, k, v, lengths, scale):
    want, tol = reference(q, k, v, lengths, scale)
    err = (got.double().cpu() - want).abs()
    info = torch.finfo(q.dtype)                       # (below the normal range: steps of tiny * eps)
    limit = tol + want.abs() * info.eps / 2 * 1.001 + info.tiny * info.eps
    assert bool((err <= limit).all()), ((err / limit).max(), err.max())


OUTLIERS = [(torch.float16, 6e4, 1e-2), (torch.float16, 6e4, 1e-4), (torch.bfloat16, 6e4, 1e-4), (torch.bfloat16, 2.0 ** 50, 1e-6)]


def outlying(dtype, D, L, at, large, small, groups=None, seed=0):
    """Keys and values of 2 heads: the tokens `at` have values `large`, and keys with a score of about -50 and -90 bits
    for queries of ones; the others' values are `small`."""
    k, v = tokens(1, 2, L, D, torch.float32, seed).clamp(-2, 2), tokens(1, 2, L, D, torch.float32, seed + 1).clamp(-3, 3) * small
    for t in at:
        k[:, 0, t], k[:, 1, t] = -50 * 0.6931 / D ** 0.5, -90 * 0.6931 / D ** 0.5
        v[:, :, t] = torch.where(torch.arange(D, device='cuda') < 32 * (groups or D), torch.linspace(0.5, 1.5, D, device='cuda') * large, v[:, :, t])
    return k.to(dtype), v.clamp(-6e4, 6e4).to(dtype) if dtype == torch.float16 else v.to(dtype)


def ones(*shape):
    """Queries of nearly equal channels, each head and token a little different."""
    n = shape[0] * shape[1] * shape[2]
    return torch.linspace(1, 1.1, n, device='cuda').view(*shape[:3], 1).expand(shape)


def decoded(q, k, v, lengths, page=32, block=32, scale=None):
    """decode() of q over a cache of k and v, and the cache's values."""
    Z, H, L, D = k.shape
    slots = -(-L // page)
    cache, pages = Guarded(Z * slots, H, D, page=page), table(Z, slots, Z * slots)
    zero = torch.zeros(Z, dtype=torch.int32, device='cuda')
    cache.write(k, v, pages, zero)
    kk, vv = cache.read(pages, zero, L, dtype=torch.float32)
    attn = SparseSelfAttention(layout=layouts.dense(1, -(-L // block)), block=block)
    return attn.decode(q, cache, pages, lengths, scale=scale), kk, vv


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,large,small', OUTLIERS)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('G,T', [(1, 1), (2, 1), (4, 1), (8, 1), (1, 3), (3, 5)])
@pytest.mark.parametrize('L,at', [(40, (0,)), (40, (7,)), (900, (0, 1, 300, 301)), (900, tuple(range(0, 900, 16)))])
def test_a_large_value_without_weight_costs_the_others_nothing(dtype, large, small, D, G, T, L, at):
    k, v = outlying(dtype, D, L, at, large, small)
    q = ones(1, 2 * G, T, D).to(dtype)
    got, kk, vv = decoded(q, k, v, ints(L))
    assert_near(got, q, kk, vv, ints(L), D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,large,small', OUTLIERS)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('G,T', [(2, 1), (8, 1), (2, 4)])
def test_queries_that_disagree_about_a_large_value(dtype, large, small, D, G, T):
    """Every other query of a tile attends to the large values, and only some groups of channels hold them."""
    L = 500
    k, v = outlying(dtype, D, L, (3, 260), large, small, groups=1)
    q = ones(1, 2 * G, T, D).to(dtype)
    q[:, 1::2] *= -1
    got, kk, vv = decoded(q, k, v, ints(L))
    assert_near(got, q, kk, vv, ints(L), D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('G', [1, 4, 8])
def test_most_weight_on_tiny_values_and_scores_that_climb(dtype, D, G):
    """The first key takes nearly all weight and has a value near zero; or scores climb by 12 bits every 50 keys, values falling."""
    L = 800
    k, v = tokens(2, 1, L, D, torch.float32).clamp(-2, 2) * 0.2, tokens(2, 1, L, D, torch.float32, 1).clamp(-3, 3)
    k[0, :, 0] += 14 * 0.6931 / D ** 0.5
    v[0, :, 0] *= 2.0 ** -18
    k[1] += (torch.arange(L, device='cuda') // 50 * 12 * 0.6931 / D ** 0.5)[:, None]
    v[1] *= torch.exp2(-(torch.arange(L, device='cuda') // 50).float())[:, None]
    q = torch.ones((2, G, 1, D), device='cuda').to(dtype)
    got, kk, vv = decoded(q, k.to(dtype), v.to(dtype), ints(L, L))
    assert_near(got, q, kk, vv, ints(L, L), D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('G,T', [(1, 1), (4, 1), (8, 1), (1, 5)])
def test_queries_up_to_the_end_of_bf16(D, G, T):
    """A power of two between the query and the scale changes no bit, up to the largest exponent; scores beyond a float's range are NaN."""
    L = 200
    k, v = tokens(1, 2, L, D, torch.bfloat16).clamp(-2, 2), tokens(1, 2, L, D, torch.bfloat16, 1)
    q = tokens(1, 2 * G, T, D, torch.bfloat16, 2).clamp(-7.5, 7.5) * 0.125
    q[..., 3] = 0.875                                   # (every query has the same exponent, so every one reaches the end)
    want, kk, vv = decoded(q, k, v, ints(L), scale=0.5)
    assert_near(want, q, kk, vv, ints(L), 0.5)
    for shift in (100, 119, 122, 125, 127):
        far = q * 2.0 ** (shift - 20) * 2.0 ** 20
        assert bool(far.isfinite().all())
        assert torch.equal(decoded(far, k, v, ints(L), scale=2.0 ** (-1 - min(shift, 120)))[0], decoded(q, k, v, ints(L), scale=2.0 ** (shift - min(shift, 120) - 1))[0])
    assert bool(decoded(q * 2.0 ** 126, k, v, ints(L), scale=1.0)[0].isnan().all())
