"""Attention over the 4-bit cache against the definition in 64 bits on the values that the cache holds.

Tolerance.  Let a_j = 16 s_j bound what the tensor cores add up for key j (codes + 8 are at most 15, values at most 8 s).
Scores: sums of D products q (c + 8) s in 32 bits with the offset taken off again, 2^-21 of the sum of their
absolute values with room for the order; exp2, the maxima and 32-bit sums 2^-20.  So a weight is off by
e_j = scale * (|q| . ak_j) * 2^-21 + 2^-20 relative, and P's rounding to half adds r = 2^-11 for bf16 (for fp16
the remainder is added back: 2^-20).  P's largest is at least 2^7 and its smallest step 2^-24, so rounding below the normal
range adds 2^-32 of the largest value for each key.  Numerator and denominator:
  |o - want| <= sum_j w_j (e_j + r + 2^-20) av_j + (sum_j w_j (e_j + 2^-20)) (sum_j w_j av_j) + n 2^-32 max_j av_j,
plus half a step of the type.
"""
import pytest
import torch

from tests.test_cache import Guarded, ints, table, tokens
from torch_blocksparse_b200 import KVCache, Rotary, SparseSelfAttention, SparsityConfig, _lib, layouts, tables

DTYPES = [torch.float16, torch.bfloat16]


def bound(x):
    """16 s of every value's group: the largest value is at least 6 s (its code is 7 unless s was rounded up)."""
    g = x.unflatten(-1, (-1, 32))
    return (g.abs().amax(-1, keepdim=True) * (16 / 6)).expand(g.shape).flatten(-2)


def decode_reference(q, k, v, there, lengths, layout, block, scale):
    """(o, tolerance) in 64 bits; k, v [Z, Hk, L, D] the cache's values; `there` [Z, L]: tokens that have a page."""
    half = 2.0 ** -11 if q.dtype == torch.bfloat16 else 2.0 ** -20
    q, k, v, layout = q.double().cpu(), k.double().cpu(), v.double().cpu(), layout.cpu() != 0
    Z, Hq, T, D = q.shape
    Hk, L = k.shape[1:3]
    o, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    ak, av = bound(k), bound(v)
    j = torch.arange(L)
    for z in range(Z):
        for t in range(T):
            pos = int(lengths[z]) - T + t
            if pos < 0 or pos // block >= layout.size(1):
                continue
            see = layout[:, pos // block][:, (j // block).clamp(max=layout.size(2) - 1)] & (j <= pos) & there[z]
            see = see.expand(Hk, L)
            for h in range(Hq):
                hk = h // (Hq // Hk)
                n = see[hk].nonzero()[:, 0]
                if n.numel() == 0:
                    continue
                w = torch.softmax((k[z, hk, n] @ q[z, h, t]) * scale, 0)
                e = abs(scale) * (ak[z, hk, n] @ q[z, h, t].abs()) * 2.0 ** -21 + 2.0 ** -20
                o[z, h, t] = w @ v[z, hk, n]
                tol[z, h, t] = ((w * (e + half + 2.0 ** -20)) @ av[z, hk, n] + (w * (e + 2.0 ** -20)).sum() * (w @ av[z, hk, n])
                                + n.numel() * 2.0 ** -32 * av[z, hk, n].amax(0))
    return o, tol


def assert_decoded(got, q, k, v, there, lengths, layout, block, scale):
    want, tol = decode_reference(q, k, v, there, lengths, layout, block, scale)
    assert got.shape == q.shape and got.dtype == q.dtype
    err = (got.double().cpu() - want).abs()
    limit = tol + want.abs() * torch.finfo(q.dtype).eps / 2 * 1.001 + torch.finfo(q.dtype).tiny
    assert bool((err <= limit).all()), ((err / limit).max(), err.max())


def filled(Z, H, L, D, page, dtype, lengths, seed=0, spare=2):
    """A cache that holds `lengths` tokens of each sequence and NaN scales everywhere else, its table, and its values."""
    slots = -(-L // page)
    cache = Guarded(Z * slots + spare, H, D, page=page)
    pages = table(Z, slots, Z * slots + spare, seed)
    k, v = tokens(Z, H, L, D, dtype, seed + 1), tokens(Z, H, L, D, dtype, seed + 2)
    start = torch.zeros(Z, dtype=torch.int32, device='cuda')
    cache.write(k, v, pages, start, lengths.clamp(max=L))
    k, v = cache.read(pages, start, L, lengths, dtype=torch.float32)
    return cache, pages, k, v


def queries(Z, H, T, D, dtype, seed=7):
    return tokens(Z, H, T, D, dtype, seed) * 0.2


def layout_of(kind, H, nb, seed=0):
    if kind == 'dense':
        return layouts.dense(1, nb)
    if kind == 'fixed':
        return layouts.fixed(H, -(-nb // 4) * 4, 4)[:, :nb, :nb].contiguous()
    if kind == 'band':
        return layouts.causal_band(H, nb, 2, 1)
    lay = (torch.rand((H, nb, nb), generator=torch.Generator().manual_seed(seed)) < 0.4).long()   # beyond the diagonal too
    lay[:, nb // 2] = 0                                                                           # a row without a block
    return lay


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('kind', ['dense', 'fixed', 'band', 'random'])
@pytest.mark.parametrize('Hq,Hk,T,block,page', [(3, 3, 1, 16, 16), (4, 4, 1, 64, 64), (8, 2, 1, 128, 32), (16, 1, 1, 32, 256),
                                                (5, 1, 3, 16, 64), (2, 2, 6, 16, 16), (6, 2, 9, 64, 128), (2, 1, 20, 16, 32)])
def test_decoded_as_in_64_bits(dtype, D, kind, Hq, Hk, T, block, page):
    L = 300
    layout = layout_of(kind, Hk, -(-L // block))
    lengths = ints(300, 1, 16, 17, 0, 129, 255, T, max(0, T - 2), 208)
    Z = lengths.numel()
    cache, pages, k, v = filled(Z, Hk, L, D, page, dtype, lengths)
    q = queries(Z, Hq, T, D, dtype)
    got = SparseSelfAttention(layout=layout, block=block).decode(q, cache, pages, lengths)
    assert_decoded(got, q, k, v, torch.ones(Z, L, dtype=torch.bool), lengths, layout, block, D ** -0.5)
    cache.check()
    # and again: the same bits
    assert torch.equal(SparseSelfAttention(layout=layout, block=block).decode(q, cache, pages, lengths), got)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('Z,H,L,kind,block', [(1, 1, 5000, 'dense', 64), (1, 2, 4999, 'fixed', 16), (2, 1, 4100, 'random', 128)])
def test_long_rows_are_split_over_a_cluster(dtype, Z, H, L, kind, block):
    lengths = ints(*([L, L - 1077][:Z]))
    layout = layout_of(kind, H, -(-L // block))
    cache, pages, k, v = filled(Z, H, L, 64, 64, dtype, lengths)
    q = queries(Z, 4 * H, 2, 64, dtype)
    got = SparseSelfAttention(layout=layout, block=block).decode(q, cache, pages, lengths, scale=0.31)
    assert_decoded(got, q, k, v, torch.ones(Z, L, dtype=torch.bool), lengths, layout, block, 0.31)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('G,T', [(1, 1), (1, 2), (2, 2), (4, 1), (8, 1)])
def test_many_sequences_with_long_rows(dtype, D, G, T):
    """As many heads as fill the GPU, each with more granules than a warp takes in sixteen steps; a few of them are checked."""
    Z, H, L, block = 300, 2, 1203, 64
    lengths = (L - torch.arange(Z) * 7 % 400).int().cuda()
    layout = layouts.dense(1, -(-L // block))
    layout[0, :, 3] = 0
    slots = -(-L // 64)
    cache, pages = Guarded(Z * slots, H, D), table(Z, slots, Z * slots)
    k, v = tokens(Z, H, L, D, dtype), tokens(Z, H, L, D, dtype, 1)
    zero = torch.zeros(Z, dtype=torch.int32, device='cuda')
    cache.write(k, v, pages, zero, lengths)
    del k, v
    q = queries(Z, H * G, T, D, dtype)
    got = SparseSelfAttention(layout=layout, block=block).decode(q, cache, pages, lengths)
    some = torch.tensor([0, 1, 57, 58, 123, 299], device='cuda')
    kk, vv = cache.read(pages[some], zero[some], L, lengths[some], dtype=torch.float32)
    assert_decoded(got[some], q[some], kk, vv, torch.ones(6, L, dtype=torch.bool), lengths[some], layout, block, D ** -0.5)
    alone = SparseSelfAttention(layout=layout, block=block).decode(q[some], cache, pages[some], lengths[some])
    assert_decoded(alone, q[some], kk, vv, torch.ones(6, L, dtype=torch.bool), lengths[some], layout, block, D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('H', [1, 74, 84, 98, 118, 148, 197, 296, 400])
def test_every_size_of_cluster(H):
    """The number of heads decides how many blocks of threads share a row: 8, 8, 7, 6, 5, 4, 3, 2 and 1 of them."""
    L, D, block = 700, 64, 32
    lengths = ints(L)
    cache, pages, k, v = filled(1, H, L, D, 64, torch.float16, lengths)
    layout = layouts.dense(1, -(-L // block))
    q = queries(1, H, 3, D, torch.float16)
    got = SparseSelfAttention(layout=layout, block=block).decode(q, cache, pages, lengths)
    some = list(range(0, H, max(1, H // 9)))
    assert_decoded(got[:, some], q[:, some], k[:, some], v[:, some], torch.ones(1, L, dtype=torch.bool), lengths, layout, block, D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_scales_and_scores_that_grow_along_the_row(dtype):
    """Later keys outweigh earlier ones by far, and later values are larger (and the other way round)."""
    Z, L, D = 2, 700, 128
    grow = torch.exp2(torch.arange(L, device='cuda') / 50 - 6)[:, None]
    cache, pages = Guarded(Z * 11, 1, D, page=64), table(Z, 11, Z * 11)
    k, v = tokens(Z, 1, L, D, torch.bfloat16), tokens(Z, 1, L, D, torch.bfloat16, 1)
    k, v = k.float().clamp(-4, 4) * grow / 16, v.float().clamp(-4, 4) * grow
    k[1], v[1] = k[1].flip(-2), v[1].flip(-2)
    v[:, :, ::3] *= 1e-3
    lengths, zero = ints(L, L), ints(0, 0)
    cache.write(k.to(dtype), v.to(dtype), pages, zero)
    kk, vv = cache.read(pages, zero, L, dtype=torch.float32)
    q = queries(Z, 8, 1, D, dtype)
    layout = layouts.dense(1, 6)
    got = SparseSelfAttention(layout=layout, block=128).decode(q, cache, pages, lengths)
    assert_decoded(got, q, kk, vv, torch.ones(Z, L, dtype=torch.bool), lengths, layout, 128, D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('L', [2, 3, 17, 64, 200])
@pytest.mark.parametrize('G', [1, 8])
def test_one_value_outweighs_the_others(dtype, D, L, G):
    """Values of very different size, by token and by channel: small results beside large terms that carry the codes' offset."""
    Z, H = 8, 4
    g = torch.Generator(device='cuda').manual_seed(L)
    def randn(*s): return torch.randn(s, generator=g, device='cuda')
    k = randn(Z, H, L, D).to(dtype)
    v = (randn(Z, H, L, D) * torch.exp2(5 * randn(Z, H, L, 1)) * torch.exp2(3 * randn(Z, H, L, D))).clamp(-30000, 30000).to(dtype)
    slots = -(-L // 64)
    cache, pages = Guarded(Z * slots, H, D), table(Z, slots, Z * slots)
    zero = torch.zeros(Z, dtype=torch.int32, device='cuda')
    cache.write(k, v, pages, zero)
    kk, vv = cache.read(pages, zero, L, dtype=torch.float32)
    q, layout = (randn(Z, H * G, 1, D) * 0.01).to(dtype), layouts.dense(1, 4)
    got = SparseSelfAttention(layout=layout, block=64).decode(q, cache, pages, zero + L)
    assert_decoded(got, q, kk, vv, torch.ones(Z, L, dtype=torch.bool), zero + L, layout, 64, D ** -0.5)


@pytest.mark.gpu
def test_missing_pages_lengths_behind_the_layout_and_the_table():
    Z, H, L, D, page = 4, 2, 256, 64, 32
    lengths = ints(256, 200, 300, 256)
    cache, pages, k, v = filled(Z, H, L, D, page, torch.float16, lengths)
    there = torch.ones(Z, L, dtype=torch.bool)
    for z, slot, number in ((0, 0, -1), (0, 3, 10 ** 6), (1, 6, 2 ** 31 - 1), (3, 2, -2 ** 31)):
        pages[z, slot] = number
        there[z, slot * page:(slot + 1) * page] = False
    pages[3] = -1                                       # nothing at all
    there[3] = False
    layout = layouts.dense(H, 8)                        # (300 lies behind the layout, and behind the table)
    q = queries(Z, H, 2, D, torch.float16)
    got = SparseSelfAttention(layout=layout, block=32).decode(q, cache, pages, lengths)
    assert_decoded(got, q, k, v, there, lengths, layout, 32, D ** -0.5)
    assert not bool(got[2].any()) and not bool(got[3].any())
    # a table that ends in front of the newest tokens: what it holds is seen
    layout = layouts.dense(1, 16)
    got = SparseSelfAttention(layout=layout, block=32).decode(q, cache, pages, lengths)
    assert_decoded(got, q, k, v, there, lengths, layout, 32, D ** -0.5)


@pytest.mark.gpu
def test_non_finite_values_reach_those_who_see_them():
    H, L, D = 1, 64, 64
    cache, pages, start = Guarded(4, H, D, page=16), table(1, 4, 4), ints(0)
    k, v = tokens(1, H, L, D, torch.bfloat16), tokens(1, H, L, D, torch.bfloat16, 1)
    k[0, 0, 20, 3], v[0, 0, 40, 40] = float('nan'), float('inf')
    cache.write(k, v, pages, start)
    layout = torch.zeros((1, 4, 4), dtype=torch.int64)
    layout[0, 3, 0] = layout[0, 3, 3] = layout[0, 2, 0] = layout[0, 2, 2] = layout[0, 1, 0] = layout[0, 1, 1] = 1
    attn = SparseSelfAttention(layout=layout, block=16)
    q = queries(1, H, 1, D, torch.bfloat16)

    def at(n):
        return attn.decode(q, cache, pages, ints(n))[0, 0, 0].isnan()

    assert not bool(at(20).any())                       # position 19: the NaN key is the next token
    assert bool(at(21).all()) and bool(at(32).all())    # its own position, and later ones of its block
    assert not bool(at(40).any())
    nan = at(41)                                        # the infinite value: its group of 32 channels alone
    assert bool(nan[32:].all()) and not bool(nan[:32].any())
    assert not bool(at(64).any())                       # rows that see neither block
    # several queries in one tile: only those that stand behind the value
    got = attn.decode(queries(1, H, 8, D, torch.bfloat16), cache, pages, ints(44))[0, 0].isnan()
    assert not bool(got[:4].any()) and bool(got[4:, 32:].all()) and not bool(got[:, :32].any())
    q[0, 0, 0, 5] = float('nan')
    assert bool(at(64).all())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('T', [1, 5])
def test_scales_of_either_sign_and_powers_of_two(dtype, T):
    Z, H, L, D = 2, 2, 150, 64
    lengths = ints(150, 77)
    cache, pages, k, v = filled(Z, H, L, D, 32, dtype, lengths)
    layout = layouts.dense(1, 5)
    attn, there = SparseSelfAttention(layout=layout, block=32), torch.ones(Z, L, dtype=torch.bool)
    q = queries(Z, 2 * H, T, D, dtype)
    for scale in (-0.2, 0.0, 3.0, 1e-3):
        assert_decoded(attn.decode(q, cache, pages, lengths, scale=scale), q, k, v, there, lengths, layout, 32, scale)
    # a power of two between the query and the scale, or on the values, changes no bit
    want = attn.decode(q, cache, pages, lengths)
    if dtype == torch.bfloat16:
        assert torch.equal(attn.decode(q * 2.0 ** -40, cache, pages, lengths, scale=D ** -0.5 * 2.0 ** 40), want)
        assert torch.equal(attn.decode(q * 2.0 ** 30, cache, pages, lengths, scale=D ** -0.5 * 2.0 ** -30), want)
        small, far = Guarded(cache.num_pages, H, D, page=32), torch.zeros(Z, dtype=torch.int32, device='cuda')
        for shift in (2.0 ** -50, 2.0 ** 50):
            small.write(k.to(dtype), (v * shift).to(dtype), pages, far, lengths)
            kk, vv = small.read(pages, far, L, lengths, dtype=torch.float32)
            assert_decoded(attn.decode(q, small, pages, lengths), q, kk, vv, there, lengths, layout, 32, D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('size', [2.0 ** 100, 2.0 ** 124, 2.0 ** -95])
def test_the_ends_of_bf16(D, size):
    lengths, H, L = ints(90), 2, 90
    cache, pages, zero = Guarded(3, H, D, page=32), table(1, 3, 3), ints(0)
    k, v = tokens(1, H, L, D, torch.bfloat16), (tokens(1, H, L, D, torch.bfloat16, 1).clamp(-7, 7) * size).to(torch.bfloat16)
    cache.write(k, v, pages, zero)
    kk, vv = cache.read(pages, zero, L, dtype=torch.float32)
    layout, there = layouts.dense(1, 3), torch.ones(1, L, dtype=torch.bool)
    for G in (1, 4, 8):
        q = queries(1, G * H, 1, D, torch.bfloat16)
        got = SparseSelfAttention(layout=layout, block=32).decode(q, cache, pages, lengths)
        assert_decoded(got, q, kk, vv, there, lengths, layout, 32, D ** -0.5)


@pytest.mark.gpu
def test_a_layout_without_blocks():
    cache, pages, _, _ = filled(1, 2, 40, 64, 16, torch.float16, ints(40))
    q = queries(1, 2, 1, 64, torch.float16)
    layout = torch.zeros((2, 3, 3), dtype=torch.int64)
    assert not bool(SparseSelfAttention(layout=layout, block=16).decode(q, cache, pages, ints(40)).any())
    with pytest.raises(ValueError):
        SparseSelfAttention(layout=layout[:1, :0, :0], block=16).decode(q, cache, pages, ints(40))


@pytest.mark.gpu
def test_pages_shared_by_sequences():
    """One prompt's pages in every sequence's table (a row expanded over the batch), read only."""
    H, L, D = 2, 100, 64
    cache, pages, k, v = filled(1, H, L, D, 32, torch.float16, ints(L))
    shared, lengths = pages.expand(3, -1), ints(100, 64, 33)
    q, layout = queries(3, H, 1, D, torch.float16), layouts.dense(1, 4)
    got = SparseSelfAttention(layout=layout, block=32).decode(q, cache, shared, lengths)
    assert_decoded(got, q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1), torch.ones(3, L, dtype=torch.bool), lengths, layout, 32, D ** -0.5)
    kk, _ = cache.read(shared, ints(0, 5, 50), 50, dtype=torch.float32)
    assert torch.equal(kk[2], k[0, :, 50:]) and torch.equal(kk[1], k[0, :, 5:55])


@pytest.mark.gpu
def test_copies_and_pickles_of_a_cache():
    import copy
    import pickle
    cache, pages, k, v = filled(1, 2, 40, 64, 16, torch.float16, ints(40))
    plain = KVCache(cache.data.size(0), 2, 64, page=16)
    plain.data.copy_(cache.data)
    attn, q = SparseSelfAttention(layout=layouts.dense(1, 3), block=16), queries(1, 2, 1, 64, torch.float16)
    want = attn.decode(q, plain, pages, ints(40))
    for other in (copy.deepcopy(plain), pickle.loads(pickle.dumps(plain))):
        assert torch.equal(copy.deepcopy(attn).decode(q, other, pages, ints(40)), want)
        other.data.fill_(0)
        assert torch.equal(attn.decode(q, plain, pages, ints(40)), want)


@pytest.mark.gpu
def test_zero_and_tiny_values():
    H, D = 2, 64
    cache, pages = Guarded(4, H, D), table(1, 4, 4)
    zero = torch.zeros((1, H, 100, D), device='cuda', dtype=torch.bfloat16)
    v = tokens(1, H, 100, D, torch.bfloat16, 1) * 2.0 ** -60
    cache.write(zero, v, pages, ints(0))
    _, vv = cache.read(pages, ints(0), 100, dtype=torch.float32)
    layout = layouts.dense(1, 2)
    attn = SparseSelfAttention(layout=layout, block=64)
    q = queries(1, H, 1, D, torch.bfloat16)
    got = attn.decode(q, cache, pages, ints(100))
    assert_decoded(got, q, zero.float(), vv, torch.ones(1, 100, dtype=torch.bool), ints(100), layout, 64, D ** -0.5)
    cache.write(zero, zero, pages, ints(0))
    assert not bool(attn.decode(q, cache, pages, ints(100)).any())
    assert not bool(attn.decode(q * 0, cache, pages, ints(100)).any())


@pytest.mark.gpu
@pytest.mark.parametrize('order', ['sequence first', 'offset', 'transposed', 'expanded'])
def test_orders_of_the_query(order):
    lengths = ints(100, 70)
    cache, pages, k, v = filled(2, 2, 100, 64, 64, torch.float16, lengths)
    q = tokens(2, 4, 3, 64, torch.float16, 5, order)
    layout = layouts.dense(1, 7)
    attn = SparseSelfAttention(layout=layout, block=16)
    assert torch.equal(attn.decode(q, cache, pages, lengths), attn.decode(q.contiguous(), cache, pages, lengths))
    wide = torch.cat((pages, pages), 1)[:, :pages.size(1)]                     # a table with gaps between its rows
    assert torch.equal(attn.decode(q, cache, wide, lengths), attn.decode(q, cache, pages, lengths))


@pytest.mark.gpu
def test_addresses_past_32_bits():
    D, H, page = 128, 8, 256
    n = (5 << 30) // (H * _lib.lib().bsp_cache_page_bytes(page, D))
    cache = KVCache(n, H, D, page=page)
    pages, lengths = ints(n - 1, 0, n - 2, n // 2).view(2, 2), ints(500, 400)
    k, v = tokens(2, H, 500, D, torch.float16), tokens(2, H, 500, D, torch.float16, 1)
    cache.write(k, v, pages, ints(0, 0), lengths)
    kk, vv = cache.read(pages, ints(0, 0), 500, dtype=torch.float32)
    q, layout = queries(2, H, 1, D, torch.float16), layouts.dense(1, 4)
    got = SparseSelfAttention(layout=layout, block=128).decode(q, cache, pages, lengths)
    assert_decoded(got, q, kk, vv, torch.ones(2, 500, dtype=torch.bool), lengths, layout, 128, D ** -0.5)


@pytest.mark.gpu
def test_captured_graphs_follow_growing_sequences():
    """Two graphs over one cache, replayed in turn and on two streams, against eager calls."""
    Z, H, L, D = 3, 4, 200, 64
    lengths = ints(100, 31, 64)
    cache, pages, _, _ = filled(Z, H, L, D, 16, torch.float16, lengths)
    attn = SparseSelfAttention(layout=layout_of('fixed', H, 13), block=16)
    new = [tokens(Z, H, 1, D, torch.float16, 20 + i) for i in range(3)]
    attn.decode(new[0], cache, pages, lengths)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.write(new[1], new[2], pages, lengths)
            out = attn.decode(new[0], cache, pages, lengths + 1)
        graphs.append((graph, out))
    twin, _, _, _ = filled(Z, H, L, D, 16, torch.float16, lengths)
    for step in range(20):
        for i, x in enumerate(new):
            x.copy_(tokens(Z, H, 1, D, torch.float16, 100 + 3 * step + i))
        graph, out = graphs[step % 2]
        graph.replay()
        twin.write(new[1], new[2], pages, lengths)
        assert torch.equal(out, attn.decode(new[0], twin, pages, lengths + 1))
        lengths.add_(1)
    torch.cuda.synchronize()
    for graph, out in graphs:
        with torch.cuda.stream(torch.cuda.Stream()):
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], graphs[1][1])


@pytest.mark.gpu
def test_a_configuration_and_changed_attributes():
    Z, H, L, D = 2, 4, 256, 64
    lengths = ints(256, 133)
    cache, pages, k, v = filled(Z, H, L, D, 64, torch.float16, lengths)
    q, there = queries(Z, H, 1, D, torch.float16), torch.ones(Z, L, dtype=torch.bool)
    attn = SparseSelfAttention(SparsityConfig(block=16, stride=64))
    layout = layouts.fixed(H, 16, 4)
    assert_decoded(attn.decode(q, cache, pages, lengths), q, k, v, there, lengths, layout, 16, D ** -0.5)
    attn = SparseSelfAttention(layout=layout, block=16)
    attn.decode(q, cache, pages, lengths)
    attn.layout = layouts.causal_band(H, 16, 2)
    assert_decoded(attn.decode(q, cache, pages, lengths), q, k, v, there, lengths, attn.layout, 16, D ** -0.5)
    attn.layout, attn.block = layouts.dense(1, 4), 64
    assert_decoded(attn.decode(q, cache, pages, lengths), q, k, v, there, lengths, attn.layout, 64, D ** -0.5)
    attn.layout = layout.cuda()                         # a layout on the device
    attn.block = 16
    assert_decoded(attn.decode(q, cache, pages, lengths), q, k, v, there, lengths, layout, 16, D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('config', [dict(), dict(stride=128, numverts=3), dict(attention='bidirectional', stride=32), dict(mode='dense')])
@pytest.mark.parametrize('page', [16, 32])
def test_a_configuration_and_a_table_that_grows_page_by_page(config, page):
    """Widths that fill no window of the layout among them; lengths behind the table see nothing."""
    H, D, most = 2, 64, 12
    config = SparsityConfig(block=16, **config)
    attn, windows = SparseSelfAttention(config), -(-most * page // config.stride)
    layout = attn.get_layout(H, windows * config.stride)
    cache, pages, k, v = filled(3, H, most * page, D, page, torch.float16, ints(*[most * page] * 3))
    q, there = queries(3, H, 2, D, torch.float16), torch.ones(3, most * page, dtype=torch.bool)
    for slots in range(1, most + 1):
        n = slots * page
        lengths = ints(n, max(0, n - 7), n + 50)
        got = attn.decode(q, cache, pages[:, :slots], lengths)
        assert_decoded(got, q, k[:, :, :n], v[:, :, :n], there[:, :n], lengths, layout[:, :n // 16, :n // 16], 16, D ** -0.5)
        assert not bool(got[2].any())
    assert not bool(attn.decode(q, cache, pages[:, :0], lengths).any())


@pytest.mark.gpu
def test_a_growing_table_builds_few_layouts():
    attn = SparseSelfAttention(SparsityConfig(block=16, stride=32))
    cache, q = KVCache(4, 1, 64, page=16), queries(1, 1, 1, 64, torch.float16)
    x = tokens(1, 1, 64, 64, torch.float16)
    cache.write(x, x, ints(0, 1, 2, 3)[None], ints(0))
    pages = ints(0, 1, 2, 3, *[-1] * 396)[None]
    before, want = tables.CACHE_STATS['misses'], attn.decode(q, cache, pages[:, :4], ints(60))
    for slots in range(4, 401):
        assert torch.equal(attn.decode(q, cache, pages[:, :slots], ints(60)), want), slots
        assert not bool(attn.decode(q, cache, pages[:, :slots], ints(16 * slots + 1)).any())    # behind the table
    assert tables.CACHE_STATS['misses'] - before <= 8 * 8


@pytest.mark.gpu
@pytest.mark.parametrize('kind', ['fixed', 'band'])
def test_rotated_written_and_decoded_as_the_whole_sequence(kind):
    """A prompt and then token after token, against forward() on the whole sequence with the cache's values."""
    from tests.util import assert_close
    Z, H, L, D, prompt, block = 2, 4, 128, 64, 100, 16
    layout = layout_of(kind, H, L // block)
    attn, rotary = SparseSelfAttention(layout=layout, block=block), Rotary(D, (16, 16))
    q, k, v = (tokens(Z, H, L, D, torch.float16, i).clamp(-3, 3) for i in range(3))
    positions = torch.stack([torch.arange(L, device='cuda') // 10, torch.arange(L, device='cuda') % 10]).int()
    cache, pages = Guarded(Z * 2, H, D), table(Z, 2, Z * 2)
    lengths = ints(0, 0)
    outs = []
    for a, b in [(0, prompt)] + [(t, t + 1) for t in range(prompt, 120)] + [(120, 128)]:
        qr, kr = rotary(q[:, :, a:b], k[:, :, a:b], positions[:, a:b])
        cache.write(kr, v[:, :, a:b], pages, lengths)
        lengths += b - a
        outs.append(attn.decode(qr, cache, pages, lengths))
    kk, vv = cache.read(pages, ints(0, 0), L)
    mask = torch.ones(L, L, device='cuda').tril()
    want = attn(rotary(q, positions=positions), kk, vv, attn_mask=mask)
    assert_close(torch.cat(outs, 2), want, kind)


@pytest.mark.gpu
def test_empty_calls():
    cache, pages, k, v = filled(2, 2, 40, 64, 16, torch.float16, ints(40, 7))
    attn = SparseSelfAttention(layout=layouts.dense(1, 3), block=16)
    for shape in ((2, 2, 0, 64), (2, 0, 1, 64)):
        assert attn.decode(torch.empty(shape, device='cuda', dtype=torch.float16), cache, pages, ints(40, 7)).shape == shape
    none = attn.decode(torch.empty((0, 2, 1, 64), device='cuda', dtype=torch.float16), cache, pages[:0], ints())
    assert none.shape == (0, 2, 1, 64)
    assert not bool(attn.decode(queries(2, 2, 1, 64, torch.float16), cache, pages[:, :0], ints(40, 7)).any())


@pytest.mark.gpu
def test_calls_one_after_the_other_see_each_other():
    """Nothing waits between them: every call finds what the calls before it have left, other operations among them."""
    from tests.test_cache import same, stands_for
    Z, H, D, n = 8, 4, 64, 300
    cache, pages = Guarded(Z * 5, H, D), table(Z, 5, Z * 5)
    attn, rotary = SparseSelfAttention(layout=layouts.dense(1, 5), block=64), Rotary(D)
    base, start = tokens(Z, H, 1, D, torch.float16), torch.zeros(Z, dtype=torch.int32, device='cuda')
    got, keys, outs, wants = [], [], [], []
    for i in range(n):
        k = rotary(base * (1 + i % 7), positions=start[:1] + i)
        cache.write(k, k, pages, start)
        keys.append(k)
        got.append(cache.read(pages, start, 1, dtype=torch.float32)[0])
        start.add_(1)
        outs.append(attn.decode(k, cache, pages, start))
        k = k + 0                                       # (memory of earlier results is used again)
    torch.cuda.synchronize()
    again = torch.zeros_like(start)
    for i in range(n):
        assert same(got[i], stands_for(keys[i])), i
        again.add_(1)
        if i % 37 == 0 or i == n - 1:
            wants.append(attn.decode(keys[i], cache, pages, again))
            torch.cuda.synchronize()
            assert torch.equal(wants[-1], outs[i]), i


# ---- refusals ----------------------------------------------------------------------------------
def test_the_library_rejects_bad_arguments():
    L = _lib.lib()
    m = tables.build_meta(torch.ones((2, 3, 3), dtype=torch.long))
    wide = tables.build_meta(torch.ones((2, 3, 4), dtype=torch.long))
    bad_magic = m.hdr.clone()
    bad_magic[0] = 0

    def call(q=16, o=16, dtype=_lib.F16, Z=1, Hq=4, Hk=2, T=1, D=64, data=16, n=1, page=64, pages=16, slots=1, lengths=16, block=16,
             hdr=m.hdr, meta=16):
        return L.bsp_cache_attn(q, o, dtype, Z, Hq, Hk, T, D, 64, 64, 64, 64, 64, 64, data, n, page, pages, 1, slots, lengths, block,
                                None if hdr is None else hdr.data_ptr(), meta, 1.0, None)

    for bad in (dict(dtype=_lib.F32), dict(Z=-1), dict(T=-1), dict(Hk=0), dict(Hq=3), dict(Hq=4, Hk=4), dict(page=40), dict(block=48),
                dict(hdr=None), dict(meta=None), dict(hdr=bad_magic), dict(hdr=wide.hdr), dict(q=None), dict(o=None), dict(lengths=None),
                dict(pages=None), dict(data=None), dict(data=8), dict(n=-1), dict(slots=-1)):
        assert call(**bad) == _lib.ERR_INVALID, bad
    for bad in (dict(D=96), dict(page=1024, slots=1 << 22), dict(Z=1 << 30, T=1 << 10), dict(T=1 << 30, Hq=1 << 10)):
        assert call(**bad) == _lib.ERR_UNSUPPORTED, bad
    assert call(Z=0, q=None, o=None, lengths=None) == _lib.OK


@pytest.mark.gpu
def test_bad_calls():
    lengths = ints(40, 7)
    cache, pages, _, _ = filled(2, 2, 40, 64, 16, torch.float16, lengths)
    attn = SparseSelfAttention(layout=layouts.dense(1, 3), block=16)
    q = queries(2, 4, 1, 64, torch.float16)
    for args in ((q.float(), cache, pages, lengths), (q[:, :3], cache, pages, lengths), (q[..., :32], cache, pages, lengths),
                 (q[0], cache, pages, lengths), (q, cache, pages.long(), lengths), (q, cache, pages[:1], lengths),
                 (q, cache, pages, lengths[:1]), (q, cache, pages, lengths.long()), (q, cache, pages[0], lengths)):
        with pytest.raises(ValueError):
            attn.decode(*args)
    for args in ((q.cpu(), cache, pages, lengths), (q, cache, pages.cpu(), lengths), (q, cache, pages, lengths.cpu())):
        with pytest.raises(RuntimeError):
            attn.decode(*args)
    with pytest.raises(NotImplementedError, match='no_grad'):
        attn.decode(q.clone().requires_grad_(), cache, pages, lengths)
    with torch.no_grad():
        attn.decode(q.clone().requires_grad_(), cache, pages, lengths)
    with pytest.raises(ValueError, match='heads'):
        SparseSelfAttention(layout=layouts.dense(3, 3), block=16).decode(q, cache, pages, lengths)
    with pytest.raises(RuntimeError, match='trace'):
        torch.jit.trace(lambda x: attn.decode(x, cache, pages, lengths), (q,), check_trace=False)


def test_the_library_rejects_rows_that_a_layout_does_not_have():
    L, m = _lib.lib(), tables.build_meta(torch.ones((2, 3, 3), dtype=torch.long))
    for rows in (-1, 4):
        assert L.bsp_cache_attn_rows(16, 16, _lib.F16, 1, 4, 2, 1, 64, 64, 64, 64, 64, 64, 64, 16, 1, 64, 16, 1, 1, 16, 16, m.hdr.data_ptr(), 16,
                                     rows, 1.0, None) == _lib.ERR_INVALID and b'rows' in L.bsp_last_error()
