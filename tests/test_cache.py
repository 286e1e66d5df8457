"""The 4-bit cache: what is written reads back as s * code, to the bit, and nothing else changes.

Codes and scales are whole decisions, so there is no tolerance: the oracle forms s = bf16(max |x| / 7) (one division
in 32 bits, one rounding) and round-half-even(x / s) with the quotient in 64 bits.  s has 8 significant bits and x at
most 11, so a quotient that is no tie is over 2^-13 away from one and 64 bits decide as exact arithmetic would;
s * code has at most 12 bits and is exact in 32, and rounded once to the type that is read.
"""
import pytest
import torch

from torch_blocksparse_b200 import KVCache, _lib

DTYPES = [torch.float16, torch.bfloat16]


def stands_for(x):
    """The values that the cache holds in place of x, in 32 bits."""
    g = x.detach().cpu().float().unflatten(-1, (-1, 32))
    amax = g.abs().amax(-1, keepdim=True)
    s = (amax / 7).bfloat16().double()
    ok = amax < float('inf')
    c = torch.where(s > 0, torch.round(g.double() / torch.where(s > 0, s, 1.0)), 0.0).clamp(-8, 7)
    return torch.where(ok, (s * torch.where(ok, c, 0.0)).float(), float('nan')).flatten(-2)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float().cpu(), 12345.0), torch.nan_to_num(b.float().cpu(), 12345.0))


def tokens(Z, H, T, D, dtype, seed=0, order='contiguous'):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn((Z, H, T, D), generator=g, device='cuda') * torch.exp(2 * torch.randn((Z, H, T, 1), generator=g, device='cuda'))
    x = x.to(dtype)
    if order == 'sequence first':
        return x.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    if order == 'offset':
        return torch.cat((x[..., :1], x, x[..., :2]), -1)[..., 1:D + 1]
    if order == 'transposed':
        return x.transpose(2, 3).contiguous().transpose(2, 3)
    if order == 'expanded':
        return x[:, :1].expand(Z, H, T, D)
    return x


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


def table(Z, slots, num_pages, seed=0):
    return torch.randperm(num_pages, generator=torch.Generator().manual_seed(seed))[:Z * slots].view(Z, slots).int().cuda()


class Guarded(KVCache):
    """A cache whose data lies between margins; every byte starts as 0xFF (scales that are NaN)."""

    def __init__(self, num_pages, *args, **kw):
        super().__init__(num_pages + 2, *args, **kw)
        self.whole = self.data.fill_(255)
        self.data = self.whole[1:-1]

    def check(self):
        assert bool((self.whole[0] == 255).all()) and bool((self.whole[-1] == 255).all()), 'written outside the cache'


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('page', [16, 64, 256])
@pytest.mark.parametrize('T,starts', [(1, (0, 15, 200)), (2, (15, 3, 16)), (16, (0, 1, 48)), (17, (15, 0, 31)), (77, (5, 64, 16)),
                                      (300, (0, 16, 9))])
def test_written_and_read(dtype, D, page, T, starts):
    H, slots = 3, -(-(T + 200) // page)
    cache = Guarded(3 * slots + 2, H, D, page=page)
    pages, start = table(3, slots, 3 * slots + 2), ints(*starts)
    k, v = tokens(3, H, T, D, dtype), tokens(3, H, T, D, dtype, 1)
    cache.write(k, v, pages, start)
    cache.check()
    for out in (torch.float32, torch.float16, torch.bfloat16):
        gk, gv = cache.read(pages, start, T, dtype=out)
        assert gk.dtype == out and same(gk, stands_for(k).to(out)) and same(gv, stands_for(v).to(out))
    # as many tokens again, one by one: the same bytes
    other = Guarded(3 * slots + 2, H, D, page=page)
    for t in range(min(T, 40)):
        other.write(k[:, :, t:t + 1], v[:, :, t:t + 1], pages, start + t)
    if T <= 40:
        assert torch.equal(other.data, cache.data)
    # a stretch from the middle
    gk, gv = cache.read(pages, start + T // 2, T - T // 2)
    assert same(gk, stands_for(k)[:, :, T // 2:].half())


@pytest.mark.gpu
@pytest.mark.parametrize('order', ['sequence first', 'offset', 'transposed', 'expanded'])
@pytest.mark.parametrize('D', [64, 128])
def test_orders_in_memory(order, D):
    cache, pages = Guarded(8, 4, D), table(2, 4, 8)
    k, v = tokens(2, 4, 33, D, torch.bfloat16, 3, order), tokens(2, 4, 33, D, torch.bfloat16, 4)
    cache.write(k, v, pages, ints(7, 160))
    gk, gv = cache.read(pages, ints(7, 160), 33, dtype=torch.float32)
    assert same(gk, stands_for(k)) and same(gv, stands_for(v))


@pytest.mark.gpu
def test_a_padded_batch_leaves_the_rest_as_it_was():
    D, H, T = 128, 2, 50
    cache, pages = Guarded(12, H, D, page=32), table(4, 3, 12)
    first = tokens(4, H, 96, D, torch.float16, 9)
    cache.write(first, first, pages, ints(0, 0, 0, 0))
    before = cache.data.clone()
    k, v = tokens(4, H, T, D, torch.float16), tokens(4, H, T, D, torch.float16, 1)
    start, count = ints(0, 21, 46, 30), ints(0, 13, 50, -4)
    k[1, :, 13:] = float('nan')                        # padding may hold anything
    cache.write(k, v, pages, start, count)
    cache.check()
    want = stands_for(first)
    for z, (s, n) in enumerate(zip(start.tolist(), count.tolist())):
        if n > 0:
            want[z, :, s:s + n] = stands_for(k)[z, :, :n]
    assert same(cache.read(pages, ints(0, 0, 0, 0), 96, dtype=torch.float32)[0], want)
    for z in (0, 3):
        assert torch.equal(cache.data[pages[z].long()], before[pages[z].long()])
    # reading stops at the count as well: zeros behind it
    got, _ = cache.read(pages, start, T, count, dtype=torch.float32)
    for z, (s, n) in enumerate(zip(start.tolist(), count.tolist())):
        n = max(0, n)
        assert same(got[z, :, :n], want[z, :, s:s + n]) and not bool(got[z, :, n:].any())


@pytest.mark.gpu
def test_tokens_without_a_place():
    """No page, ids out of range, positions in front of the sequence and behind the table."""
    D, H, T = 64, 2, 70
    cache = Guarded(4, H, D, page=16)
    pages = ints(0, -1, 2, 4, 1, 2 ** 31 - 1, -2 ** 31, 3).view(2, 4)
    k, v = tokens(2, H, T, D, torch.bfloat16), tokens(2, H, T, D, torch.bfloat16, 1)
    start = ints(-5, 2)
    cache.write(k, v, pages, start)
    cache.check()
    want = torch.zeros_like(stands_for(k))
    for z in range(2):
        for t in range(T):
            pos = int(start[z]) + t
            if 0 <= pos < 64 and 0 <= int(pages[z, pos // 16]) < 4:
                want[z, :, t] = stands_for(k)[z, :, t]
    assert same(cache.read(pages, start, T, dtype=torch.float32)[0], want)
    for far in (2 ** 31 - 1, -2 ** 31):
        before = cache.data.clone()
        cache.write(k, v, pages, ints(far, far))
        assert torch.equal(cache.data, before) and not bool(cache.read(pages, ints(far, far), T)[0].any())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_every_value_against_many_scales(dtype):
    """Each of the type's positive and negative values as one of a group whose largest is another, ties among them."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    every = every[every.isfinite()]
    g = torch.Generator().manual_seed(0)
    tops = [7.0, 3.5, 1.0, 7 * 2.0 ** -10, 448.0, 1.09375, 0.8203125, 113.0, 60000.0, 2.0 ** -14, 3 * 2.0 ** -24]
    tops += torch.randn(40, generator=g).abs().tolist()
    if dtype == torch.bfloat16:
        tops += [3e38, 1e-38, 1e-30, 9e-41, 1e-20]
    rows = []
    for top in torch.tensor(tops).to(dtype):
        x = every[every.abs() <= top]
        x = x[torch.randperm(x.numel(), generator=g)][:31 * 4 * 256]
        x = torch.nn.functional.pad(x, (0, -x.numel() % 124)).view(-1, 4, 31)
        rows.append(torch.cat((x, top.expand(x.size(0), 4, 1)), -1).flatten(1))
    x = torch.cat(rows)[None, None].cuda()             # [1, 1, T, 128]
    T = x.size(2)
    cache = KVCache(-(-T // 64), 1, 128)
    pages = table(1, cache.num_pages, cache.num_pages)
    cache.write(x, -x, pages, ints(0))
    k, v = cache.read(pages, ints(0), T, dtype=torch.float32)
    assert same(k, stands_for(x)) and same(v, stands_for(-x))


@pytest.mark.gpu
def test_non_finite_values_stay_in_their_group():
    cache, pages = KVCache(2, 1, 128), ints(1, 0).view(1, 2)
    k = tokens(1, 1, 40, 128, torch.bfloat16)
    want = stands_for(k)
    k[0, 0, 3, 33], k[0, 0, 17, 127], k[0, 0, 30, 0] = float('nan'), float('inf'), float('-inf')
    cache.write(k, k, pages, ints(0))
    want[0, 0, 3, 32:64] = want[0, 0, 17, 96:] = want[0, 0, 30, :32] = float('nan')
    for got in cache.read(pages, ints(0), 40, dtype=torch.float32):
        assert same(got, want)


@pytest.mark.gpu
def test_addresses_past_32_bits():
    D, H, page = 128, 8, 256
    n = (5 << 30) // (H * _lib.lib().bsp_cache_page_bytes(page, D))
    cache = KVCache(n, H, D, page=page)
    assert cache.data.numel() > 2 ** 32
    pages = ints(n - 1, n // 2, 1, n - 2).view(2, 2)
    k, v = tokens(2, H, 300, D, torch.float16), tokens(2, H, 300, D, torch.float16, 1)
    cache.write(k, v, pages, ints(100, 3))
    gk, gv = cache.read(pages, ints(100, 3), 300, dtype=torch.float32)
    assert same(gk, stands_for(k)) and same(gv, stands_for(v))
    untouched = cache.data[:4].clone()
    untouched[1] = 0
    assert not bool(untouched.any())


@pytest.mark.gpu
def test_captured_with_moving_starts_and_on_another_stream():
    cache, pages = KVCache(8, 2, 64, page=16), table(2, 4, 8)
    k, v = tokens(2, 2, 5, 64, torch.float16), tokens(2, 2, 5, 64, torch.float16, 1)
    start = ints(0, 30)
    cache.write(k, v, pages, start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(k, v, pages, start)
        got = cache.read(pages, start, 5, dtype=torch.float32)
        start.add_(7)
    for seed in range(2, 5):
        k.copy_(tokens(2, 2, 5, 64, torch.float16, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert same(got[0], stands_for(k))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.write(v, k, pages, start)
        got = cache.read(pages, start, 5, dtype=torch.float32)
    side.synchronize()
    assert same(got[0], stands_for(v)) and same(got[1], stands_for(k))


@pytest.mark.gpu
def test_empty_calls():
    cache, pages = KVCache(2, 1, 64), ints(0, 1).view(1, 2)
    none = torch.empty((1, 1, 0, 64), device='cuda', dtype=torch.float16)
    cache.write(none, none, pages, ints(0))
    assert cache.read(pages, ints(0), 0)[0].shape == (1, 1, 0, 64)
    assert cache.read(pages[:0], ints(), 3)[0].shape == (0, 1, 3, 64)
    one = torch.ones((1, 1, 4, 64), device='cuda', dtype=torch.float16)
    cache.write(one, one, pages[:, :0], ints(0))       # a table without a slot
    assert not bool(cache.data.any())
    empty = KVCache(0, 1, 64)
    empty.write(one, one, pages, ints(0))
    assert not bool(empty.read(pages, ints(0), 4)[0].any())


# ---- refusals ----------------------------------------------------------------------------------
def test_bad_constructions():
    with pytest.raises(NotImplementedError):
        KVCache(1, 1, 96)
    for page in (0, 8, 48, 2048):
        with pytest.raises(ValueError):
            KVCache(1, 1, 64, page=page)
    for pages, heads in ((-1, 1), (1, 0)):
        with pytest.raises(ValueError):
            KVCache(pages, heads, 64)
    with pytest.raises(RuntimeError, match='CUDA'):
        KVCache(1, 1, 64, device='cpu')


def test_the_library_rejects_bad_arguments():
    L = _lib.lib()
    assert L.bsp_cache_page_bytes(64, 128) == 4 * 18 * 128 and L.bsp_cache_page_bytes(48, 64) == -1 and L.bsp_cache_page_bytes(64, 32) == -1

    def call(fn, k=16, v=16, dtype=_lib.F16, Z=1, H=1, T=1, D=64, st=64, data=16, n=1, page=64, pages=16, slots=1, start=16):
        return fn(k, v, dtype, Z, H, T, D, st, st, st, st, st, st, data, n, page, pages, 1, slots, start, None, None)

    for fn in (L.bsp_cache_write, L.bsp_cache_read):
        for bad in (dict(dtype=7), dict(Z=-1), dict(H=0), dict(T=-1), dict(n=-1), dict(slots=-1), dict(page=24), dict(page=8),
                    dict(k=None), dict(v=None), dict(data=None), dict(data=24), dict(pages=None), dict(start=None)):
            assert call(fn, **bad) == _lib.ERR_INVALID, bad
        assert call(fn, D=96) == _lib.ERR_UNSUPPORTED
        assert call(fn, page=1024, slots=1 << 22) == _lib.ERR_UNSUPPORTED
        assert call(fn, Z=1 << 30, H=1 << 20, T=1 << 20) == _lib.ERR_UNSUPPORTED
        assert call(fn, Z=0, k=None, v=None, start=None) == _lib.OK
    assert call(L.bsp_cache_write, dtype=_lib.F32) == _lib.ERR_INVALID
    assert call(L.bsp_cache_read, k=24) == _lib.ERR_INVALID and b'aligned' in L.bsp_last_error()


@pytest.mark.gpu
def test_bad_calls():
    cache, pages, start = KVCache(4, 2, 64), table(2, 2, 4), ints(0, 0)
    k = tokens(2, 2, 5, 64, torch.float16)
    for bad in ((k.float(), k.float(), pages, start), (k, k.bfloat16(), pages, start), (k[:, :1], k[:, :1], pages, start),
                (k, k[:, :, :4], pages, start), (k[..., :32], k[..., :32], pages, start), (k, k, pages.long(), start),
                (k, k, pages[:1], start), (k, k, pages.t(), start), (k, k, pages, start[:1]), (k, k, pages, start.long()),
                (k, k, pages, ints(0, 1, 2, 3)[::2]), (k, k, pages, start, ints(1)), (k[0], k[0], pages, start)):
        with pytest.raises(ValueError):
            cache.write(*bad)
    for bad in ((k, k, pages.cpu(), start), (k, k, pages, start.cpu()), (k.cpu(), k.cpu(), pages, start)):
        with pytest.raises(RuntimeError):
            cache.write(*bad)
    with pytest.raises(NotImplementedError, match='no_grad'):
        cache.write(k.clone().requires_grad_(), k, pages, start)
    with torch.no_grad():
        cache.write(k.clone().requires_grad_(), k, pages, start)
    with pytest.raises(ValueError):
        cache.read(pages, start, -1)
    with pytest.raises(ValueError):
        cache.read(pages, start, 5, dtype=torch.float64)
    with pytest.raises(RuntimeError, match='trace'):
        torch.jit.trace(lambda x: cache.read(pages, start, 5)[0] + x, (k,), check_trace=False)
    cache.data = cache.data[:, :1]
    with pytest.raises(ValueError, match='contiguous'):
        cache.read(pages, start, 5)


@pytest.mark.gpu
def test_more_tokens_than_an_int_counts_are_refused():
    """An operand whose rows share memory can be as long; none of it is written."""
    cache, pages = KVCache(2, 1, 64, page=16), ints(0, 1)[None]
    x = tokens(1, 1, 1, 64, torch.float16).expand(1, 1, 2 ** 32 + 5, 64)
    with pytest.raises(NotImplementedError):
        cache.write(x, x, pages, ints(0))
    assert not bool(cache.data.any())
