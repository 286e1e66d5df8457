"""Rotary positions against the rotation in 64 bits: types, orders in memory, axes, far positions, gradients.

Tolerance of a turned pair, before the result is rounded to its type: the angle's fraction of a turn is
rounded to 2^-25 of half a turn (pi * 2^-25 = 9.4e-8), sincospif is off by at most 2 ulp (1.2e-7), and the two
products and the sum in 32 bits by 2^-24 each: below 4e-7 (|x0| + |x1|).  The oracle's own angle, a product
of doubles, is off by 2^-52 of itself.  The final rounding adds half a step of the type.
"""
import math

import pytest
import torch

from torch_blocksparse_b200 import MultiheadAttention, Rotary, _lib, layouts

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def turn(rotary, x, positions, sign=1):
    """x turned in 64 bits, and the bound on the error of the same in 32."""
    Z, H, L, D = x.shape
    x = x.detach().double().cpu()
    pos = torch.arange(L)[None] if positions is None else positions.cpu()
    if pos.dim() == 1:
        pos = pos[None]
    if pos.dim() == 2:
        pos = pos[:, None]
    pos = pos.expand(-1, Z, -1).double()
    pairs = sum(rotary.sections)
    freq = rotary.frequencies or [float(rotary.base) ** (-i / n) for n in rotary.sections for i in range(n)]
    axis = [a for a, n in enumerate(rotary.sections) for _ in range(n)]
    y, tol = x.clone(), torch.zeros_like(x)
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if rotary.interleaved else (i, pairs + i)
        t = sign * (pos[axis[i]] * freq[i])[:, None]
        y[..., a] = x[..., a] * t.cos() - x[..., b] * t.sin()
        y[..., b] = x[..., b] * t.cos() + x[..., a] * t.sin()
        tol[..., a] = tol[..., b] = (x[..., a].abs() + x[..., b].abs()) * (4e-7 + t.abs() * 2.0 ** -52)
    return y, tol


def assert_turned(got, rotary, x, positions, sign=1):
    want, tol = turn(rotary, x, positions, sign)
    assert got.shape == x.shape and got.dtype == x.dtype
    err = (got.detach().double().cpu() - want).abs()
    # a value below the type's normal range is rounded to a fixed step
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    assert bool((err <= tol + want.abs() * torch.finfo(x.dtype).eps / 2 * (1 + 1e-6) + tiny).all()), err.max()


def operand(shape, dtype, order='contiguous', seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    Z, H, L, D = shape
    def randn(*s): return torch.randn(s, generator=g, device='cuda').to(dtype)
    if order == 'sequence first':                     # [L, Z, H * D], as a projection writes it
        return randn(L, Z, H * D).view(L, Z, H, D).permute(1, 2, 0, 3)
    if order == 'chunk':                              # the middle third of a joint projection
        return randn(Z, L, 3 * H * D).chunk(3, dim=-1)[1].view(Z, L, H, D).transpose(1, 2)
    if order == 'offset':                             # starts off any 16-byte boundary, odd strides
        return randn(Z, H, L, D + 3)[..., 1:D + 1]
    if order == 'transposed':                         # unit stride on L
        return randn(Z, H, D, L).transpose(2, 3)
    if order == 'expanded':
        return randn(Z, 1, L, D).expand(Z, H, L, D)
    return randn(Z, H, L, D)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('shape,kv,sections', [
    ((1, 1, 1, 2), 1, None), ((2, 3, 7, 64), 3, None), ((1, 12, 1, 128), 2, (16, 24, 24)), ((5, 4, 33, 80), 1, (16, 16)),
    ((2, 2, 9, 48), 2, (7, 0, 6)), ((3, 1, 257, 96), 4, (48,)), ((64, 2, 1, 256), 2, (64, 64)), ((1, 2, 5, 254), 2, (1,)),
    ((2, 16, 1100, 64), 16, (10, 11, 11))])
def test_turned_as_in_64_bits(dtype, interleaved, shape, kv, sections):
    Z, H, L, D = shape
    rotary = Rotary(D, sections, interleaved=interleaved)
    axes = len(rotary.sections)
    g = torch.Generator(device='cuda').manual_seed(1)
    positions = torch.randint(0, 5000, (axes, Z, L), generator=g, device='cuda', dtype=torch.int32)
    q, k = operand(shape, dtype), operand((Z, kv, L, D), dtype, seed=2)
    yq, yk = rotary(q, k, positions)
    assert_turned(yq, rotary, q, positions)
    assert_turned(yk, rotary, k, positions)
    assert torch.equal(rotary(q, positions=positions), yq)


@pytest.mark.gpu
@pytest.mark.parametrize('order', ['sequence first', 'chunk', 'offset', 'transposed', 'expanded'])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_orders_in_memory(order, interleaved, dtype):
    rotary = Rotary(64, (12, 12), interleaved=interleaved)
    positions = torch.stack([torch.arange(19, device='cuda') // 5, torch.arange(19, device='cuda') % 5])
    q, k = operand((3, 4, 19, 64), dtype, order), operand((3, 2, 19, 64), dtype, order, 1)
    yq, yk = rotary(q, k, positions)
    assert_turned(yq, rotary, q, positions)
    assert_turned(yk, rotary, k, positions)
    if order == 'sequence first':
        assert yq.permute(2, 0, 1, 3).is_contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize('kind', [torch.int32, torch.int64])
def test_far_and_negative_positions(kind):
    rotary = Rotary(128)
    far = [0, 1, -1, 2 ** 20 - 1, 2 ** 31 - 1, -2 ** 31, 12345678] + ([2 ** 40 + 3, -2 ** 41] if kind == torch.int64 else [])
    positions = torch.tensor(far, device='cuda', dtype=kind)
    q = operand((2, 3, len(far), 128), torch.float32)
    assert_turned(rotary(q, positions=positions), rotary, q, positions)
    strided = torch.stack([positions, positions + 1], -1)[:, 0]                   # every other element
    assert torch.equal(rotary(q, positions=strided), rotary(q, positions=positions))
    shared = positions.view(1, 1, -1)
    assert torch.equal(rotary(q, positions=shared), rotary(q, positions=positions))


@pytest.mark.gpu
@pytest.mark.parametrize('interleaved', [False, True])
def test_small_sines_and_cosines_keep_their_bits(interleaved):
    """Angles next to whole quarters of a turn, turning (1, 0): the result is the cosine and the sine alone.

    sincospif is off by at most 2 ulp (2^-22), its argument by 2^-24 of itself, which at most an eighth of a turn
    away from a quarter is 1.1 * 2^-24 of the sine and less of the cosine: below 2^-21 together.  The table's rounding
    adds |position| * 2^-62, the oracle's product of doubles 2^-52 of the angle."""
    near = [k * math.pi / 2 + s * d for k in range(-4, 5) for d in (2.0 ** -20, 1e-4, 0.03) for s in (1, -1)]
    rotary = Rotary(2 * len(near), frequencies=near, interleaved=interleaved)
    positions = torch.tensor([1, -1, 5, 1001], device='cuda')
    x = torch.zeros((1, 1, 4, 2 * len(near)), device='cuda')
    first, second = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, len(near)), slice(len(near), None))
    x[..., first] = 1
    y = rotary(x, positions=positions)[0, 0].double().cpu()
    angle = positions.double().cpu()[:, None] * torch.tensor(near, dtype=torch.float64)
    for got, want in ((y[:, first], angle.cos()), (y[:, second], angle.sin())):
        limit = want.abs() * 2.0 ** -21 + positions.cpu().abs()[:, None] * 2.0 ** -62 + angle.abs() * 2.0 ** -52
        assert bool(((got - want).abs() <= limit).all()), ((got - want).abs() / limit).max()


@pytest.mark.gpu
def test_given_frequencies_and_default_positions():
    rotary = Rotary(32, (5, 4), frequencies=[0.0, 1.0, 3.5, -2.0, 1e-9, 6.2, 0.5, 0.25, 7.0])
    positions = torch.arange(2 * 3 * 11, device='cuda').view(2, 3, 11)
    x = operand((3, 2, 11, 32), torch.float32)
    assert_turned(rotary(x, positions=positions), rotary, x, positions)
    plain = Rotary(32)
    assert_turned(plain(x), plain, x, None)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('interleaved', [False, True])
def test_gradient_is_the_turn_back(dtype, interleaved):
    rotary = Rotary(40, (8, 10), interleaved=interleaved)
    positions = torch.randint(0, 999, (2, 1, 21), device='cuda')
    q, k = operand((2, 4, 21, 40), dtype).requires_grad_(), operand((2, 1, 21, 40), dtype, seed=1).requires_grad_()
    dq, dk = operand(q.shape, dtype, seed=2), operand(k.shape, dtype, 'transposed', seed=3)
    yq, yk = rotary(q, k, positions)
    torch.autograd.backward((yq, yk), (dq, dk))
    assert_turned(q.grad, rotary, dq, positions, -1)
    assert_turned(k.grad, rotary, dk, positions, -1)
    # one of the two alone: the other neither needs nor gets a gradient
    yq, yk = rotary(q.detach(), k, positions)
    g, = torch.autograd.grad(yk, k, dk)
    assert torch.equal(g, k.grad) and not (yq.requires_grad and yq.grad_fn is None)
    g, = torch.autograd.grad(rotary(q, k, positions)[0], q, dq)
    assert torch.equal(g, q.grad)
    # a broadcast gradient (of a sum)
    g, = torch.autograd.grad(rotary(q, positions=positions).sum(), q)
    assert_turned(g, rotary, torch.ones_like(q), positions, -1)


@pytest.mark.gpu
@pytest.mark.parametrize('tracked', ['q', 'k'])
def test_an_operand_that_needs_no_gradient(tracked):
    """Its result needs none either, and none is turned back for it, also where both results are used."""
    rotary = Rotary(16, (4, 4))
    positions = torch.randint(0, 50, (2, 5), device='cuda')
    x = {n: operand((1, 2, 5, 16), torch.float32, seed=i) for i, n in enumerate('qk')}
    x[tracked].requires_grad_()
    y = dict(zip('qk', rotary(x['q'], x['k'], positions)))
    other = 'k' if tracked == 'q' else 'q'
    assert y[tracked].requires_grad and not y[other].requires_grad and y[other].grad_fn is None
    assert torch.equal(y[other], rotary(x[other], positions=positions))
    d = operand((1, 2, 5, 16), torch.float32, seed=5)
    g, = torch.autograd.grad((y[tracked] * y[other].cos()).sum() + (y[tracked] * d).sum(), x[tracked])
    assert_turned(g, rotary, d + y[other].cos(), positions, -1)
    # differentiated again with respect to one incoming gradient of two
    z = {n: t.detach().requires_grad_() for n, t in x.items()}
    w = {n: d.clone().requires_grad_(n == tracked) for n in 'qk'}
    yq, yk = rotary(z['q'], z['k'], positions)
    g = dict(zip('qk', torch.autograd.grad((yq, yk), (z['q'], z['k']), (w['q'], w['k']), create_graph=True)))
    assert g[tracked].requires_grad and not g[other].requires_grad
    gg, = torch.autograd.grad(g[tracked], w[tracked], d)
    assert_turned(gg, rotary, d, positions)


@pytest.mark.gpu
def test_tangents_and_batched_transforms_are_refused():
    """Passing them by would drop a derivative without a word."""
    import torch.autograd.forward_ad as fwad
    rotary, x, t = Rotary(16), operand((1, 2, 5, 16), torch.float32), operand((1, 2, 5, 16), torch.float32, seed=1)
    with fwad.dual_level():
        dual = fwad.make_dual(x, t)
        for args in ((dual,), (dual, x), (x, dual), (x.clone().requires_grad_(), dual)):
            with pytest.raises(RuntimeError, match='jvp'):
                rotary(*args)
    with pytest.raises(RuntimeError):
        torch.func.vmap(rotary)(torch.stack([x, t]))


@pytest.mark.gpu
def test_gradient_against_differences_and_again():
    rotary = Rotary(16, (4, 4))
    positions = torch.randint(0, 50, (2, 5), device='cuda')
    x, d = operand((1, 2, 5, 16), torch.float32).requires_grad_(), operand((1, 2, 5, 16), torch.float32, seed=5)
    w = operand((1, 2, 5, 16), torch.float32, seed=6)
    g, = torch.autograd.grad((rotary(x, positions=positions) * w).sum(), x, create_graph=True)
    # the map is linear, so a step of 2^-3 has no error but rounding: 160 products of values below 16, 2^-23 each
    h = 2.0 ** -3
    with torch.no_grad():
        f = [(rotary(x + s * h * d, positions=positions).double() * w.double()).sum().item() for s in (1, -1)]
    assert abs((f[0] - f[1]) / (2 * h) - (g.double() * d.double()).sum().item()) < 160 * 16 * 2.0 ** -23 / h * 2
    # differentiated again with respect to the incoming gradient: the turn itself
    w2 = w.clone().requires_grad_()
    g, = torch.autograd.grad(rotary(x, positions=positions), x, w2, create_graph=True)
    gg, = torch.autograd.grad(g, w2, d)
    assert_turned(gg, rotary, d, positions)


@pytest.mark.gpu
def test_a_position_changed_before_the_backward_is_noticed():
    rotary = Rotary(16)
    x, positions = operand((1, 1, 4, 16), torch.float32).requires_grad_(), torch.arange(4, device='cuda')
    y = rotary(x, positions=positions)
    positions.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    rotary = Rotary(64, (16, 16))
    x, positions = operand((2, 2, 30, 64), torch.float16).requires_grad_(), torch.randint(0, 99, (2, 2, 30), device='cuda')
    dy = operand(x.shape, torch.float16, seed=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rotary(x, positions=positions)
        y = rotary(x, positions=positions)
    torch.cuda.current_stream().wait_stream(side)
    assert_turned(y, rotary, x, positions)
    leaf = x.detach().clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rotary(leaf, positions=positions)
        g, = torch.autograd.grad(y, leaf, dy)
    with torch.no_grad():
        leaf.copy_(operand(x.shape, torch.float16, seed=7))
        positions.add_(17)
    graph.replay()
    torch.cuda.synchronize()
    assert_turned(y, rotary, leaf, positions)
    assert_turned(g, rotary, dy, positions, -1)


@pytest.mark.gpu
def test_empty_operands_and_non_finite_values():
    rotary = Rotary(64)
    for shape in ((0, 2, 3, 64), (2, 0, 3, 64), (2, 2, 0, 64)):
        assert rotary(torch.empty(shape, device='cuda', dtype=torch.float16)).shape == shape
    x = operand((1, 2, 5, 64), torch.float32)
    want = rotary(x)
    x[0, 1, 3, 7] = float('nan')
    got = rotary(x)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, 1, 3, [7, 39]] = True                       # its pair, nothing else
    assert bool(got[bad].isnan().all()) and torch.equal(got[~bad], want[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize('order', ['contiguous', 'sequence first'])
def test_addresses_past_32_bits(order):
    L, H, D = (1 << 23) + 5, 3, 96                     # 2.4 G elements
    assert L * H * D > 2 ** 31
    rotary = Rotary(D, (16, 16))
    x = torch.empty((1, H, L, D) if order == 'contiguous' else (L, 1, H, D), device='cuda', dtype=torch.bfloat16).normal_()
    x = x if order == 'contiguous' else x.permute(1, 2, 0, 3)
    positions = torch.stack([torch.arange(L, device='cuda') // 1000, torch.arange(L, device='cuda') % 1000])
    y = rotary(x, positions=positions)
    for at in (slice(0, 9), slice(L // 2, L // 2 + 9), slice(L - 9, L)):
        assert_turned(y[:, :, at], rotary, x[:, :, at], positions[:, at])


@pytest.mark.gpu
def test_copies_and_pickles():
    import copy
    import pickle
    rotary, x = Rotary(32, (8, 8), interleaved=True), operand((1, 2, 7, 32), torch.float32)
    positions = torch.randint(0, 99, (2, 7), device='cuda')
    want = rotary(x, positions=positions)
    for other in (copy.deepcopy(rotary), pickle.loads(pickle.dumps(rotary))):
        assert torch.equal(other(x, positions=positions), want)
    rotary.interleaved = False                          # an attribute that is changed counts
    assert_turned(rotary(x, positions=positions), rotary, x, positions)


@pytest.mark.gpu
def test_traced():
    rotary = Rotary(32, (8, 8))
    q, k, positions = operand((2, 3, 6, 32), torch.float32), operand((2, 1, 6, 32), torch.float32), torch.randint(0, 9, (2, 6), device='cuda')
    traced = torch.jit.trace(lambda q, k, p: rotary(q, k, p), (q, k, positions), check_trace=False)
    q2, k2, p2 = q + 1, k - 1, positions + 3
    for got, want in zip(traced(q2, k2, p2), rotary(q2, k2, p2)):
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_a_trace_refuses_what_a_call_refuses():
    rotary, q = Rotary(32), operand((2, 3, 6, 32), torch.float16)
    for k in (q.float(), q[:, :, :5], q[:1], q[..., :30]):
        with pytest.raises(ValueError):
            rotary(q, k)
        with pytest.raises(ValueError):
            torch.jit.trace(lambda a, b: rotary(a, b), (q, k), check_trace=False)


@pytest.mark.gpu
@pytest.mark.parametrize('train', [False, True])
def test_multihead_attention_with_positions(train):
    L, B, E, H = 64, 2, 128, 2
    torch.manual_seed(0)
    rotary = Rotary(64, (16, 16))
    mha = MultiheadAttention(E, H, layouts.dense(H, L // 16), 16, rotary=rotary).cuda().half()
    x = torch.randn(L, B, E, device='cuda').half().requires_grad_(train)
    positions = torch.stack([torch.arange(L, device='cuda') // 8, torch.arange(L, device='cuda') % 8])
    out, _ = mha(x, x, x, positions=positions)
    xd = x.detach().double().cpu().requires_grad_(train)
    p = {n: t.detach().double().cpu() for n, t in mha.named_parameters()}
    q, k, v = (xd @ p['in_proj_weight'].T + p['in_proj_bias']).chunk(3, -1)
    q, k, v = (t.view(L, B, H, 64).permute(1, 2, 0, 3) for t in (q, k, v))

    def turned(t):
        n = 32
        f = torch.cat([positions[a].cpu().double()[:, None] * 10000.0 ** (-torch.arange(16).double() / 16) for a in range(2)], -1)
        a, b = t[..., :n], t[..., n:]
        return torch.cat((a * f.cos() - b * f.sin(), b * f.cos() + a * f.sin()), -1)

    w = torch.softmax(turned(q) @ turned(k).transpose(-1, -2) / 8, -1) @ v
    want = w.permute(2, 0, 1, 3).reshape(L, B, E) @ p['out_proj.weight'].T + p['out_proj.bias']
    from tests.util import assert_close
    assert_close(out, want.detach().to(out.dtype), 'out')
    if train:
        d = torch.randn_like(out)
        out.backward(d)
        want.backward(d.double().cpu())
        assert_close(x.grad, xd.grad.to(x.dtype), 'dx')
    plain = MultiheadAttention(E, H, layouts.dense(H, L // 16), 16).cuda().half()
    with pytest.raises(ValueError, match='without rotary'):
        plain(x, x, x, positions=positions)


# ---- refusals ----------------------------------------------------------------------------------
def test_bad_constructions():
    for args in ((63,), (0,), (258,), (64, (20, 20)), (64, ()), (64, (0, 0)), (64, (-1, 8))):
        with pytest.raises(ValueError):
            Rotary(*args)
    with pytest.raises(ValueError):
        Rotary(64, (16,), frequencies=[1.0] * 15)
    with pytest.raises(ValueError):
        Rotary(64, base=0)
    with pytest.raises(RuntimeError, match='CUDA'):
        Rotary(64)(torch.zeros(1, 1, 1, 64))
    with pytest.raises(ValueError, match='channels'):
        MultiheadAttention(128, 2, layouts.dense(2, 1), 16, rotary=Rotary(32))


def test_a_turn_is_exact_to_64_bits():
    turns = Rotary(128).turns()
    assert len(turns) == 64 and all(-2 ** 63 <= t < 2 ** 63 for t in turns)
    for i, t in enumerate(turns):          # (rounded to a whole 2^-64 of a turn: off by at most pi * 2^-64 rad)
        assert math.isclose(t * 2.0 ** -64 * 2 * math.pi, 10000.0 ** (-i / 64), rel_tol=1e-15, abs_tol=math.pi * 2.0 ** -64)


def test_the_library_rejects_bad_arguments():
    L = _lib.lib()

    def call(q=16, out=16, H=1, dtype=_lib.F16, Z=1, length=1, D=64, pairs=32, table=16, axes=1, pos=16, pos_bytes=4, inter=0, sl=64, k=None, Hk=0):
        return L.bsp_rotary(q, out, H, sl, sl, sl, 64, 64, 64, k, k, Hk, 0, 0, 0, 0, 0, 0, dtype, Z, length, D, pairs, inter, table, axes,
                            pos, pos_bytes, 0, 0, 1, 0, None)

    assert call(dtype=5) == _lib.ERR_INVALID and b'dtype' in L.bsp_last_error()
    for bad in (dict(Z=-1), dict(length=-1), dict(H=-1), dict(D=258), dict(D=0), dict(pairs=33), dict(pairs=0), dict(axes=0),
                dict(pos_bytes=2), dict(pos_bytes=0, axes=2), dict(pos=None), dict(table=None), dict(q=None), dict(out=None), dict(Hk=1)):
        assert call(**bad) == _lib.ERR_INVALID, bad
    assert call(q=18, inter=1) == _lib.ERR_INVALID and b'even' in L.bsp_last_error()
    assert call(Z=2, sl=65, inter=1) == _lib.ERR_INVALID
    assert call(H=1 << 21) == _lib.ERR_UNSUPPORTED
    assert call(Z=0, q=None) == _lib.OK               # nothing to do


@pytest.mark.gpu
def test_bad_calls():
    rotary = Rotary(64, (16, 16))
    q, positions = operand((2, 2, 5, 64), torch.float16), torch.zeros(2, 5, dtype=torch.int32, device='cuda')
    for bad in (dict(positions=None), dict(positions=positions.float()), dict(positions=positions[:, :4]), dict(positions=positions[:1]),
                dict(positions=positions[0]), dict(positions=positions[:, None].expand(2, 3, 5)), dict(key=q.float(), positions=positions),
                dict(key=q[:, :, :4], positions=positions), dict(key=q[:1], positions=positions)):
        with pytest.raises(ValueError):
            rotary(q, **bad)
    with pytest.raises(ValueError):
        rotary(q[..., :32], positions=positions)
    with pytest.raises(ValueError):
        rotary(q.double(), positions=positions)
    with pytest.raises(ValueError):
        rotary(q[0], positions=positions)
    with pytest.raises(RuntimeError):
        rotary(q, positions=positions.cpu())
    with pytest.raises(RuntimeError):
        rotary(q, q.cpu(), positions)


@pytest.mark.gpu
def test_more_tokens_than_an_int_counts_are_refused():
    x = torch.zeros((1, 1, 1, 2), device='cuda', dtype=torch.float16)
    for shape in ((1, 1, 2 ** 32 + 5, 2), (2 ** 32 + 5, 1, 1, 2), (1, 2 ** 32 + 5, 1, 2)):
        with pytest.raises(NotImplementedError):
            Rotary(2)(x.expand(shape))
