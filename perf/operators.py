"""Cases of the serving side of sparse attention: rotary positions, the 4-bit key / value cache and attention over it.

    Rotary                       rotation of queries and keys by positions with one or several axes, and its gradient
    KVCache.write / .read        keys and values quantised to 4 bits as they enter a paged cache, and read back
    SparseSelfAttention.decode   attention of the newest tokens over such a cache, along the rows of a sparse layout

listed() names eleven cases, draw() gives more of the same ranges.  With `own` false, run() computes a case in
elementary torch operations; with `own` true it makes the package's calls.  Inputs are synthetic, drawn from a seed.

The cache holds, for each token, head and group of 32 channels, s = bf16(max |x| / 7) and the integers
rint(x / s) in [-8, 7]; it stands for the values s * integer.
"""
import math

import torch

own = False

DTYPES = {'fp32': torch.float32, 'fp16': torch.float16, 'bf16': torch.bfloat16}
GROUP = 32


def listed():
    return [
        # One new token for each of 64 sequences, up to a million positions in: latency.
        dict(name='rotary_decode', op='rotary', dtype='fp16', train=False, batch=64, heads=16, kv_heads=16, length=1,
             head_dim=64, axes=1, partial=0, interleaved=False, far=1 << 20),
        # Training on video: 8 frames of 32 x 32 patches, three axes, forward and backward.
        dict(name='rotary_video_train', op='rotary', dtype='bf16', train=True, batch=2, heads=16, kv_heads=16, length=8192,
             head_dim=128, axes=3, partial=0, interleaved=False, far=0),
        # Training on images of 37 x 29 patches in 32 bits: an odd length, neighbouring pairs, 16 channels left as they are.
        dict(name='rotary_image_fp32', op='rotary', dtype='fp32', train=True, batch=3, heads=10, kv_heads=5, length=1073,
             head_dim=80, axes=2, partial=16, interleaved=True, far=0),
        # The newest token of 64 sequences enters the cache and is read back: latency.
        dict(name='cache_append', op='write', dtype='bf16', batch=64, heads=16, length=1, head_dim=128, page=64, past=4000),
        # Ragged prompts of up to 8192 tokens enter an empty cache and are read back for their own attention.
        dict(name='cache_prompt', op='write', dtype='fp16', batch=8, heads=16, length=8192, head_dim=64, page=64, past=0),
        # Long sequences are read back whole.
        dict(name='cache_read_long', op='read', dtype='bf16', batch=4, heads=16, length=16384, head_dim=128, page=128, past=0),
        # One short sequence generates: all latency.
        dict(name='decode_short', op='decode', dtype='fp16', batch=1, heads=12, kv_heads=12, tokens=1, length=1024,
             head_dim=64, block=64, page=64, layout='fixed'),
        # The benchmark's attention workload, serving a ragged batch: windows of 4 blocks, the last of each global.
        dict(name='decode_8k', op='decode', dtype='fp16', batch=8, heads=16, kv_heads=16, tokens=1, length=8192,
             head_dim=64, block=64, page=64, layout='fixed'),
        # Six drafted tokens are verified at once on the default block 16, windows of 64.
        dict(name='decode_verify', op='decode', dtype='fp16', batch=4, heads=8, kv_heads=8, tokens=6, length=2048,
             head_dim=64, block=16, page=64, layout='fixed'),
        # The benchmark's BigBird-style workload at its full batch and length.
        dict(name='decode_bigbird', op='decode', dtype='bf16', batch=32, heads=16, kv_heads=16, tokens=1, length=16384,
             head_dim=128, block=128, page=128, layout='bigbird'),
        # A dense layer among the sparse ones: four query heads share each head of a long cache.
        dict(name='decode_dense_grouped', op='decode', dtype='bf16', batch=16, heads=32, kv_heads=8, tokens=1,
             length=32768, head_dim=128, block=128, page=128, layout='dense'),
    ]


# ---- drawn cases ------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choices(['rotary', 'write', 'read', 'decode'], [3, 2, 1, 4])[0]
    if op == 'rotary':
        head_dim = rng.choice([32, 48, 64, 64, 80, 96, 128, 128])
        axes = rng.choice([1, 2, 3])
        kv = rng.choice([1, 2, 4, 5, 8, 16])
        return dict(op=op, dtype=rng.choice(['fp32', 'fp16', 'bf16']), train=rng.random() < 0.6, batch=_log(rng, 1, 64),
                    heads=kv * rng.choice([1, 1, 2, 4]), kv_heads=kv, length=_log(rng, 1, 16384), head_dim=head_dim, axes=axes,
                    partial=rng.choice([0, 0, 8, 16]), interleaved=rng.random() < 0.5, far=rng.choice([0, 1 << 14, 1 << 20]))
    head_dim = rng.choice([64, 128])
    dtype = rng.choice(['fp16', 'bf16'])
    page = rng.choice([16, 32, 64, 128])
    if op in ('write', 'read'):
        return dict(op=op, dtype=dtype, batch=_log(rng, 1, 64), heads=rng.choice([1, 2, 4, 8, 12, 16]),
                    length=_log(rng, 1, 16384), head_dim=head_dim, page=page, past=rng.choice([0, 0, 1, 77, 1000]))
    block = rng.choice([16, 32, 64, 64, 128])
    layout = rng.choice(['fixed', 'fixed', 'band', 'bigbird', 'dense'])
    kv = rng.choice([1, 2, 4, 8, 12, 16])
    length = _log(rng, 100, 32768)
    if layout != 'dense':
        length = min(length, 512 * block)
    return dict(op=op, dtype=dtype, batch=_log(rng, 1, 32), heads=kv * rng.choice([1, 1, 1, 2, 4, 8]), kv_heads=kv,
                tokens=rng.choice([1, 1, 1, 2, 5, 16]), length=length, head_dim=head_dim, block=block, page=page, layout=layout)


def _moved(case):
    """Bytes that the plain form of a case would hold at once, roughly: what bounds a drawn case."""
    if case['op'] == 'decode':
        return case['batch'] * case['kv_heads'] * case['length'] * case['head_dim']
    return case['batch'] * case['heads'] * case['length'] * case['head_dim']


def draw(rng):
    most = max(work(c)['bytes'] for c in listed())
    hold = max(_moved(c) for c in listed() if c['op'] == 'decode')
    while True:
        case = _draw(rng)
        if _moved(case) <= hold and work(case)['bytes'] <= most:
            return case


# ---- what a case is made of -------------------------------------------------------------------
def _layout(case):
    """The layout of a decode case, [heads or 1, blocks, blocks], on the CPU; its last row holds the longest sequence."""
    nb, H, block = -(-case['length'] // case['block']), case['kv_heads'], case['block']
    i, j = torch.arange(nb)[:, None], torch.arange(nb)[None, :]
    if case['layout'] == 'dense':
        return torch.ones((1, nb, nb), dtype=torch.int64)
    if case['layout'] == 'fixed':           # windows of 4 blocks, and the last block of every earlier window
        one = (i >= j) & ((i // 4 == j // 4) | (j % 4 == 3))
    else:                                   # a band of 4 blocks and the first block
        one = (i >= j) & ((i - j < 4) | (j == 0))
    one = one.long()
    if case['layout'] != 'bigbird':
        return one.expand(H, nb, nb).contiguous()
    g = torch.Generator().manual_seed(0)    # 3 blocks around the row, 2 global rows and columns, 3 random ones
    lay = ((i - j).abs() <= 1) | (i < 2) | (j < 2)
    lay = lay.long().expand(H, nb, nb).contiguous()
    return lay.scatter_(2, torch.randint(nb, (H, nb, 3), generator=g), 1)


def _counts(case):
    """How many tokens each sequence of a batch has: the longest first, the others down to half of it, odd sizes among them."""
    Z, L, least = case['batch'], case['length'], case.get('tokens', 1)
    return [max(least, L - z * (L // 2) // Z - (z % 3 if z else 0)) for z in range(Z)]


def _rows(case):
    """The block-rows that the newest tokens of each sequence lie in, first and last."""
    return [((n - case['tokens']) // case['block'], (n - 1) // case['block']) for n in _counts(case)]


def _sections(case):
    """Pairs of channels for each axis: all but `partial` channels, split as evenly as whole pairs allow."""
    pairs, axes = (case['head_dim'] - case['partial']) // 2, case['axes']
    return [pairs // axes + (1 if a < pairs % axes else 0) for a in range(axes)]


def _slots(case):
    """Pages that each sequence of a cache case has room for."""
    return -(-(case['length'] + case.get('past', 0)) // case['page'])


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device='cuda', dtype=dtype)


def _keys_values(case, g, heads):
    """Keys whose channels differ in size and have a mean, as they come out of a projection, and plain values."""
    Z, L, D, dtype = case['batch'], case['length'], case['head_dim'], DTYPES[case['dtype']]
    size = torch.exp(0.5 * _randn(g, heads, 1, D))
    k = (_randn(g, Z, heads, L, D, dtype=dtype) * size.to(dtype) + _randn(g, heads, 1, D).to(dtype))
    return k, _randn(g, Z, heads, L, D, dtype=dtype)


def _inputs(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    Z, D, dtype = case['batch'], case['head_dim'], DTYPES[case['dtype']]
    if case['op'] == 'rotary':
        L, A = case['length'], case['axes']
        side = max(1, int(round(L ** (1 / A))))
        flat = torch.arange(L, device='cuda')
        pos = torch.stack([flat // side ** (A - 1 - a) % (side if a else L) for a in range(A)])        # a grid, row by row
        start = torch.randint(case['far'] + 1, (A, Z, 1), generator=g, device='cuda')
        x = dict(q=_randn(g, Z, case['heads'], L, D, dtype=dtype), k=_randn(g, Z, case['kv_heads'], L, D, dtype=dtype),
                 positions=(pos[:, None] + start).int())
        if case['train']:
            x.update(dq=torch.randn_like(x['q']), dk=_randn(g, Z, case['kv_heads'], L, D, dtype=dtype))
            x['dq'] = _randn(g, Z, case['heads'], L, D, dtype=dtype)
        return x
    heads = case['kv_heads'] if case['op'] == 'decode' else case['heads']
    k, v = _keys_values(case, g, heads)
    slots = _slots(case)
    x = dict(k=k, v=v, pages=torch.randperm(Z * slots, generator=g, device='cuda').view(Z, slots).int(),
             start=torch.full((Z,), case.get('past', 0), dtype=torch.int32, device='cuda'),
             count=torch.tensor(_counts(case), dtype=torch.int32, device='cuda'))
    if case['op'] == 'decode':
        x['q'] = _randn(g, Z, case['heads'], case['tokens'], D, dtype=dtype)
    return x


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    Z, D = case['batch'], case['head_dim']
    if case['op'] == 'rotary':
        if own:
            from torch_blocksparse_b200 import Rotary
            s['rotary'] = Rotary(D, sections=_sections(case), interleaved=case['interleaved'])
            if case['train']:
                s['q'].requires_grad_()
                s['k'].requires_grad_()
        return s
    heads, pages = s['k'].size(1), Z * _slots(case)
    if own:
        from torch_blocksparse_b200 import KVCache, SparseSelfAttention
        s['cache'] = KVCache(pages, heads, D, page=case['page'], device='cuda')
        if case['op'] != 'write':
            s['cache'].write(s['k'], s['v'], s['pages'], s['start'], s['count'])
        if case['op'] == 'decode':
            s['attention'] = SparseSelfAttention(layout=_layout(case), block=case['block'])
    else:
        # (one more page than there are: what lies past a sequence's end goes there)
        for n in 'kv':
            s[n + '_codes'] = torch.zeros((pages + 1, heads, case['page'], D), dtype=torch.int8, device='cuda')
            s[n + '_scales'] = torch.zeros((pages + 1, heads, case['page'], D // GROUP), dtype=torch.bfloat16, device='cuda')
        if case['op'] != 'write':
            _plain_write(s)
    if case['op'] == 'decode':
        layout = _layout(case)
        if not own:
            s['layout'] = layout.cuda()
            s['widest'] = max(int((layout[:, a] | layout[:, b]).sum(-1).max()) for a, b in _rows(case))   # blocks to look at
        s['lengths'] = s['count']
    if case['op'] != 'write':
        del s['k'], s['v']
    return s


# ---- plain forms ------------------------------------------------------------------------------
def _plain_angles(case, positions):
    """cos and sin of every position and pair, [Z, 1, L, pairs], in 32 bits from angles in 64."""
    angle = []
    for a, n in enumerate(_sections(case)):
        freq = 10000.0 ** (-torch.arange(n, device='cuda', dtype=torch.float64) / n)
        angle.append(positions[a].double()[:, None, :, None] * freq)
    angle = torch.cat(angle, -1)
    return angle.cos().float(), angle.sin().float()


def _plain_rotate(case, x, cos, sin):
    n = 2 * cos.size(-1)
    y, turned = x.float(), x[..., :n].float()
    if case['interleaved']:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :n // 2], turned[..., n // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., n:]), -1).to(x.dtype)


def _plain_quantise(x):
    """Codes and scales of a [..., D] tensor, a scale for each 32 channels."""
    g = x.float().unflatten(-1, (-1, GROUP))
    s = (g.abs().amax(-1) / 7).bfloat16()
    c = (g / s.float()[..., None]).round().nan_to_num(0).clamp(-8, 7)
    return c.flatten(-2).to(torch.int8), s


def _plain_values(codes, scales):
    return (codes.float().unflatten(-1, (-1, GROUP)) * scales.float()[..., None]).flatten(-2)


def _plain_places(s, T):
    """Page and place in it of the tokens start .. start + T - 1 of every sequence, [Z, T]; which of them there are."""
    page = s['case']['page']
    t = torch.arange(T, device='cuda')
    at = s['start'].long()[:, None] + t
    there = t < s['count'][:, None]
    ids = s['pages'].long().gather(1, (at // page).clamp(max=s['pages'].size(1) - 1))
    return torch.where(there, ids, s['k_codes'].size(0) - 1), at % page, there


def _plain_write(s):
    ids, at, _ = _plain_places(s, s['k'].size(2))
    for n in 'kv':
        codes, scales = _plain_quantise(s[n])
        s[n + '_codes'][ids, :, at] = codes.transpose(1, 2)
        s[n + '_scales'][ids, :, at] = scales.transpose(1, 2)


def _plain_read(s):
    ids, at, there = _plain_places(s, s['case']['length'])
    dtype = DTYPES[s['case']['dtype']]
    out = [_plain_values(s[n + '_codes'][ids, :, at], s[n + '_scales'][ids, :, at]) for n in 'kv']
    return tuple((x * there[..., None, None]).to(dtype).transpose(1, 2).contiguous() for x in out)


def _plain_decode(s):
    """Every sequence's blocks gathered out of the pages, then scores, softmax and weighted sum in 32 bits."""
    c, q, layout = s['case'], s['q'], s['layout']
    Z, Hq, T, D = q.shape
    Hk, block, page = c['kv_heads'], c['block'], c['page']
    pos = s['lengths'].long()[:, None] - T + torch.arange(T, device='cuda')             # [Z, T]
    sees = layout.expand(Hk, -1, -1)[:, pos // block].transpose(0, 1) != 0              # [Z, Hk, T, blocks]
    used = sees.any(2).int().argsort(dim=-1, descending=True, stable=True)[..., :s['widest']]
    sees = sees.gather(3, used[:, :, None].expand(-1, -1, T, -1))
    token = (used[..., None] * block + torch.arange(block, device='cuda')).flatten(-2)  # [Z, Hk, N]
    ok = sees.repeat_interleave(block, -1) & (token[:, :, None] <= pos[:, None, :, None])
    slot = (token // page).clamp(max=s['pages'].size(1) - 1)
    ids = s['pages'].long()[torch.arange(Z, device='cuda')[:, None, None], slot]
    head = torch.arange(Hk, device='cuda')[None, :, None]
    k, v = (_plain_values(s[n + '_codes'][ids, head, token % page], s[n + '_scales'][ids, head, token % page]) for n in 'kv')
    qf = q.float().unflatten(1, (Hk, -1)).flatten(2, 3)                                 # [Z, Hk, G * T, D]
    score = (qf @ k.transpose(-1, -2)) * D ** -0.5
    score = score.masked_fill(~ok.repeat(1, 1, Hq // Hk, 1), float('-inf'))
    w = torch.exp(score - score.amax(-1, keepdim=True))
    out = (w @ v) / w.sum(-1, keepdim=True)
    return out.view(Z, Hq, T, D).to(q.dtype)


def run(state):
    s, c = state, state['case']
    if c['op'] == 'rotary':
        if own:
            q, k = s['rotary'](s['q'], s['k'], s['positions'])
            if not c['train']:
                return q, k
            return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (s['q'], s['k']), (s['dq'], s['dk']))
        cos, sin = _plain_angles(c, s['positions'])
        out = _plain_rotate(c, s['q'], cos, sin), _plain_rotate(c, s['k'], cos, sin)
        if c['train']:
            out += _plain_rotate(c, s['dq'], cos, -sin), _plain_rotate(c, s['dk'], cos, -sin)
        return out
    if c['op'] == 'decode':
        return s['attention'].decode(s['q'], s['cache'], s['pages'], s['lengths']) if own else _plain_decode(s)
    if c['op'] == 'write':
        s['cache'].write(s['k'], s['v'], s['pages'], s['start'], s['count']) if own else _plain_write(s)
    if own:
        return s['cache'].read(s['pages'], s['start'], c['length'], s['count'], dtype=DTYPES[c['dtype']])
    return _plain_read(s)


def work(case):
    Z, D, e = case['batch'], case['head_dim'], 4 if case['dtype'] == 'fp32' else 2
    token = D // 2 + D // GROUP * 2                       # bytes of one key or value in the cache
    if case['op'] == 'rotary':
        n = Z * (case['heads'] + case['kv_heads']) * case['length'] * D * (2 if case['train'] else 1)
        return {'bytes': 2 * e * n + 4 * case['axes'] * Z * case['length'], 'flops': 3 * n}
    if case['op'] == 'decode':
        layout, tokens = _layout(case), 0
        for n, (a, b) in zip(_counts(case), _rows(case)):
            blocks = (layout[:, a] | layout[:, b]).nonzero()[:, 1] * case['block']
            tokens += int((n - blocks).clamp(0, case['block']).sum()) * (case['kv_heads'] // layout.size(0))
        q = Z * case['heads'] * case['tokens'] * D
        return {'bytes': 2 * token * tokens + 2 * e * q,
                'flops': 4 * tokens * D * (case['heads'] // case['kv_heads']) * case['tokens']}
    n, there = case['heads'], sum(_counts(case))
    moved = 2 * n * (there * token + Z * case['length'] * D * e)          # read: the cache in, every row out
    if case['op'] == 'write':
        moved += 2 * n * there * (token + D * e)
    return {'bytes': moved, 'flops': 2 * n * there * D}


# ---- the definitions in 64 bits ----------------------------------------------------------------
def _exact_cached(x):
    """The values that a 4-bit cache stands for, from the definition."""
    x = x.double()
    parts = []
    for c0 in range(0, x.size(-1), GROUP):
        p = x[..., c0:c0 + GROUP]
        s = torch.div(p.abs().max(-1, keepdim=True).values, 7).to(torch.bfloat16).double()
        n = torch.where(s > 0, torch.round(p / torch.where(s > 0, s, 1.0)), 0.0)
        parts.append(s * torch.clip(n, -8, 7))
    return torch.cat(parts, -1)


def _exact_turn(case, x, positions, sign):
    sections, pairs = _sections(case), sum(_sections(case))
    y, i = x.double().clone(), 0
    for a, n in enumerate(sections):
        for m in range(n):
            angle = sign * positions[a].double() * math.exp(-math.log(10000.0) * m / n)
            one, two = (2 * i, 2 * i + 1) if case['interleaved'] else (i, i + pairs)
            z = torch.complex(x[..., one].double(), x[..., two].double()) * torch.polar(torch.ones_like(angle), angle)[:, None]
            y[..., one], y[..., two] = z.real, z.imag
            i += 1
    return y


def exact(case, seed):
    x = _inputs(case, seed)
    if case['op'] == 'rotary':
        out = [_exact_turn(case, x[n], x['positions'], 1) for n in 'qk']
        if case['train']:
            out += [_exact_turn(case, x[n], x['positions'], -1) for n in ('dq', 'dk')]
        return tuple(out)
    if case['op'] != 'decode':
        out = []
        for n in 'kv':
            y = _exact_cached(x[n])
            for z, there in enumerate(_counts(case)):
                y[z, :, there:] = 0
            out.append(y)
        return tuple(out)
    layout = _layout(case).cuda().bool()
    Z, Hq, T, D = x['q'].shape
    Hk, out = case['kv_heads'], torch.zeros(x['q'].shape, dtype=torch.float64, device='cuda')
    for z, n in enumerate(_counts(case)):
        k, v = _exact_cached(x['k'][z, :, :n]), _exact_cached(x['v'][z, :, :n])
        block_of = torch.arange(n, device='cuda') // case['block']
        for t in range(T):
            pos = n - T + t
            sees = layout[:, pos // case['block']][:, block_of].expand(Hk, n)
            sees = sees & (torch.arange(n, device='cuda') <= pos)
            q = x['q'][z, :, t].double().view(Hk, Hq // Hk, D)
            score = torch.einsum('hgd,hnd->hgn', q, k) / math.sqrt(D)
            w = torch.softmax(score.masked_fill(~sees[:, None], -math.inf), -1)
            out[z, :, t] = torch.einsum('hgn,hnd->hgd', w, v).view(Hq, D)
    return out
