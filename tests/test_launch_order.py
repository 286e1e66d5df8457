"""Rotary, cache write, cache read and decode right behind copies, other kernels and events of other streams, called and captured.

The four kernels are launched before the work in front of them has ended and wait for it themselves; whatever that work is,
they have to find what it leaves.
"""
import pytest
import torch

from tests.test_cache import ints, table, tokens
from torch_blocksparse_b200 import KVCache, Rotary, SparseSelfAttention, layouts

Z, H, L, D, PAGE = 4, 4, 96, 64, 32


class Step:
    """A prompt rotated, written and read, its last token decoded, from inputs that something else fills first."""

    def __init__(self):
        self.attn, self.rotary = SparseSelfAttention(layout=layouts.dense(1, 6), block=16), Rotary(D)
        self.cache, self.pages = KVCache(Z * 3, H, D, page=PAGE), table(Z, 3, Z * 3)
        self.q, self.k, self.v = (torch.zeros((Z, H, L, D), device='cuda', dtype=torch.float16) for _ in range(3))
        self.start, self.lengths = ints(*[0] * Z), ints(*[0] * Z)

    def inputs(self):
        return [self.q, self.k, self.v, self.lengths]

    def __call__(self):
        q, k = self.rotary(self.q, self.k)
        self.cache.write(k, self.v, self.pages, self.start, self.lengths)
        kk, vv = self.cache.read(self.pages, self.start, L, self.lengths)
        return q, kk, vv, self.attn.decode(q[:, :, -1:], self.cache, self.pages, self.lengths)


def values(i):
    return [tokens(Z, H, L, D, torch.float16, 3 * i + n) for n in range(3)] + [(torch.arange(Z, device='cuda') * 7 + 60 + i % 9).int()]


def expected(i):
    step = Step()
    for x, y in zip(step.inputs(), values(i)):
        x.copy_(y)
    torch.cuda.synchronize()
    out = [t.clone() for t in step()]
    torch.cuda.synchronize()
    return out


def fill_by(way, step, source, side):
    """Brings source's tensors into the step's inputs, on the current stream or, joined by events, on another."""
    def copies():
        for x, y in zip(step.inputs(), source):
            if way == 'kernels':
                torch.add(y, 0, out=x)
            else:
                x.copy_(y, non_blocking=True)
    if way != 'another stream':
        return copies()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200000)
        copies()
    torch.cuda.current_stream().wait_stream(side)


WAYS = ['copies', 'kernels', 'another stream']


@pytest.mark.gpu
@pytest.mark.parametrize('way', WAYS)
def test_called_behind(way):
    step, side = Step(), torch.cuda.Stream()
    sources = [values(i) for i in range(6)]
    step()
    got = []
    for source in sources:
        fill_by(way, step, source, side)
        got.append(step())
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, expected(i))), i


@pytest.mark.gpu
@pytest.mark.parametrize('way', WAYS)
def test_captured_behind(way):
    step, side, source = Step(), torch.cuda.Stream(), [x.clone() for x in values(0)]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fill_by(way, step, source, side)
        out = step()
    for i in range(6):
        for x, y in zip(source, values(i)):
            x.copy_(y)
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, expected(i))), i


@pytest.mark.gpu
def test_two_captured_steps_replayed_on_two_streams_at_once():
    """They share no memory but the layout's tables; each finds its own inputs."""
    steps, graphs = [Step(), Step()], []
    for i, step in enumerate(steps):
        for x, y in zip(step.inputs(), values(i)):
            x.copy_(y)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(50):
        for stream, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for i, (_, out) in enumerate(graphs):
        assert all(torch.equal(a, b) for a, b in zip(out, expected(i))), i
