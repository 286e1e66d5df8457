"""Attributes of an attention module or a cache that are set between its calls: every later call follows them."""
import pytest
import torch

from tests.test_cache import ints, table, tokens
from torch_blocksparse_b200 import KVCache, SparseSelfAttention, SparsityConfig, layouts


def test_tables_follow_the_layout_and_the_configuration():
    a = SparseSelfAttention(layout=layouts.dense(2, 4), block=16)
    old = a.get_ops(2, 64)
    assert a.get_ops(2, 64) is old
    a.layout = layouts.causal_band(2, 4, 2)
    new = a.get_ops(2, 64)
    assert new is not old and new[0].meta.nnz == int(a.layout.sum()) and a.get_ops(2, 64) is new
    assert a.tiles[(2, 64)] is new[0].attn_tiles
    a = SparseSelfAttention(SparsityConfig(block=16, stride=64))
    old = a.get_ops(2, 256)
    a.sparsity_config = SparsityConfig(block=32, stride=128)
    new = a.get_ops(2, 256)
    assert a.block == 32 and new[0].block == 32 and new[0].meta.nnz == int(layouts.fixed(2, 8, 4).sum())
    a.block = 64
    assert a.get_ops(2, 256)[0].block == 64
    # an explicit layout keeps its block whatever the configuration says
    a = SparseSelfAttention(layout=layouts.dense(2, 4), block=16)
    a.sparsity_config = SparsityConfig(block=32, stride=128)
    assert a.block == 16


def test_tables_built_while_the_layout_changes_are_not_kept():
    class Changing(SparseSelfAttention):
        def get_layout(self, H, L):
            found = super().get_layout(H, L)
            if self.layout is first:
                self.layout = second               # (as another thread would)
            return found

    first, second = layouts.dense(2, 4), layouts.causal_band(2, 4, 2)
    a = Changing(layout=first, block=16)
    a.get_ops(2, 64)
    assert a.get_ops(2, 64)[0].meta.nnz == int(second.sum()) and a.tiles[(2, 64)] is a.get_ops(2, 64)[0].attn_tiles


@pytest.mark.gpu
@pytest.mark.parametrize('fused', [True, False])
def test_forward_and_decode_follow_a_changed_layout(fused):
    H, L, D = 2, 64, 64
    q, k, v = (tokens(1, H, L, D, torch.float16, i).clamp(-3, 3) for i in range(3))
    cache, pages = KVCache(4, H, D, page=16), table(1, 4, 4)
    cache.write(k, v, pages, ints(0))
    attn = SparseSelfAttention(layout=layouts.dense(H, 4), block=16, fused=fused)
    steps = [(lambda a: setattr(a, 'layout', layouts.causal_band(H, 4, 1))), (lambda a: setattr(a, 'layout', layouts.causal_band(H, 4, 2)))]
    for step in [lambda a: None] + steps:
        step(attn)
        fresh = SparseSelfAttention(layout=attn.layout, block=16, fused=fused)
        assert torch.equal(attn(q, k, v), fresh(q, k, v))
        assert torch.equal(attn.decode(q[:, :, -1:], cache, pages, ints(L)), fresh.decode(q[:, :, -1:], cache, pages, ints(L)))
    attn = SparseSelfAttention(SparsityConfig(block=16, stride=64), fused=fused)
    attn(q, k, v), attn.decode(q[:, :, -1:], cache, pages, ints(L))
    attn.sparsity_config = SparsityConfig(block=32, stride=32)
    fresh = SparseSelfAttention(SparsityConfig(block=32, stride=32), fused=fused)
    assert torch.equal(attn(q, k, v), fresh(q, k, v))
    assert torch.equal(attn.decode(q[:, :, -1:], cache, pages, ints(L)), fresh.decode(q[:, :, -1:], cache, pages, ints(L)))


@pytest.mark.gpu
def test_operations_built_while_an_attribute_changes_are_not_kept():
    class ChangingCache(KVCache):
        armed = False

        @property
        def head_dim(self):
            if self.armed:                             # (as another thread would, while the operation is built)
                self.armed = False
                self.data = other
            return 64

        @head_dim.setter
        def head_dim(self, value):
            pass

    cache = ChangingCache(2, 1, 64, page=16)
    other = torch.zeros_like(cache.data)
    cache.armed = True
    cache._op()
    x = tokens(1, 1, 16, 64, torch.float16)
    cache.write(x, x, table(1, 2, 2), ints(0))
    assert bool(other.any())

    class Changing(SparseSelfAttention):
        def _decode_op(self, ops, key, cache, device):
            op = super()._decode_op(ops, key, cache, device)
            if self.layout is first:
                self.layout = second
                ops[key] = op                          # (as a thread that was interrupted before it stored the operation)
            return op

    first, second = layouts.dense(1, 2), layouts.causal_band(1, 2, 1)
    attn, cache, pages = Changing(layout=first, block=16), KVCache(2, 1, 64, page=16), table(1, 2, 2)
    k = tokens(1, 1, 32, 64, torch.float16)
    cache.write(k, k, pages, ints(0))
    attn.decode(k[:, :, -1:], cache, pages, ints(32))
    want = SparseSelfAttention(layout=second, block=16).decode(k[:, :, -1:], cache, pages, ints(32))
    assert torch.equal(attn.decode(k[:, :, -1:], cache, pages, ints(32)), want)
