"""Sparse self-attention wrapper with the reference's interface.

Mirrors torch_blocksparse/deepspeedsparseselfattention.py:
  SparsityConfig(mode, block, stride, attention, numverts, vertsize)          (8-26)
  DeepSpeedSparseSelfAttention(sparsity_config, key_padding_mask_mode='add',
                               attn_mask_mode='mul')                          (109-117)
  forward(query, key, value, rpe=None, key_padding_mask=None, attn_mask=None) (135-166)
and is also exported as SparseSelfAttention.

Differences, all additive:
  * an explicit `layout` (with `block`) may be given instead of a SparsityConfig,
    for layouts the config cannot describe (e.g. BigBird-style);
  * the op cache is per instance and keyed on (heads, sequence length), not a
    class-level dict keyed on the length alone (deepspeedsparseselfattention.py:67-106),
    so two modules with different layouts never share tables;
  * `fused=True` (default) computes scores, softmax and the product with V in
    one kernel without storing the score tensor; `fused=False` runs the
    reference's three-op chain sdd -> softmax -> dsd.
"""
import weakref

import torch
import torch.nn as nn

from . import _lib, fused, tables
from .matmul import MatMul
from .softmax import Softmax


class SparsityConfig:
    """deepspeedsparseselfattention.py:8-26."""

    def __init__(self, mode='fixed', block=16, stride=64, attention='unidirectional', numverts=1, vertsize=1):
        if mode != 'dense' and mode != 'fixed':
            raise NotImplementedError('only "dense" and "fixed" modes are supported for now')
        self.mode = mode
        self.block = block
        self.stride = stride
        if attention != 'unidirectional' and attention != 'bidirectional':
            raise NotImplementedError('only "uni/bi-directional" attentions are supported for now')
        self.attention = attention
        self.numverts = numverts
        self.vertsize = vertsize


class DeepSpeedSparseSelfAttention(_lib.WithOps, nn.Module):

    _op_cache = '_attn'
    _op_attributes = frozenset(('block', 'layout', 'sparsity_config'))

    @staticmethod
    def _make_layout(num_heads, num_blocks, mode, block_stride, attention, numverts, vertsize):
        """deepspeedsparseselfattention.py:51-65, built natively."""
        return tables.make_fixed_layout(num_heads, num_blocks, mode, block_stride, attention, numverts, vertsize)

    def __init__(self, sparsity_config=None, key_padding_mask_mode='add', attn_mask_mode='mul',
                 layout=None, block=None, fused=True):
        super().__init__()
        if layout is not None:
            if block is None:
                raise ValueError('an explicit layout needs its block size')
            if layout.dim() != 3 or layout.size(1) != layout.size(2):
                raise ValueError('an attention layout must be [heads, L/block, L/block]')
        self.sparsity_config = sparsity_config if sparsity_config is not None else SparsityConfig()
        self.layout = layout
        self.block = block if layout is not None else self.sparsity_config.block
        self.key_padding_mask_mode = key_padding_mask_mode
        self.attn_mask_mode = attn_mask_mode
        self.fused = fused
        self.ops = dict()
        self.tiles = dict()
        self._attn = _lib.OpCache()       # native attention per (heads, length, device index)
        self._causal_cache = dict()
        self.causal_checks = 0            # comparisons of a mask against the causal one made so far

    def __setattr__(self, name, value):
        # The tables of a layout go with it, before the operations made of them do (so that no call puts an operation of the
        # old tables into the new cache), and a configuration brings its block.  (An explicit layout that no longer fits
        # a changed block keeps its tables, which every call then refuses.)
        known = self.__dict__
        if 'ops' in known and (name in ('layout', 'sparsity_config') or (name == 'block' and known.get('layout') is None)):
            super(_lib.WithOps, self).__setattr__(name, value)
            self.ops, self.tiles = dict(), dict()
            if name == 'sparsity_config' and known.get('layout') is None:
                self.block = value.block
        super().__setattr__(name, value)

    def get_layout(self, H, L):
        """The [H, L/block, L/block] layout used for H heads and sequence length L."""
        block = self.block
        if L % block != 0:
            raise ValueError(f'Sequence length {L} must be dividable by block size {block}')
        if self.layout is not None:
            if self.layout.size(0) != H or self.layout.size(1) * block != L:
                raise ValueError(f'layout {tuple(self.layout.shape)} with block {block} does not fit {H} heads of length {L}')
            return self.layout
        cfg = self.sparsity_config
        if cfg.stride % block != 0:
            raise ValueError(f'Stride {cfg.stride} must be dividable by block size {block}')
        return DeepSpeedSparseSelfAttention._make_layout(H, L // block, cfg.mode, cfg.stride // block,
                                                         cfg.attention, cfg.numverts, cfg.vertsize)

    def get_ops(self, H, L):
        """(sdd_nt, dsd_nn, softmax) for H heads of length L, built once
        (deepspeedsparseselfattention.py:67-106)."""
        key, ops, tiles = (H, L), self.ops, self.tiles      # (before the attributes: see __setattr__)
        found = ops.get(key)
        if found is None:
            layout, block = self.get_layout(H, L), self.block
            sdd_nt = MatMul(layout, block, 'sdd', trans_a=False, trans_b=True)
            dsd_nn = MatMul(layout, block, 'dsd', trans_a=False, trans_b=False)
            dsd_nn._meta = sdd_nt.meta            # one metadata buffer per layout
            found = (sdd_nt, dsd_nn, Softmax(layout, block))
            tiles[key] = sdd_nt.attn_tiles = tables.build_attn_tiles(layout, block) if self.fused else None
            ops[key] = found
        return found

    def _attn_op(self, query, H, L):
        """The fused attention with this module's tables on the device of `query`."""
        ops = self._attn
        sdd_nt, _, _ = self.get_ops(H, L)
        tiles = sdd_nt.attn_tiles if hasattr(sdd_nt, 'attn_tiles') else self.tiles[(H, L)]   # (in modules saved earlier)
        op = fused.Attention(sdd_nt.meta, tiles, self.block, query.device)
        ops[(H, L, query.get_device())] = op
        return op

    def _is_causal(self, attn_mask, owner=None):
        """True when a 'mul' attention mask is exactly the lower-triangular (causal) mask: the
        fused kernels then derive it from the indices.  The answer is remembered per tensor
        object and version (not per address: a freed tensor's address is reused).  `owner` is
        the tensor the caller handed in when `attn_mask` is a view or a converted copy made from
        it on the way here (forward() squeezes and casts the mask, which creates a new tensor
        object on every call): the answer is then remembered for the caller's tensor.  A caller
        that builds a new mask tensor for every call pays the comparison every time."""
        key = attn_mask if owner is None else owner
        entry = self._causal_cache.get(id(key))
        if entry is not None and entry[0]() is key and entry[1] == key._version:
            return entry[2]
        self.causal_checks += 1
        L = attn_mask.size(-1)
        hit = (attn_mask.dim() == 2 and attn_mask.size(0) == L and
               bool(torch.equal(attn_mask != 0, torch.ones((L, L), dtype=torch.bool, device=attn_mask.device).tril())))
        if len(self._causal_cache) > 16:
            self._causal_cache.clear()
        self._causal_cache[id(key)] = (weakref.ref(key), key._version, hit)
        return hit

    def graphed(self, query, key, value, dout, scale=None):
        """Forward + backward on the given [bsz, heads, L, head_dim] buffers as one CUDA graph (see
        fused.GraphedStep): `step = module.graphed(q, k, v, do)`, then `step.replay()` per step;
        results in step.o, step.dq, step.dk, step.dv.  No rpe / masks."""
        bsz, num_heads, tgt_len, head_dim = query.size()
        sdd_nt, _, _ = self.get_ops(num_heads, tgt_len)
        tiles = self.tiles.get((num_heads, tgt_len))
        return fused.GraphedStep(sdd_nt.meta, tiles, self.block, float(head_dim) ** -0.5 if scale is None else float(scale),
                                 query, key, value, dout)

    def transpose_key_for_scores(self, x, L):
        """deepspeedsparseselfattention.py:119-123: a key given as [.., hd, L] is
        viewed back as [.., L, hd]."""
        bsz, num_heads, seq_len, head_dim = x.size()
        if seq_len != L:
            return x.permute(0, 1, 3, 2)
        return x

    def transpose_mask_for_sparse(self, qtype, x, is_key_padding_mask=False):
        """deepspeedsparseselfattention.py:125-132."""
        if x.dtype != qtype:
            x = x.to(qtype)
        if x.dim() == 2 and 1 not in x.shape:
            return x
        if is_key_padding_mask:
            xdim = x.dim()
            for d in range(xdim - 1, 0, -1):
                x = x.squeeze(dim=d)
            return x
        return x.squeeze()

    def forward(self, query, key, value, rpe=None, key_padding_mask=None, attn_mask=None):
        key = _lib.ops().attention_key(query, key, value)       # (a key given as [.., hd, L] is viewed back)
        if key_padding_mask is not None:
            key_padding_mask = self.transpose_mask_for_sparse(query.dtype, key_padding_mask, is_key_padding_mask=True)
            if key_padding_mask.dim() == 1:
                key_padding_mask = key_padding_mask.unsqueeze(0)
        mask_owner = attn_mask
        if attn_mask is not None:
            attn_mask = self.transpose_mask_for_sparse(query.dtype, attn_mask)
        head_dim = query.size(3)
        if type(head_dim) is not int:                 # (torch.jit.trace: sizes are tensors)
            head_dim = int(head_dim)
        return self.attend(query, key, value, head_dim ** -0.5, rpe, key_padding_mask, attn_mask,
                           mask_owner=mask_owner)

    def attend(self, query, key, value, scaling, rpe=None, key_padding_mask=None, attn_mask=None, mask_owner=None,
               seq_first_out=False):
        """The attention core on [bsz, heads, L, head_dim] operands with an explicit score scale
        (masks already in the dtype of the operands).  `mask_owner`: the caller's own attention
        mask tensor when `attn_mask` was derived from it (see _is_causal).  `seq_first_out`: the
        fused kernel writes its result in [L, bsz, heads * head_dim] memory order (returned as the
        [bsz, heads, L, head_dim] view of it)."""
        _, num_heads, tgt_len, _ = query.shape
        if type(tgt_len) is not int:                  # (torch.jit.trace: sizes are tensors, each one a key of its own)
            num_heads, tgt_len = int(num_heads), int(tgt_len)
        if key_padding_mask is not None and key_padding_mask.dtype != query.dtype:
            key_padding_mask = key_padding_mask.to(query.dtype)
        if attn_mask is not None and attn_mask.dtype != query.dtype:
            if mask_owner is None:
                mask_owner = attn_mask
            attn_mask = attn_mask.to(query.dtype)
        if self.fused and fused.fused_supported(query, self.block):
            am_mode = self.attn_mask_mode
            if attn_mask is not None and am_mode == 'mul' and self._is_causal(attn_mask, mask_owner):
                am_mode = 'causal'
            op = self._attn.get((num_heads, tgt_len, query.get_device())) or self._attn_op(query, num_heads, tgt_len)
            return fused.attention(op, query, key, value, scaling, rpe, key_padding_mask, attn_mask,
                                   self.key_padding_mask_mode, am_mode, seq_first_out)
        sdd_nt, dsd_nn, softmax = self.get_ops(num_heads, tgt_len)
        w = sdd_nt(query, key)
        w = softmax(w, scale=scaling, rpe=rpe, key_padding_mask=key_padding_mask, attn_mask=attn_mask,
                    key_padding_mask_mode=self.key_padding_mask_mode, attn_mask_mode=self.attn_mask_mode)
        return dsd_nn(w, value)


    def decode(self, query, cache, pages, lengths, scale=None):
        """Attention of the newest tokens of every sequence over a KVCache that holds their keys and values
        already.  query [Z, heads, T, head_dim] (FP16 or BF16; heads a multiple of the cache's, neighbouring
        ones share a head of it); pages int32 [Z, slots], the sequences' page table (see KVCache);
        lengths int32 [Z], tokens of each sequence, the T new ones included.  Returns [Z, heads, T, head_dim].

        Query t stands at position lengths[z] - T + t and sees the keys up to its own position that lie in
        the nonzero blocks of its block-row: what forward() gives for that row under a causal
        attn_mask.  The layout is the module's own, [heads of the cache or 1, ...], or its configuration's for
        sequences as long as the page table; rows behind its end see nothing.  Positions below zero
        (sequences shorter than T) and queries that see nothing give zeros.  scale: head_dim ** -0.5
        (1.0 for queries that are scaled already, as MultiheadAttention scales them in front of its `core`);
        where scale times a query's largest channel is above 2 ** 119 its result is NaN.

        One kernel, without workspace, on the current stream of the cache's device; no gradient.  Lengths
        and tables are read on the device, so that a captured call can be replayed as sequences grow (the
        first call for a layout uploads its tables: not inside a capture)."""
        cache_op = cache._op()
        ops = self._attn
        key = (cache_op.heads, query.get_device(), None if self.layout is not None else pages.size(-1) * cache.page, 'decode')
        op = ops.get(key) or self._decode_op(ops, key, cache, query.device)
        return op(query, cache_op, pages, lengths, scale)

    def _decode_op(self, ops, key, cache, device):
        layout = self.layout
        if layout is None:
            # Layouts are made of whole windows; about 8 sizes between one power of two and the next serve tables of any
            # width (a table that grows page by page builds one now and then), each by its first rows.
            rows, block = max(1, -(-key[2] // self.block)), self.block
            window = max(1, self.sparsity_config.stride // block)
            step = window * max(1, (1 << rows.bit_length() >> 4) // window)
            size = -(-rows // step) * step
            meta = ops.get((*key[:2], size, 'rows'))
            if meta is None:
                meta = ops[(*key[:2], size, 'rows')] = tables.build_meta(self.get_layout(cache.num_heads, size * block))
        else:
            if layout.size(0) not in (1, cache.num_heads):
                raise ValueError(f'a layout of {layout.size(0)} heads does not fit a cache of {cache.num_heads}')
            rows, block, meta = layout.size(1), self.block, tables.build_meta(layout)
        op = ops[key] = _lib.ops().CacheAttentionOp(meta.hdr, meta.on(device), block, rows)
        return op


SparseSelfAttention = DeepSpeedSparseSelfAttention
