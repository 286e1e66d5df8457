"""A paged cache of keys and values in 4 bits, for serving what SparseSelfAttention trains.

The reference has no cache: it computes whole sequences.  SparseSelfAttention.decode attends over this
one.  The checks and launches are in csrc/torch/serving.cpp, the kernels in csrc/cache.cu and
csrc/cache_attn.cu, the format in csrc/cache.cuh.
"""
import torch

from . import _lib
from .tracing import recording


class KVCache(_lib.WithOps):
    """KVCache(num_pages, num_heads, head_dim, page=64, device='cuda')

    Room for num_pages pages of `page` tokens (a power of two from 16 to 1024) of num_heads heads of 64
    or 128 channels, 4.5 bits a value: for each token, head and 32 channels a scale s = bf16(max |x| / 7)
    and codes rint(x / s) in [-8, 7], standing for s * code.  A group with an infinity or a NaN reads
    back as NaN.  `data` (uint8, zeros at first, which reads as numbers) is the whole of it, in a format of its own.

    Which page holds which tokens is the caller's table: `pages`, int32 [Z, slots] on the cache's device,
    names the page of tokens slot * page .. slot * page + page - 1 of every sequence; an entry that is no
    page (-1, or any number outside 0 .. num_pages - 1) has none: its tokens are not written, read as zeros and
    are not attended to.  Pages may be shared by sequences that only read them.

    Calls run on the current stream of the cache's device, do not synchronise and can be captured
    into a graph; tables and lengths are read on the device.  Nothing here is differentiable.
    """

    _op_attributes = frozenset(('data', 'page', 'head_dim'))

    def __init__(self, num_pages, num_heads, head_dim, page=64, device='cuda'):
        if head_dim not in (64, 128):
            raise NotImplementedError(f'head dimension {head_dim} (64 and 128 are supported)')
        size = _lib.lib().bsp_cache_page_bytes(page, head_dim)
        if size < 0:
            raise ValueError(f'pages of {page} tokens (a power of two from 16 to 1024 is needed)')
        if num_pages < 0 or num_heads < 1 or num_pages >= 2 ** 31:
            raise ValueError(f'a cache of {num_pages} pages of {num_heads} heads')
        device = torch.device(device)
        if device.type != 'cuda':
            raise RuntimeError(f'torch_blocksparse_b200 runs on CUDA tensors only (got device {device})')
        self.head_dim = head_dim
        self.page = page
        self.data = torch.zeros((num_pages, num_heads, size), dtype=torch.uint8, device=device)
        self._ops = _lib.OpCache()

    @property
    def num_pages(self):
        return self.data.size(0)

    @property
    def num_heads(self):
        return self.data.size(1)

    def _op(self):
        if recording() is not None:
            raise RuntimeError('a KVCache changes between calls, which torch.jit.trace cannot replay')
        ops = self._ops                      # (before the attributes: see WithOps)
        op = ops.get('op')
        if op is None:
            d = self.data
            if d.dtype != torch.uint8 or not d.is_cuda or d.dim() != 3 or not d.is_contiguous() or \
                    d.size(2) != _lib.lib().bsp_cache_page_bytes(self.page, self.head_dim):
                raise ValueError('data must be a contiguous uint8 CUDA tensor [pages, heads, bytes of a page]')
            op = ops['op'] = _lib.ops().CacheOp(d, self.page, self.head_dim)
        return op

    def write(self, key, value, pages, start, count=None):
        """Quantises key and value [Z, num_heads, T, head_dim] (FP16 or BF16, any strides) into positions
        start[z] .. of every sequence; start, and count where only the first count[z] of the T tokens are
        there (a padded batch), are int32 [Z].  What else the cache holds stays as it is.  Sequences of one
        call must not share pages that are written."""
        self._op().write(key, value, pages, start, count)

    def read(self, pages, start, length, count=None, dtype=torch.float16):
        """Keys and values of positions start[z] .. start[z] + length - 1 as two [Z, num_heads, length,
        head_dim] tensors of dtype (FP32, FP16 or BF16); zeros from token count[z] on."""
        return self._op().read(pages, start, length, count, dtype)
