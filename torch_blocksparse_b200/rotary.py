"""Rotary positions: pairs of channels of queries and keys turned by angles that grow with a token's position.

Next to the attention of this package, which knows of no positions beyond its layout (the reference
has none either): turned queries and keys make their products depend on distances.  One axis is the
position in a text; two are the rows and columns of an image's patches, three a video's frames as
well.  The checks, the autograd function and the launch are in csrc/torch/serving.cpp.
"""
from fractions import Fraction

import torch

from . import _lib, tracing
from .tracing import recording

_TWO_PI = 2 * Fraction(3141592653589793238462643383279502884197, 10 ** 39)


class Rotary(_lib.WithOps):
    """Rotary(head_dim, sections=None, base=10000., interleaved=False, frequencies=None)

    sections     pairs of channels for each axis, in order; the first 2 * sum(sections) channels are
                 turned, the others left as they are.  None: one axis over all channels.
    base         pair i of an axis with n pairs turns by position * base ** (-i / n).
    interleaved  a pair is two neighbouring channels (0, 1), (2, 3), ...; otherwise channel i and
                 channel sum(sections) + i.
    frequencies  radians per position for every pair of all sections, in place of base's.

    rotary(query, key=None, positions=None) takes [Z, H, L, head_dim] operands of one type (FP32, FP16
    or BF16; any strides; the numbers of heads may differ) and returns the turned query, or query and
    key, as new tensors in their operands' memory order.  positions: int32 or int64 on the same device,
    [axes, L] or [axes, Z, L], or [L] for one axis, negative ones too; None: 0, 1, .. L - 1 on one axis.
    Angles are off by at most |position| * 2^-62 radians, sines and cosines beyond that by 2^-21 of themselves.
    Both operands are differentiable (the gradient is turned back), positions are not.  The first call on a
    device uploads a table: not inside a capture.
    """

    _op_attributes = frozenset(('head_dim', 'sections', 'base', 'interleaved', 'frequencies'))

    def __init__(self, head_dim, sections=None, base=10000., interleaved=False, frequencies=None):
        if head_dim < 2 or head_dim > 256 or head_dim % 2 != 0:
            raise ValueError('head_dim must be even and at most 256')
        sections = (head_dim // 2,) if sections is None else tuple(int(n) for n in sections)
        if not sections or min(sections) < 0 or sum(sections) < 1 or 2 * sum(sections) > head_dim:
            raise ValueError(f'sections {sections} must be numbers of pairs, at most {head_dim // 2} in all')
        if frequencies is not None and len(frequencies) != sum(sections):
            raise ValueError(f'{len(frequencies)} frequencies for {sum(sections)} pairs')
        if not base > 0:
            raise ValueError('base must be positive')
        self.head_dim = head_dim
        self.sections = sections
        self.base = base
        self.interleaved = interleaved
        self.frequencies = None if frequencies is None else tuple(float(f) for f in frequencies)
        self._ops = _lib.OpCache()           # native operation per device index

    def turns(self):
        """For every pair, what a position adds to its angle as a 64-bit fraction of a whole turn."""
        freq = self.frequencies
        if freq is None:
            freq = [float(self.base) ** (-i / n) for n in self.sections for i in range(n)]
        turns = [round(Fraction(f) / _TWO_PI * 2 ** 64) % 2 ** 64 for f in freq]
        return [t - 2 ** 64 if t >= 2 ** 63 else t for t in turns]

    def _op(self, device):
        ops = self._ops
        axis = [a for a, n in enumerate(self.sections) for _ in range(n)]
        table = torch.tensor([self.turns(), axis], dtype=torch.int64).to(device)
        op = _lib.ops().RotaryOp(table, self.head_dim, len(self.sections), self.interleaved)
        ops[device.index] = op
        return op

    def __call__(self, query, key=None, positions=None):
        if not query.is_cuda:
            raise RuntimeError(f'torch_blocksparse_b200 runs on CUDA tensors only (got a {query.device} tensor)')
        op = self._ops.get(query.get_device()) or self._op(query.device)
        if recording() is not None:
            op.check(query, key)
            q = tracing.call(op, 'one', query, positions)
            return q if key is None else (q, tracing.call(op, 'one', key, positions))
        q, k = op(query, key, positions)
        return q if key is None else (q, k)
