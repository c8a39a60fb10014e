"""``SparseDropout``: dropout whose decisions come from a counter and are never stored (``sparta_dropout``,
``sparta_dropout_blocks``).  The reference has no dropout; a training step of an attention layer needs it on the
attention probabilities, which this package keeps as block values or never forms at all."""
from typing import NamedTuple, Optional

import torch

from sparta_b200 import _lib
from sparta_b200.tesa import BCSIndexes


class DropoutKey(NamedTuple):
    """What selects the random numbers of one call: ``rng`` on the device, or the two host numbers."""
    rng: Optional[torch.Tensor]
    seed: int
    call: int


def check_probability(p: float) -> float:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f'dropout probability has to be between 0 and 1, got {p}')
    return p


def signed64(seed: int) -> int:
    """The lower 64 bits of a seed as a signed number."""
    seed &= (1 << 64) - 1
    return seed - (1 << 64) if seed >> 63 else seed


class _Counter(object):
    """Host-side random state of a module: a seed and the number of training calls so far."""

    def __init__(self, seed: Optional[int]):
        self.drawn = seed is None
        self.seed = int(torch.randint(0, 1 << 62, (), dtype=torch.int64)) if seed is None else int(seed)
        self.calls = 0

    def __deepcopy__(self, memo) -> '_Counter':
        """A copied layer is another layer: it drops other positions, unless its seed was chosen."""
        copy = _Counter(None if self.drawn else self.seed)
        if not self.drawn:
            copy.calls = self.calls
        return copy

    def next(self, rng: Optional[torch.Tensor]) -> DropoutKey:
        if rng is not None:
            return DropoutKey(rng, 0, 0)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError('a captured graph would repeat the same dropout at every replay: pass rng, an int64 '
                               'tensor (seed, call number) on the GPU, and rewrite it between replays')
        key = DropoutKey(None, signed64(self.seed), self.calls)
        self.calls += 1
        return key


def sparse_dropout(x: torch.Tensor, p: float, key: DropoutKey, indexes: Optional[BCSIndexes] = None) -> torch.Tensor:
    """Dropout of ``x`` with the random numbers of ``key``; see ``SparseDropout``."""
    if indexes is None:
        return _lib.torch_ops().dropout(x, p, key.rng, key.seed, key.call, None, None, 0, 0, 0)
    if indexes.batched or not indexes.BCSR:
        raise ValueError('dropout of block values needs the BCSR indexes of one 2-D mask')
    if indexes.block_W < 8:
        raise ValueError(f'dropout of block values needs blocks at least 8 wide, got {indexes.block_W}')
    if indexes.bcsr_buf.device != x.device:
        raise ValueError(f'the indexes are on {indexes.bcsr_buf.device}, the input on {x.device}')
    if x.dim() == 0 or x.shape[-1] != indexes.val_stride_blocks * indexes.block_H * indexes.block_W:
        raise ValueError(f'the input of shape {tuple(x.shape)} does not hold the block values of these indexes')
    return _lib.torch_ops().dropout(x, p, key.rng, key.seed, key.call, indexes.bcsr_buf, indexes.nnz_dev, indexes.block_H,
                                    indexes.block_W, indexes.val_stride_blocks)


class SparseDropout(torch.nn.Module):
    r"""Dropout :math:`y = x \cdot keep / (1 - p)` with decisions from a counter-based generator.

    Whether position (batch element, row, column) of a call is kept depends on those three numbers, a seed and the
    call's number alone: the backward pass draws the same decisions again, nothing is stored, and dense tensors,
    block values of any block size and the fused attention agree.  ``p`` is rounded to a multiple of 1 / 65536.

    Args:
        p: probability that an element is dropped.
        seed: 64-bit seed (default: drawn from torch's generator, again for every deep copy of the module).  Modules
            with one seed drop alike.

    Shape: any shape (columns up to 2^30), float32 / float16 / bfloat16; the last two dimensions are rows and columns,
    those before them together the batch.  With ``indexes`` (``get_sparse_indexes()`` of an operator) the input holds block values
    :math:`(*, nnz \cdot BH \cdot BW)`.

    ``forward(x, rng=None, indexes=None)``: without ``rng`` the module's seed and its count of calls select the
    numbers; ``rng``, an int64 tensor (seed, call number) on the GPU, replaces both and is what a captured graph
    needs, and a forward pass that is run again for its gradients (activation checkpointing).  In evaluation mode, and for ``p == 0``, the input is returned.
    """

    def __init__(self, p: float = 0.5, seed: Optional[int] = None):
        super().__init__()
        self.p = check_probability(p)
        self._counter = _Counter(seed)

    def forward(self, x: torch.Tensor, rng: Optional[torch.Tensor] = None,
                indexes: Optional[BCSIndexes] = None) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x
        _lib.require_cuda(x)
        return sparse_dropout(x, self.p, self._counter.next(rng), indexes)

    def get_extra_state(self):
        return {'seed': self._counter.seed, 'calls': self._counter.calls}

    def set_extra_state(self, state):
        self._counter.seed, self._counter.calls = int(state['seed']), int(state['calls'])

    def extra_repr(self) -> str:
        return f'p={self.p}'
