"""``RotaryEmbedding``: rotary positions on queries and keys (``sparta_rotary``).  The reference's attention knows no
positions; the layer around it turns queries and keys before it calls the operator."""
import math
from decimal import Decimal, localcontext
from typing import Dict, List, Optional, Tuple, Union

import torch

from sparta_b200 import _lib

_SCALINGS = ('none', 'linear', 'ntk', 'yarn')
_TWO_PI = Decimal('6.28318530717958647692528676655900576839433879875')


def rotary_frequencies(rotary_dim: int, base: float, scaling: str, factor: float,
                       original_length: Optional[int]) -> Tuple[List[float], float]:
    """(angle per position of every pair, factor on the turned values).

    'linear' divides the positions by ``factor``; 'ntk' raises the base so that the lowest frequency is divided by
    ``factor``; 'yarn' (Peng, Quesnelle, Fan, Shippole, "YaRN: efficient context window extension", 2023) divides the
    frequencies that turn less than once in ``original_length`` positions, keeps those that turn more than 32 times,
    blends between, and scales the values by 0.1 ln(factor) + 1."""
    if scaling == 'ntk' and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    magnitude = 1.0
    if scaling == 'linear':
        freq = [f / factor for f in freq]
    elif scaling == 'yarn':
        def blend(f):
            whole = min(1.0, max(0.0, (original_length * f / (2 * math.pi) - 1.0) / 31.0))
            return f / factor * (1.0 - whole) + f * whole
        freq = [blend(f) for f in freq]
        magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    return freq, magnitude


def as_turns(freq: List[float]) -> List[int]:
    """Angles per position as 64-bit fractions of a turn, in two's complement."""
    with localcontext() as context:
        context.prec = 60
        whole = [int((Decimal(f) / _TWO_PI * (1 << 64)).to_integral_value()) % (1 << 64) for f in freq]
    return [w - (1 << 64) if w >= 1 << 63 else w for w in whole]


class RotaryEmbedding(torch.nn.Module):
    r"""Rotary positions: each pair of the first ``rotary_dim`` elements of a head is turned by
    :math:`position \cdot f_i`, :math:`f_i = base^{-2 i / rotary\_dim}`; the rest of the head is copied.

    Args:
        head_dim: elements of a head.
        rotary_dim: elements that are turned (even; default: all).
        base: base of the frequencies.
        interleaved: pairs are (2 i, 2 i + 1); default (i, i + rotary_dim / 2).
        scaling: 'none', 'linear', 'ntk' or 'yarn' by ``factor`` (see ``rotary_frequencies``); 'yarn' needs
            ``original_length``.

    ``forward(query, key=None, positions=None, key_positions=None)``: tensors (..., N, E) in the attention's order --
    (B, H, N, E) or (B * H, N, E) -- of any strides with contiguous heads, float32 / float16 / bfloat16; both are
    turned in one launch.  ``positions``: int32 or int64, (N,) or one row per sequence (B, N); default 0, 1, 2 ...
    Keys take the queries' positions unless ``key_positions`` is given.  Outputs are contiguous.  Angles are exact to
    about 2e-7 radians for positions of up to 31 bits.
    """

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, interleaved: bool = False,
                 scaling: str = 'none', factor: float = 1.0, original_length: Optional[int] = None):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim <= 0 or rotary_dim <= 0 or rotary_dim > head_dim or rotary_dim % 2:
            raise ValueError(f'rotary_dim has to be even and at most head_dim, got {rotary_dim} of {head_dim}')
        if scaling not in _SCALINGS:
            raise ValueError(f'scaling has to be one of {_SCALINGS}, got {scaling!r}')
        if not base > 0 or not factor > 0 or not math.isfinite(base) or not math.isfinite(factor):
            raise ValueError('base and factor have to be positive numbers')
        if scaling == 'yarn' and not (original_length and original_length > 0):
            raise ValueError("scaling 'yarn' needs original_length")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, bool(interleaved)
        self.scaling, self.factor, self.base, self.original_length = scaling, factor, base, original_length
        freq, self.magnitude = rotary_frequencies(rotary_dim, base, scaling, factor, original_length)
        self._turn_list = as_turns(freq)
        self._turns_of: Dict[torch.device, torch.Tensor] = {}

    def _turns(self, device: torch.device) -> torch.Tensor:
        if device not in self._turns_of:
            self._turns_of[device] = torch.tensor(self._turn_list, dtype=torch.int64, device=device)
        return self._turns_of[device]

    def forward(self, query: torch.Tensor, key: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                key_positions: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        _lib.require_cuda(query)
        out = _lib.torch_ops().rotary(query, key, positions, key_positions, self._turns(query.device), self.head_dim,
                                      self.rotary_dim, self.interleaved, self.magnitude)
        return out[0] if key is None else (out[0], out[1])

    def extra_repr(self) -> str:
        return (f'head_dim={self.head_dim}, rotary_dim={self.rotary_dim}, base={self.base}, '
                f'interleaved={self.interleaved}, scaling={self.scaling!r}')
