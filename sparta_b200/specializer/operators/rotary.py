"""``RotaryEmbedding``: rotary positions on queries and keys (``sparta_rotary``).  The reference's attention knows no
positions; the layer around it turns queries and keys before it calls the operator."""
import math
from decimal import Decimal, localcontext
from typing import Dict, List, Optional, Sequence, Tuple, Union

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


def _record(x: torch.Tensor, y: torch.Tensor, positions: Optional[torch.Tensor]):
    """(tensor to keep alive, ``sparta_rotary_tensor``): (..., N, E) as [batch, heads, n, dim] with strides, next to its
    positions."""
    if x.dim() > 4:
        x = x.flatten(0, -3)
    if x.stride(-1) != 1:
        x = x.contiguous()
    shape, s = x.shape, x.stride()
    n, rows, pos = shape[-2], 1, None
    if positions is not None:
        pos = positions.data_ptr()
        if positions.dim() == 2:
            rows = positions.shape[0]
        if positions.shape[-1] != n:
            raise ValueError(f'{positions.shape[-1]} positions for {n} tokens')
    if len(shape) == 4:
        batch, heads = shape[0], shape[1]
        if rows != 1 and rows != batch:
            raise ValueError(f'positions of {rows} sequences for a batch of {batch}')
        sb, sh, sn = s[0], s[1], s[2]
    elif len(shape) == 3:
        if shape[0] % rows:
            raise ValueError(f'positions of {rows} sequences for {shape[0]} heads')
        batch, heads = rows, shape[0] // rows
        sb, sh, sn = heads * s[0], s[0], s[1]
    else:
        if rows != 1:
            raise ValueError(f'positions of {rows} sequences for one')
        batch, heads, sb, sh, sn = 1, 1, 0, 0, s[0]
    return x, _lib.RotaryTensor(x.data_ptr(), y.data_ptr(), pos, sb, sh, sn, batch, heads, n, 1 if rows > 1 else 0)


_Two = _lib.RotaryTensor * 2


def _launch(module: 'RotaryEmbedding', tensors: Sequence[torch.Tensor], positions: Sequence[Optional[torch.Tensor]],
            backward: bool) -> List[torch.Tensor]:
    outs, records, keep, wide = [], [], [], 0
    for x, pos in zip(tensors, positions):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        outs.append(y)
        if x.numel() > 0:
            held, record = _record(x, y, pos)
            keep.append(held)
            records.append(record)
            if pos is not None:
                wide = pos.dtype == torch.int64
    if records:
        x = keep[0]
        device = x.device
        with _lib.on_device(device):
            _lib.check(_lib.lib().sparta_rotary(
                _Two(*records), len(records), module._turns(device).data_ptr(), module.head_dim, module.rotary_dim,
                module.interleaved, module.magnitude, backward, wide, _lib.dtype_code(x), _lib.stream_ptr(device)),
                'sparta_rotary')
    return outs


class RotaryFunc(torch.autograd.Function):

    @staticmethod
    def forward(ctx, module: 'RotaryEmbedding', backward: bool, query_positions, key_positions, *tensors):
        ctx.module, ctx.reverse = module, not backward
        ctx.save_for_backward(query_positions, key_positions)
        ctx.set_materialize_grads(False)
        return tuple(_launch(module, tensors, (query_positions, key_positions), backward))

    @staticmethod
    def backward(ctx, *grads):
        positions = ctx.saved_tensors
        wanted = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[4 + i]]
        out: List[Optional[torch.Tensor]] = [None] * len(grads)
        if wanted:
            pos, given = [positions[i] for i in wanted] + [None], [grads[i] for i in wanted]
            # linear: the gradient's own gradient is the same operator; the plain launch skips autograd's bookkeeping
            turned = (RotaryFunc.apply(ctx.module, ctx.reverse, pos[0], pos[1], *given) if torch.is_grad_enabled()
                      else _launch(ctx.module, given, pos, ctx.reverse))
            for i, g in zip(wanted, turned):
                out[i] = g
        return (None, None, None, None, *out)


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
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, int(bool(interleaved))
        self.scaling, self.factor, self.base, self.original_length = scaling, factor, base, original_length
        freq, self.magnitude = rotary_frequencies(rotary_dim, base, scaling, factor, original_length)
        self._turn_list = as_turns(freq)
        self._turns_of: Dict[torch.device, torch.Tensor] = {}

    def _turns(self, device: torch.device) -> torch.Tensor:
        if device not in self._turns_of:
            self._turns_of[device] = torch.tensor(self._turn_list, dtype=torch.int64, device=device)
        return self._turns_of[device]

    def _check(self, x: torch.Tensor, positions: Optional[torch.Tensor], first: torch.Tensor):
        _lib.require_cuda(x)
        _lib.dtype_code(x)
        if x.dim() < 2 or x.shape[-1] != self.head_dim:
            raise ValueError(f'expected (..., N, {self.head_dim}), got {tuple(x.shape)}')
        if x.dtype != first.dtype or x.device != first.device:
            raise ValueError('queries and keys have to be of one type on one device')
        if positions is not None:
            if positions.dtype not in (torch.int32, torch.int64) or positions.dim() not in (1, 2):
                raise ValueError('positions have to be int32 or int64, (N,) or (B, N)')
            if positions.device != x.device:
                raise ValueError(f'positions are on {positions.device}, the input on {x.device}')

    def forward(self, query: torch.Tensor, key: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                key_positions: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        if key is not None and key_positions is None:
            key_positions = positions
        if key_positions is not positions and key_positions is not None and positions is not None \
                and key_positions.dtype != positions.dtype:
            positions, key_positions = positions.long(), key_positions.long()
        self._check(query, positions, query)
        if positions is not None:
            positions = positions.contiguous()
        if key is None:
            return RotaryFunc.apply(self, False, positions, None, query)[0]
        self._check(key, key_positions, query)
        if key_positions is not None:
            key_positions = key_positions.contiguous()
        return RotaryFunc.apply(self, False, positions, key_positions, query, key)

    def extra_repr(self) -> str:
        return (f'head_dim={self.head_dim}, rotary_dim={self.rotary_dim}, base={self.base}, '
                f'interleaved={bool(self.interleaved)}, scaling={self.scaling!r}')
