"""Host side of the counter-based dropout and the rotary positions: the oracle's generator against published vectors,
refusals, frequencies.  No GPU."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_training as oracle
from sparta_b200 import _lib
from sparta_b200.nn import RotaryEmbedding, SparseDropout
from sparta_b200.specializer.operators.rotary import as_turns, rotary_frequencies

FAKE = 0x1000  # never dereferenced: the calls below are refused first


def test_philox_known_answer():
    """First vector of the generator's published known-answer list (seven rounds, all zeros)."""
    got = oracle.philox4x32([0, 0, 0, 0], [0, 0])
    assert [int(v) for v in got] == [0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48]


@pytest.mark.parametrize('p', [0.0, 0.1, 0.5, 0.93, 1.0])
def test_kept_share(p):
    """The kept share lies within six standard deviations of 1 - p (n = 2^17 decisions)."""
    keep = oracle.dropout_keep(5, 3, 2, 64, 1024, p)
    n = keep.numel()
    assert abs(keep.double().mean().item() - (1 - p)) <= 6 * math.sqrt(p * (1 - p) / n) + 1 / 131072
    assert abs((1 - oracle.dropout_threshold(p) / 65536) * oracle.dropout_scale(p) - (p < 1)) < 1e-12


def test_dropout_refusals():
    L = _lib.lib()
    ok = (FAKE, FAKE, 1, 4, 8)
    assert L.sparta_dropout(None, FAKE, 1, 4, 8, 0.5, None, 0, 0, 0, None) == -1
    assert L.sparta_dropout(FAKE, None, 1, 4, 8, 0.5, None, 0, 0, 0, None) == -1
    assert L.sparta_dropout(FAKE, FAKE, 0, 4, 8, 0.5, None, 0, 0, 0, None) == -1
    for p in (-0.1, 1.1, math.nan):
        assert L.sparta_dropout(*ok, p, None, 0, 0, 0, None) == -1
    assert L.sparta_dropout(*ok, 0.5, None, 0, 0, 3, None) == -1
    assert L.sparta_dropout(FAKE, FAKE + 8, 1, 4, 8, 0.5, None, 0, 0, 0, None) == -5
    assert L.sparta_dropout(FAKE + 1, FAKE, 1, 4, 8, 0.5, None, 0, 0, 1, None) == -5
    assert L.sparta_dropout(*ok, 0.5, FAKE + 4, 0, 0, 0, None) == -5
    assert L.sparta_dropout(FAKE, FAKE, 1 << 30, 1 << 30, 1 << 30, 0.5, None, 0, 0, 0, None) == -2
    blocks = (FAKE, FAKE, FAKE, FAKE, 1, 32, 32, 4)
    assert L.sparta_dropout_blocks(FAKE, FAKE, None, FAKE, 1, 32, 32, 4, 0.5, None, 0, 0, 0, None) == -1
    assert L.sparta_dropout_blocks(FAKE, FAKE, FAKE, FAKE, 1, 32, 4, 4, 0.5, None, 0, 0, 0, None) == -2
    assert L.sparta_dropout_blocks(FAKE, FAKE, FAKE, FAKE, 1, 24, 32, 4, 0.5, None, 0, 0, 0, None) == -2
    assert L.sparta_dropout_blocks(FAKE, FAKE, FAKE, FAKE, 65536, 32, 32, 4, 0.5, None, 0, 0, 0, None) == -2
    assert L.sparta_dropout_blocks(*blocks, 2.0, None, 0, 0, 0, None) == -1
    for p in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError):
            SparseDropout(p)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        SparseDropout(0.5)(torch.ones(4))
    x = torch.ones(4)
    assert SparseDropout(0.0)(x) is x and SparseDropout(0.5).eval()(x) is x


def test_dropout_state_round_trip():
    a, b = SparseDropout(0.5, seed=7), SparseDropout(0.5, seed=8)
    a._counter.calls = 41
    b.load_state_dict(a.state_dict())
    assert (b._counter.seed, b._counter.calls) == (7, 41)
    torch.manual_seed(3)
    first = SparseDropout(0.5)._counter.seed
    torch.manual_seed(3)
    assert SparseDropout(0.5)._counter.seed == first


def test_copies_of_a_module_drop_other_positions():
    import copy
    import pickle
    drawn, chosen = SparseDropout(0.5), SparseDropout(0.5, seed=3)
    drawn._counter.calls = chosen._counter.calls = 5
    one, other = copy.deepcopy(drawn), copy.deepcopy(drawn)
    assert len({drawn._counter.seed, one._counter.seed, other._counter.seed}) == 3 and one._counter.calls == 0
    same = copy.deepcopy(chosen)
    assert (same._counter.seed, same._counter.calls) == (3, 5)
    stored = pickle.loads(pickle.dumps(drawn))
    assert (stored._counter.seed, stored._counter.calls) == (drawn._counter.seed, 5)


@pytest.mark.parametrize('scaling', ['none', 'linear', 'ntk', 'yarn'])
def test_rotary_frequencies(scaling):
    freq, magnitude = rotary_frequencies(64, 10000.0, scaling, 8.0, 4096)
    plain, _ = rotary_frequencies(64, 10000.0, 'none', 1.0, None)
    assert len(freq) == 32 and all(a > b for a, b in zip(freq, freq[1:]))
    lowest = {'none': 1.0, 'linear': 8.0, 'ntk': 8.0, 'yarn': 8.0}[scaling]
    assert math.isclose(plain[-1] / freq[-1], lowest, rel_tol=1e-12)
    highest = 8.0 if scaling == 'linear' else 1.0
    assert math.isclose(plain[0] / freq[0], highest, rel_tol=1e-12)
    assert math.isclose(magnitude, 0.1 * math.log(8.0) + 1.0 if scaling == 'yarn' else 1.0)


def test_turns_are_exact():
    """Position times the 64-bit fraction of a turn, modulo a turn, against the angle in 64-bit floating point: they may
    differ by the latter's rounding, position * f * 2^-52, and by position * 2^-65 turns."""
    freq, _ = rotary_frequencies(128, 10000.0, 'none', 1.0, None)
    for f, turn in zip(freq, as_turns(freq)):
        for pos in (0, 1, 77, 4095, 1 << 20, (1 << 24) + 1, -5):
            angle = (turn * pos) % (1 << 64) / 2.0 ** 64 * 2 * math.pi
            far = abs(math.remainder(angle - pos * f, 2 * math.pi))
            assert far <= abs(pos) * (f * 2.0 ** -51 + 2 * math.pi * 2.0 ** -65) + 1e-14


def test_rotary_refusals():
    L = _lib.lib()
    def rec(**kw):
        d = dict(x=FAKE, y=FAKE, positions=FAKE, stride_batch=64, stride_head=64, stride_token=64, batch=1, heads=1, n=4,
                 positions_per_batch=0)
        d.update(kw)
        return (_lib.RotaryTensor * 1)(_lib.RotaryTensor(**d))
    def call(r, count=1, turns=FAKE, dim=64, rotary=64, pos64=1, dtype=0):
        return L.sparta_rotary(r, count, turns, dim, rotary, 0, 1.0, 0, pos64, dtype, None)
    assert call(None) == -1 and call(rec(), count=3) == -1 and call(rec(), turns=None) == -1
    assert call(rec(x=None)) == -1 and call(rec(y=None)) == -1 and call(rec(n=0)) == -1 and call(rec(heads=-1)) == -1
    assert call(rec(), dtype=3) == -1
    assert call(rec(), rotary=66) == -2 and call(rec(), rotary=31) == -2
    assert call(rec(x=FAKE + 2)) == -5 and call(rec(positions=FAKE + 4)) == -5 and call(rec(), turns=FAKE + 4) == -5
    assert call(rec(batch=1 << 30, n=1 << 30, heads=1 << 30)) == -2
    for bad in (dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=31), dict(head_dim=64, rotary_dim=0),
                dict(head_dim=7), dict(head_dim=64, scaling='other'), dict(head_dim=64, base=0.0),
                dict(head_dim=64, factor=-1.0), dict(head_dim=64, scaling='yarn'), dict(head_dim=64, base=math.inf)):
        with pytest.raises(ValueError):
            RotaryEmbedding(**bad)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        RotaryEmbedding(8)(torch.ones(2, 3, 8))
