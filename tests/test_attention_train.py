"""Host side of the attention training step: refusals of the C entries, struct layout.  No GPU."""
import ctypes

from sparta_b200 import _lib

FAKE = 0x10000  # never dereferenced: the calls below are refused first


def args(**kw):
    d = dict(Q=FAKE, K=FAKE, V=FAKE, O=FAKE, lse=FAKE, dO=FAKE, dQ=FAKE, dK=FAKE, dV=FAKE, workspace=FAKE, workspace_bytes=1 << 40,
             row_ptr=FAKE, bcsr_idx=FAKE, dropout=0.0, scale=0.125, heads=4, kv_heads=2, Nt=128, Ns=192, D=64, BLK=64, dtype=1,
             status=FAKE)
    d.update(kw)
    return ctypes.byref(_lib.AttnTrainArgs(**d))


def test_struct_layout():
    assert ctypes.sizeof(_lib.AttnTrainArgs) == 15 * 8 + 3 * 8 + 8 + 8 + 8 * 4
    assert ctypes.sizeof(_lib.RotaryTensor) == 3 * 8 + 3 * 8 + 4 * 4


def test_refusals():
    L = _lib.lib()
    for fn in (L.sparta_attn_train_fwd, L.sparta_attn_train_bwd):
        assert fn(None, None) == -1
        for name in ('Q', 'K', 'V', 'O', 'row_ptr', 'bcsr_idx'):
            assert fn(args(**{name: None}), None) == -1
        for name in ('heads', 'kv_heads', 'Nt', 'Ns'):
            assert fn(args(**{name: 0}), None) == -1
        for p in (-0.5, 1.5, float('nan')):
            assert fn(args(dropout=p), None) == -1
        assert fn(args(dtype=0), None) == -3 and fn(args(D=96), None) == -3 and fn(args(BLK=32), None) == -3
        assert fn(args(scale=0.0), None) == -3 and fn(args(Ns=65536 + 64), None) == -3
        assert fn(args(Nt=100), None) == -2 and fn(args(Ns=100), None) == -2 and fn(args(kv_heads=3), None) == -2
        assert fn(args(heads=1 << 26, kv_heads=1 << 26), None) == -2
        for name in ('Q', 'K', 'V', 'O', 'mask'):
            assert fn(args(**{name: FAKE + 8}), None) == -5
        assert fn(args(rng=FAKE + 4), None) == -5 and fn(args(lse=FAKE + 2), None) == -5
    bwd = L.sparta_attn_train_bwd
    for kw in (dict(lse=None), dict(dO=None), dict(dK=None), dict(dV=None), dict(dQ=None, dK=None, dV=None)):
        assert bwd(args(**kw), None) == -1
    for name in ('dO', 'dQ', 'dK', 'dV', 'workspace'):
        assert bwd(args(**{name: FAKE + 8}), None) == -5
    need = L.sparta_attn_train_bwd_workspace_bytes(4, 2, 128, 192, 64, 0)
    assert need >= 2 * 4 * 128 * 4 + 2 * 3
    assert bwd(args(workspace_bytes=need - 1), None) == -4 and bwd(args(workspace=None), None) == -4
    assert bwd(args(Nt=65536 + 64), None) == -3
    assert bwd(args(nnz_hint=-1), None) == -1
    for bad in ((0, 1, 128, 128, 64, 0), (4, 3, 128, 128, 64, 0), (4, 2, 128, 128, 96, 0), (4, 2, 128, 128, 64, -1)):
        assert L.sparta_attn_train_bwd_workspace_bytes(*bad) == 0
    # tiles that several CTAs share leave partial sums in the workspace: it grows with the kept blocks up to a bound
    long = (4, 1, 65536, 65536, 128)
    sizes = [L.sparta_attn_train_bwd_workspace_bytes(*long, n) for n in (0, 2000, 20000, 1 << 20)]
    assert sizes[0] < sizes[1] and sizes[0] == sizes[3] and max(sizes) <= sizes[0] + (256 << 20)
    assert bwd(args(workspace_bytes=need, nnz_hint=0, workspace=None), None) == -4


def test_room_for_dropout_decisions():
    f = _lib.lib().sparta_attn_train_bwd_dropout_bytes
    assert f(16, 100) == 16 * 100 * 64 * 64 // 8  # a bit per kept score
    assert f(0, 100) == 0 and f(-1, 100) == 0 and f(16, 0) == 0 and f(16, -5) == 0
    # a bound, and whole blocks of every head below it
    assert f(16, 1 << 40) <= 1 << 30 and f(16, 1 << 40) % (16 * 512) == 0 and f(1 << 30, 1) == 0
