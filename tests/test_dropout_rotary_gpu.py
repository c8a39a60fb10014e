"""Counter-based dropout and rotary positions on the GPU against the 64-bit oracle."""
import itertools

import pytest
import torch

from oracle import attention_training as oracle
from sparta_b200.nn import RotaryEmbedding, SparseDropout
from sparta_b200.specializer.operators.rotary import rotary_frequencies
from sparta_b200.tesa import get_bcs_function

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def rng(seed, call):
    return torch.tensor([seed, call], dtype=torch.int64, device='cuda')


def close(got, want, dtype, absolute=0.0):
    """One rounding of the type, and of the 32-bit product before it: half a step each, relative to the value."""
    rel = torch.finfo(dtype).eps / 2 + torch.finfo(torch.float32).eps
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # half a step of the subnormal numbers and more
    off = (got.double().cpu() - want).abs()
    assert bool((off <= rel * want.abs() * (1 + 1e-6) + tiny + absolute).all()), (off - rel * want.abs()).max().item()


# ---- dropout ---------------------------------------------------------------------------------------------------
SHAPES = [(1,), (7,), (8,), (5, 1), (3, 4, 5), (2, 3, 8), (1, 1, 1024), (2, 5, 1001), (3, 33, 257), (1, 2, 4093), (2, 2, 3, 40),
          (1, 700, 3), (1, 1, 1023), (4, 1, 9), (2, 16, 2048)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_dropout_forward_and_backward(shape, dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(shape, generator=g).to(dtype)
    dy = torch.randn(shape, generator=g).to(dtype)
    seed, call, p = (1 << 61) + 12345, 7, 0.3
    three = (1,) * (3 - len(shape)) + shape if len(shape) <= 3 else (-1,) + shape[-2:]
    view = x.reshape(three)
    keep = oracle.dropout_keep(seed, call, *view.shape, p).reshape(shape)
    xc = x.cuda().requires_grad_()
    y = SparseDropout(p)(xc, rng=rng(seed, call))
    dx, = torch.autograd.grad(y, xc, dy.cuda())
    assert y.dtype == dtype and y.shape == x.shape
    for got, src in ((y.detach(), x), (dx, dy)):
        assert torch.equal(got.cpu() != 0, keep & (src != 0))
        close(got, src.double() * keep * oracle.dropout_scale(p), dtype)


# Many rows, so that a thread takes several of them: segments of a warp on rows of their own, rows in several chunks, a
# change of batch element inside a thread's rows, ends of rows within and at the end of the tensor, an odd first address.
MANY = [(3, 50700, 9), (2, 4740, 257), (1, 3792, 1001), (2, 37900, 64), (19000, 8, 11), (1, 152000, 8), (5, 30001, 7)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', MANY)
@pytest.mark.parametrize('offset', [0, 3])
def test_dropout_of_many_rows(shape, offset, dtype):
    n = shape[0] * shape[1] * shape[2]
    g = torch.Generator(device='cuda').manual_seed(2)
    x = torch.randn(n + offset, generator=g, device='cuda').to(dtype)[offset:].view(shape)
    p, seed, call = 0.2, 99, 3
    keep = oracle.dropout_keep(seed, call, *shape, p)
    y = SparseDropout(p)(x, rng=rng(seed, call))
    want = x.double().cpu() * keep * oracle.dropout_scale(p)
    assert torch.equal(y.cpu() != 0, keep & (x.cpu() != 0))
    close(y, want, dtype)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('offset,cols', [(1, 64), (3, 61), (8, 64), (5, 8)])
def test_dropout_of_unaligned_and_strided_inputs(offset, cols, dtype):
    base = torch.randn(offset + 6 * cols, device='cuda').to(dtype)
    x = base[offset:].view(6, cols)
    keep = oracle.dropout_keep(3, 1, 1, 6, cols, 0.5)[0]
    y = SparseDropout(0.5)(x, rng=rng(3, 1))
    close(y, x.double().cpu() * keep * 2, dtype)
    t = SparseDropout(0.5)(x.t(), rng=rng(3, 1))  # rows and columns of the view, not of the memory
    close(t, x.t().double().cpu() * oracle.dropout_keep(3, 1, 1, cols, 6, 0.5)[0] * 2, dtype)


def test_dropout_ends_of_the_range():
    x = torch.tensor([float('nan'), float('inf'), -float('inf'), 1.0] * 64, device='cuda')
    assert torch.equal(SparseDropout(1.0)(x, rng=rng(0, 0)), torch.zeros_like(x))
    keep = oracle.dropout_keep(9, 2, 1, 1, 256, 0.5)[0, 0].cuda()
    y = SparseDropout(0.5)(x, rng=rng(9, 2))
    assert torch.equal(torch.isnan(y), torch.isnan(x) & keep) and bool((y[~keep] == 0).all())
    assert torch.equal(SparseDropout(1e-9)(torch.ones(64, device='cuda'), rng=rng(0, 0)), torch.ones(64, device='cuda'))
    assert SparseDropout(0.5)(torch.empty((0, 8), device='cuda'), rng=rng(0, 0)).shape == (0, 8)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('block', [(8, 8), (32, 16), (64, 64), (4, 128)])
def test_dropout_of_block_values_agrees_with_dense(block, dtype):
    H, W = 256, 384
    g = torch.Generator().manual_seed(2)
    coarse = (torch.rand((H // block[0], W // block[1]), generator=g) < 0.4).to(torch.uint8)
    coarse[0] = 0
    mask = coarse.repeat_interleave(block[0], 0).repeat_interleave(block[1], 1).cuda()
    indexes = get_bcs_function(*block, True, False).build_indexes(mask)
    dense = (torch.randn((3, H, W), generator=g).cuda() * mask).to(dtype)
    drop = SparseDropout(0.25)
    x = indexes.convert(dense).requires_grad_()
    y = drop(x, rng=rng(4, 9), indexes=indexes)
    want = drop(dense, rng=rng(4, 9))
    assert torch.equal(indexes.inverse(y.detach()), want)
    dx, = torch.autograd.grad(y, x, x.detach())
    assert torch.equal(dx, y.detach())


def test_dropout_counts_calls_and_refuses():
    x = torch.ones(4096, device='cuda')
    a, b = SparseDropout(0.5, seed=5), SparseDropout(0.5, seed=5)
    first, second = a(x), a(x)
    assert not torch.equal(first, second)
    assert torch.equal(b(x), first) and torch.equal(b(x), second)
    assert torch.equal(first, SparseDropout(0.5)(x, rng=rng(5, 0)))
    for bad in (torch.zeros(2, device='cuda'), torch.zeros(3, dtype=torch.int64, device='cuda'), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(ValueError):
            a(x, rng=bad)
    with pytest.raises(TypeError):
        a(x.double())
    indexes = get_bcs_function(32, 32, True, False).build_indexes(torch.ones((64, 64), dtype=torch.uint8, device='cuda'))
    with pytest.raises(ValueError):
        a(x[:100], indexes=indexes)
    narrow = get_bcs_function(8, 4, True, False).build_indexes(torch.ones((64, 64), dtype=torch.uint8, device='cuda'))
    with pytest.raises(ValueError):
        a(x, indexes=narrow)
    # numbers that were rewritten between forward and backward would drop other positions: autograd refuses
    numbers = rng(1, 1)
    leaf = x.clone().requires_grad_()
    y = a(leaf, rng=numbers)
    numbers.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_dropout_in_a_graph():
    x = torch.ones((64, 1000), device='cuda')
    drop, numbers = SparseDropout(0.5), rng(6, 0)
    drop(x, rng=numbers)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = drop(x, rng=numbers)
    for call in (0, 1, 5):
        numbers.copy_(rng(6, call))
        graph.replay()
        assert torch.equal(y, drop(x, rng=rng(6, call)))
    torch.cuda.synchronize()
    refused = []
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        torch.zeros(1, device='cuda')
        try:
            drop(x)
        except RuntimeError as e:
            refused.append(str(e))
    assert refused and 'rng' in refused[0]


def test_dropout_on_another_stream():
    x = torch.randn((512, 4096), device='cuda')
    want = SparseDropout(0.5)(x, rng=rng(1, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = SparseDropout(0.5)(x, rng=rng(1, 2))
    side.synchronize()
    assert torch.equal(got, want)


# ---- rotary positions --------------------------------------------------------------------------------------------
def rotary_close(got, want, dtype, magnitude, x):
    """Angle off by at most 2.2e-7 radians (half a step of a 32-bit number below 1/2 turn, 2^-25 of a half turn, times
    pi, and sincospi's own error of 2 steps), two 32-bit products and a sum, one rounding: in units of the pair's norm."""
    norm = x.double().abs().amax() * 2 * magnitude
    close(got, want, dtype, absolute=float(norm) * 6e-7)


CASES = [  # dim, rotary_dim, interleaved, scaling
    (64, 64, False, 'none'), (128, 96, True, 'yarn'), (128, 96, False, 'linear'), (80, 40, True, 'ntk'), (24, 10, False, 'none'),
    (7, 6, True, 'none'), (2, 2, False, 'yarn'), (256, 2, True, 'ntk'), (40, 16, False, 'yarn')]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim,rotary_dim,interleaved,scaling', CASES)
@pytest.mark.parametrize('token_major', [False, True])
def test_rotary_forward_and_backward(dim, rotary_dim, interleaved, scaling, token_major, dtype):
    b, hq, hk, n = 2, 6, 3, 37
    g = torch.Generator().manual_seed(4)
    freq, magnitude = rotary_frequencies(rotary_dim, 10000.0, scaling, 4.0, 512)
    rot = RotaryEmbedding(dim, rotary_dim, interleaved=interleaved, scaling=scaling, factor=4.0, original_length=512)
    pos = torch.randint(0, 1 << 22, (b, n), generator=g)
    make = lambda h: ((lambda t: t.transpose(1, 2) if token_major else t)(  # noqa: E731
        torch.randn((b, n, h, dim) if token_major else (b, h, n, dim), generator=g).to(dtype)))
    q, k = make(hq), make(hk)
    dq, dk = (torch.randn((b, h, n, dim), generator=g).to(dtype) for h in (hq, hk))
    qc, kc = (t.cuda().requires_grad_() for t in (q, k))
    yq, yk = rot(qc, kc, positions=pos.cuda())
    gq, gk = torch.autograd.grad((yq, yk), (qc, kc), (dq.cuda(), dk.cuda()))
    for got, src, sign in ((yq, q, 1.0), (yk, k, 1.0), (gq, dq, -1.0), (gk, dk, -1.0)):
        assert got.dtype == dtype
        rotary_close(got.detach(), oracle.rotary(src, pos, freq, magnitude, interleaved, sign), dtype, magnitude, src)


@pytest.mark.parametrize('positions', ['none', 'shared32', 'shared64', 'rows', 'negative'])
@pytest.mark.parametrize('flat', [False, True])
def test_rotary_positions_and_layouts(positions, flat):
    b, h, n, dim = 3, 4, 9, 32
    x = torch.randn((b, h, n, dim))
    pos = torch.arange(n)
    if positions in ('rows', 'negative'):
        pos = torch.randint(-1000 if positions == 'negative' else 0, 1 << 30, (b, n))
    want = oracle.rotary(x, pos.expand(b, n), rotary_frequencies(dim, 500.0, 'none', 1.0, None)[0], 1.0, False)
    rot = RotaryEmbedding(dim, base=500.0)
    given = {'none': None, 'shared32': pos.int().cuda(), 'shared64': pos.cuda()}.get(positions, pos.cuda())
    xc = x.cuda().flatten(0, 1) if flat else x.cuda()
    rotary_close(rot(xc, positions=given).view(b, h, n, dim), want, torch.float32, 1.0, x)
    if positions == 'none':
        rotary_close(rot(x[0, 0].cuda()), want[0, 0], torch.float32, 1.0, x)
        rotary_close(rot(x[None].cuda())[0], want, torch.float32, 1.0, x)


def test_rotary_one_token_and_unaligned():
    rot = RotaryEmbedding(64)
    x = torch.randn((5, 8, 1, 64)).to(torch.bfloat16)
    pos = torch.tensor([[0], [1 << 20], [7], [(1 << 31) - 1], [99]])
    freq = rotary_frequencies(64, 10000.0, 'none', 1.0, None)[0]
    # 31-bit positions: the oracle's own angles are off by position * 2^-53 radians, 2.4e-7
    rotary_close(rot(x.cuda(), positions=pos.cuda()), oracle.rotary(x, pos, freq, 1.0, False), torch.bfloat16, 1.0, x)
    base = torch.randn(1 + 4 * 64)
    u = base.cuda()[1:].view(4, 64)
    rotary_close(rot(u), oracle.rotary(base[1:].view(1, 1, 4, 64), torch.arange(4)[None], freq, 1.0, False)[0, 0], torch.float32, 1.0, base)
    wide = torch.randn((4, 128))
    v = wide.cuda()[:, ::2]  # elements of a head apart in memory
    rotary_close(rot(v), oracle.rotary(wide[None, None, :, ::2], torch.arange(4)[None], freq, 1.0, False)[0, 0], torch.float32, 1.0, wide)
    assert rot(torch.empty((2, 0, 64), device='cuda')).shape == (2, 0, 64)


def test_rotary_is_undone_by_its_gradient_and_by_differences():
    """The operator is linear and orthogonal: its gradient applied to its output gives the input back, and
    <dy, R x> = <R^T dy, x>."""
    rot = RotaryEmbedding(64, 48, interleaved=True)
    x = torch.randn((2, 3, 50, 64), device='cuda', requires_grad=True)
    y = rot(x)
    back, = torch.autograd.grad(y, x, y.detach(), create_graph=True)
    assert (back - x).abs().max().item() < 5e-6 * x.abs().max().item()
    dy = torch.randn_like(y)
    dx, = torch.autograd.grad(rot(x), x, dy)
    a, b = (dy.double() * y.double()).sum().item(), (dx.double() * x.double()).sum().item()
    assert abs(a - b) < 1e-5 * (dy.double().norm() * y.double().norm()).item()


def test_rotary_partly_used_and_shared():
    """Only one of the two outputs is used; a broadcast input collects the gradients of its copies; keys with positions
    of their own."""
    rot = RotaryEmbedding(32)
    q = torch.randn((2, 4, 5, 32), device='cuda', requires_grad=True)
    k1 = torch.randn((1, 1, 6, 32), device='cuda', requires_grad=True)
    kp = torch.arange(6, device='cuda') + 11
    yq, yk = rot(q, k1.expand(2, 3, 6, 32), positions=torch.arange(5, device='cuda'), key_positions=kp)
    dk = torch.randn_like(yk)
    gq, gk = torch.autograd.grad(yk, (q, k1), dk, allow_unused=True)
    assert gq is None
    freq = rotary_frequencies(32, 10000.0, 'none', 1.0, None)[0]
    want = oracle.rotary(dk.cpu(), kp.cpu().expand(2, 6), freq, 1.0, False, -1.0).sum((0, 1), keepdim=True)
    assert (gk.double().cpu() - want).abs().max() < 6 * 6e-7 * dk.abs().max().item() * 2 + 1e-6
    y32, = [rot(q, positions=torch.arange(5, device='cuda', dtype=torch.int32))]
    assert torch.equal(y32, yq)


def test_rotary_refuses():
    rot = RotaryEmbedding(32)
    q = torch.randn((2, 4, 5, 32), device='cuda')
    bad = [dict(query=q[..., :16]), dict(query=q.double()), dict(query=q, key=q.half()), dict(query=q[0, 0, 0]),
           dict(query=q, positions=torch.arange(5)), dict(query=q, positions=torch.arange(5., device='cuda')),
           dict(query=q, positions=torch.arange(4, device='cuda')), dict(query=q, positions=torch.zeros((3, 5), dtype=torch.int64, device='cuda')),
           dict(query=q.flatten(0, 1), positions=torch.zeros((3, 5), dtype=torch.int64, device='cuda')),
           dict(query=q[0, 0], positions=torch.zeros((2, 5), dtype=torch.int64, device='cuda')),
           dict(query=q, key=q[:, :, :4], positions=torch.arange(5, device='cuda'))]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            rot(**kw)


def test_rotary_in_a_graph():
    rot = RotaryEmbedding(64)
    x, pos = torch.randn((2, 3, 1, 64), device='cuda'), torch.zeros((2, 1), dtype=torch.int64, device='cuda')
    rot(x, positions=pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rot(x, positions=pos)
    for at in (3, 700):
        pos.fill_(at)
        x.normal_()
        graph.replay()
        assert torch.equal(y, rot(x, positions=pos))


def test_rotary_many_heads_and_long():
    """More tokens x heads than one wave: several heads per thread, a ragged last group of heads."""
    rot = RotaryEmbedding(64)
    x = torch.randn((1, 13, 40000, 64), device='cuda').to(torch.float16)
    y = rot(x)
    want = oracle.rotary(x[:, :, -50:].cpu(), torch.arange(39950, 40000)[None], rotary_frequencies(64, 10000.0, 'none', 1.0, None)[0], 1.0, False)
    rotary_close(y[:, :, -50:], want, torch.float16, 1.0, x)
    assert torch.equal(rot(x[:, 12:].contiguous()), y[:, 12:])
