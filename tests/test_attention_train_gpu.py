"""Training step of the fused sparse attention -- forward with log-sum-exp, backward that recomputes the probabilities,
dropout on the probabilities, shared key / value heads, rotary positions -- against the 64-bit oracle."""
import math

import pytest
import torch

from oracle import attention_training as oracle
from oracle import oracle as masks
from sparta_b200 import _lib
from sparta_b200.nn import RotaryEmbedding, SparseAttention
from sparta_b200.specializer.operators.rotary import rotary_frequencies
from sparta_b200.tesa import get_bcs_function

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def config(tile=64):
    mm = {'_impl': 'sparta', 'BLOCK_SIZE_M_VALUE': tile, 'BLOCK_SIZE_K_VALUE': tile, 'BLOCK_SIZE_N_VALUE': tile}
    sm = {'_impl': 'sparta', 'BLOCK_SIZE_H_VALUE': tile, 'BLOCK_SIZE_W_VALUE': tile, 'ROW_TILE_VALUE': 4}
    cfg = {f'{op}/{k}': mm for op in ('qk', 'out') for k in ('forward:C', 'backward:A', 'backward:B')}
    return {**cfg, 'sm/forward:y': sm, 'sm/backward:x': sm}


def rng(seed, call):
    return torch.tensor([seed, call], dtype=torch.int64, device='cuda')


def inputs(dtype, heads, kv_heads, nt, ns, dim, seed=1, qscale=1.0):
    g = torch.Generator().manual_seed(seed)
    q, do = ((torch.randn((heads, nt, dim), generator=g) * s).to(dtype) for s in (qscale, 1.0))
    k, v = (torch.randn((kv_heads, ns, dim), generator=g).to(dtype) for _ in range(2))
    return q, k, v, do


def block_mask(nt, ns, share, seed=2, elements=False):
    g = torch.Generator().manual_seed(seed)
    m = (torch.rand((nt // 64, ns // 64), generator=g) < share).to(torch.uint8).repeat_interleave(64, 0).repeat_interleave(64, 1)
    if elements:
        m = m * (torch.rand((nt, ns), generator=g) < 0.6).to(torch.uint8)
    return m


def want_and_bounds(q, k, v, do, mask, keep=None, up=1.0):
    """The oracle's out, dq, dk, dv and how far a computation may be off that rounds P' and dS once to the type, O once
    before delta, each result once (u = eps / 2 of the type), holds everything else in 32 bits, and takes the
    exponential with a relative error of 2^-21.  Worst case, element by element, first order in u."""
    heads, dim = q.shape[0], q.shape[2]
    group = heads // k.shape[0]
    scale = 1 / math.sqrt(dim)
    out, dq, dk, dv, lse = oracle.attention(q, k, v, do, mask, scale, keep, up)
    u, e32 = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    tiny = torch.finfo(q.dtype).smallest_normal * u  # rounding below the normal range
    Q, K, V, dO = q.double(), k.double().repeat_interleave(group, 0), v.double().repeat_interleave(group, 0), do.double()
    w = torch.ones(()) if keep is None else keep.double() * up
    p = torch.exp((Q @ K.transpose(1, 2) * scale).masked_fill(mask == 0, -math.inf) - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
    n = mask.shape[1] + mask.shape[0]
    # the exponent: a 32-bit dot product of length D, the log-sum-exp (a sum of up to n terms), two roundings of the sum
    size = Q.abs() @ K.abs().transpose(1, 2) * scale
    rel_p = (dim + 8) * e32 * (size + size.amax(-1, keepdim=True)) + (lse.abs()[..., None].nan_to_num(0, 0, 0) * 4 + 40 + n) * e32 + 2.0 ** -21
    used = p * w
    e_used = used * (u + rel_p) + tiny * (p > 0) * (up if keep is not None else 1.0)
    e_out = e_used @ V.abs() + n * e32 * (used @ V.abs()) + u * out.abs() + tiny
    dp = (dO @ V.transpose(1, 2)) * w
    delta = (p * dp).sum(-1, keepdim=True)
    e_delta = (dO.abs() * e_out).sum(-1, keepdim=True) + dim * e32 * (dO.abs() * out.abs()).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_ds = ds.abs() * (u + rel_p + 4 * e32) + p * ((dim + 2) * e32 * ((dO.abs() @ V.abs().transpose(1, 2)) * w) + e_delta) + tiny * (p > 0)
    e_dq = scale * (e_ds @ K.abs() + n * e32 * (ds.abs() @ K.abs())) + u * dq.abs() + tiny
    fold = lambda t: t.view(k.shape[0], group, *t.shape[1:]).sum(1)  # noqa: E731
    e_dk = fold(scale * (e_ds.transpose(1, 2) @ Q.abs() + group * n * e32 * (ds.abs().transpose(1, 2) @ Q.abs()))) + u * dk.abs() + tiny
    e_dv = fold(e_used.transpose(1, 2) @ dO.abs() + group * n * e32 * (used.transpose(1, 2) @ dO.abs())) + u * dv.abs() + tiny
    return (out, dq, dk, dv), (e_out, e_dq, e_dk, e_dv)


def check(got, want, bounds):
    for name, x, y, b in zip(('out', 'dq', 'dk', 'dv'), got, want, bounds):
        x = x.detach().double().cpu().view(y.shape)
        assert torch.isfinite(x).all(), name
        over = ((x - y).abs() - 1.01 * b).max().item()
        assert over <= 0, f'{name}: {over} over the bound, worst {(x - y).abs().max().item()}'
        norm = y.norm().item()
        if norm > 0:  # the errors of single elements do not all point one way: the whole is far nearer than the worst case
            rel = (x - y).norm().item() / norm
            assert rel <= 4 * torch.finfo(got[0].dtype).eps / 2, f'{name}: {rel} off as a whole'


def build(mask, q, k, v, fused=True, **kw):
    op = SparseAttention(mask.cuda(), fused=fused, **kw)
    op.build(config(), sample_inputs=[q, k, v])
    op.check_status = True
    return op


def step(op, q, k, v, do, **kw):
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = op(*leaves, **kw)
    return (out,) + torch.autograd.grad(out, leaves, do.cuda())


SHAPES = [  # heads, kv_heads, nt, ns, share of blocks, element mask
    (1, 1, 64, 64, 1.0, False), (2, 2, 128, 128, 1.0, False), (3, 3, 64, 192, 1.0, False), (2, 2, 320, 64, 0.7, False),
    (2, 1, 256, 448, 0.5, False), (6, 2, 192, 320, 0.5, True), (4, 4, 512, 512, 0.3, False), (1, 1, 128, 1088, 0.6, True),
    (8, 2, 576, 256, 0.4, False), (2, 2, 256, 256, 0.4, True),
    # few tiles with many steps: several CTAs share a tile and add their partial sums
    (1, 1, 2048, 192, 0.8, False), (4, 1, 1088, 128, 0.9, True), (2, 2, 64, 4096, 0.7, False), (1, 1, 4160, 4032, 0.5, False)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('shape', SHAPES)
def test_forward_and_gradients(shape, dim, dtype):
    heads, kv_heads, nt, ns, share, elements = shape
    q, k, v, do = inputs(dtype, heads, kv_heads, nt, ns, dim)
    mask = block_mask(nt, ns, share, elements=elements)
    op = build(mask, q, k, v)
    assert op._use_fused
    got = step(op, q, k, v, do)
    check(got, *want_and_bounds(q, k, v, do, mask))
    again = step(op, q, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), 'a second pass adds in another order'


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('p', [0.1, 0.75, 0.9999])
@pytest.mark.parametrize('shape', [(2, 2, 256, 256, 0.6, False), (4, 2, 192, 448, 0.6, True), (2, 1, 512, 128, 1.0, False),
                                   (2, 1, 2048, 192, 0.8, True), (1, 1, 64, 4096, 0.9, False)])
def test_dropout(shape, p, dim, dtype):
    heads, kv_heads, nt, ns, share, elements = shape
    q, k, v, do = inputs(dtype, heads, kv_heads, nt, ns, dim)
    mask = block_mask(nt, ns, share, elements=elements)
    op = build(mask, q, k, v, dropout=p)
    seed, call = (1 << 61) + 99, 1 << 31
    keep = oracle.dropout_keep(seed, call, heads, nt, ns, p)
    got = step(op, q, k, v, do, rng=rng(seed, call))
    check(got, *want_and_bounds(q, k, v, do, mask, keep, oracle.dropout_scale(p)))
    with torch.no_grad():  # dropout without gradients, and none in evaluation mode
        assert torch.equal(op(q.cuda(), k.cuda(), v.cuda(), rng=rng(seed, call)), got[0])
        plain = SparseAttention.forward(op.eval(), q.cuda(), k.cuda(), v.cuda())
        assert torch.equal(plain, build(mask, q, k, v)(q.cuda(), k.cuda(), v.cuda()))


@pytest.mark.parametrize('dim', [64, 128])
def test_everything_dropped(dim):
    q, k, v, do = inputs(torch.float16, 2, 2, 128, 256, dim)
    op = build(block_mask(128, 256, 1.0), q, k, v, dropout=1.0)
    for x in step(op, q, k, v, do, rng=rng(1, 1)):
        assert bool((x == 0).all())


@pytest.mark.parametrize('dim', [64, 128])
def test_masks_that_leave_rows_and_columns_empty(dim):
    """No block at all; whole tiles without blocks along either side; rows without an element inside kept blocks."""
    q, k, v, do = inputs(torch.bfloat16, 2, 2, 384, 512, dim)
    none = torch.zeros((384, 512), dtype=torch.uint8)
    holes = block_mask(384, 512, 0.7)
    holes[128:256] = 0
    holes[:, 256:384] = 0
    holes[300:340] = 0   # inside blocks
    holes[:, 20:30] = 0
    holes[5, :] = 0
    one = none.clone()
    one[383, 511] = 1
    op = build(none, q, k, v)
    for mask in (none, holes, one, torch.ones_like(none)):
        op.update_mask(mask.cuda())
        got = step(op, q, k, v, do)
        check(got, *want_and_bounds(q, k, v, do, mask))
        rows, cols = mask.sum(1) == 0, mask.sum(0) == 0
        assert bool((got[0][:, rows] == 0).all()) and bool((got[1][:, rows] == 0).all())
        assert bool((got[2][:, cols] == 0).all()) and bool((got[3][:, cols] == 0).all())


@pytest.mark.parametrize('dim', [64, 128])
def test_large_scores(dim):
    """Scores of several tens: one key takes almost all of a row."""
    q, k, v, do = inputs(torch.float16, 2, 2, 256, 512, dim, qscale=6.0)
    mask = block_mask(256, 512, 1.0)
    got = step(build(mask, q, k, v), q, k, v, do)
    want, bounds = want_and_bounds(q, k, v, do, mask)
    for x, y, b in zip(got, want, bounds):  # the gradients nearly cancel: only the worst case holds
        assert ((x.detach().double().cpu() - y).abs() <= 1.01 * b).all()


def test_directional_differences():
    """<gradient, direction> against central differences of the oracle's forward in 64 bits."""
    q, k, v, do = inputs(torch.float16, 2, 1, 128, 192, 64)
    mask = block_mask(128, 192, 0.8, elements=True)
    keep, up = oracle.dropout_keep(3, 4, 2, 128, 192, 0.2), oracle.dropout_scale(0.2)
    got = step(build(mask, q, k, v, dropout=0.2), q, k, v, do, rng=rng(3, 4))
    _, bounds = want_and_bounds(q, k, v, do, mask, keep, up)
    g = torch.Generator().manual_seed(8)
    for at in range(3):
        d = torch.randn((q, k, v)[at].shape, generator=g).double()
        eps = 1e-5

        def loss(sign):
            x = [t.double() for t in (q, k, v)]
            x[at] = x[at] + sign * eps * d
            return (oracle.attention(*x, do, mask, 0.125, keep, up)[0] * do.double()).sum().item()
        slope = (loss(1) - loss(-1)) / (2 * eps)
        have = (got[1 + at].double().cpu() * d).sum().item()
        assert abs(have - slope) <= (bounds[1 + at] * d.abs()).sum().item() + 1e-4 * abs(slope) + 1e-6


def test_composed_path_takes_the_same_dropout_and_shared_heads():
    """32-bit inputs run on the three operators; dropout, shared heads and four dimensions work there alike."""
    q, k, v, do = (t.float() for t in inputs(torch.float16, 6, 2, 192, 128, 64))
    mask = block_mask(192, 128, 0.7, elements=True)
    op = SparseAttention(mask.cuda(), dropout=0.3)
    four = lambda t: t.view(2, -1, *t.shape[1:])  # noqa: E731
    op.build(config(32), sample_inputs=[four(q).cuda(), four(k).cuda(), four(v).cuda()])
    assert not op._use_fused
    keep = oracle.dropout_keep(5, 6, 6, 192, 128, 0.3)
    got = step(op, four(q), four(k), four(v), four(do), rng=rng(5, 6))
    assert got[0].shape == four(q).shape
    want = oracle.attention(q, k, v, do, mask, 0.125, keep, oracle.dropout_scale(0.3))
    for x, y in zip(got, want):  # 32-bit kernels; the repository's bar for them
        torch.testing.assert_close(x.detach().double().cpu().view(y.shape), y, atol=1e-4, rtol=1e-4)


@pytest.mark.parametrize('dtype', DTYPES)
def test_auto_takes_the_fused_kernels_for_training(dtype, monkeypatch):
    q, k, v, do = inputs(dtype, 2, 2, 128, 128, 64)
    mask = block_mask(128, 128, 1.0)
    op = build(mask, q, k, v, fused='auto')
    monkeypatch.setattr(op._matmul_qk, 'forward', None)  # the composed path is not to be called
    check(step(op, q, k, v, do), *want_and_bounds(q, k, v, do, mask))


def test_layouts_and_partial_gradients():
    """Four dimensions, token-major views, misaligned storage, an expanded output gradient, a broadcast key head, and
    gradients of some inputs only."""
    dtype, dim = torch.bfloat16, 64
    q, k, v, do = inputs(dtype, 8, 4, 128, 192, dim)
    mask = block_mask(128, 192, 0.7)
    want, bounds = want_and_bounds(q, k, v, do, mask)
    op = build(mask, q, k, v)
    four = lambda t: t.view(2, -1, *t.shape[1:])  # noqa: E731
    major = lambda t: four(t).cuda().transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    leaves = [major(t).requires_grad_() for t in (q, k, v)]
    out = op(*leaves)
    assert out.shape == (2, 4, 128, dim)
    check((out,) + torch.autograd.grad(out, leaves, major(do)), want, bounds)
    # storage that begins off a 16-byte boundary
    off = lambda t: torch.cat([torch.zeros(1, dtype=dtype), t.flatten()]).cuda()[1:].view(t.shape)  # noqa: E731
    leaves = [off(t).requires_grad_() for t in (q, k, v)]
    out = op(*leaves)
    check((out,) + torch.autograd.grad(out, leaves, off(do)), want, bounds)
    # an output gradient of strides 0
    ones = torch.ones_like(do)
    want1, bounds1 = want_and_bounds(q, k, v, ones, mask)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = op(*leaves)
    check((out,) + torch.autograd.grad(out.sum(), leaves), want1, bounds1)
    # subsets
    full = step(op, q, k, v, do)
    for subset in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.cuda().requires_grad_(i in subset) for i, t in enumerate((q, k, v))]
        out = op(*leaves)
        grads = torch.autograd.grad(out, [leaves[i] for i in subset], do.cuda())
        assert all(torch.equal(g, full[1 + i]) for g, i in zip(grads, subset))
    # one key head broadcast by hand over all of them
    k1 = k[:1].cuda().requires_grad_()
    out = op(q.cuda(), k1.expand(4, 192, dim), v.cuda())
    got, = torch.autograd.grad(out, k1, do.cuda())
    parts, part_bounds = want_and_bounds(q, k[:1].expand(4, 192, dim), v, do, mask)
    u = torch.finfo(dtype).eps / 2
    total, bound = parts[2].sum(0, keepdim=True), part_bounds[2].sum(0, keepdim=True)  # autograd adds the rounded parts in the type
    bound = bound + 4 * u * parts[2].abs().sum(0, keepdim=True)
    assert ((got.double().cpu() - total).abs() <= bound).all()


def test_two_steps_at_once_and_masks_that_change():
    """Two forward passes before either backward pass, with another mask and other random numbers in between."""
    q, k, v, do = inputs(torch.float16, 2, 2, 256, 256, 64)
    a, b = block_mask(256, 256, 0.5, seed=3), block_mask(256, 256, 0.5, seed=4)
    op = build(a, q, k, v, dropout=0.2)
    la = [t.cuda().requires_grad_() for t in (q, k, v)]
    lb = [t.cuda().requires_grad_() for t in (q, k, v)]
    oa = op(*la, rng=rng(1, 1))
    op.update_mask(b.cuda())
    ob = op(*lb, rng=rng(1, 2))
    ga, gb = torch.autograd.grad(oa, la, do.cuda()), torch.autograd.grad(ob, lb, do.cuda())
    up = oracle.dropout_scale(0.2)
    check((oa,) + ga, *want_and_bounds(q, k, v, do, a, oracle.dropout_keep(1, 1, 2, 256, 256, 0.2), up))
    check((ob,) + gb, *want_and_bounds(q, k, v, do, b, oracle.dropout_keep(1, 2, 2, 256, 256, 0.2), up))
    # the module's own numbers: every call drops other positions, forward and backward agree
    with torch.no_grad():
        assert not torch.equal(op(*la), op(*la))
    seed, call = op._dropout._counter.seed, op._dropout._counter.calls
    got = step(op, q, k, v, do)
    check(got, *want_and_bounds(q, k, v, do, b, oracle.dropout_keep(seed, call, 2, 256, 256, 0.2), up))


def test_dynamic_mask():
    q, k, v, do = inputs(torch.float16, 2, 2, 128, 256, 64)
    mask = block_mask(128, 256, 0.5, seed=5, elements=True).cuda()
    op = build(mask, q, k, v)
    op.set_dynamic()
    for seed in (6, 7):
        mask.copy_(block_mask(128, 256, 0.6, seed=seed, elements=True))
        check(step(op, q, k, v, do), *want_and_bounds(q, k, v, do, mask.cpu()))
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = op(*leaves)
    mask.zero_()  # the backward pass would read other elements than the forward pass did
    with pytest.raises(RuntimeError):
        out.backward(do.cuda())


def test_captured_step():
    q, k, v, do = inputs(torch.bfloat16, 4, 2, 192, 256, 128)
    mask = block_mask(192, 256, 0.6, elements=True)
    op = build(mask, q, k, v, dropout=0.1)
    op.check_status = False
    leaves, d, numbers = [t.cuda().requires_grad_() for t in (q, k, v)], do.cuda(), rng(2, 0)

    def run():
        out = op(*leaves, rng=numbers)
        return (out,) + torch.autograd.grad(out, leaves, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for call in (4, 5):
        numbers.copy_(rng(2, call))
        with torch.no_grad():
            leaves[0].copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(call)).to(q.dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step(op, leaves[0].detach().cpu(), k, v, do, rng=rng(2, call))))
    assert op.fused_status() == [0, 0, 0, 0]


def test_another_stream():
    q, k, v, do = inputs(torch.float16, 8, 8, 512, 512, 64)
    op = build(block_mask(512, 512, 0.5), q, k, v)
    want = step(op, q, k, v, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(op, q, k, v, do)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [64, 128])
def test_rotary_dropout_and_attention_together(dim, dtype):
    """A whole layer's step: rotary positions on token-major projections, attention with dropout over shared heads,
    backward through both, against the oracle's chain on the rounded rotary outputs."""
    b, h, hk, n = 2, 4, 2, 192
    g = torch.Generator().manual_seed(9)
    make = lambda heads: torch.randn((b, n, heads, dim), generator=g).to(dtype)  # noqa: E731
    q, k, v, do = make(h), make(hk), make(hk), make(h).transpose(1, 2)
    mask = block_mask(n, n, 0.8, elements=True)
    pos = torch.randint(0, 1 << 20, (b, n), generator=g)
    rotary = RotaryEmbedding(dim, dim // 2, interleaved=True)
    op = SparseAttention(mask.cuda(), dropout=0.15, rotary=rotary)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    views = [t.transpose(1, 2) for t in leaves]
    op.build(config(), sample_inputs=views)
    out = op(*views, rng=rng(7, 8), positions=pos.cuda())
    got = (out,) + torch.autograd.grad(out, leaves, do.cuda())
    assert op.fused_status() == [0, 0, 0, 0]
    freq, _ = rotary_frequencies(dim // 2, 10000.0, 'none', 1.0, None)
    with torch.no_grad():
        rq, rk = (t.cpu().flatten(0, 1) for t in rotary(*(t.detach() for t in views[:2]), positions=pos.cuda()))
    flat = lambda t: t.transpose(1, 2).flatten(0, 1)  # noqa: E731
    keep = oracle.dropout_keep(7, 8, b * h, n, n, 0.15)
    want, bounds = want_and_bounds(rq, rk, flat(v), do.flatten(0, 1), mask, keep, oracle.dropout_scale(0.15))
    u = torch.finfo(dtype).eps / 2
    turn = lambda t, sign: oracle.rotary(t.view(b, -1, n, dim), pos, freq, 1.0, True, sign)  # noqa: E731
    for at, (x, y, e) in enumerate(zip(got, want, bounds)):
        x = x.detach().double().cpu()
        x = x if at == 0 else x.transpose(1, 2)
        y, e = y.view(x.shape), e.view(x.shape)
        if at in (1, 2):  # turned back: a pair's errors add up to at most sqrt(2) of the larger, plus one more rounding
            y = turn(y, -1.0)
            pair = e[..., :dim // 2].unflatten(-1, (-1, 2)).amax(-1, keepdim=True).expand(-1, -1, -1, -1, 2).flatten(-2) * math.sqrt(2)
            e = torch.cat([pair, e[..., dim // 2:]], -1) * (1 + u) + u * y.abs() + 1e-6
        assert ((x - y).abs() <= 1.01 * e).all(), at


def test_refusals():
    q, k, v, do = (t.cuda() for t in inputs(torch.float16, 4, 2, 128, 128, 64))
    op = build(block_mask(128, 128, 1.0), q, k, v)
    for bad in ((q[:3], k, v), (q, k, v[:1]), (q, k[:, :64], v), (q[..., :32], k[..., :32], v[..., :32])):
        with pytest.raises((ValueError, AssertionError)):
            op(*bad)
    with pytest.raises(TypeError):
        op(q, k.bfloat16(), v)
    with pytest.raises(ValueError):
        op(q, k, v, positions=torch.arange(128, device='cuda'))
    with pytest.raises(ValueError):
        build(block_mask(128, 128, 1.0), q, k, v, dropout=0.5)(q, k, v, rng=torch.zeros(2, device='cuda'))
    leaf = q.clone().requires_grad_()
    grad, = torch.autograd.grad(op(leaf, k, v), leaf, do, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_offsets_beyond_32_bits():
    """2^31 elements and more in each tensor: the last heads come out as they do alone."""
    heads, n, dim = 4100, 8192, 64
    mask = torch.zeros((n, n), dtype=torch.uint8)
    for i in range(0, n // 64, 3):
        mask[i * 64:(i + 1) * 64, i * 64:(i + 1) * 64] = 1
    d = torch.Generator(device='cuda').manual_seed(1)
    make = lambda: torch.randn((heads, n, dim), generator=d, device='cuda', dtype=torch.float16)  # noqa: E731
    q, k, v, do = make(), make(), make(), make()
    op = build(mask, q[:1], k[:1], v[:1])
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = op(*leaves)
    grads = torch.autograd.grad(out, leaves, do)
    small = [t[-3:].detach().clone().requires_grad_() for t in (q, k, v)]
    out1 = op(*small)
    grads1 = torch.autograd.grad(out1, small, do[-3:])
    for a, b in zip((out,) + grads, (out1,) + grads1):
        assert torch.equal(a[-3:], b)


def test_nan_reaches_the_gradients():
    """A NaN in one query row makes that row's output and dQ, and the dK, dV of the keys it sees, NaN: none turns into a
    number.  Blocks of other pairs of block rows and columns do not see it."""
    q, k, v, do = inputs(torch.bfloat16, 1, 1, 256, 256, 64)
    q[0, 7, 3] = float('nan')
    mask = torch.zeros((256, 256), dtype=torch.uint8)
    for i in range(0, 256, 64):
        mask[i:i + 64, i:i + 64] = 1
    out, dq, dk, dv = step(build(mask, q, k, v), q, k, v, do)
    for x in (out, dq):
        assert bool(torch.isnan(x[0, 7]).all()) and bool(torch.isfinite(x[0, 8:]).all())
    for x in (dk, dv):
        assert bool(torch.isnan(x[0, :64]).all()) and bool(torch.isfinite(x[0, 128:]).all())


def test_two_graphs_replayed_in_turn():
    """Two captured steps of one operator keep apart: neither's buffers are the other's."""
    q, k, v, do = inputs(torch.float16, 2, 2, 256, 256, 64)
    op = build(block_mask(256, 256, 0.6), q, k, v, dropout=0.2)
    op.check_status = False
    eager = [t.cuda().requires_grad_() for t in (q, k, v)]
    alive = op(*eager, rng=rng(0, 0))  # an eager graph of its own that lives on
    cases = []
    for seed in (1, 2):
        leaves = [t.cuda().requires_grad_() for t in inputs(torch.float16, 2, 2, 256, 256, 64, seed=seed)[:3]]
        d, numbers = do.cuda(), rng(seed, 5)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(op(*leaves, rng=numbers), leaves, d)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = op(*leaves, rng=numbers)
            held = (out,) + torch.autograd.grad(out, leaves, d)
        want = step(op, *(t.detach().cpu() for t in leaves), do, rng=rng(seed, 5))
        cases.append((graph, held, want, leaves, d, numbers))
    for _ in range(2):
        for graph, *_ in cases:
            graph.replay()
    torch.cuda.synchronize()
    for _, held, want, *_ in cases:
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(alive, eager, do.cuda()))


@pytest.mark.parametrize('dtype', DTYPES)
def test_half_precision_on_the_three_operators(dtype):
    """fused=False, built through sparta.nn.build: dropout and shared heads, at the repository's bar for half types."""
    import sparta_b200
    q, k, v, do = inputs(dtype, 4, 2, 128, 192, 64)
    mask = block_mask(128, 192, 0.7, elements=True)
    op = SparseAttention(mask.cuda(), fused=False, dropout=0.25)
    sparta_b200.nn.build(op, [q.cuda(), k.cuda(), v.cuda()], {'root': config()})
    keep = oracle.dropout_keep(3, 9, 4, 128, 192, 0.25)
    got = step(op, q, k, v, do, rng=rng(3, 9))
    want = oracle.attention(q, k, v, do, mask, 0.125, keep, oracle.dropout_scale(0.25))
    for x, y in zip(got, want):
        scale = max(1.0, y.abs().max().item())  # the scores' gradients pass through the type three times
        torch.testing.assert_close(x.detach().double().cpu() / scale, y / scale, atol=2e-2, rtol=2e-2)
    fused = build(mask, q, k, v, dropout=0.25)
    out = step(fused, q, k, v, do, rng=rng(3, 9))[0]
    torch.testing.assert_close(out, got[0], atol=2e-2, rtol=2e-2)


def test_random_state_travels_with_the_module():
    q, k, v, do = inputs(torch.float16, 2, 2, 128, 128, 64)
    mask = block_mask(128, 128, 1.0)
    a, b = (build(mask, q, k, v, dropout=0.5) for _ in range(2))
    a(q.cuda(), k.cuda(), v.cuda())
    b.load_state_dict(a.state_dict())
    assert torch.equal(a(q.cuda(), k.cuda(), v.cuda()), b(q.cuda(), k.cuda(), v.cuda()))
    a.eval(), b.eval()
    assert torch.equal(a(q.cuda(), k.cuda(), v.cuda()), build(mask, q, k, v)(q.cuda(), k.cuda(), v.cuda()))


def test_long_sequences_with_global_tokens():
    """Tiles launched head by head (queries and keys beyond L2) and shared by several CTAs (global rows and columns):
    two heads against 64 bits on the GPU, with the mask's blocks as elements."""
    heads, n, dim = 16, 16384, 128
    block = torch.zeros((n // 64, n // 64), dtype=torch.bool)
    i = torch.arange(n // 64)
    block |= (i[:, None] - i[None, :]).abs() <= 2
    block[0], block[:, 0] = True, True
    mask = block.cuda().to(torch.uint8).repeat_interleave(64, 0).repeat_interleave(64, 1)
    d = torch.Generator(device='cuda').manual_seed(2)
    q, do = (torch.randn((heads, n, dim), generator=d, device='cuda').bfloat16() for _ in range(2))
    k, v = (torch.randn((heads // 2, n, dim), generator=d, device='cuda').bfloat16() for _ in range(2))
    op = build(mask, q, k, v)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = op(*leaves)
    got = (out,) + torch.autograd.grad(out, leaves, do)
    kept = mask.bool()
    for kv in (0, heads // 2 - 1):
        h = slice(2 * kv, 2 * kv + 2)
        kk, vv = k[kv].detach().double(), v[kv].detach().double()
        parts = []
        for a in range(2 * kv, 2 * kv + 2):
            p = torch.softmax((q[a].detach().double() @ kk.T / dim ** 0.5).masked_fill(~kept, -math.inf), -1)
            o, dv = p @ vv, p.T @ do[a].double()
            ds = p * (do[a].double() @ vv.T - (o * do[a].double()).sum(-1, keepdim=True)) / dim ** 0.5
            parts.append((o, ds @ kk, ds.T @ q[a].detach().double(), dv))
        want = [torch.stack([x[j] for x in parts]) for j in range(4)]
        want[2], want[3] = want[2].sum(0), want[3].sum(0)
        for name, x, y in zip(('out', 'dq', 'dk', 'dv'), (got[0][h], got[1][h], got[2][kv], got[3][kv]), want):
            rel = ((x.detach().double() - y).norm() / y.norm()).item()
            assert rel <= 4 * torch.finfo(torch.bfloat16).eps / 2, f'{name} of head {kv}: {rel}'


@pytest.mark.parametrize('elements', [False, True])
@pytest.mark.parametrize('dim', [64, 128])
def test_dropout_decisions_made_once_or_in_every_pass(dim, elements):
    """Room for the decisions of all kept blocks, of all but one, of none: the same gradients bit for bit, and nothing
    is written behind the workspace."""
    heads, kv_heads, nt, ns = 6, 2, 320, 448
    q, k, v, do = (t.cuda() for t in inputs(torch.float16, heads, kv_heads, nt, ns, dim))
    mask = block_mask(nt, ns, 0.5, elements=elements).cuda()
    idx = get_bcs_function(64, 64, True, False).build_indexes(mask)
    L, n, numbers = _lib.lib(), idx.block_nnz, rng(5, 9)
    out, lse = torch.empty_like(q), torch.empty((heads, nt), device='cuda')
    status = torch.zeros(4, dtype=torch.int32, device='cuda')
    stream = torch.cuda.current_stream().cuda_stream
    a = _lib.AttnTrainArgs(Q=q.data_ptr(), K=k.data_ptr(), V=v.data_ptr(), O=out.data_ptr(), lse=lse.data_ptr(), dO=do.data_ptr(),
                           row_ptr=idx.row_ptr.data_ptr(), bcsr_idx=idx.bcsr_buf.data_ptr(), mask=mask.data_ptr() if elements else None,
                           rng=numbers.data_ptr(), status=status.data_ptr(), dropout=0.25, scale=dim ** -0.5, heads=heads,
                           kv_heads=kv_heads, Nt=nt, Ns=ns, D=dim, BLK=64, dtype=_lib.F16)
    assert L.sparta_attn_train_fwd(a, stream) == 0
    base = L.sparta_attn_train_bwd_workspace_bytes(heads, kv_heads, nt, ns, dim, 0)
    every = L.sparta_attn_train_bwd_dropout_bytes(heads, n)
    assert every == heads * n * 512
    results = []
    for extra in (0, 1, every - 512, every - 1, every, every + 4096, 2 * heads * nt * ns):
        room = torch.full((base + extra + 256,), 0xa5, dtype=torch.uint8, device='cuda')
        grads = [torch.full_like(t, math.nan) for t in (q, k, v)]
        a.workspace, a.workspace_bytes = room.data_ptr(), base + extra
        a.dQ, a.dK, a.dV = (t.data_ptr() for t in grads)
        assert L.sparta_attn_train_bwd(a, stream) == 0
        assert bool((room[base + extra:] == 0xa5).all()) and not status.any()
        results.append(grads)
    for grads in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(grads, results[0]))
    keep = oracle.dropout_keep(5, 9, heads, nt, ns, 0.25)
    want, bounds = want_and_bounds(q.cpu(), k.cpu(), v.cpu(), do.cpu(), mask.cpu(), keep, oracle.dropout_scale(0.25))
    for got, w, e in zip([out] + results[0], want, bounds):
        assert bool(((got.double().cpu() - w).abs() <= e).all())
