"""Workloads of the attention-training operators and their plain forms.

A training step of a layer built on ``SparseAttention`` turns queries and keys by their positions, runs the
block-sparse attention with dropout on its probabilities, drops out activations, and takes all of it backward.
The cases below are those three operators alone:

* ``attention``: forward and backward pass of softmax_mask(Q K^T / sqrt(E)) V over the kept blocks of a mask,
  with shared key / value heads and dropout on the probabilities;
* ``dropout``: forward and backward pass of dropout whose decisions come from a counter (Philox4x32-7, Salmon et
  al., "Parallel random numbers: as easy as 1, 2, 3", 2011) and are never stored;
* ``rotary``: rotary positions on queries and keys, both layouts, part of the head, scaled for long contexts.

``own`` selects the operators of this package (true) or elementary torch operations in 32 bits (false).
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {'fp32': torch.float32, 'fp16': torch.float16, 'bf16': torch.bfloat16}


# ---- cases -----------------------------------------------------------------------------------------------------
def _attention(name, dtype, batch, heads, kv_heads, nt, ns, dim, keep, mask, dropout):
    """``mask``: 'band' (8 blocks either side of the diagonal, first block row and column, ``keep`` of the rest),
    'blocks' (``keep`` of the 64 x 64 blocks) or 'elements' (8 x 8 pieces on top of it)."""
    return {'name': name, 'kind': 'attention', 'dtype': dtype, 'batch': batch, 'heads': heads, 'kv_heads': kv_heads,
            'nt': nt, 'ns': ns, 'dim': dim, 'keep': keep, 'mask': mask, 'dropout': dropout}


def _dropout(name, dtype, batch, rows, cols, p):
    return {'name': name, 'kind': 'dropout', 'dtype': dtype, 'batch': batch, 'rows': rows, 'cols': cols, 'p': p}


def _rotary(name, dtype, batch, heads, kv_heads, n, dim, rotary_dim, interleaved, scaling, far, token_major, backward):
    """``far``: first position of a sequence lies below it; ``token_major``: tensors arrive as views of
    [batch, n, heads, dim], as a projection leaves them."""
    return {'name': name, 'kind': 'rotary', 'dtype': dtype, 'batch': batch, 'heads': heads, 'kv_heads': kv_heads, 'n': n,
            'dim': dim, 'rotary_dim': rotary_dim, 'interleaved': interleaved, 'scaling': scaling, 'far': far,
            'token_major': token_major, 'backward': backward}


def listed():
    return [
        # one short sequence of a small model: a training step bound by the latency of its launches
        _attention('attention_short', 'fp16', 1, 4, 4, 256, 256, 64, 0.6, 'blocks', 0.0),
        # the attention workload of this repository's benchmark: B4 H16 S4096 D64, band + global + random blocks
        _attention('attention_b4h16s4096', 'fp16', 4, 16, 16, 4096, 4096, 64, 0.05, 'band', 0.0),
        # the same with dropout on the probabilities, as a model that is trained with it runs it
        _attention('attention_b4h16s4096_dropout', 'bf16', 4, 16, 16, 4096, 4096, 64, 0.05, 'band', 0.1),
        # the long-sequence configuration (S8192 D128 bf16) on one GPU's share of heads, four query heads to a key head
        _attention('attention_h16s8192_shared', 'bf16', 1, 16, 4, 8192, 8192, 128, 0.05, 'band', 0.0),
        # cross attention with an odd number of blocks, holes inside the blocks and dropout
        _attention('attention_cross_odd', 'bf16', 2, 8, 2, 1088, 2240, 128, 0.4, 'elements', 0.1),
        # activations of a small batch with odd sizes: launch latency counts
        _dropout('dropout_small', 'fp32', 3, 33, 1001, 0.25),
        # hidden states of a training step: 16 sequences of 2048 tokens, 4096 wide
        _dropout('dropout_hidden', 'bf16', 16, 2048, 4096, 0.1),
        # activations whose rows are no multiple of a vector
        _dropout('dropout_odd', 'fp16', 8, 1777, 4093, 0.5),
        # one new token of 64 sequences at far positions: a serving step
        _rotary('rotary_token', 'bf16', 64, 16, 4, 1, 128, 128, False, 'none', 1 << 20, False, False),
        # queries and keys of the B4 H16 S4096 D64 attention, forward and backward
        _rotary('rotary_b4h16s4096', 'fp16', 4, 16, 16, 4096, 64, 64, False, 'none', 1, False, True),
        # a long context: scaled frequencies, three quarters of the head turned, token-major projections
        _rotary('rotary_long_partial', 'bf16', 1, 32, 8, 16384, 128, 96, True, 'yarn', 1 << 17, True, True),
        # 32-bit training with an odd number of tokens and linear scaling
        _rotary('rotary_fp32_odd', 'fp32', 2, 8, 8, 1777, 80, 40, True, 'linear', 1 << 16, True, True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(['attention', 'dropout', 'rotary'])
    if kind == 'attention':
        dim = rng.choice([64, 128])
        kv_heads, group, batch = log_int(1, 8), rng.choice([1, 1, 2, 4]), log_int(1, 4)
        nt, ns = 64 * log_int(1, 96), 64 * log_int(1, 96)
        while batch * kv_heads * group * nt * ns * dim > 64 * 4096 * 4096 * 64:
            nt, ns = max(64, nt // 128 * 64), max(64, ns // 128 * 64)
        mask = rng.choice(['band', 'blocks', 'elements'])
        c = _attention('', rng.choice(['fp16', 'bf16']), batch, kv_heads * group, kv_heads, nt, ns, dim,
                       round(rng.uniform(0.02, 0.2) if mask == 'band' else rng.uniform(0.1, 1.0), 3), mask,
                       rng.choice([0.0, 0.0, 0.1, 0.35]))
    elif kind == 'dropout':
        batch, rows, cols = log_int(1, 16), log_int(1, 2048), log_int(1, 4096)
        c = _dropout('', rng.choice(['fp32', 'fp16', 'bf16']), batch, rows, cols, round(rng.uniform(0.02, 0.9), 3))
    else:
        dim = 8 * log_int(2, 32)
        kv_heads, group, batch, n = log_int(1, 8), rng.choice([1, 2, 4]), log_int(1, 16), log_int(1, 16384)
        while batch * kv_heads * group * n * dim > 32 * 16384 * 128:
            n = max(1, n // 2)
        c = _rotary('', rng.choice(['fp32', 'fp16', 'bf16']), batch, kv_heads * group, kv_heads, n, dim,
                    rng.choice([dim, 2 * log_int(1, dim // 2)]), rng.random() < 0.5,
                    rng.choice(['none', 'linear', 'ntk', 'yarn']), log_int(1, 1 << 22), rng.random() < 0.5, rng.random() < 0.7)
    del c['name']
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------
def _block_mask(c, g):
    rows, cols = c['nt'] // 64, c['ns'] // 64
    keep = torch.rand((rows, cols), generator=g) < c['keep']
    if c['mask'] == 'band':
        i, j = torch.arange(rows)[:, None], torch.arange(cols)[None, :]
        keep = keep | ((i - j).abs() <= 8) | (i == 0) | (j == 0)
    mask = keep.to('cuda', torch.uint8).repeat_interleave(64, 0).repeat_interleave(64, 1)
    if c['mask'] == 'elements':
        fine = (torch.rand((c['nt'] // 8, c['ns'] // 8), generator=g) < 0.7).to('cuda', torch.uint8)
        mask = mask * fine.repeat_interleave(8, 0).repeat_interleave(8, 1)
    return mask.contiguous()


def _attention_config():
    mm = {'_impl': 'sparta', 'BLOCK_SIZE_M_VALUE': 64, 'BLOCK_SIZE_K_VALUE': 64, 'BLOCK_SIZE_N_VALUE': 64}
    sm = {'_impl': 'sparta', 'BLOCK_SIZE_H_VALUE': 64, 'BLOCK_SIZE_W_VALUE': 64, 'ROW_TILE_VALUE': 4}
    return {'qk/forward:C': mm, 'qk/backward:A': mm, 'qk/backward:B': mm, 'out/forward:C': mm, 'out/backward:A': mm,
            'out/backward:B': mm, 'sm/forward:y': sm, 'sm/backward:x': sm}


def _random_pair(seed, device):
    """The counter generator's inputs: a 64-bit seed and a call number."""
    return torch.tensor([seed * 0x9E3779B97F4A7C15 % (1 << 62), 11 + seed % 1000], dtype=torch.int64, device=device)


def prepare(case, seed):
    c = case
    g = torch.Generator().manual_seed(seed)
    d = torch.Generator(device='cuda').manual_seed(seed + 1)
    t = _DTYPES[c['dtype']]

    def normal(*shape):
        return torch.randn(shape, generator=d, device='cuda', dtype=torch.float32).to(t)

    s = {'case': c, 'rng': _random_pair(seed, 'cuda')}
    if c['kind'] == 'attention':
        b, h, k, dim = c['batch'], c['heads'], c['kv_heads'], c['dim']
        s['mask'] = _block_mask(c, g)
        s['q'] = normal(b, h, c['nt'], dim).requires_grad_()
        s['k'], s['v'] = (normal(b, k, c['ns'], dim).requires_grad_() for _ in range(2))
        s['dout'] = normal(b, h, c['nt'], dim)
        if own:
            from sparta_b200.nn import SparseAttention
            s['op'] = SparseAttention(s['mask'], dropout=c['dropout'])
            s['op'].build(_attention_config(), sample_inputs=[s['q'], s['k'], s['v']])
    elif c['kind'] == 'dropout':
        s['x'] = normal(c['batch'], c['rows'], c['cols']).requires_grad_()
        s['dout'] = normal(c['batch'], c['rows'], c['cols'])
        if own:
            from sparta_b200.nn import SparseDropout
            s['op'] = SparseDropout(c['p'])
    else:
        b, n, dim = c['batch'], c['n'], c['dim']
        for name, h in (('q', c['heads']), ('k', c['kv_heads'])):
            x = normal(b, n, h, dim).transpose(1, 2) if c['token_major'] else normal(b, h, n, dim)
            s[name] = x.requires_grad_(c['backward'])
            s['d' + name] = normal(b, h, n, dim)
        start = torch.randint(0, c['far'], (b, 1), generator=g)
        s['positions'] = (start + torch.arange(n)[None, :]).to('cuda', torch.int64)
        s['turn'], s['magnitude'] = _frequencies(c)
        if own:
            from sparta_b200.nn import RotaryEmbedding
            s['op'] = RotaryEmbedding(dim, rotary_dim=c['rotary_dim'], base=10000.0, interleaved=c['interleaved'],
                                      scaling=c['scaling'], factor=8.0, original_length=4096)
    return s


def _frequencies(c):
    """Angle per position of every pair (fp64, on the GPU) and the factor on the turned values."""
    r = c['rotary_dim']
    i = torch.arange(r // 2, dtype=torch.float64, device='cuda')
    factor, length, magnitude = 8.0, 4096.0, 1.0
    base = 10000.0
    if c['scaling'] == 'ntk' and r > 2:
        base = base * factor ** (r / (r - 2))
    freq = base ** (-2.0 * i / r)
    if c['scaling'] == 'linear':
        freq = freq / factor
    if c['scaling'] == 'yarn':
        turns = length * freq / (2 * math.pi)
        ramp = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        freq = freq / factor * (1 - ramp) + freq * ramp
        magnitude = 0.1 * math.log(factor) + 1.0
    return freq, magnitude


# ---- one pass --------------------------------------------------------------------------------------------------
def run(state):
    s = state
    c = s['case']
    if c['kind'] == 'attention':
        if own:
            out = s['op'](s['q'], s['k'], s['v'], rng=s['rng'])
            return (out.detach(),) + torch.autograd.grad(out, (s['q'], s['k'], s['v']), s['dout'])
        return _plain_attention(s, c)
    if c['kind'] == 'dropout':
        if own:
            out = s['op'](s['x'], rng=s['rng'])
            return (out.detach(),) + torch.autograd.grad(out, (s['x'],), s['dout'])
        keep, scale = _plain_keep(s['rng'], c['batch'], c['rows'], c['cols'], c['p'])
        x, dy = s['x'].detach(), s['dout']
        return tuple(torch.where(keep, v.float() * scale, torch.zeros((), device='cuda')).to(v.dtype) for v in (x, dy))
    if own:
        q, k = s['op'](s['q'], s['k'], positions=s['positions'])
        if not c['backward']:
            return q, k
        return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (s['q'], s['k']), (s['dq'], s['dk']))
    out = (_plain_rotary(s['q'].detach(), s, c, 1.0), _plain_rotary(s['k'].detach(), s, c, 1.0))
    if not c['backward']:
        return out
    return out + (_plain_rotary(s['dq'], s, c, -1.0), _plain_rotary(s['dk'], s, c, -1.0))


def _plain_mul32(a, b):
    """(high, low) 32-bit words of the product of two 32-bit words held in int64."""
    low = (a * b) & 0xFFFFFFFF
    high = (a * (b >> 16) + ((a * (b & 0xFFFF)) >> 16)) >> 16
    return high, low


def _plain_keep(rng, batch, rows, cols, p):
    """Which positions of a [batch, rows, cols] tensor are kept: 16 random bits each, eight positions of a row to a
    counter (column / 8, row, batch, call number) under the key `seed`; kept when not below round(65536 p)."""
    seed, call = rng[0], rng[1] & 0xFFFFFFFF
    groups = (cols + 7) // 8
    ar = lambda n: torch.arange(n, dtype=torch.int64, device=rng.device)  # noqa: E731
    shape = (batch, rows, groups)
    x = [ar(groups).view(1, 1, -1).expand(shape), ar(rows).view(1, -1, 1).expand(shape),
         ar(batch).view(-1, 1, 1).expand(shape), call.expand(shape)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for i in range(7):  # the generator's seven rounds
        h0, l0 = _plain_mul32(0xD2511F53, x[0])
        h1, l1 = _plain_mul32(0xCD9E8D57, x[2])
        x = [h1 ^ x[1] ^ k0, l1, h0 ^ x[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([w & 0xFFFF if half == 0 else w >> 16 for w in x for half in (0, 1)], -1)
    threshold = int(math.floor(p * 65536 + 0.5))
    keep = words.reshape(batch, rows, groups * 8)[:, :, :cols] >= threshold
    return keep, 65536.0 / (65536 - threshold)


def _plain_attention(s, c):
    b, h, kv, nt, ns, dim = (c[n] for n in ('batch', 'heads', 'kv_heads', 'nt', 'ns', 'dim'))
    g = h // kv
    q, do = (s[n].detach().float().view(b * kv, g * nt, dim) for n in ('q', 'dout'))  # heads that share keys side by side
    k, v = (s[n].detach().float().view(b * kv, ns, dim) for n in ('k', 'v'))
    mask = s['mask'] != 0
    scale = 1.0 / math.sqrt(dim)
    x = (q @ k.transpose(1, 2)).view(b * h, nt, ns).mul_(scale).masked_fill_(~mask, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    prob = x.div_(torch.where(total == 0, torch.ones_like(total), total))
    if c['dropout'] > 0:
        keep, up = _plain_keep(s['rng'], b * h, nt, ns, c['dropout'])
        used = prob * keep * up
    else:
        used = prob
    flat = used.view(b * kv, g * nt, ns)
    out = flat @ v
    dv = flat.transpose(1, 2) @ do
    dp = (do @ v.transpose(1, 2)).view(b * h, nt, ns)
    if c['dropout'] > 0:
        dp = dp.mul_(keep).mul_(up)
    delta = (out * do).sum(-1).view(b * h, nt, 1)
    ds = dp.sub_(delta).mul_(prob).mul_(scale).view(b * kv, g * nt, ns)
    dq, dk = ds @ k, ds.transpose(1, 2) @ q
    t = s['q'].dtype
    return (out.view(b, h, nt, dim).to(t), dq.view(b, h, nt, dim).to(t), dk.view(b, kv, ns, dim).to(t),
            dv.view(b, kv, ns, dim).to(t))


def _plain_rotary(x, s, c, sign):
    r = c['rotary_dim']
    angle = s['positions'].double()[:, None, :, None] * s['turn']  # far positions need 64 bits
    cos, sin = (torch.cos(angle) * s['magnitude']).float(), (torch.sin(angle) * (sign * s['magnitude'])).float()
    y = x.float()
    part, rest = y[..., :r], y[..., r:]
    if c['interleaved']:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part[..., :r // 2], part[..., r // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1).to(x.dtype)


# ---- what a pass cannot do without -----------------------------------------------------------------------------
def _kept_share(c):
    """Expected share of kept blocks."""
    if c['mask'] != 'band':
        return c['keep']
    rows, cols = c['nt'] // 64, c['ns'] // 64
    sure = sum(1 for i in range(rows) for j in range(cols) if abs(i - j) <= 8 or i == 0 or j == 0)
    return (sure + c['keep'] * (rows * cols - sure)) / (rows * cols)


def work(case):
    c = case
    size = 4 if c['dtype'] == 'fp32' else 2
    if c['kind'] == 'attention':
        query = c['batch'] * c['heads'] * c['nt'] * c['dim'] * size
        key = c['batch'] * c['kv_heads'] * c['ns'] * c['dim'] * size
        # q, dout in; out, dq out; k, v in; dk, dv out; the mask once.  Two products forward, five backward
        share = _kept_share(c)
        return {'bytes': 4 * query + 4 * key + c['nt'] * c['ns'],
                'flops': 7 * 2 * c['batch'] * c['heads'] * c['nt'] * c['ns'] * c['dim'] * share}
    if c['kind'] == 'dropout':
        n = c['batch'] * c['rows'] * c['cols']
        return {'bytes': 4 * n * size, 'flops': 2 * n}  # x and dy in, y and dx out
    n = c['batch'] * (c['heads'] + c['kv_heads']) * c['n'] * c['dim']
    passes = 2 if c['backward'] else 1
    return {'bytes': passes * (2 * n * size + 8 * c['batch'] * c['n']), 'flops': passes * 3 * n * c['rotary_dim'] / c['dim']}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------
def _exact_keep(seed, batch, rows, cols, p):
    pair = _random_pair(seed, 'cpu').numpy().astype(np.uint64)
    groups = -(-cols // 8)
    low = np.uint64(0xFFFFFFFF)
    col, row, lead = np.meshgrid(np.arange(groups), np.arange(rows), np.arange(batch), indexing='ij')
    c0, c1, c2 = (v.transpose(2, 1, 0).reshape(-1).astype(np.uint64) for v in (col, row, lead))
    c3 = np.full_like(c0, pair[1] & low)
    key = [int(pair[0] & low), int(pair[0] >> np.uint64(32))]
    for i in range(7):
        p0, p1 = np.uint64(0xD2511F53) * c0, np.uint64(0xCD9E8D57) * c2
        c0, c1, c2, c3 = ((p1 >> np.uint64(32)) ^ c1 ^ np.uint64(key[0]), p1 & low,
                          (p0 >> np.uint64(32)) ^ c3 ^ np.uint64(key[1]), p0 & low)
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    bits = np.stack([c0, c1, c2, c3], 1).astype('<u4').view('<u2').reshape(batch, rows, groups * 8)[:, :, :cols]
    cut = math.floor(65536 * p + 0.5)
    return torch.from_numpy(bits.astype(np.int32) >= cut).cuda(), 65536 / (65536 - cut)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c['kind'] == 'attention':
        return _exact_attention(s, c, seed)
    if c['kind'] == 'dropout':
        keep, up = _exact_keep(seed, c['batch'], c['rows'], c['cols'], c['p'])
        return s['x'].detach().double() * keep * up, s['dout'].double() * keep * up
    return _exact_rotary(s, c)


def _exact_attention(s, c, seed):
    if c['dropout'] > 0 and c['batch'] * c['heads'] * c['nt'] * c['ns'] > 200e6:
        return None  # the generator on the host would take over 20 seconds
    group = c['heads'] // c['kv_heads']
    q, do = s['q'].detach().double(), s['dout'].double()
    k, v = (s[n].detach().double().repeat_interleave(group, 1) for n in ('k', 'v'))
    sc = torch.einsum('bhid,bhjd->bhij', q, k) / c['dim'] ** 0.5
    kept = s['mask'].bool()
    lse = torch.logsumexp(sc.masked_fill_(~kept, -math.inf), -1, keepdim=True)
    p = sc.sub_(lse.masked_fill(lse == -math.inf, 0.0)).exp_()
    del sc
    w = torch.ones((), dtype=torch.float64, device='cuda')
    if c['dropout'] > 0:
        keep, up = _exact_keep(seed, c['batch'] * c['heads'], c['nt'], c['ns'], c['dropout'])
        w = keep.view(c['batch'], c['heads'], c['nt'], c['ns']) * up
    used = p * w
    out = torch.einsum('bhij,bhjd->bhid', used, v)
    dv = torch.einsum('bhij,bhid->bhjd', used, do)
    del used
    dp = torch.einsum('bhid,bhjd->bhij', do, v) * w
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / c['dim'] ** 0.5
    del dp, p
    dq, dk = torch.einsum('bhij,bhjd->bhid', ds, k), torch.einsum('bhij,bhid->bhjd', ds, q)
    shape = (c['batch'], c['kv_heads'], group, c['ns'], c['dim'])
    return out, dq, dk.reshape(shape).sum(2), dv.reshape(shape).sum(2)


def _exact_rotary(s, c):
    r, base, factor, length = c['rotary_dim'], 10000.0, 8.0, 4096.0
    freq, magnitude = [], 1.0
    for i in range(r // 2):
        if c['scaling'] == 'ntk' and r > 2:
            f = math.pow(base * math.pow(factor, r / (r - 2)), -2 * i / r)
        else:
            f = math.pow(base, -2 * i / r)
        if c['scaling'] == 'linear':
            f /= factor
        if c['scaling'] == 'yarn':
            whole = min(1.0, max(0.0, (length * f / (2 * math.pi) - 1) / 31))
            f = whole * f + (1 - whole) * f / factor
            magnitude = 1 + 0.1 * math.log(factor)
        freq.append(f)
    freq = np.array(freq, dtype=np.float64)
    angle = s['positions'].cpu().numpy().astype(np.float64)[:, None, :, None] * freq
    turn = torch.from_numpy(np.cos(angle) + 1j * np.sin(angle)).cuda() * magnitude

    def turned(x, t):
        y = x.detach().double()
        head = y[..., :r]
        pairs = head.unflatten(-1, (r // 2, 2)) if c['interleaved'] else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * t)
        z = z.flatten(-2) if c['interleaved'] else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, y[..., r:]], -1)

    out = (turned(s['q'], turn), turned(s['k'], turn))
    if not c['backward']:
        return out
    return out + (turned(s['dq'], turn.conj()), turned(s['dk'], turn.conj()))
