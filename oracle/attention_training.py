"""64-bit oracle of the attention-training operators: counter-based dropout, rotary positions and the gradients of masked
attention.  Plain numpy / torch on the CPU, independent of the package."""
import math

import numpy as np
import torch

_LOW = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key, rounds=7):
    """Philox4x32 (Salmon et al., SC 2011) on arrays of 32-bit words; four arrays of words."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    for _ in range(rounds):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & _LOW, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & _LOW]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def dropout_keep(seed, call, batch, rows, cols, p):
    """Boolean [batch, rows, cols] of the kept positions."""
    b, r, g = np.meshgrid(np.arange(batch), np.arange(rows), np.arange((cols + 7) // 8), indexing='ij')
    seed &= (1 << 64) - 1
    words = philox4x32([g, r, b, np.full(g.shape, call & 0xFFFFFFFF)], [seed & 0xFFFFFFFF, seed >> 32])
    values = np.stack([v for w in words for v in (w & np.uint64(0xFFFF), w >> np.uint64(16))], -1)
    values = values.reshape(batch, rows, -1)[:, :, :cols].astype(np.int64)
    return torch.from_numpy(values >= dropout_threshold(p))


def dropout_threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def dropout_scale(p):
    t = dropout_threshold(p)
    return 65536.0 / (65536 - t) if t < 65536 else 0.0


def rotary(x, positions, freq, magnitude, interleaved, sign=1.0):
    """x [batch, heads, n, dim]; positions [batch, n] integers; freq: angle per position of each pair."""
    y = x.double().clone()
    angle = positions.double()[:, None, :, None] * torch.tensor(freq, dtype=torch.float64)
    cos, sin = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude * sign
    half = len(freq)
    ia, ib = ((slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half)))
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia] = a * cos - b * sin
    y[..., ib] = b * cos + a * sin
    return y


def attention(q, k, v, dout, mask, scale, keep=None, up=1.0):
    """out, dq, dk, dv, lse of masked attention in 64 bits.  q, dout [heads, Nt, D]; k, v [kv_heads, Ns, D], heads a
    multiple of kv_heads; mask [Nt, Ns]; keep [heads, Nt, Ns] booleans of dropout with scale `up`."""
    group = q.shape[0] // k.shape[0]
    q, dout = q.double(), dout.double()
    kk, vv = k.double().repeat_interleave(group, 0), v.double().repeat_interleave(group, 0)
    s = (q @ kk.transpose(1, 2) * scale).masked_fill(mask == 0, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
    w = torch.ones_like(p) if keep is None else keep.double() * up
    out = (p * w) @ vv
    dv = (p * w).transpose(1, 2) @ dout
    dp = (dout @ vv.transpose(1, 2)) * w
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    dq, dk = ds @ kk, ds.transpose(1, 2) @ q
    fold = lambda t: t.view(k.shape[0], group, *t.shape[1:]).sum(1)  # noqa: E731
    return out, dq, fold(dk), fold(dv), lse
