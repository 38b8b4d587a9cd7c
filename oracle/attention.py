"""64-bit statements of the dropout and the cross attention (test infrastructure only; no reference kernels:
the stock blocks run ``nn.Dropout``, ``nn.GELU`` and SDPA).

Nothing is rounded to a storage dtype here: the tests' bars count the rounding.
"""

from __future__ import annotations

import math

import numpy as np

__all__ = ["philox4x32", "dropout_bits", "dropout_factors", "gelu", "gelu_grad", "dropout_forward", "dropout_backward",
           "cross_attention_forward", "cross_attention_backward"]

_M32 = 0xFFFFFFFF


def philox4x32(counter, key, rounds: int = 7):
    """Philox4x32 (Salmon et al., SC 2011) of one counter (4 words) and key (2 words), in Python integers."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & _M32, (p0 >> 32) ^ c[3] ^ k[1], p0 & _M32]
        k = [(k[0] + 0x9E3779B9) & _M32, (k[1] + 0xBB67AE85) & _M32]
    return c


def dropout_bits(first_block: int, blocks: int, seed: int, offset: int) -> np.ndarray:
    """The 16 random bits of elements ``8 first_block ...`` (``8 blocks`` of them), vectorised over blocks."""
    g = np.arange(first_block, first_block + blocks, dtype=np.uint64)
    m32, sh = np.uint64(_M32), np.uint64(32)
    c = [g & m32, g >> sh, np.full_like(g, offset & _M32), np.full_like(g, (offset >> 32) & _M32)]
    k = [seed & _M32, (seed >> 32) & _M32]
    for _ in range(7):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> sh) ^ c[1] ^ np.uint64(k[0]), p1 & m32, (p0 >> sh) ^ c[3] ^ np.uint64(k[1]), p0 & m32]
        k = [(k[0] + 0x9E3779B9) & _M32, (k[1] + 0xBB67AE85) & _M32]
    w = np.stack(c, axis=1)
    return np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], axis=2).reshape(-1).astype(np.int64)


def dropout_factors(count: int, p: float, seed: int, offset: int) -> np.ndarray:
    """0 for a dropped element, 65536 / (65536 - round(65536 p)) for a kept one."""
    limit = min(int(math.floor(p * 65536 + 0.5)), 65535)
    keep = dropout_bits(0, -(-count // 8), seed, offset)[:count] >= limit
    return np.where(keep, 65536.0 / (65536 - limit), 0.0)


_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def gelu(x):
    return x * 0.5 * _erfc(-x / math.sqrt(2.0))


def gelu_grad(x):
    return 0.5 * _erfc(-x / math.sqrt(2.0)) + x * np.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi)


def dropout_forward(x, p, seed, offset, activation=None, residual=None):
    y = gelu(x) if activation == "gelu" else x
    f = dropout_factors(x.size, p, seed, offset).reshape(x.shape)
    y = np.where(f > 0, y * f, 0.0)
    return y if residual is None else y + residual


def dropout_backward(grad, p, seed, offset, x=None, activation=None):
    d = grad * gelu_grad(x) if activation == "gelu" else grad
    f = dropout_factors(grad.size, p, seed, offset).reshape(grad.shape)
    return np.where(f > 0, d * f, 0.0)


def _weights(q, k, scale, seen):
    """One head: ``(P[N, M], lse[N])``; a row that sees nothing has no weight and lse -inf."""
    s = np.where(seen[None, :], (q @ k.T) * scale, -np.inf)
    top = s.max(axis=1, initial=-np.inf)
    e = np.exp(s - np.where(np.isfinite(top), top, 0.0)[:, None])
    total = e.sum(axis=1)
    with np.errstate(divide="ignore"):
        lse = np.where(total > 0, np.log(total) + np.where(np.isfinite(top), top, 0.0), -np.inf)
    return e / np.where(total > 0, total, 1.0)[:, None], lse


def _seen(b, m, key_mask, key_lengths):
    seen = np.ones((b, m), dtype=bool)
    if key_mask is not None:
        seen &= np.asarray(key_mask, dtype=bool)
    if key_lengths is not None:
        seen &= np.arange(m)[None, :] < np.clip(np.asarray(key_lengths), 0, m)[:, None]
    return seen


def _keep(b, n, m, h, p, seed, offset):
    if p == 0.0:
        return None
    pitch = -(-m // 8) * 8
    return dropout_factors(b * h * n * pitch, p, seed, offset).reshape(b, h, n, pitch)[..., :m]


def cross_attention_forward(q, k, v, key_mask=None, key_lengths=None, scale=None, p=0.0, seed=0, offset=0):
    """``q[B, N, H, D]``, ``k`` / ``v[B, M, Hk, D]`` -> ``(out[B, N, H, D], lse[B, H, N])``; masked keys and
    values are never read."""
    b, n, h, d = q.shape
    m, hk = k.shape[1:3]
    scale = d**-0.5 if scale is None else scale
    seen, keep = _seen(b, m, key_mask, key_lengths), _keep(b, n, m, h, p, seed, offset)
    out, lse = np.zeros((b, n, h, d)), np.zeros((b, h, n))
    for i in range(b):
        for j in range(h):
            kk, vv = (np.where(seen[i][:, None], t[i, :, j // (h // hk)], 0.0) for t in (k, v))
            w, lse[i, j] = _weights(q[i, :, j], kk, scale, seen[i])
            out[i, :, j] = (w if keep is None else w * keep[i, j]) @ vv
    return out, lse


def cross_attention_backward(grad, q, k, v, key_mask=None, key_lengths=None, scale=None, p=0.0, seed=0, offset=0):
    """``(grad_q, grad_k, grad_v)``; heads that share a key head add up, masked keys get zeros."""
    b, n, h, d = q.shape
    m, hk = k.shape[1:3]
    scale = d**-0.5 if scale is None else scale
    seen, keep = _seen(b, m, key_mask, key_lengths), _keep(b, n, m, h, p, seed, offset)
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    for i in range(b):
        for j in range(h):
            c = j // (h // hk)
            kk, vv = (np.where(seen[i][:, None], t[i, :, c], 0.0) for t in (k, v))
            w, _ = _weights(q[i, :, j], kk, scale, seen[i])
            f = 1.0 if keep is None else keep[i, j]
            g = grad[i, :, j]
            dv[i, :, c] += (w * f).T @ g
            dw = (g @ vv.T) * f
            ds = w * (dw - (w * dw).sum(axis=1, keepdims=True)) * scale
            dq[i, :, j] = ds @ kk
            dk[i, :, c] += ds.T @ q[i, :, j]
    return dq, dk, dv
