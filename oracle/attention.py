"""64-bit statements of the dropout, the cross attention and the local attention (test infrastructure only; no reference kernels:
the stock blocks run ``nn.Dropout``, ``nn.GELU`` and SDPA).

Nothing is rounded to a storage dtype here: the tests' bars count the rounding.
"""

from __future__ import annotations

import math

import numpy as np

__all__ = ["philox4x32", "dropout_bits", "dropout_factors", "gelu", "gelu_grad", "dropout_forward", "dropout_backward",
           "cross_attention_forward", "cross_attention_backward", "local_attention_forward", "local_attention_backward",
           "local_attention_step"]

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


# ---------------------------------------------------------------------- local attention


def local_seen(b, n, m, left=None, right=None, sinks=0, starts=None, key_mask=None, key_lengths=None):
    """``[B, N, M]``: whether query ``n`` of batch row ``b`` sees frame ``m``."""
    p = np.arange(n)[None, :, None] + (0 if starts is None else np.asarray(starts, dtype=np.int64)[:, None, None])
    j = np.arange(m)[None, None, :]
    seen = np.repeat(_seen(b, m, key_mask, key_lengths)[:, None, :], n, axis=1)
    if right is not None:
        seen &= j <= p + right
    if left is not None:
        seen &= (j >= p - left) | (j < sinks)
    return seen


def bias_numbers(bias):
    """The bias's entries as they count: those of -1e30 or less hide, others are cut to +-2^20."""
    return np.where(bias <= -1e30, -np.inf, np.clip(bias, -(2.0**20), 2.0**20))


def _local_bias(bias, bucket_of, distance):
    """``(bias[..., H], bucket)`` of an array of distances."""
    most = (len(bucket_of) - 1) // 2
    bucket = np.asarray(bucket_of)[np.clip(distance, -most, most) + most]
    return bias_numbers(bias)[bucket], bucket


def _local_weights(q, k, scale, seen, added):
    """One head: ``(P[N, M], lse[N])`` of the scores ``scale q k^T + added`` where ``seen``."""
    s = np.where(seen, (q @ k.T) * scale + added, -np.inf)
    top = s.max(axis=1, initial=-np.inf)
    e = np.exp(s - np.where(np.isfinite(top), top, 0.0)[:, None])
    total = e.sum(axis=1)
    with np.errstate(divide="ignore"):
        lse = np.where(total > 0, np.log(total) + np.where(np.isfinite(top), top, 0.0), -np.inf)
    return e / np.where(total > 0, total, 1.0)[:, None], lse


def _local_parts(q, k, v, left, right, sinks, bias, bucket_of, key_mask, key_lengths, starts, scale):
    """For every batch row and head: its index, K and V without what no query may read, the seen pairs, the added
    bias and the pairs' buckets."""
    b, n, h, d = q.shape
    m, hk = k.shape[1:3]
    kept = _seen(b, m, key_mask, key_lengths)
    seen = local_seen(b, n, m, left, right, sinks, starts, key_mask, key_lengths)
    for i in range(b):
        p = np.arange(n)[:, None] + (0 if starts is None else int(starts[i]))
        added, bucket = (np.zeros((n, m, h)), None) if bias is None else _local_bias(bias, bucket_of, np.arange(m)[None] - p)
        for j in range(h):
            c = j // (h // hk)
            kk, vv = (np.where(kept[i][:, None], t[i, :, c], 0.0) for t in (k, v))
            yield i, j, c, kk, vv, seen[i], added[..., j], bucket


def local_attention_forward(q, k, v, left=None, right=None, sinks=0, bias=None, bucket_of=None, key_mask=None,
                            key_lengths=None, starts=None, scale=None):
    """``q[B, N, H, D]`` over ``k`` / ``v[B, M, Hk, D]`` -> ``(out[B, N, H, D], lse[B, H, N])``."""
    b, n, h, d = q.shape
    scale = d**-0.5 if scale is None else scale
    out, lse = np.zeros((b, n, h, d)), np.zeros((b, h, n))
    for i, j, c, kk, vv, seen, added, _ in _local_parts(q, k, v, left, right, sinks, bias, bucket_of, key_mask, key_lengths,
                                                        starts, scale):
        w, lse[i, j] = _local_weights(q[i, :, j], kk, scale, seen, added)
        out[i, :, j] = w @ vv
    return out, lse


def local_attention_backward(grad, q, k, v, left=None, right=None, sinks=0, bias=None, bucket_of=None, key_mask=None,
                             key_lengths=None, starts=None, scale=None):
    """``(grad_q, grad_k, grad_v, grad_bias or None)``."""
    d = q.shape[3]
    scale = d**-0.5 if scale is None else scale
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    db = None if bias is None else np.zeros(bias.shape)
    for i, j, c, kk, vv, seen, added, bucket in _local_parts(q, k, v, left, right, sinks, bias, bucket_of, key_mask,
                                                             key_lengths, starts, scale):
        w, _ = _local_weights(q[i, :, j], kk, scale, seen, added)
        g = grad[i, :, j]
        dv[i, :, c] += w.T @ g
        dw = g @ vv.T
        ds = w * (dw - (w * dw).sum(axis=1, keepdims=True))
        dq[i, :, j] = ds @ kk * scale
        dk[i, :, c] += ds.T @ q[i, :, j] * scale
        if bias is not None:
            np.add.at(db[:, j], bucket, ds)
    return dq, dk, dv, db


def ring_slot(frame: int, sinks: int, ring: int) -> int:
    return frame if frame < sinks else sinks + (frame - sinks) % ring


def local_attention_step(q, k, v, k_cache, v_cache, positions, left, sinks=0, bias=None, bucket_of=None, scale=None):
    """``(out[B, N, H, D], k_cache, v_cache)``; the caches given are left as they are."""
    b, n, h, d = q.shape
    hk, ring = k.shape[2], k_cache.shape[1] - sinks
    scale = d**-0.5 if scale is None else scale
    out, kc, vc = np.zeros((b, n, h, d)), k_cache.copy(), v_cache.copy()
    for i in range(b):
        p = int(positions[i])
        if p < 0:
            continue
        for x in range(n):
            at = ring_slot(p + x, sinks, ring)
            kc[i, at], vc[i, at] = k[i, x], v[i, x]
        frames = np.array([f for f in range(p + n) if f < sinks or f >= p - left])
        slots = np.array([ring_slot(int(f), sinks, ring) for f in frames])
        distance = frames[None, :] - (p + np.arange(n))[:, None]
        seen = (distance <= 0) & ((distance >= -left) | (frames < sinks)[None, :])
        added = np.zeros((n, len(frames), h)) if bias is None else _local_bias(bias, bucket_of, distance)[0]
        for j in range(h):
            w, _ = _local_weights(q[i, :, j], kc[i, slots, j // (h // hk)], scale, seen, added[..., j])
            out[i, :, j] = w @ vc[i, slots, j // (h // hk)]
    return out, kc, vc
