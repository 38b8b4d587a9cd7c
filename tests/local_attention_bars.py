"""The local attention in 64 bits with the largest error that the kernels' arithmetic allows, per element.

The derivation is that of ``attention_bars`` with three things more:

* the bias starts the score's fp32 sum, so its magnitude joins that of the products;
* the bias's gradient is summed from fp32 ``dS``, unrounded, with ``D`` corrected by what a row's ``dS`` adds up to:
  with ``P'`` the computed weights (``eps`` relative, their sum 1 within ``eps``), ``dP'`` the computed products
  (``(D + 4) u32`` of ``|dO| |V|``) and ``D'`` the first ``D``, ``D' + sum P' (dP' - D')`` is off by
  ``eps (sum P |dP| + |D'|) + (D + 4) u32 sum P |dO| |V|`` and the sum's own ``(M + 8) u32 sum P (|dP| + |D'|)``;
  the bins, buckets and blocks add ``L u32`` of the sum of ``|dS|``, ``L`` the additions that follow each other;
* a step keeps its weights in fp32 and scales q before the products (``u32`` more).
"""

from __future__ import annotations

import numpy as np

import oracle.attention as oa
from tests.attention_bars import HALF, LOST, U32, check  # noqa: F401


def _score_eps(s, mag, d, m, lse):
    """The rows' relative error bounds of their weights."""
    top = np.where(mag > 0, mag * (d + 8) + np.abs(s) * 4, 0.0).max(axis=1, initial=0.0)
    return 2 * (top + np.abs(np.where(np.isfinite(lse), lse, 0)) * 4 + m + 16)[:, None] * U32


def reference(dt, q, k, v, grad=None, bias_dt="f32", left=None, right=None, sinks=0, bias=None, bucket_of=None, key_mask=None,
              key_lengths=None, starts=None, scale=None):
    """``{name: (value, bar)}`` for ``out``, ``lse`` and, with ``grad``, ``dq``, ``dk``, ``dv`` (and ``db`` with a bias)."""
    b, n, h, d = q.shape
    m, hk = k.shape[1:3]
    g = h // hk
    scale = d**-0.5 if scale is None else scale
    u = HALF[dt]
    u16 = 0.0 if dt == "f32" else u
    tiny = 2.0**-25 if dt == "f16" else 1e-37
    args = (left, right, sinks, bias, bucket_of, key_mask, key_lengths, starts, scale)
    out, lse = oa.local_attention_forward(q, k, v, *args)
    bar_out, bar_lse = np.zeros(out.shape), np.zeros(lse.shape)
    res = {}
    if grad is not None:
        dq, dk, dv, db = oa.local_attention_backward(grad, q, k, v, *args)
        bq, bk, bv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
        bb, total = (None, None) if bias is None else (np.zeros(db.shape), np.zeros(db.shape))
    for i, j, c, kk, vv, seen, added, bucket in oa._local_parts(q, k, v, *args):
        w, _ = oa._local_weights(q[i, :, j], kk, scale, seen, added)
        off = np.where(np.isfinite(added), np.abs(added), 0.0)
        s = np.where(seen, np.abs(q[i, :, j] @ kk.T) * scale + off, 0.0)
        mag = np.where(seen, np.abs(q[i, :, j]) @ np.abs(kk).T * scale + off, 0.0)
        eps = _score_eps(s, mag, d, m, lse[i, j])
        av = np.abs(vv)
        wmax = w.max(axis=1, initial=0.0)[:, None]
        low = 2.0**-31 * wmax * (seen @ av) if dt == "f16" else 0.0
        ref = np.abs(out[i, :, j])
        inner = (u16 + eps + m * U32) * (w @ av) + low + LOST * (seen @ av)
        bar_out[i, :, j] = inner + (u + 4 * U32) * (ref + inner) + tiny
        bar_lse[i, j] = eps[:, 0] + 4 * U32 * (1 + np.abs(np.where(np.isfinite(lse[i, j]), lse[i, j], 0)))
        if grad is None:
            continue
        dO, rows = np.abs(grad[i, :, j]), g * n
        gv, gav = grad[i, :, j] @ vv.T, dO @ av.T
        D = (grad[i, :, j] * out[i, :, j]).sum(axis=1)
        dD = (dO * bar_out[i, :, j]).sum(axis=1) + d * U32 * (dO * (ref + bar_out[i, :, j])).sum(axis=1)
        inside = np.abs(gv - D[:, None])
        if bias is not None:
            near = np.abs(D) + dD
            fixed = (eps[:, 0] * ((w * np.abs(gv)).sum(axis=1) + near) + (d + 4) * U32 * (w * gav).sum(axis=1)
                     + (m + 8) * U32 * (w * (np.abs(gv) + near[:, None])).sum(axis=1))
            e32 = w * (eps * inside + (d + 4) * U32 * gav + fixed[:, None] + 4 * U32 * inside) + LOST * inside * seen
            np.add.at(bb[:, j], bucket, e32)
            np.add.at(total[:, j], bucket, w * inside)
            dD = np.maximum(dD, fixed)  # the keys' gradients have the corrected D, the queries' the first
        ds = w * inside
        bound = 2 * dO.sum(axis=1).max(initial=0.0) * av.max(initial=0.0)
        low_s = 2.0**-38 * bound * seen if dt == "f16" else 0.0
        e_ds = w * (eps * inside + (d + 4) * U32 * gav + dD[:, None])
        e_ds = e_ds + u16 * (ds + e_ds) + low_s + LOST * inside * seen
        low_p = 2.0**-38 if dt == "f16" else 0.0
        e_p = (u16 + eps + 2 * U32) * w + (low_p + LOST) * seen
        bq[i, :, j] = scale * ((e_ds + (m + 4) * U32 * ds) @ np.abs(kk))
        bk[i, :, c] += scale * ((e_ds + (rows + 4) * U32 * ds).T @ np.abs(q[i, :, j]))
        bv[i, :, c] += (e_p + (rows + 4) * U32 * w).T @ dO
    res["out"], res["lse"] = (out, bar_out), (lse, bar_lse)
    if grad is not None:
        for name, x, bar in (("dq", dq, bq), ("dk", dk, bk), ("dv", dv, bv)):
            res[name] = (x, bar + (u + 4 * U32) * (np.abs(x) + bar) + tiny)
        if bias is not None:
            span = len(bucket_of)
            chain = n + 4 * span + b * (m // 64 + 2) + 64
            bar = bb + chain * U32 * (total + bb)
            ub = HALF[bias_dt]
            res["db"] = (db, bar + (ub + 4 * U32) * (np.abs(db) + bar) + (2.0**-25 if bias_dt == "f16" else 1e-37))
    return res


def step_reference(dt, q, k, v, k_cache, v_cache, positions, left, sinks=0, bias=None, bucket_of=None, scale=None):
    """``(out, bar), k_cache, v_cache`` of a step."""
    b, n, h, d = q.shape
    hk, ring = k.shape[2], k_cache.shape[1] - sinks
    scale = d**-0.5 if scale is None else scale
    out, kc, vc = oa.local_attention_step(q, k, v, k_cache, v_cache, positions, left, sinks, bias, bucket_of, scale)
    bar = np.zeros(out.shape)
    for i in range(b):
        p = int(positions[i])
        if p < 0:
            continue
        frames = np.array([f for f in range(p + n) if f < sinks or f >= p - left])
        slots = np.array([oa.ring_slot(int(f), sinks, ring) for f in frames])
        distance = frames[None, :] - (p + np.arange(n))[:, None]
        seen = (distance <= 0) & ((distance >= -left) | (frames < sinks)[None, :])
        added = np.zeros((n, len(frames), h)) if bias is None else oa._local_bias(bias, bucket_of, distance)[0]
        for j in range(h):
            kk, vv = kc[i, slots, j // (h // hk)], vc[i, slots, j // (h // hk)]
            w, lse = oa._local_weights(q[i, :, j], kk, scale, seen, added[..., j])
            off = np.where(np.isfinite(added[..., j]), np.abs(added[..., j]), 0.0)
            s = np.where(seen, np.abs(q[i, :, j] @ kk.T) * scale + off, 0.0)
            mag = np.where(seen, np.abs(q[i, :, j]) @ np.abs(kk).T * scale + off, 0.0)
            eps = _score_eps(s, mag, d + 1, len(frames), lse)
            inner = (eps + len(frames) * U32) * (w @ np.abs(vv)) + LOST * (seen @ np.abs(vv))
            bar[i, :, j] = inner + (HALF[dt] + 4 * U32) * (np.abs(out[i, :, j]) + inner)
    return (out, bar + (2.0**-25 if dt == "f16" else 1e-37)), kc, vc
