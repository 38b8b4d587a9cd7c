"""The cross attention in 64 bits with the largest error that the kernels' arithmetic allows, per element.

Derivation (``u`` = half a step of the storage dtype, ``u32`` = 2^-24; ``w`` the weights, ``f`` the dropout's
factors, ``x`` an input's magnitude):

* a score is a sum of ``D`` products in fp32, scaled and shifted in log2 units: off by at most ``(D + 8) u32`` of
  ``scale |q| |k|`` and ``4 u32`` of itself; exp2 adds 2 ``u32``, the row's sum ``M u32``, so a weight is off by
  ``eps_i`` (the row's largest such bound) relative, twice that with the normalisation;
* 16 bits: weights (and dS) are rounded once, ``u`` relative; what lies below fp16's normal numbers is off by half
  of 2^-24 over the scale it is held at (a row's largest weight is held at 2^6 or more in the forward, weights at
  2^14 and dS at 2^14 over its bound in the backward);
* exp2 gives 0 below fp32's normal numbers: a weight of less than 2^-126 may be lost whole, and is then off by
  2^-126 at most (a row whose scores spread over hundreds has such weights; their share of dK is
  2^-126 |dP - D| |q|, and |dP - D| is in the tens);
* ``D_i = sum dO o O`` takes the stored O, with its own error;
* every sum over ``M`` (or the rows) in fp32 adds its length times ``u32``; the result is rounded, ``u``.
"""

from __future__ import annotations

import numpy as np

import oracle.attention as oa

U32 = 2.0**-24
LOST = 2.0**-126
HALF = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def reference(dt, q, k, v, grad=None, key_mask=None, key_lengths=None, scale=None, p=0.0, seed=0, offset=0):
    """``{name: (value, bar)}`` for ``out``, ``lse`` and, with ``grad``, ``dq``, ``dk``, ``dv``."""
    b, n, h, d = q.shape
    m, hk = k.shape[1:3]
    g = h // hk
    scale = d**-0.5 if scale is None else scale
    u = HALF[dt]
    u16 = 0.0 if dt == "f32" else u
    tiny = 2.0**-25 if dt == "f16" else 1e-37
    seen = oa._seen(b, m, key_mask, key_lengths)
    keep = oa._keep(b, n, m, h, p, seed, offset)
    fmax = 1.0 if keep is None or not keep.size else max(1.0, float(keep.max()))
    out, lse = oa.cross_attention_forward(q, k, v, key_mask, key_lengths, scale, p, seed, offset)
    bar_out, bar_lse = np.zeros(out.shape), np.zeros(lse.shape)
    res = {}
    if grad is not None:
        dq, dk, dv = oa.cross_attention_backward(grad, q, k, v, key_mask, key_lengths, scale, p, seed, offset)
        bq, bk, bv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    for i in range(b):
        for j in range(h):
            c = j // g
            kk, vv = (np.where(seen[i][:, None], t[i, :, c], 0.0) for t in (k, v))
            w, _ = oa._weights(q[i, :, j], kk, scale, seen[i])
            f = np.ones((n, m)) if keep is None else keep[i, j]
            s = np.abs(q[i, :, j] @ kk.T) * scale
            mag = np.abs(q[i, :, j]) @ np.abs(kk).T * scale
            top = (mag * (d + 8) + s * 4).max(axis=1, initial=0.0) + np.abs(np.where(np.isfinite(lse[i, j]), lse[i, j], 0)) * 4
            eps = 2 * (top + m + 16)[:, None] * U32
            wf, av = w * f, np.abs(vv)
            wmax = w.max(axis=1, initial=0.0)[:, None]
            low = 2.0**-31 * fmax * wmax * av.sum(axis=0)[None] if dt == "f16" else 0.0
            ref = np.abs(out[i, :, j])
            inner = (u16 + eps + m * U32) * (wf @ av) + low + LOST * fmax * av.sum(axis=0)[None]
            bar_out[i, :, j] = inner + (u + 4 * U32) * (ref + inner) + tiny
            bar_lse[i, j] = eps[:, 0] + 4 * U32 * (1 + np.abs(np.where(np.isfinite(lse[i, j]), lse[i, j], 0)))
            if grad is None:
                continue
            dO, rows = np.abs(grad[i, :, j]), g * n
            gv = grad[i, :, j] @ vv.T
            dD = (dO * bar_out[i, :, j]).sum(axis=1) + d * U32 * (dO * (ref + bar_out[i, :, j])).sum(axis=1)
            D = (grad[i, :, j] * out[i, :, j]).sum(axis=1)
            inside = np.abs(gv * f - D[:, None])
            ds = w * inside
            bound = 2 * dO.sum(axis=1).max(initial=0.0) * av.max(initial=0.0) * fmax
            low_s = 2.0**-38 * bound * (seen[i][None, :] & np.ones((n, 1), bool)) if dt == "f16" else 0.0
            e_ds = w * (eps * inside + (d + 4) * U32 * f * (dO @ av.T) + dD[:, None])
            e_ds = e_ds + u16 * (ds + e_ds) + low_s + LOST * inside
            low_p = 2.0**-38 if dt == "f16" else 0.0
            e_pf = (u16 + eps + 2 * U32) * wf + (low_p + LOST * fmax) * (f > 0)
            bq[i, :, j] = scale * ((e_ds + (m + 4) * U32 * ds) @ np.abs(kk))
            bk[i, :, c] += scale * ((e_ds + (rows + 4) * U32 * ds).T @ np.abs(q[i, :, j]))
            bv[i, :, c] += (e_pf + (rows + 4) * U32 * wf).T @ dO
    res["out"], res["lse"] = (out, bar_out), (lse, bar_lse)
    if grad is not None:
        for name, x, bar in (("dq", dq, bq), ("dk", dk, bk), ("dv", dv, bv)):
            res[name] = (x, bar + (u + 4 * U32) * (np.abs(x) + bar) + tiny)
    return res


def check(actual, ref_bar, what):
    ref, bar = ref_bar
    a = actual.detach().double().cpu().numpy()
    assert a.shape == ref.shape, (what, a.shape, ref.shape)
    fin = np.isfinite(ref)
    assert np.array_equal(a[~fin], ref[~fin]), what
    if not fin.any():
        return
    err, lim = np.abs(a[fin] - ref[fin]), bar[fin]
    k = int(np.argmax(err / lim))
    assert np.all(err <= lim), (what, "error", err[k], "bar", lim[k], "of", ref[fin][k])
