"""Local attention where the learned bias hides frames: a query that is left with one frame learns nothing from it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle.attention as oa
from tests import local_attention_bars as bars
from tests.conftest import dt_name, to_np
from tests.test_gpu_local_attention import _inputs

_F = [torch.float32, torch.bfloat16, torch.float16]


def _table(distance, shown, heads, per_head=True):
    """A bucket a distance; ``shown`` are the distances whose entries are finite in the even heads, all of them in the odd."""
    g = torch.Generator().manual_seed(3)
    table = torch.randn(2 * distance + 1, heads, generator=g)
    hidden = torch.tensor([d not in shown for d in range(-distance, distance + 1)])
    table[hidden, ::2 if per_head else 1] = -torch.inf
    return table


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape", [(2, 150, 150, 4, 2, 64), (130, 45, 45, 4, 2, 32), (130, 64, 64, 2, 2, 128), (1, 70, 300, 2, 1, 128),
                                   (1, 1, 9, 2, 2, 8)])
@pytest.mark.parametrize("distance,shown,rule", [
    (12, [0], {}),                                      # itself alone
    (12, [-2, 7], dict(left=5, right=7, sinks=1)),      # one or two of a window
    (5, [-5], dict(right=0)),                           # those far behind: the first queries see none, then one, then more
    (40, [-40, 3], dict(left=60, sinks=2, masked=True)),
    (3, [], {}),                                        # none
])
def test_a_frame_that_the_bias_leaves_alone(hip_ext, dtype, shape, distance, shown, rule):
    """Exact zeros in dQ where window, sinks, masks and bias leave a query one frame (or none), and in dK and the bias's
    gradient where only such queries see a frame or a bucket; everything within the bars of the 64-bit statement."""
    rule = dict(rule)
    b, n, m, h, hk, d = shape
    q, k, v, do, km, kl = _inputs(shape, dtype, "both" if rule.pop("masked", False) else "none", seed=12)
    table = _table(distance, shown, h)
    plan = hip_ext.relative_bias_plan(2 * distance + 1, distance, "cuda", bucket_of=list(range(2 * distance + 1)))
    kw = dict(rule, bias=table.cuda(), bias_plan=plan, key_mask=km, key_lengths=kl)
    out, lse = hip_ext.local_attention_forward(q, k, v, need_lse=True, **kw)
    results = (out, lse, *hip_ext.local_attention_backward(do, q, k, v, out, lse, **kw))
    masks = [None if t is None else t.cpu().numpy() for t in (km, kl)]
    ref = bars.reference(dt_name(dtype), *map(to_np, (q, k, v, do)), "f32", rule.get("left"), rule.get("right"), rule.get("sinks", 0),
                         to_np(table), np.arange(2 * distance + 1), *masks)
    for name, t in zip(("out", "lse", "dq", "dk", "dv", "db"), results):
        bars.check(t, ref[name], (name, shape, dtype, distance, shown, rule))
    window = oa.local_seen(b, n, m, rule.get("left"), rule.get("right"), rule.get("sinks", 0), None, *masks)
    bucket = np.clip(np.arange(m)[None] - np.arange(n)[:, None], -distance, distance) + distance
    seen = window[..., None] & np.isfinite(to_np(table))[bucket][None]  # [B, N, M, H]
    learns = seen & (seen.sum(axis=2, keepdims=True) > 1)
    assert bool((to_np(results[2])[~learns.any(axis=2)] == 0).all())
    assert bool((to_np(results[3])[~learns.any(axis=1).reshape(b, m, hk, h // hk).any(axis=3)] == 0).all())
    unlearnt = np.ones(table.shape, dtype=bool)
    for c in range(2 * distance + 1):
        unlearnt[c] = ~learns[:, bucket == c].any(axis=(0, 1))
    assert bool((to_np(results[5])[unlearnt] == 0).all())
