"""Local attention (windows, sinks, learned relative bias, frame-by-frame steps) against the 64-bit statement; the bars
are derived in ``local_attention_bars``."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle.attention as oa
from pymsst_amd.extension import relative_buckets
from tests import local_attention_bars as bars
from tests.conftest import dt_name, to_np

_F = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(shape, dtype, mask="none", seed=0):
    b, n, m, h, hk, d = shape
    g = torch.Generator().manual_seed(seed)
    q, do = (torch.randn(b, n, h, d, generator=g).to(dtype).cuda() for _ in range(2))
    k, v = (torch.randn(b, m, hk, d, generator=g).to(dtype).cuda() for _ in range(2))
    km = kl = None
    if mask in ("keys", "both"):
        km = torch.rand(b, m, generator=g) < 0.6
        km[0] = False  # one batch row that sees nothing
        km = km.cuda()
    if mask in ("lengths", "both"):
        kl = torch.randint(0, m + 1, (b,), generator=g, dtype=torch.int32)
        kl[-1] = m + 5  # cut to m
        kl = kl.cuda()
    return q, k, v, do, km, kl


def _none_or(f, t):
    return None if t is None else f(t)


def _bias(ext, h, buckets, distance, two_sided, dtype, seed=5):
    if not buckets:
        return None, None
    g = torch.Generator().manual_seed(seed)
    table = (torch.randn(buckets, h, generator=g) * 0.7).to(dtype).cuda()
    return table, ext.relative_bias_plan(buckets, distance, "cuda", bidirectional=two_sided)


def check_attention(ext, shape, dtype, left=None, right=None, sinks=0, buckets=0, distance=0, mask="none", starts=None, seed=0,
                    scale=None, bias_dtype=torch.float32, edit=None):
    q, k, v, do, km, kl = _inputs(shape, dtype, mask, seed)
    if edit is not None:
        q, k, v, do = edit(q, k, v, do)
    bias, plan = _bias(ext, shape[3], buckets, distance, right != 0, bias_dtype)
    qs = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    kw = dict(left=left, right=right, sinks=sinks, bias=bias, bias_plan=plan, key_mask=km, key_lengths=kl, query_starts=qs,
              scale=scale)
    out, lse = ext.local_attention_forward(q, k, v, need_lse=True, **kw)
    grads = ext.local_attention_backward(do, q, k, v, out, lse, **kw)
    ref = bars.reference(dt_name(dtype), to_np(q), to_np(k), to_np(v), to_np(do), dt_name(bias_dtype), left, right, sinks,
                         _none_or(to_np, bias), _none_or(lambda p: p.bucket_of.cpu().numpy(), plan),
                         _none_or(lambda t: t.cpu().numpy(), km), _none_or(lambda t: t.cpu().numpy(), kl), starts, scale)
    what = (shape, dtype, left, right, sinks, buckets, distance, mask, starts)
    for name, t in zip(("out", "lse", "dq", "dk", "dv", "db"), (out, lse, *grads)):
        bars.check(t, ref[name], (name, what))
    return out, lse, grads


# ---------------------------------------------------------------------- GPU

_SHAPES = [
    # b, n, m, h, hk, d
    (2, 70, 70, 4, 2, 64),
    (1, 1, 1, 1, 1, 8),
    (3, 130, 130, 2, 1, 32),
    (2, 33, 257, 6, 3, 40),
    (1, 258, 258, 2, 2, 128),
    (2, 62, 62, 8, 8, 64),
    (1, 300, 300, 3, 1, 72),
]
_RULES = [
    # left, right, sinks, buckets, distance
    (None, None, 0, 32, 24),
    (None, 0, 0, 0, 0),
    (20, 0, 3, 16, 48),
    (17, 40, 2, 0, 0),
    (40, 9, 35, 32, 128),
    (0, 0, 1, 8, 5),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape", _SHAPES)
@pytest.mark.parametrize("rule", _RULES)
@pytest.mark.parametrize("mask", ["none", "both"])
def test_forward_and_backward(hip_ext, dtype, shape, rule, mask):
    check_attention(hip_ext, shape, dtype, *rule, mask=mask, bias_dtype=dtype if mask == "both" else torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape", [(33, 62, 62, 8, 8, 64), (65, 70, 33, 8, 4, 32), (260, 5, 64, 2, 1, 128), (129, 130, 1, 2, 2, 40)])
@pytest.mark.parametrize("rule", [(None, None, 0, 32, 24), (9, 12, 3, 16, 40), (20, 0, 2, 0, 0)])
@pytest.mark.parametrize("mask", ["none", "both"])
def test_few_frames_of_many_pairs(hip_ext, dtype, shape, rule, mask):
    check_attention(hip_ext, shape, dtype, *rule, mask=mask, seed=2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape,rule,starts", [
    ((2, 40, 900, 2, 2, 64), (300, 0, 4, 32, 128), [860, 333]),   # a chunk over a longer cache: split forward
    ((2, 3, 2000, 8, 2, 64), (None, 0, 0, 32, 64), [1997, -2]),
    ((1, 513, 513, 4, 1, 64), (60, 11, 5, 16, 1000), None),       # the sinks' later queries in blocks of their own
    ((2, 700, 640, 2, 2, 32), (130, 0, 140, 0, 0), [5, -100]),    # two tiles of sinks, split
    ((3, 100, 90, 2, 1, 128), (30, 20, 2, 8, 9), [10**9, -(10**9), 80]),  # queries that see sinks alone, or nothing
    ((1, 600, 600, 2, 2, 64), (0, 0, 0, 8, 6), None),             # a frame sees itself
    ((1, 200, 200, 2, 2, 64), (None, None, 0, 8, 1024), None),    # distances beyond every pair
])
@pytest.mark.parametrize("mask", ["none", "lengths"])
def test_windows_starts_and_splits(hip_ext, dtype, shape, rule, starts, mask):
    check_attention(hip_ext, shape, dtype, *rule, mask=mask, starts=starts, seed=4)


def _step_case(shape, dtype, slots, positions, seed=0):
    b, n, h, hk, d = shape
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, n, h, d, generator=g).to(dtype).cuda()
    k, v = (torch.randn(b, n, hk, d, generator=g).to(dtype).cuda() for _ in range(2))
    kc, vc = (torch.randn(b, slots, hk, d, generator=g).to(dtype).cuda() for _ in range(2))
    return q, k, v, kc, vc, torch.tensor(positions, dtype=torch.int32, device="cuda")


def check_step(ext, shape, dtype, left, sinks, ring, positions, buckets=0, distance=0, seed=0, bias_dtype=torch.float32, edit=None):
    q, k, v, kc, vc, pos = _step_case(shape, dtype, sinks + ring, positions, seed)
    if edit is not None:
        q, k, v, kc, vc = edit(q, k, v, kc, vc)
    bias, plan = _bias(ext, shape[2], buckets, distance, False, bias_dtype)
    ref, want_k, want_v = bars.step_reference(dt_name(dtype), *map(to_np, (q, k, v, kc, vc)), positions, left, sinks,
                                              _none_or(to_np, bias), _none_or(lambda p: p.bucket_of.cpu().numpy(), plan))
    out = ext.local_attention_step(q, k, v, kc, vc, pos, left, sinks, bias=bias, bias_plan=plan)
    what = (shape, dtype, left, sinks, ring, positions, buckets)
    assert np.array_equal(to_np(kc), want_k) and np.array_equal(to_np(vc), want_v), what
    bars.check(out, ref, what)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape,left,sinks,ring,positions", [
    ((1, 1, 4, 4, 32), 64, 2, 65, [500]),
    ((4, 1, 8, 8, 64), 30, 4, 31, [0, 3, 34, -1]),
    ((5, 1, 4, 2, 128), 100, 0, 120, [99, 100, 101, 1000003, 1]),
    ((3, 4, 8, 2, 40), 21, 5, 40, [2, 44, 10000]),
    ((2, 7, 6, 1, 96), 50, 3, 57, [52, 7]),
    ((2, 3, 16, 2, 8), 9, 0, 12, [8, 100]),
    ((2, 1, 1, 1, 64), 0, 0, 1, [0, 5]),
    ((1, 1, 2, 2, 64), 5000, 8, 5010, [60001]),  # split over the frames
    ((1, 2, 12, 2, 72), 3000, 40, 3002, [2999]),
])
@pytest.mark.parametrize("buckets,distance", [(0, 0), (16, 48)])
def test_step(hip_ext, dtype, shape, left, sinks, ring, positions, buckets, distance):
    check_step(hip_ext, shape, dtype, left, sinks, ring, positions, buckets, distance,
               bias_dtype=torch.float32 if buckets == 16 and shape[1] == 1 else dtype)
