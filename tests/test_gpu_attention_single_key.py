"""Queries that see exactly one key: the weight is 1 whatever the score, so neither the score's gradient nor, through
it, the query's or the key's can be anything but zero."""

from __future__ import annotations

import pytest
import torch

from tests import attention_bars as bars
from tests.conftest import dt_name, to_np

_F = [torch.float32, torch.bfloat16, torch.float16]
_SEED, _OFFSET = 0x1234567_89ABCDEF, 0x7000000_00000005


def _inputs(shape, dtype, seed=0):
    b, n, m, h, hk, d = shape
    g = torch.Generator().manual_seed(seed)
    q, do = (torch.randn(b, n, h, d, generator=g).to(dtype).cuda() for _ in range(2))
    k, v = (torch.randn(b, m, hk, d, generator=g).to(dtype).cuda() for _ in range(2))
    return q, k, v, do


def _run(ext, q, k, v, do, km, kl, p):
    kw = dict(key_mask=km, key_lengths=kl, dropout_p=p,
              rng=torch.tensor([_SEED, _OFFSET], dtype=torch.int64, device="cuda") if p else None)
    out, lse = ext.cross_attention_forward(q, k, v, need_lse=True, **kw)
    return (out, lse, *ext.cross_attention_backward(do, q, k, v, out, lse, **kw))


def _check(results, q, k, v, do, km, kl, p, rows=slice(None)):
    ref = bars.reference(dt_name(q.dtype), *(to_np(t) for t in (q, k, v, do)), None if km is None else km.cpu().numpy(),
                         None if kl is None else kl.cpu().numpy(), None, p, _SEED, _OFFSET)
    for name, t in zip(("out", "lse", "dq", "dk", "dv"), results):
        bars.check(t, ref[name], (name, tuple(q.shape), tuple(k.shape), p))


_SHAPES = [
    # b, n, m, h, hk, d
    (1, 1, 1, 1, 1, 8),
    (2, 70, 1, 4, 2, 64),
    (1, 700, 1, 8, 8, 64),
    (3, 5, 1, 2, 2, 128),
    (2, 33, 2, 4, 2, 64),
    (2, 130, 64, 3, 1, 40),
    (2, 37, 65, 4, 4, 32),
    (2, 70, 700, 4, 2, 64),    # keys split over blocks, in the queries' kernel too
    (1, 900, 66, 2, 1, 128),   # rows split
    (2, 1, 3000, 2, 2, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape", _SHAPES)
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("by", ["mask", "lengths", "both"])
def test_gradients_of_queries_and_keys_are_zero(hip_ext, dtype, shape, p, by):
    b, _, m = shape[:3]
    if m == 1 and by != "mask":
        by = "none"
    places = [m - 1] if m == 1 else [0, m // 2, m - 1] if by == "mask" else [0]
    for place in places:
        km = kl = None
        if by in ("mask", "both"):
            km = torch.zeros(b, m, dtype=torch.bool, device="cuda")
            km[:, place] = True
            if by == "both":
                km[:, 1:] = True
        if by in ("lengths", "both"):
            kl = torch.ones(b, dtype=torch.int32, device="cuda")
        q, k, v, do = _inputs(shape, dtype, seed=place)
        q = q * 4  # scores of tens, whose log-sums are rounded further from them
        results = _run(hip_ext, q, k, v, do, km, kl, p)
        assert bool((results[2] == 0).all()), ("dq", place, results[2].abs().max())
        assert bool((results[3] == 0).all()), ("dk", place, results[3].abs().max())
        _check(results, q, k, v, do, km, kl, p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("m", [40, 150, 1500])
def test_batch_rows_of_none_one_two_and_all_keys(hip_ext, dtype, m):
    """Each batch row has its own count: one key gives zeros, two (in one tile, in two tiles, at the ends) do not."""
    q, k, v, do = _inputs((6, 45, m, 4, 2, 64), dtype, seed=m)
    km = torch.zeros(6, m, dtype=torch.bool, device="cuda")
    for row, keys in enumerate(([], [m // 3], [3, 4], [0, m - 1], [m - 40, m - 1], list(range(m)))):
        km[row, keys] = True
    for p in (0.0, 0.3):
        results = _run(hip_ext, q, k, v, do, km, None, p)
        _check(results, q, k, v, do, km, None, p)
        for grad in results[2:4]:
            assert bool((grad[:2] == 0).all())
            for row in range(3, 6) if p == 0 else (5,):
                assert bool((grad[row] != 0).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("m", [1, 200])
def test_a_gradient_that_is_no_number_stays_one(hip_ext, dtype, m):
    """NaN minus itself is no zero: a row whose incoming gradient holds one says so in its query's gradient."""
    q, k, v, do = _inputs((1, 9, m, 2, 2, 32), dtype)
    do[0, 4, 1, 3] = float("nan")
    kl = torch.ones(1, dtype=torch.int32, device="cuda")
    dq, dk = _run(hip_ext, q, k, v, do, None, kl, 0.0)[2:4]
    assert bool(torch.isnan(dq[0, 4, 1]).all()) and bool(torch.isnan(dk[0, 0, 1]).all())
    rest = torch.ones(dq.shape[:3], dtype=torch.bool, device="cuda")
    rest[0, 4, 1] = False
    assert bool((dq[rest] == 0).all()) and bool((dk[0, :, 0] == 0).all())
