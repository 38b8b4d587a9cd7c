"""Cross attention where its tiles end: rows past the last query, group sizes that do not divide a tile, every way the
blocks are numbered, and fp16's powers of two over row tiles of different magnitudes.  Values and gradients against
the 64-bit statement, with the bars of ``attention_bars``."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle.attention as oa
from tests import attention_bars as bars
from tests.conftest import dt_name, to_np

_F = [torch.float32, torch.bfloat16, torch.float16]
_SEED, _OFFSET = 0x1234567_89ABCDEF, 0x7000000_00000005


def _rng():
    return torch.tensor([_SEED, _OFFSET], dtype=torch.int64, device="cuda")


def _inputs(shape, dtype, seed=0):
    b, n, m, h, hk, d = shape
    g = torch.Generator().manual_seed(seed)
    q, do = (torch.randn(b, n, h, d, generator=g).to(dtype).cuda() for _ in range(2))
    k, v = (torch.randn(b, m, hk, d, generator=g).to(dtype).cuda() for _ in range(2))
    return q, k, v, do


def _run(ext, q, k, v, do, **kw):
    out, lse = ext.cross_attention_forward(q, k, v, need_lse=True, **kw)
    return (out, lse, *ext.cross_attention_backward(do, q, k, v, out, lse, **kw))


_NAMES = ("out", "lse", "dq", "dk", "dv")


# ---------------------------------------------------------------------- rows past the last query


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape", [(1, 5, 40, 2, 2, 64), (1, 5, 90, 2, 1, 64), (2, 65, 64, 3, 1, 32), (1, 130, 300, 2, 2, 128),
                                   (1, 700, 20, 2, 2, 40)])
def test_an_infinite_gradient_in_the_last_row_reaches_dv_as_one(hip_ext, dtype, shape):
    """dV is P^T dO: where one dO is infinite, so is every key's dV in that column (P > 0 here), in the tile's last
    row as in any other."""
    n, h, hk = shape[1], shape[3], shape[4]
    for row in (n - 1, 0):
        q, k, v, do = _inputs(shape, dtype)
        do[-1, row, h - 1, 3] = float("inf")
        dv = _run(hip_ext, q, k, v, do)[4]
        assert bool((dv[-1, :, hk - 1, 3] == torch.inf).all()), row
        dv[-1, :, hk - 1, 3] = 0
        assert bool(torch.isfinite(dv).all())
