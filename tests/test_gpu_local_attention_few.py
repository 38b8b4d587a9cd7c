"""Local attention over up to 64 frames of many batch rows (one backward kernel): queries that stand anywhere, and many of
them."""

from __future__ import annotations

import random

import pytest
import torch

from tests.test_gpu_local_attention import check_attention


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,far", [((130, 70, 60, 4, 2, 64), 90), ((260, 1, 64, 2, 1, 32), 40), ((130, 1100, 33, 2, 2, 40), 1000), ((64, 130, 64, 4, 4, 128), 200)])
@pytest.mark.parametrize("rule", [dict(left=20, right=5, sinks=3, buckets=16, distance=30), dict(right=0, buckets=8, distance=12), dict(left=9, right=70),
                                  dict(left=40, sinks=70, buckets=32, distance=100, mask="both")])
def test_queries_that_stand_anywhere(hip_ext, dtype, shape, far, rule):
    """Starts before the first frame, among the frames and past the last one, so that rows see none, some or all of them."""
    rng = random.Random(17)
    starts = [rng.randint(-far, far) for _ in range(shape[0])]
    starts[:3] = [2**29, -(2**31), 0]
    check_attention(hip_ext, shape, dtype, starts=starts, **rule)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_queries_over_few_frames(hip_ext, dtype):
    check_attention(hip_ext, (64, 2100, 50, 4, 4, 32), dtype, left=2000, right=0, sinks=2, buckets=16, distance=60)
