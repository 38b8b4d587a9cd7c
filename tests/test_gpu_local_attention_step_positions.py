"""A step of the local attention at the ends of its positions."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_local_attention import _bias, _step_case


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,left,sinks,ring", [(1, 20, 3, 21), (5, 2, 0, 9), (4, 300, 5, 310)])
def test_streams_at_the_last_position(hip_ext, dtype, n, left, sinks, ring):
    """A ring behind its sinks repeats every ``ring`` frames, so a stream at the last position answers and writes what one
    as many rings before does, bit for bit; the lowest position is an idle stream's."""
    most = 2**31 - n
    near = most - ring * ((most - 3 * ring - sinks) // ring)
    q, k, v, kc, vc, pos = _step_case((3, n, 4, 2, 64), dtype, sinks + ring, [0, 0, -1])
    bias, plan = _bias(hip_ext, 4, 16, 40, False, torch.float32)
    results = []
    for positions in ([most, near, -1], [near, most, -(2**31)]):
        pos.copy_(torch.tensor(positions, dtype=torch.int64).to(torch.int32))
        caches = [t.clone() for t in (kc, vc)]
        out = hip_ext.local_attention_step(q, k, v, *caches, pos, left=left, sinks=sinks, bias=bias, bias_plan=plan)
        results.append([out, *caches])
    assert all(torch.equal(x, y) for x, y in zip(*results))
    assert bool((results[0][0][:2] != 0).any()) and bool((results[0][0][2] == 0).all())
    assert torch.equal(results[0][1][2], kc[2]) and not torch.equal(results[0][1][:2], kc[:2])
