"""A step of the local attention beside autograd: its writes into the caches are known to it."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_local_attention import _step_case


@pytest.mark.gpu
def test_a_backward_that_has_saved_a_cache_fails_after_a_step(hip_ext):
    q, k, v, kc, vc, pos = _step_case((2, 1, 4, 2, 64), torch.float32, 24, [5, 70])
    for place in (0, 1):
        w = torch.randn_like(kc, requires_grad=True)
        loss = ((kc, vc)[place] * w).sum()  # saves the cache
        hip_ext.local_attention_step(q, k, v, kc, vc, pos, left=20, sinks=3)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    # parts of one buffer share its counter, and an idle call counts too (what it writes is known on the device alone)
    both = torch.randn(2, 2, 24, 2, 64, device="cuda")
    before = both._version
    hip_ext.local_attention_step(q, k, v, both[0], both[1], torch.full_like(pos, -1), left=20, sinks=3)
    assert both._version > before


@pytest.mark.gpu
def test_caches_and_gradients(hip_ext):
    """Caches that require a gradient are refused, as torch refuses to write into a leaf; without gradients, and with tensors
    of inference mode, the step is the same; its output requires none."""
    q, k, v, kc, vc, pos = _step_case((2, 1, 4, 2, 64), torch.bfloat16, 24, [5, 70])
    caches = [t.clone() for t in (kc, vc)]
    want = hip_ext.local_attention_step(q, k, v, kc, vc, pos, left=20, sinks=3)
    leaf = caches[0].clone().requires_grad_()
    for bad in ((leaf, caches[1]), (caches[1], leaf), (leaf * 1, caches[1])):
        with pytest.raises(RuntimeError, match="require a gradient"):
            hip_ext.local_attention_step(q, k, v, *bad, pos, left=20, sinks=3)
    assert torch.equal(leaf, caches[0])
    with torch.no_grad():
        assert torch.equal(hip_ext.local_attention_step(q, k, v, leaf, caches[1].clone(), pos, left=20, sinks=3), want)
    with torch.inference_mode():
        frozen = [t.clone() for t in caches]
        assert torch.equal(hip_ext.local_attention_step(q, k, v, *frozen, pos, left=20, sinks=3), want)
    got = hip_ext.local_attention_step(q.clone().requires_grad_(), k, v, *[t.clone() for t in caches], pos, left=20, sinks=3)
    assert torch.equal(got, want) and not got.requires_grad
