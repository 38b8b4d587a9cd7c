"""The local attention's memory: the workspace that the sizes ask for, and calls that need none."""

from __future__ import annotations

import ctypes

import pytest
import torch

from pymsst_amd import _lib
from tests import local_attention_bars as bars
from tests.conftest import dt_name, to_np
from tests.test_gpu_local_attention import _inputs


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_backward_that_needs_no_workspace_takes_none(hip_ext, dtype):
    """Many batch rows of up to 64 frames without a bias, through the C entry: size 0, and a null workspace (or one at any
    address) is taken."""
    b, n, m, h, hk, d = 256, 9, 21, 2, 1, 32
    lib, code = _lib.load_library(), {torch.float16: 1, torch.bfloat16: 2}[dtype]
    q, k, v, do, _, _ = _inputs((b, n, m, h, hk, d), dtype, seed=4)
    out, lse = hip_ext.local_attention_forward(q, k, v, left=6, right=4, sinks=2, need_lse=True)
    ref = bars.reference(dt_name(dtype), *map(to_np, (q, k, v, do)), left=6, right=4, sinks=2)
    assert lib.pmsst_local_attention_backward_workspace_size(b, n, m, h, hk, d, 6, 4, 2, 0, -1, code) == 0
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for workspace in (None, ctypes.c_void_p(out.data_ptr() + 2)):  # of no bytes: nothing is written there
        grads = [torch.full_like(t, float("nan")) for t in (q, k, v)]
        rc = lib.pmsst_local_attention_backward(_p(do), None, _p(q), None, _p(k), None, _p(v), None, _p(out), _p(lse), None, 0,
                                                None, None, 6, 4, 2, None, 0, None, None, None, 0, 0, *map(_p, grads), None, b, n, m,
                                                h, hk, d, d**-0.5, code, workspace, 0, stream)
        assert rc == 0, lib.pmsst_last_error()
        for name, t in zip(("dq", "dk", "dv"), grads):
            bars.check(t, ref[name], (name, dtype))
