"""The local attention's memory: the workspace that the sizes ask for, and calls that need none."""

from __future__ import annotations

import ctypes

import pytest
import torch

from pymsst_amd import _lib
from pymsst_amd import extension as ext_mod
from tests import local_attention_bars as bars
from tests.conftest import dt_name, to_np
from tests.test_gpu_guard_writes import _GuardedTorch
from tests.test_gpu_local_attention import _inputs, check_attention


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


def _backward_bytes(b, n, h, hk, d, left, right, sinks, dtype, distance=-1):
    return _lib.load_library().pmsst_local_attention_backward_workspace_size(b, n, n, h, hk, d, left, right, sinks, 0, distance, dtype)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("b,h,hk,d,left,right,sinks", [(1, 8, 8, 64, 128, 128, 4), (1, 8, 1, 64, 64, 64, 4), (16, 8, 8, 64, 128, 128, 2048),
                                                       (2, 16, 4, 128, 300, 0, 700), (40, 4, 4, 32, 20, 5, 1)])
def test_the_sinks_parts_do_not_grow_with_the_square_of_the_frames(b, h, hk, d, left, right, sinks, dtype):
    """The backward's workspace with sinks: statistics of the rows (two fp32 each, and a bit), fp16's maxima, the parts of
    split blocks (up to 1024 blocks of 128 frames, dK and dV) or of the sinks' own blocks, and the sinks' later rows',
    which are sums of the sinks alone: 64 MB, one part, or as much as dK and dV in fp32."""
    sizes = []
    for n in (8064, 16128, 32256, 64512):
        need = _backward_bytes(b, n, h, hk, d, left, right, sinks, dtype)
        row = 8 * d * b * hk  # bytes of a frame's dK and dV of all pairs, in fp32
        stat = 9 * b * h * (n + 64) + 128 * b * hk + 4096
        own = max(1024 * 128 * 8 * d, (sinks + 128) * row)
        assert need <= stat + own + max(64 << 20, sinks * row, n * row), (n, need)
        sizes.append(need)
    assert sizes[3] - sizes[2] <= 2.2 * (sizes[2] - sizes[1]) + (64 << 20), sizes


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,left,sinks", [((4, 1100, 1100, 8, 2, 128), 10, 1024), ((1, 900, 900, 4, 1, 64), 30, 5),
                                              ((1, 500, 400, 4, 2, 40), 9, 450), ((70, 300, 300, 4, 4, 32), 12, 130)])
def test_gradients_of_sinks_that_several_blocks_share(hip_ext, monkeypatch, dtype, shape, left, sinks):
    """Blocks split over their queries beside the sinks' own blocks, many sinks (whose parts are fewer than their tiles
    ask for), more sinks than frames, unsplit blocks; nothing is written outside the workspace."""
    guard = _GuardedTorch(torch)
    monkeypatch.setattr(ext_mod, "torch", guard)
    check_attention(hip_ext, shape, dtype, left=left, right=3, sinks=sinks)
    assert not guard.damaged()


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
