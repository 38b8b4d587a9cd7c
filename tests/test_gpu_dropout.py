"""The counter-based dropout (alone, behind a GELU, before a residual sum), forward and backward.

Bars, derived from the arithmetic (``u`` = half a step of the storage dtype, relative; 0 below is the fp32
computation, whose steps are 2^-24):

* without an activation: one product by a rounded factor and, with a residual, one sum: 3 * 2^-24 of the
  magnitudes that enter, then ``u`` of the result;
* the GELU's two terms (``cdf`` and ``x phi``): 1.2e-6 of their magnitudes in fp32 (polynomial and its
  evaluation 4e-7, exp and reciprocal 1 ulp each, four products), 1.2e-5 in 16 bits (polynomial 7.3e-6,
  exponent's rounding 40 * 2^-24 where the tail is still above fp16's smallest number), then ``u``;
* fp16's and fp32's smallest numbers: half of 2^-24, and 1e-37.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import oracle.attention as oa
from pymsst_amd import _lib
from tests.conftest import to_np

_F = [torch.float32, torch.bfloat16, torch.float16]
_SEED, _OFFSET = 0x1234567_89ABCDEF, 0x7000000_00000005


def _rng(device, seed=_SEED, offset=_OFFSET):
    return torch.tensor([seed, offset], dtype=torch.int64, device=device)


def _check(actual, ref, dtype, inner, what):
    """``inner``: absolute bound of the fp32 computation's error, per element."""
    half = torch.finfo(dtype).eps / 2
    floor = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-25}[dtype]
    err = np.abs(to_np(actual) - ref)
    bar = inner + half * (np.abs(ref) + inner) + floor
    worst = np.argmax(err / bar)
    assert err.flat[worst] <= bar.flat[worst], (what, worst, to_np(actual).flat[worst], ref.flat[worst])


# ---------------------------------------------------------------------- CPU


def test_philox_known_answers():
    """The published 7-round vectors' zero case, and the oracle's vector form against its integer form."""
    assert oa.philox4x32((0, 0, 0, 0), (0, 0)) == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    assert oa.philox4x32((0, 0, 0, 0), (0, 0), 10) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    first = 2**32 - 2  # the counter's second word changes inside
    bits = oa.dropout_bits(first, 4, _SEED, _OFFSET).reshape(4, 8)
    for i in range(4):
        g = first + i
        words = oa.philox4x32((g & 0xFFFFFFFF, g >> 32, _OFFSET & 0xFFFFFFFF, _OFFSET >> 32),
                              (_SEED & 0xFFFFFFFF, _SEED >> 32))
        assert [w >> s & 0xFFFF for w in words for s in (0, 16)] == list(bits[i])


def test_oracle_gelu_gradient_against_differences():
    x = np.linspace(-6, 6, 241)
    h = 1e-5
    assert np.max(np.abs((oa.gelu(x + h) - oa.gelu(x - h)) / (2 * h) - oa.gelu_grad(x))) < 1e-9


def test_c_abi_refusals():
    lib = _lib.load_library()
    one = ctypes.c_void_p(16)  # never dereferenced: every call below is refused first
    assert lib.pmsst_dropout_forward(one, None, one, 8, 0.1, one, 0, 7, None) == -2
    for p in (-0.1, 1.0, float("nan")):
        assert lib.pmsst_dropout_forward(one, None, one, 8, p, one, 0, 0, None) == -1
        assert "probability" in _lib.last_error()
    assert lib.pmsst_dropout_forward(one, None, one, 8, 0.1, one, 1, 0, None) == -1  # tanh is not its activation
    assert lib.pmsst_dropout_forward(None, None, one, 8, 0.1, one, 0, 0, None) == -1
    assert lib.pmsst_dropout_forward(one, None, one, 8, 0.1, None, 0, 0, None) == -1
    assert "rng" in _lib.last_error()
    assert lib.pmsst_dropout_forward(one, None, one, -1, 0.1, one, 0, 0, None) == -1
    assert lib.pmsst_dropout_forward(one, None, one, 2**60, 0.1, one, 0, 0, None) == -1  # more than one grid
    assert lib.pmsst_dropout_backward(one, None, one, 8, 0.1, one, 2, 0, None) == -1  # GELU needs x
    assert lib.pmsst_dropout_forward(None, None, None, 0, 0.1, one, 0, 0, None) == 0  # nothing to do


def test_calls_past_the_grid_are_refused():
    """A launch has less than 2^32 work-items: more elements are an argument error, not a launch's."""
    lib = _lib.load_library()
    one = ctypes.c_void_p(16)  # never dereferenced
    assert lib.pmsst_dropout_forward(one, None, one, 2**40, 0.1, one, 0, 0, None) == -1
    assert "too many" in _lib.last_error()


# ---------------------------------------------------------------------- GPU


def _inputs(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (3.0 * torch.randn(shape, generator=g)).to(dtype)
    return x, torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (130, 64), (61, 67), (3, 4097), (1031, 192)])
@pytest.mark.parametrize("form", ["plain", "residual", "gelu", "gelu_residual"])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5])
def test_forward_and_backward(hip_ext, dtype, shape, form, p):
    x, dy, res = (t.cuda() for t in _inputs(shape, dtype, 5))
    act = "gelu" if "gelu" in form else None
    residual = res if "residual" in form else None
    rng = _rng("cuda")
    y = hip_ext.dropout_forward(x, p, rng, activation=act, residual=residual)
    dx = hip_ext.dropout_backward(dy, p, rng, x=x if act else None, activation=act)
    assert y.shape == dx.shape == x.shape and y.dtype == dx.dtype == dtype
    xn, dn = to_np(x), to_np(dy)
    f = oa.dropout_factors(xn.size, p, _SEED, _OFFSET).reshape(xn.shape)
    ref = oa.dropout_forward(xn, p, _SEED, _OFFSET, act, None if residual is None else to_np(residual))
    gref = oa.dropout_backward(dn, p, _SEED, _OFFSET, xn, act)
    if act:
        rel = 1.2e-6 if dtype == torch.float32 else 1.2e-5
        phi = xn * np.exp(-0.5 * xn * xn) / np.sqrt(2 * np.pi)
        inner, ginner = rel * f * np.abs(oa.gelu(xn)), rel * f * np.abs(dn) * (np.abs(oa.gelu_grad(xn) - phi) + np.abs(phi))
    else:
        inner, ginner = 2.0**-23 * f * np.abs(xn), 2.0**-23 * f * np.abs(dn)
    if residual is not None:
        inner = inner + 2.0**-24 * (np.abs(ref) + inner)
    _check(y, ref, dtype, inner, "y")
    _check(dx, gref, dtype, ginner, "dx")
    if residual is None:
        assert bool(((y == 0) | (torch.from_numpy(f).cuda() > 0)).all())  # what is dropped is 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_tails_and_special_values(hip_ext, dtype):
    """The GELU's tails, the infinities and NaN; a dropped NaN is 0."""
    x = torch.cat([torch.linspace(-14, 14, 4001), torch.tensor([float("inf"), float("nan"), -3e4, 3e4])]).to(dtype).cuda()
    y = hip_ext.dropout_forward(x, 0.0, None, activation="gelu")
    ref = oa.gelu(to_np(x[:4001]))
    rel = 1.2e-6 if dtype == torch.float32 else 2e-5  # (14^2 / 2 log2 e) 2^-24 in the exponent, 16 bits
    _check(y[:4001], ref, dtype, rel * np.abs(ref), "tail")
    assert y[4001] == float("inf") and torch.isnan(y[4002]) and y[4003] == 0 and y[4004] == x[4004]
    dx = hip_ext.dropout_backward(torch.ones_like(x), 0.0, None, x=x, activation="gelu")
    assert torch.isnan(dx[4002]) and dx[4003] == 0 and dx[4004] == 1
    bad = torch.full((4096,), float("nan"), dtype=dtype, device="cuda")
    z = hip_ext.dropout_forward(bad, 0.5, _rng("cuda"))
    kept = torch.from_numpy(oa.dropout_factors(4096, 0.5, _SEED, _OFFSET) > 0).cuda()
    assert bool((z[~kept] == 0).all()) and bool(torch.isnan(z[kept]).all())


@pytest.mark.gpu
def test_probability_is_held(hip_ext):
    """The share of a long row that is dropped, and of each of its 8 places: within 6 standard deviations."""
    for p in (0.01, 0.1, 0.9):
        y = hip_ext.dropout_forward(torch.ones(8 * 200_000, device="cuda"), p, _rng("cuda", 11, 3)).reshape(-1, 8)
        dropped = (y == 0).double().mean(dim=0).cpu()
        assert float((dropped - p).abs().max()) < 6 * (p * (1 - p) / 200_000) ** 0.5 + 2.0**-17
        assert abs(float(y.double().mean()) - 1) < 6 * (p / (1 - p) / 1_600_000) ** 0.5 + 1e-6


@pytest.mark.gpu
def test_views_streams_and_captured_replays(hip_ext):
    """A view that starts between 16 bytes, a transposed one, another stream, and a captured call whose seed and
    offset change between replays."""
    x = torch.randn(4001, device="cuda").to(torch.bfloat16)
    rng = _rng("cuda", 3, 4)
    a = hip_ext.dropout_forward(x[1:], 0.3, rng, activation="gelu", residual=x[:-1])
    b = hip_ext.dropout_forward(x[1:].clone(), 0.3, rng, activation="gelu", residual=x[:-1].clone())
    assert torch.equal(a, b)
    t = torch.randn(40, 33, device="cuda")
    assert torch.equal(hip_ext.dropout_forward(t.t(), 0.3, rng), hip_ext.dropout_forward(t.t().contiguous(), 0.3, rng))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = hip_ext.dropout_forward(x, 0.3, rng)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c, hip_ext.dropout_forward(x, 0.3, rng))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hip_ext.dropout_forward(x, 0.3, rng)
        dx = hip_ext.dropout_backward(y, 0.3, rng)
    for step in range(4):
        rng.copy_(_rng("cuda", 3 + step // 2, 40 + step))
        graph.replay()
        torch.cuda.synchronize()
        want = hip_ext.dropout_forward(x, 0.3, rng)
        assert torch.equal(y, want) and torch.equal(dx, hip_ext.dropout_backward(want, 0.3, rng))


@pytest.mark.gpu
def test_refusals(hip_ext):
    x = torch.zeros(8, device="cuda")
    rng = _rng("cuda")
    for call in (
        lambda: hip_ext.dropout_forward(x.cpu(), 0.1, rng),
        lambda: hip_ext.dropout_forward(x, 1.0, rng),
        lambda: hip_ext.dropout_forward(x, float("nan"), rng),
        lambda: hip_ext.dropout_forward(x, 0.1, None),
        lambda: hip_ext.dropout_forward(x, 0.1, rng.cpu()),
        lambda: hip_ext.dropout_forward(x, 0.1, rng.int()),
        lambda: hip_ext.dropout_forward(x, 0.1, rng[:1]),
        lambda: hip_ext.dropout_forward(x, 0.1, rng, residual=x[:4]),
        lambda: hip_ext.dropout_forward(x, 0.1, rng, residual=x.half()),
        lambda: hip_ext.dropout_forward(x.double(), 0.1, rng),
        lambda: hip_ext.dropout_backward(x, 0.1, rng, activation="gelu"),
        lambda: hip_ext.dropout_backward(x, 0.1, rng, x=x[:4], activation="gelu"),
    ):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        hip_ext.dropout_forward(x, 0.1, rng, activation="tanh")
    assert hip_ext.dropout_forward(x[:0], 0.1, rng).numel() == 0
