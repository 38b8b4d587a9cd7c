"""Cross attention, forward and backward, against the 64-bit statement; the bars are derived in
``attention_bars``."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import oracle.attention as oa
from pymsst_amd import _lib
from pymsst_amd import extension as ext_mod
from tests import attention_bars as bars
from tests.conftest import dt_name, to_np
from tests.test_gpu_guard_writes import _GuardedTorch

_F = [torch.float32, torch.bfloat16, torch.float16]
_SEED, _OFFSET = 0x1234567_89ABCDEF, 0x7000000_00000005


def _rng():
    return torch.tensor([_SEED, _OFFSET], dtype=torch.int64, device="cuda")


def _inputs(shape, dtype, mask="none", seed=0, scale=1.0):
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


def _check(ext, shape, dtype, mask="none", p=0.0, seed=0, scale=None, edit=None):
    q, k, v, do, km, kl = _inputs(shape, dtype, mask, seed)
    if edit is not None:
        q, k, v, do = edit(q, k, v, do)
    kw = dict(key_mask=km, key_lengths=kl, scale=scale, dropout_p=p, rng=_rng() if p else None)
    out, lse = ext.cross_attention_forward(q, k, v, need_lse=True, **kw)
    grads = ext.cross_attention_backward(do, q, k, v, out, lse, **kw)
    ref = bars.reference(dt_name(dtype), to_np(q), to_np(k), to_np(v), to_np(do), _none_or(lambda t: t.cpu().numpy(), km),
                         _none_or(lambda t: t.cpu().numpy(), kl), scale, p, _SEED, _OFFSET)
    for name, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        if name != "lse":
            assert t.dtype == dtype
        bars.check(t, ref[name], (name, shape, dtype, mask, p))
    return out, lse, grads


# ---------------------------------------------------------------------- CPU


def test_oracle_against_autograd_and_differences():
    """The hand-written backward against torch's autograd of the formula and against differences, in 64 bits."""
    g = torch.Generator().manual_seed(1)
    b, n, m, h, hk, d, p = 2, 5, 11, 4, 2, 8, 0.3
    q, do = (torch.randn(b, n, h, d, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(b, m, hk, d, generator=g, dtype=torch.float64) for _ in range(2))
    km = torch.rand(b, m, generator=g) < 0.7
    keep = torch.from_numpy(oa._keep(b, n, m, h, p, 3, 4))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    kk, vv = (t.repeat_interleave(h // hk, dim=2) for t in leaves[1:])
    s = torch.einsum("bnhd,bmhd->bhnm", leaves[0], kk) * d**-0.5
    w = torch.softmax(s.masked_fill(~km[:, None, None], -torch.inf), dim=-1) * keep
    out = torch.einsum("bhnm,bmhd->bnhd", w, vv)
    want = torch.autograd.grad(out, leaves, do)
    args = [t.numpy() for t in (q, k, v)]
    got_out, _ = oa.cross_attention_forward(*args, km.numpy(), None, None, p, 3, 4)
    got = oa.cross_attention_backward(do.numpy(), *args, km.numpy(), None, None, p, 3, 4)
    assert np.allclose(got_out, out.detach().numpy(), atol=1e-13)
    for x, y in zip(got, want):
        assert np.allclose(x, y.numpy(), atol=1e-13)
    rng = np.random.default_rng(0)
    for i in range(3):
        step = rng.standard_normal(args[i].shape)
        lo, hi = list(args), list(args)
        lo[i], hi[i] = args[i] - 1e-5 * step, args[i] + 1e-5 * step
        vals = [(oa.cross_attention_forward(*x, km.numpy(), None, None, p, 3, 4)[0] * do.numpy()).sum() for x in (lo, hi)]
        assert abs((vals[1] - vals[0]) / 2e-5 - (got[i] * step).sum()) < 1e-8


def test_c_abi_refusals():
    lib = _lib.load_library()
    one = ctypes.c_void_p(4096)  # never dereferenced: every call below is refused first
    odd = ctypes.c_void_p(4104)

    def fwd(q=one, qs=None, k=one, ks=None, v=one, out=one, b=1, n=2, m=3, h=4, hk=2, d=64, scale=1.0, p=0.0, rng=None,
            dtype=2, ws=None, size=0):
        return lib.pmsst_cross_attention_forward(q, qs, k, ks, v, None, None, 0, None, out, None, b, n, m, h, hk, d, scale,
                                                 p, rng, dtype, ws, size, None)

    def bwd(grad=one, q=one, out=one, lse=one, dq=one, n=2, m=3, d=64, p=0.0, rng=None, ws=one, size=1 << 40, dtype=2):
        return lib.pmsst_cross_attention_backward(grad, None, q, None, one, None, one, None, out, lse, None, 0, None, dq, one,
                                                  one, 1, n, m, 4, 2, d, 1.0, p, rng, dtype, ws, size, None)

    assert fwd(dtype=9) == -2 and bwd(dtype=9) == -2
    for bad in (dict(hk=3), dict(hk=0), dict(d=4), dict(d=12), dict(d=136), dict(b=-1), dict(n=-1), dict(m=-1),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(p=1.0),
                dict(p=-0.5), dict(p=0.5), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=odd),
                dict(out=odd), dict(b=2**31), dict(n=2**30), dict(m=2**31),
                dict(qs=(ctypes.c_int64 * 3)(512, 260, 64)), dict(ks=(ctypes.c_int64 * 3)(512, 128, 4))):
        assert fwd(**bad) == -1, bad
    for bad in (dict(n=0), dict(n=-1), dict(d=12), dict(p=0.5), dict(p=1.5), dict(grad=None), dict(out=None), dict(lse=None),
                dict(dq=None), dict(dq=odd), dict(grad=odd)):
        assert bwd(**bad) == -1, bad
    assert bwd(m=300, ws=None) == -4 and bwd(m=300, size=16) == -4
    need = lib.pmsst_cross_attention_forward_workspace_size(1, 1, 20000, 8, 8, 64, 2)
    assert need > 0 and fwd(n=1, m=20000, h=8, hk=8, ws=one, size=need - 1) == -4
    assert lib.pmsst_cross_attention_forward_workspace_size(1, 1, 20000, 8, 3, 64, 2) == 0  # no such call
    assert fwd(b=0) == 0 and fwd(n=0) == 0  # nothing to do


def test_calls_past_the_grid_are_refused():
    """A launch has less than 2^32 work-items, 2^24 blocks of 256: more tiles are an argument error, not a launch's."""
    lib = _lib.load_library()
    one = ctypes.c_void_p(4096)  # never dereferenced

    def fwd(b, n):
        return lib.pmsst_cross_attention_forward(one, None, one, None, one, None, None, 0, None, one, None, b, n, 3, 8, 8, 8, 1.0,
                                                 0.0, None, 2, None, 0, None)

    def bwd(b, n, m, dtype):
        return lib.pmsst_cross_attention_backward(one, None, one, None, one, None, one, None, one, one, None, 0, None, one, one,
                                                  one, b, n, m, 8, 8, 8, 1.0, 0.0, None, dtype, one, 1 << 60, None)

    assert fwd(2**21, 1) == fwd(2**14, 2**14) == -1
    assert bwd(2**21, 1, 3, 2) == bwd(2**14, 2**14, 65, 1) == bwd(2**14, 1, 2**14, 0) == -1


@pytest.mark.parametrize("pairs", [1, 7, 8, 16, 63, 65, 100, 512, 513, 576, 992, 2047, 2048, 2049, 8256])
@pytest.mark.parametrize("per", [1, 3, 8])
def test_block_numbering_visits_every_tile_once(pairs, per):
    """The numbering of ``attention.h`` (blocks of a pair on one XCD, many pairs eight at a time), restated."""
    by_xcd, by_eight = pairs % 8 == 0 or pairs >= 64, pairs >= 2048 or (pairs >= 512 and pairs % 64 == 0)
    step = 64 if by_eight else 8 if by_xcd else 1
    seen = []
    for x in range(-(-pairs // step) * step * per):
        i, xcd = divmod(x, 8)
        local, sub = divmod(i, per) if by_xcd else divmod(x, per)
        pair = ((local // 8) * 8 + xcd) * 8 + local % 8 if by_eight else local * 8 + xcd if by_xcd else local
        if pair < pairs:
            seen.append((pair, sub))
    assert len(seen) == pairs * per == len(set(seen))


# ---------------------------------------------------------------------- GPU

_SHAPES = [
    # b, n, m, h, hk, d
    (2, 70, 150, 4, 2, 64),
    (1, 1, 1, 1, 1, 8),
    (3, 130, 64, 2, 1, 32),
    (2, 33, 257, 6, 3, 40),
    (1, 65, 31, 4, 4, 72),
    (1, 258, 129, 2, 2, 128),
    (2, 62, 62, 8, 8, 64),
    (2, 9, 64, 3, 3, 96),
    (2, 64, 65, 2, 2, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape", _SHAPES)
@pytest.mark.parametrize("mask,p", [("none", 0.0), ("both", 0.0), ("keys", 0.3), ("lengths", 0.1)])
def test_forward_and_backward(hip_ext, dtype, shape, mask, p):
    _check(hip_ext, shape, dtype, mask, p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape", [
    (2, 1, 1500, 4, 4, 64),    # single queries: keys split, dQ split
    (1, 1, 3001, 8, 2, 128),   # with shared heads
    (1, 4, 2100, 2, 2, 32),
    (1, 2, 1025, 4, 2, 80),
    (1, 1900, 5, 4, 1, 64),    # few keys under many rows: dK and dV split
    (1, 1100, 40, 2, 2, 128),
])
@pytest.mark.parametrize("mask,p", [("none", 0.0), ("lengths", 0.2), ("keys", 0.0)])
def test_split_axes(hip_ext, dtype, shape, mask, p):
    if mask == "keys" and shape[0] == 1:
        mask = "lengths"
    _check(hip_ext, shape, dtype, mask, p, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_rows_and_batches_without_keys(hip_ext, dtype):
    """No keys at all, a length of zero, a negative one, a mask that leaves nothing: zeros and -inf, bit for bit."""
    for m, lengths, masked in ((0, None, False), (40, [0, -3], False), (700, None, True), (700, [0, 0], False)):
        for n in (1, 70):
            q, k, v, do, _, _ = _inputs((2, n, m, 4, 2, 64), dtype)
            kl = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
            km = torch.zeros(2, m, dtype=torch.bool, device="cuda") if masked else None
            k.fill_(float("nan"))
            v.fill_(float("inf"))
            out, lse = hip_ext.cross_attention_forward(q, k, v, km, kl, need_lse=True)
            assert bool((out == 0).all()) and bool((lse == -torch.inf).all())
            for t in hip_ext.cross_attention_backward(do, q, k, v, out, lse, km, kl):
                assert bool((t == 0).all())
    q, k, v, do, _, _ = _inputs((2, 0, 30, 4, 2, 64), dtype)
    out, lse = hip_ext.cross_attention_forward(q, k, v, need_lse=True)
    dq, dk, dv = hip_ext.cross_attention_backward(do, q, k, v, out, lse)
    assert out.shape == dq.shape == q.shape and bool((dk == 0).all()) and bool((dv == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("n", [1, 90])
def test_what_masked_places_hold_is_never_seen(hip_ext, dtype, n):
    q, k, v, do, km, kl = _inputs((3, n, 600, 4, 2, 64), dtype, "both", seed=9)
    seen = km & (torch.arange(600, device="cuda")[None] < kl[:, None])
    results = []
    for junk in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
        kj, vj = (torch.where(seen[..., None, None], t, torch.full_like(t, junk)) for t in (k, v))
        out, lse = hip_ext.cross_attention_forward(q, kj, vj, km, kl, dropout_p=0.1, rng=_rng(), need_lse=True)
        grads = hip_ext.cross_attention_backward(do, q, kj, vj, out, lse, km, kl, dropout_p=0.1, rng=_rng())
        assert bool((grads[1][~seen] == 0).all()) and bool((grads[2][~seen] == 0).all())
        results.append((out, lse, *grads))
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_infinite_and_nan_inputs_reach_their_rows_only(hip_ext, dtype):
    q, k, v, do, _, _ = _inputs((1, 70, 90, 2, 2, 64), dtype)
    clean = hip_ext.cross_attention_forward(q, k, v)[0]
    q2 = q.clone()
    q2[0, 5, 0, 3] = float("nan")
    out = hip_ext.cross_attention_forward(q2, k, v)[0]
    assert bool(torch.isnan(out[0, 5, 0]).all())
    out[0, 5, 0] = clean[0, 5, 0]
    assert torch.equal(out, clean)
    v2 = v.clone()
    v2[0, 7, 1, 2] = float("inf")
    out = hip_ext.cross_attention_forward(q, k, v2)[0]
    assert bool((out[0, :, 1, 2] == torch.inf).all())
    out[0, :, 1, 2] = clean[0, :, 1, 2]
    assert torch.equal(out, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_large_scores_and_scales(hip_ext, dtype):
    """Scores of hundreds (one key takes a row), and a scale of its own."""
    _check(hip_ext, (1, 40, 300, 2, 2, 64), dtype, edit=lambda q, k, v, do: (q * 16, k, v, do))
    _check(hip_ext, (1, 1, 1500, 2, 2, 64), dtype, edit=lambda q, k, v, do: (q * 16, k, v, do))
    _check(hip_ext, (1, 40, 300, 2, 2, 64), dtype, scale=0.37)
    # scores that climb from tile to tile, by less and by more than the maximum may lag
    for slope in (0.02, 0.5):
        def ramp(q, k, v, do, slope=slope):
            q, k = torch.zeros_like(q), k * 0.05
            q[..., 0] = 8
            k[..., 0] = (torch.arange(k.shape[1], device="cuda") * slope)[None, :, None].to(k.dtype)
            return q, k, v, do
        _check(hip_ext, (1, 33, 500, 2, 2, 64), dtype, edit=ramp)


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("factors", [(1e-5, 1.0), (1.0, 300.0), (300.0, 30.0), (1e-4, 1e-3)])
def test_fp16_gradients_of_any_size(hip_ext, p, factors):
    """Gradients and values far from 1: P and dS keep their digits as fp16 operands and do not overflow."""
    def edit(q, k, v, do):
        return q, k, v * factors[1], do * factors[0]
    for shape in ((1, 50, 1500, 2, 1, 64), (2, 40, 70, 2, 2, 32)):
        _check(hip_ext, shape, torch.float16, p=p, seed=4, edit=edit)


@pytest.mark.gpu
def test_fp16_gradients_where_values_would_overflow_the_operand(hip_ext):
    q, k, v, do, _, _ = _inputs((1, 64, 200, 2, 2, 64), torch.float16)
    v, do = torch.full_like(v, 3e4), torch.full_like(do, 0.5) * (1 + torch.arange(64, device="cuda") % 2)
    v[:, ::2] *= -1
    out, lse = hip_ext.cross_attention_forward(q, k, v, need_lse=True)
    dq, dk, dv = hip_ext.cross_attention_backward(do.half(), q, k, v, out, lse)
    want = oa.cross_attention_backward(to_np(do.half()), to_np(q), to_np(k), to_np(v))
    assert bool(torch.isfinite(dv).all())
    for got, ref in zip((dq, dk), want):  # what fp16 can hold of them is there
        fits = np.abs(ref) < 6e4
        assert np.isfinite(to_np(got)[fits]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dropout_bits_are_those_of_the_dropout_op(hip_ext, dtype):
    b, n, m, h, d, p = 2, 37, 150, 3, 32, 0.3
    q, k, v, _, _, _ = _inputs((b, n, m, h, h, d), dtype)
    pitch = (m + 7) // 8 * 8
    keep = hip_ext.dropout_forward(torch.ones(b, h, n, pitch, device="cuda"), p, _rng())[..., :m].double()
    s = torch.matmul(q.double().transpose(1, 2), k.double().permute(0, 2, 3, 1).contiguous()) * d**-0.5
    want = torch.matmul(torch.softmax(s, dim=-1) * keep, v.double().transpose(1, 2).contiguous()).transpose(1, 2)
    got = hip_ext.cross_attention_forward(q, k, v, dropout_p=p, rng=_rng())[0].double()
    err = float((got - want).norm() / want.norm())
    # two roundings of half a step, uniform (rms 1 / sqrt 3 of the half step each); fp32: sums of 150 terms
    assert err < (1e-6 if dtype == torch.float32 else 2 * 2.0**-8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_views_are_read_in_place(hip_ext, dtype):
    """Slices of a fused projection, a [B, H, N, D] layout, an expanded batch, and tensors that have to be copied
    give the bits of dense ones; their gradients too."""
    b, n, h, d = 2, 75, 4, 64
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(b, n, 3, h, d, generator=g).to(dtype).cuda()
    do = torch.randn(b, h, n, d, generator=g).to(dtype).cuda().transpose(1, 2)
    q, k, v = qkv.unbind(2)
    dense = [t.contiguous() for t in (q, k, v)]
    out, lse = hip_ext.cross_attention_forward(q, k, v, need_lse=True)
    want, wlse = hip_ext.cross_attention_forward(*dense, need_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    for x, y in zip(hip_ext.cross_attention_backward(do, q, k, v, out, lse),
                    hip_ext.cross_attention_backward(do.contiguous(), *dense, want, wlse)):
        assert torch.equal(x, y)
    shared = [t[:1].expand(b, -1, -1, -1) for t in (k, v)]
    out, lse = hip_ext.cross_attention_forward(q, *shared, need_lse=True)
    want, wlse = hip_ext.cross_attention_forward(dense[0], *[t.contiguous() for t in shared], need_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    wide = torch.randn(b, n, h, d + 3, generator=g).to(dtype).cuda()  # rows of no whole 16 bytes: copied
    assert torch.equal(hip_ext.cross_attention_forward(wide[..., 1:d + 1], k, v)[0],
                       hip_ext.cross_attention_forward(wide[..., 1:d + 1].contiguous(), k, v)[0])
    km = (torch.rand(n, b, generator=g) < 0.5).cuda().t()
    assert torch.equal(hip_ext.cross_attention_forward(q, k, v, km)[0],
                       hip_ext.cross_attention_forward(q, k, v, km.contiguous().to(torch.uint8))[0])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_offsets_past_32_bits(hip_ext, n):
    """Keys and values whose rows lie up to 3e9 elements apart (one shared buffer of 6 GB)."""
    d, m, step = 64, 90, 2**25
    pool = torch.empty(m * step + 4 * d, dtype=torch.bfloat16, device="cuda")
    k = pool.as_strided((1, m, 2, d), (0, step, d, 1), 0)
    v = pool.as_strided((1, m, 2, d), (0, step, d, 1), 2 * d)
    g = torch.Generator().manual_seed(1)
    kd, vd = (torch.randn(1, m, 2, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    k.copy_(kd)
    v.copy_(vd)
    q, do = (torch.randn(1, n, 4, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    out, lse = hip_ext.cross_attention_forward(q, k, v, need_lse=True)
    want, wlse = hip_ext.cross_attention_forward(q, kd, vd, need_lse=True)
    assert torch.equal(out, want)
    for x, y in zip(hip_ext.cross_attention_backward(do, q, k, v, out, lse),
                    hip_ext.cross_attention_backward(do, q, kd, vd, want, wlse)):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 100, 300, 4, 2, 64), (1, 1, 3000, 4, 4, 64)])
def test_captured_replays_with_new_seeds_and_lengths(hip_ext, shape):
    """Forward and backward in one graph, replayed with other inputs, seeds, offsets and lengths, each replay against
    the eager call; two graphs' workspaces are their own."""
    q, k, v, do, km, kl = _inputs(shape, torch.bfloat16, "both" if shape[0] > 1 else "lengths")
    rng = _rng()

    def both():
        kw = dict(key_mask=km, key_lengths=kl, dropout_p=0.2, rng=rng)
        out, lse = hip_ext.cross_attention_forward(q, k, v, need_lse=True, **kw)
        return [out, lse, *hip_ext.cross_attention_backward(do, q, k, v, out, lse, **kw)]

    both()
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(both())
    for step in range(4):
        q.copy_(torch.randn(q.shape).to(q.dtype))
        rng.add_(step + 1)
        kl.copy_(torch.randint(0, shape[2] + 1, (shape[0],), dtype=torch.int32))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = both()
        for got in held:
            assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
def test_streams_and_repeated_calls(hip_ext):
    """Two calls at once on two streams, and the same call again: the same bits."""
    q, k, v, do, km, kl = _inputs((2, 300, 700, 4, 2, 64), torch.float16, "both")

    def call():
        out, lse = hip_ext.cross_attention_forward(q, k, v, km, kl, need_lse=True)
        return [out, lse, *hip_ext.cross_attention_backward(do, q, k, v, out, lse, km, kl)]

    want = call()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    for res in got:
        assert all(torch.equal(x, y) for x, y in zip(res, want))


@pytest.mark.gpu
def test_more_pairs_than_a_row_of_the_maxima(hip_ext):
    """2^20 + 8 pairs: the fp16 maxima alone are 2^24 blocks.  The first and the last batch rows against 64 bits."""
    b, n, m, h, d = 2**17 + 1, 1, 65, 8, 8
    g = torch.Generator(device="cuda").manual_seed(5)
    q, do = (torch.randn(b, n, h, d, generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    k, v = (torch.randn(b, m, h, d, generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    out, lse = hip_ext.cross_attention_forward(q, k, v, need_lse=True)
    grads = hip_ext.cross_attention_backward(do, q, k, v, out, lse)
    for rows in (slice(0, 2), slice(2**15 - 1, 2**15 + 1), slice(b - 2, b)):
        ref = bars.reference("f16", *(to_np(t[rows]) for t in (q, k, v, do)), None, None, None, 0.0, 0, 0)
        for name, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
            bars.check(t[rows], ref[name], (name, rows))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_no_write_outside_the_outputs(hip_ext, monkeypatch, dtype):
    """Outputs and workspaces between guard patterns, at odd shapes of every route (split forward and backward, few
    keys, wide rows, cut head dimensions)."""
    guard = _GuardedTorch(torch)
    monkeypatch.setattr(ext_mod, "torch", guard)
    for shape in ((2, 70, 150, 4, 2, 64), (1, 1, 3000, 4, 2, 72), (1, 900, 33, 3, 1, 40), (2, 33, 200, 2, 2, 128),
                  (1, 5, 1500, 2, 1, 128), (2, 129, 65, 6, 2, 24)):
        for p in (0.0, 0.2):
            q, k, v, do, km, kl = _inputs(shape, dtype, "lengths", seed=1)
            kw = dict(key_lengths=kl, dropout_p=p, rng=_rng() if p else None)
            out, lse = hip_ext.cross_attention_forward(q, k, v, need_lse=True, **kw)
            hip_ext.cross_attention_backward(do, q, k, v, out, lse, **kw)
            assert not guard.damaged(), shape
    x = torch.randn(4099, device="cuda").to(dtype)
    hip_ext.dropout_forward(x, 0.3, _rng(), activation="gelu", residual=x)
    hip_ext.dropout_backward(x, 0.3, _rng(), x=x, activation="gelu")
    assert not guard.damaged()


@pytest.mark.gpu
def test_refusals(hip_ext):
    q, k, v, do, _, _ = _inputs((2, 5, 9, 4, 2, 64), torch.bfloat16)
    out, lse = hip_ext.cross_attention_forward(q, k, v, need_lse=True)
    km = torch.ones(2, 9, dtype=torch.bool, device="cuda")
    kl = torch.ones(2, dtype=torch.int32, device="cuda")
    f, bw = hip_ext.cross_attention_forward, hip_ext.cross_attention_backward
    for call in (
        lambda: f(q.cpu(), k, v), lambda: f(q[0], k, v), lambda: f(q, k.float(), v), lambda: f(q, k, v[:, :5]),
        lambda: f(q[:1], k, v), lambda: f(q[..., :32], k, v), lambda: f(q[:, :, :3], k, v),
        lambda: f(q[..., :12], k[..., :12], v[..., :12]), lambda: f(q, k.cpu(), v), lambda: f(q, k[:, :, :0], v[:, :, :0]),
        lambda: f(q.double(), k.double(), v.double()), lambda: f(q, k, v, km[:, :5]), lambda: f(q, k, v, km.float()),
        lambda: f(q, k, v, km.cpu()), lambda: f(q, k, v, None, kl.long()), lambda: f(q, k, v, None, kl[:1]),
        lambda: f(q, k, v, scale=0.0), lambda: f(q, k, v, scale=float("nan")), lambda: f(q, k, v, dropout_p=1.0, rng=_rng()),
        lambda: f(q, k, v, dropout_p=0.1), lambda: bw(do[:1], q, k, v, out, lse), lambda: bw(do.float(), q, k, v, out, lse),
        lambda: bw(do, q, k, v, out[:, :3], lse), lambda: bw(do, q, k, v, out, lse.double()),
        lambda: bw(do, q, k, v, out, lse[:, :, :3]),
    ):
        with pytest.raises(RuntimeError):
            call()
