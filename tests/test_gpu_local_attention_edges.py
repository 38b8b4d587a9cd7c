"""Local attention where it can go wrong: nothing to see, junk in masked places, special bias entries, strides, far
offsets, graphs, streams, guarded writes, refusals; a stream's steps against the whole sequence; the differentiable
function.  Values against the 64-bit statement with the bars of ``local_attention_bars``."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import oracle.attention as oa
from pymsst_amd import _lib
from pymsst_amd import extension as ext_mod
from pymsst_amd import fused_roformer as fr
from pymsst_amd.extension import HipFusedExtension, relative_buckets
from tests import local_attention_bars as bars
from tests.conftest import dt_name, to_np
from tests.test_gpu_guard_writes import _GuardedTorch
from tests.test_gpu_local_attention import _bias, _inputs, _step_case, check_attention, check_step

_F = [torch.float32, torch.bfloat16, torch.float16]


def _run(ext, q, k, v, do, **kw):
    out, lse = ext.local_attention_forward(q, k, v, need_lse=True, **kw)
    return [out, lse, *ext.local_attention_backward(do, q, k, v, out, lse, **kw)]


# ---------------------------------------------------------------------- CPU


def test_oracle_against_autograd_and_differences():
    """The hand-written backward against torch's autograd of the formula and against differences, in 64 bits."""
    g = torch.Generator().manual_seed(1)
    b, n, h, hk, d, left, right, sinks = 2, 11, 4, 2, 8, 3, 2, 2
    q, do = (torch.randn(b, n, h, d, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(b, n, hk, d, generator=g, dtype=torch.float64) for _ in range(2))
    table = torch.randn(8, h, generator=g, dtype=torch.float64)
    of = np.array(relative_buckets(8, 5))
    km = torch.rand(b, n, generator=g) < 0.8
    starts = np.array([0, 2], dtype=np.int32)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    kk, vv = (t.repeat_interleave(h // hk, dim=2) for t in leaves[1:3])
    delta = torch.arange(n)[None, None, :] - torch.arange(n)[None, :, None] - torch.from_numpy(starts).long()[:, None, None]
    s = torch.einsum("bnhd,bmhd->bhnm", leaves[0], kk) * d**-0.5
    s = s + leaves[3][torch.from_numpy(of)[delta.clamp(-5, 5) + 5]].permute(0, 3, 1, 2)
    seen = (delta <= right) & ((delta >= -left) | (torch.arange(n) < sinks)) & km[:, None, :]
    w = torch.softmax(s.masked_fill(~seen[:, None], -torch.inf), dim=-1).nan_to_num(0.0)
    out = torch.einsum("bhnm,bmhd->bnhd", w, vv)
    want = torch.autograd.grad(out, leaves, do)
    args = [t.numpy() for t in (q, k, v)]
    rest = (left, right, sinks, table.numpy(), of, km.numpy(), None, starts)
    assert np.allclose(oa.local_attention_forward(*args, *rest)[0], out.detach().numpy(), atol=1e-13)
    got = oa.local_attention_backward(do.numpy(), *args, *rest)
    for x, y in zip(got, want):
        assert np.allclose(x, y.numpy(), atol=1e-13)
    rng = np.random.default_rng(0)
    for i in range(4):
        base = [*args, table.numpy()]
        step = rng.standard_normal(base[i].shape)
        vals = []
        for sign in (-1, 1):
            x = list(base)
            x[i] = base[i] + sign * 1e-5 * step
            vals.append((oa.local_attention_forward(*x[:3], left, right, sinks, x[3], *rest[4:])[0] * do.numpy()).sum())
        assert abs((vals[1] - vals[0]) / 2e-5 - (got[i] * step).sum()) < 1e-8


@pytest.mark.parametrize("buckets,most,two", [(32, 128, True), (32, 128, False), (8, 5, True), (320, 800, True), (4, 2, True), (2, 2, False)])
def test_buckets_follow_the_formula(buckets, most, two):
    """Away from borders the logarithm's own value; on them the bucket that begins there."""
    of = relative_buckets(buckets, most, two)
    side = buckets // 2 if two else buckets
    near = side // 2
    assert len(of) == 2 * most + 1 and min(of) == 0 and max(of) < buckets
    for i, got in enumerate(of):
        d = i - most
        f = abs(d) if two else max(-d, 0)
        offset = side if two and d > 0 else 0
        if f < near:
            assert got == offset + f
            continue
        x = near + np.log(f / near) / np.log(most / near) * (side - near)
        allowed = {min(int(np.floor(x + e)), side - 1) for e in (-1e-9, 1e-9)}
        assert got - offset in allowed
        if abs(x - round(x)) < 1e-9:
            assert got - offset == min(round(x), side - 1)


def test_plans_are_checked():
    plan = HipFusedExtension.relative_bias_plan(32, 128, "cpu")
    of, order, first = (t.tolist() for t in plan[:3])
    assert of == relative_buckets(32, 128) and sorted(order) == list(range(257)) and first[0] == 0 and first[-1] == 257
    for c in range(32):
        assert [of[i] for i in order[first[c]:first[c + 1]]] == [c] * of.count(c)
    own = HipFusedExtension.relative_bias_plan(5, 2, "cpu", bucket_of=[4, 0, 2, 0, 1])
    assert own.bucket_of.tolist() == [4, 0, 2, 0, 1] and own.first.tolist() == [0, 2, 3, 4, 4, 5]
    for bad in (dict(num_buckets=3, max_distance=9), dict(num_buckets=2, max_distance=9), dict(num_buckets=8, max_distance=2),
                dict(num_buckets=8, max_distance=1025), dict(num_buckets=1026, max_distance=1000), dict(num_buckets=0, max_distance=9),
                dict(num_buckets=4, max_distance=1, bucket_of=[0, 4, 1]), dict(num_buckets=4, max_distance=1, bucket_of=[0, -1, 1]),
                dict(num_buckets=4, max_distance=1, bucket_of=[0, 1])):
        with pytest.raises(RuntimeError):
            HipFusedExtension.relative_bias_plan(**bad, device="cpu")


def test_c_abi_refusals():
    lib = _lib.load_library()
    one, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4104)  # never dereferenced: every call below is refused first
    strides = lambda *s: (ctypes.c_int64 * 3)(*s)  # noqa: E731

    def fwd(q=one, qs=None, k=one, v=one, out=one, b=1, n=2, m=3, h=4, hk=2, d=64, scale=1.0, dtype=2, ws=None, size=0, left=-1,
            right=-1, sinks=0, starts=None, bias=None, bias_dtype=0, of=one, buckets=8, most=4):
        return lib.pmsst_local_attention_forward(q, qs, k, None, v, None, None, 0, None, starts, left, right, sinks, bias,
                                                 bias_dtype, of, buckets, most, out, None, b, n, m, h, hk, d, scale, dtype, ws,
                                                 size, None)

    def bwd(grad=one, q=one, out=one, lse=one, dq=one, n=2, m=3, d=64, ws=one, size=1 << 40, dtype=2, bias=None, dbias=one,
            order=one, first=one, sinks=0, left=-1):
        return lib.pmsst_local_attention_backward(grad, None, q, None, one, None, one, None, out, lse, None, 0, None, None, left,
                                                  -1, sinks, bias, 0, one, order, first, 8, 4, dq, one, one, dbias, 1, n, m, 4, 2,
                                                  d, 1.0, dtype, ws, size, None)

    def step(q=one, k=one, kc=one, vc=one, pos=one, out=one, b=2, n=1, slots=20, left=9, sinks=4, d=64, dtype=2, kcs=None,
             bias=None, ws=None, size=0, scale=1.0):
        return lib.pmsst_local_attention_step(q, None, k, None, one, None, kc, kcs, vc, None, pos, left, sinks, bias, 0, one, 8, 4,
                                              out, b, n, slots, 4, 2, d, scale, dtype, ws, size, None)

    assert fwd(dtype=9) == -2 and bwd(dtype=9) == -2 and step(dtype=9) == -2
    assert fwd(bias=one, bias_dtype=1) == -2  # fp16 bias of bf16 queries
    for bad in (dict(hk=3), dict(d=12), dict(b=-1), dict(n=-1), dict(m=-1), dict(scale=0.0), dict(scale=float("nan")), dict(q=None),
                dict(k=None), dict(out=None), dict(q=odd), dict(out=odd), dict(n=2**28 + 1), dict(m=2**28 + 1), dict(left=-2),
                dict(right=-2), dict(left=2**29 + 1), dict(right=2**29 + 1), dict(sinks=-1), dict(sinks=2**28 + 1),
                dict(bias=one, of=None), dict(bias=one, buckets=0), dict(bias=one, buckets=1025), dict(bias=one, most=-1),
                dict(bias=one, most=1025), dict(bias=one, scale=2.0**-21), dict(bias=one, scale=2.0**21), dict(qs=strides(512, 260, 64))):
        assert fwd(**bad) == -1, bad
    for bad in (dict(n=0), dict(n=-1), dict(d=12), dict(grad=None), dict(out=None), dict(lse=None), dict(dq=None), dict(dq=odd),
                dict(bias=one, dbias=None), dict(bias=one, order=None), dict(bias=one, first=None)):
        assert bwd(**bad) == -1, bad
    assert bwd(ws=None) == -4 and bwd(size=16) == -4 and bwd(bias=one, size=16) == -4
    for bad in (dict(q=None), dict(k=None), dict(kc=None), dict(vc=None), dict(pos=None), dict(out=None), dict(kc=odd), dict(left=-1),
                dict(slots=13), dict(sinks=11), dict(left=16), dict(n=8), dict(n=-1), dict(d=20), dict(scale=-1.0),
                dict(kcs=strides(2560, 132, 64)), dict(sinks=-1)):
        assert step(**bad) == -1, bad
    need = lib.pmsst_local_attention_step_workspace_size(1, 1, 4, 2, 64, 20000, 4, 2)
    assert need > 0 and step(b=1, left=20000, slots=20010, ws=one, size=need - 1) == -4
    assert lib.pmsst_local_attention_step_workspace_size(1, 1, 4, 3, 64, 20000, 4, 2) == 0  # no such call
    need = lib.pmsst_local_attention_forward_workspace_size(1, 4, 20000, 8, 8, 64, -1, 0, 0, 1, 2)
    assert need > 0 and fwd(n=4, m=20000, h=8, hk=8, right=0, starts=one, ws=one, size=need - 1) == -4
    assert fwd(b=0) == 0 and fwd(n=0) == 0 and step(b=0) == 0 and step(n=0) == 0  # nothing to do


def test_one_cache_for_keys_and_values_is_refused():
    """Each would be written over the other."""
    lib = _lib.load_library()
    one = ctypes.c_void_p(4096)  # never dereferenced
    rc = lib.pmsst_local_attention_step(one, None, one, None, one, None, one, None, one, None, one, 9, 4, None, 0, None, 0, 0, one,
                                        2, 1, 20, 4, 2, 64, 1.0, 2, None, 0, None)
    assert rc == -1 and b"one place" in lib.pmsst_last_error()


def test_calls_past_the_grid_are_refused():
    lib = _lib.load_library()
    one = ctypes.c_void_p(4096)  # never dereferenced
    for b, n in ((2**21, 1), (2**14, 2**14)):
        assert lib.pmsst_local_attention_forward(one, None, one, None, one, None, None, 0, None, None, -1, -1, 0, None, 0, None, 0, 0,
                                                 one, None, b, n, 3, 8, 8, 8, 1.0, 2, None, 0, None) == -1
        assert lib.pmsst_local_attention_backward(one, None, one, None, one, None, one, None, one, one, None, 0, None, None, -1, -1,
                                                  0, None, 0, None, None, None, 0, 0, one, one, one, None, b, n, 3, 8, 8, 8, 1.0, 0,
                                                  one, 1 << 60, None) == -1
    assert lib.pmsst_local_attention_step(one, None, one, None, one, None, one, None, one, None, one, 1, 0, None, 0, None, 0, 0, one,
                                          2**21, 1, 4, 8, 8, 8, 1.0, 2, None, 0, None) == -1


# ---------------------------------------------------------------------- GPU: nothing to see, junk


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_rows_and_batches_without_frames(hip_ext, dtype):
    """No frames at all, lengths of zero and below, masks that leave nothing, windows that lie past the end: zeros and
    -inf, bit for bit, and a bias that learns nothing."""
    plan = hip_ext.relative_bias_plan(8, 20, "cuda")
    bias = torch.randn(8, 4, device="cuda")
    for m, lengths, masked, starts in ((0, None, False, None), (40, [0, -3], False, None), (300, None, True, None),
                                       (300, None, False, [5000, -400]), (60, None, False, [10**9, -(10**9)])):
        for n in (1, 70):
            q, k, v, do, _, _ = _inputs((2, n, m, 4, 2, 64), dtype)
            kl = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
            km = torch.zeros(2, m, dtype=torch.bool, device="cuda") if masked else None
            qs = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
            if starts is None:
                k.fill_(float("nan"))
                v.fill_(float("inf"))
            kw = dict(left=30, right=3, key_mask=km, key_lengths=kl, query_starts=qs, bias=bias, bias_plan=plan)
            out, lse, *grads = _run(hip_ext, q, k, v, do, **kw)
            assert bool((out == 0).all()) and bool((lse == -torch.inf).all())
            assert len(grads) == 4 and all(bool((t == 0).all()) for t in grads)
    for b, n in ((2, 0), (0, 5)):
        q, k, v, do, _, _ = _inputs((b, n, 30, 4, 2, 64), dtype)
        out, lse, *grads = _run(hip_ext, q, k, v, do, left=4, bias=bias, bias_plan=plan)
        assert out.shape == q.shape and all(bool((t == 0).all()) for t in grads) and grads[3].shape == bias.shape
    pos = torch.full((2,), -1, dtype=torch.int32, device="cuda")
    q, k, v, kc, vc, _ = _step_case((2, 0, 4, 2, 64), dtype, 9, [0, 0])
    assert hip_ext.local_attention_step(q, k, v, kc, vc, pos, left=3).shape == (2, 0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("b,n", [(3, 1), (3, 90), (140, 40)])
def test_what_masked_places_hold_is_never_seen(hip_ext, dtype, b, n):
    m = 600 if b == 3 else 60
    q, k, v, do, km, kl = _inputs((b, n, m, 4, 2, 64), dtype, "both", seed=9)
    seen = km & (torch.arange(m, device="cuda")[None] < kl[:, None])
    bias, plan = _bias(hip_ext, 4, 16, 30, True, torch.float32)
    kw = dict(left=70, right=9, sinks=3, key_mask=km, key_lengths=kl, bias=bias, bias_plan=plan)
    results = []
    for junk in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
        kj, vj = (torch.where(seen[..., None, None], t, torch.full_like(t, junk)) for t in (k, v))
        results.append(_run(hip_ext, q, kj, vj, do, **kw))
        assert bool((results[-1][3][~seen] == 0).all()) and bool((results[-1][4][~seen] == 0).all())
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_unseen_slots_of_a_cache_are_not_read(hip_ext, dtype):
    """Slots that hold no frame a query sees: not written yet, left behind by the window, an idle stream's."""
    shape, left, sinks, ring = (4, 2, 4, 2, 64), 20, 3, 40
    positions = [0, 17, 1000, -1]
    q, k, v, kc, vc, pos = _step_case(shape, dtype, sinks + ring, positions)
    held = torch.zeros(4, sinks + ring, dtype=torch.bool)
    for i, p in enumerate(positions):
        for f in range(max(p, 0)):
            if f < sinks or f >= p - left:
                held[i, oa.ring_slot(f, sinks, ring)] = True
    held = held.cuda()[..., None, None]
    outs = []
    for junk in (0.0, float("nan"), float("inf")):
        kj, vj = (torch.where(held, t, torch.full_like(t, junk)) for t in (kc, vc))
        want = [t.clone() for t in (kj, vj)]
        outs.append(hip_ext.local_attention_step(q, k, v, kj, vj, pos, left, sinks))
        for i, p in enumerate(positions):  # and nothing but the new frames' slots is written
            for x in range(2 if p >= 0 else 0):
                at = oa.ring_slot(p + x, sinks, ring)
                want[0][i, at], want[1][i, at] = k[i, x], v[i, x]
        assert all(torch.equal(a.view(torch.uint8), w.view(torch.uint8)) for a, w in zip((kj, vj), want))
    assert all(torch.equal(outs[0], t) for t in outs[1:]) and bool((outs[0][3] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape,kw", [((2, 70, 70, 4, 2, 64), dict(left=0, right=0)), ((1, 200, 200, 2, 2, 32), dict(left=0, right=0)),
                                      ((2, 150, 150, 2, 1, 64), dict(right=0)), ((130, 40, 40, 2, 2, 64), dict(left=3, right=0))])
def test_a_frame_seen_alone_leaves_exact_zeros(hip_ext, dtype, shape, kw):
    """Where a query sees one frame, its weight is 1 whatever the score: dQ is zero, and where all that see a frame do,
    so is its dK; the bias learns nothing from such pairs."""
    b, n = shape[:2]
    bias, plan = _bias(hip_ext, shape[3], 8, 6, False, torch.float32)
    q, k, v, do, _, _ = _inputs(shape, dtype, seed=3)
    out, lse, dq, dk, dv, db = _run(hip_ext, q, k, v, do, bias=bias, bias_plan=plan, **kw)
    if kw.get("left") == 0:
        assert all(bool((t == 0).all()) for t in (dq, dk, db))
    else:
        assert bool((dq[:, 0] == 0).all()) and bool((dq[:, 1:] != 0).any())
        masked = torch.ones(b, n, dtype=torch.bool, device="cuda")
        masked[:, ::2] = False  # every second frame hidden: query 1 and 2 see frame 1 alone
        _, _, dq, _, _, _ = _run(hip_ext, q, k, v, do, bias=bias, bias_plan=plan, key_mask=masked, **kw)
        assert bool((dq[:, :3] == 0).all())


# ---------------------------------------------------------------------- GPU: the bias's own edges


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("shape", [(2, 130, 130, 4, 2, 64), (66, 60, 60, 4, 4, 64)])
def test_special_bias_entries(hip_ext, dtype, shape):
    """-inf and the lowest number of a type hide a bucket's frames, huge entries are cut; a hidden bucket learns nothing."""
    b, n, m, h, hk, d = shape
    q, k, v, do, _, _ = _inputs(shape, dtype, seed=6)
    plan = hip_ext.relative_bias_plan(16, 40, "cuda")
    of = plan.bucket_of.cpu().numpy()
    table = torch.randn(16, h, generator=torch.Generator().manual_seed(1))
    table[3, 0], table[9, 1], table[15, 2], table[7, 3] = -torch.inf, torch.finfo(torch.float32).min, -2e30, -torch.inf
    kw = dict(bias=table.cuda(), bias_plan=plan)
    results = _run(hip_ext, q, k, v, do, **kw)
    ref = bars.reference(dt_name(dtype), *map(to_np, (q, k, v, do)), "f32", bias=to_np(table), bucket_of=of)
    for name, t in zip(("out", "lse", "dq", "dk", "dv", "db"), results):
        bars.check(t, ref[name], (name, shape, dtype))
    assert all(float(results[5][c, i]) == 0.0 for c, i in ((3, 0), (9, 1), (15, 2), (7, 3)))
    table = torch.full((16, h), -torch.inf)  # nothing is seen
    out, lse, *grads = _run(hip_ext, q, k, v, do, bias=table.cuda(), bias_plan=plan)
    assert bool((out == 0).all()) and bool((lse == -torch.inf).all()) and all(bool((t == 0).all()) for t in grads)
    table = torch.zeros(16, h)
    table[5] = 3e38  # cut to 2^20: takes every row that has it
    out, lse, *grads = _run(hip_ext, q, k, v, do, bias=table.cuda(), bias_plan=plan)
    assert all(bool(torch.isfinite(t).all()) for t in (out, lse, *grads))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_own_buckets_and_many_of_them(hip_ext, dtype):
    """A bucket a distance (1024 of them are the most), buckets without distances, one bucket for all: its gradient is 0
    within the bars."""
    q, k, v, do, _, _ = _inputs((2, 150, 150, 2, 1, 64), dtype, seed=8)
    g = torch.Generator().manual_seed(4)
    for buckets, most, of in ((601, 300, list(range(601))), (1024, 511, [min(i, 1023) for i in range(1023)]), (5, 3, [4, 4, 0, 0, 2, 2, 4]),
                              (1, 0, [0])):
        plan = hip_ext.relative_bias_plan(buckets, most, "cuda", bucket_of=of)
        table = torch.randn(buckets, 2, generator=g)
        results = _run(hip_ext, q, k, v, do, left=90, right=40, bias=table.cuda(), bias_plan=plan)
        ref = bars.reference(dt_name(dtype), *map(to_np, (q, k, v, do)), "f32", 90, 40, 0, to_np(table), np.array(of))
        for name, t in zip(("out", "lse", "dq", "dk", "dv", "db"), results):
            bars.check(t, ref[name], (name, buckets, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("rule", [dict(), dict(left=120, right=0, sinks=2)])
def test_an_fp32_bias_gradient_of_many_pairs(hip_ext, dtype, rule):
    """The bars bound every rounding at its worst; what leans to one side adds up long before that.  A row's weights are off
    by at most about 40 roundings of 2^-24 (scores of 5, lse of 7, sums of 258), 2.4e-6, each row to its own side: over the
    6192 rows of a head the sums' errors fall below a tenth of that, and the fp32 sums of a bin's up to 2 10^5 terms add
    their square root in roundings, 2.7e-5 / sqrt(terms) of a sum of |dS| that is sqrt(terms) times the signed sum's
    size or less: 2e-6 of the gradient's norm holds both with room, the 3e-4 of a D from a rounded output does not."""
    b, n, h = 24, 258, 4
    q, k, v, do, _, _ = _inputs((b, n, n, h, h, 64), dtype, seed=21)
    bias, plan = _bias(hip_ext, h, 32, 128, rule.get("right") != 0, torch.float32)
    db = _run(hip_ext, q, k, v, do, bias=bias, bias_plan=plan, **rule)[5]
    want = oa.local_attention_backward(*map(to_np, (do, q, k, v)), bias=to_np(bias), bucket_of=plan.bucket_of.cpu().numpy(), **rule)[3]
    assert np.linalg.norm(to_np(db) - want) <= 2e-6 * np.linalg.norm(want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("d", [64, 128])
def test_the_largest_distance(hip_ext, dtype, d):
    """1024 frames either way: the most that the tables in LDS hold, beside the largest tiles; and steps over as many."""
    check_attention(hip_ext, (1, 1100, 1100, 1, 1, d), dtype, buckets=64, distance=1024)
    check_step(hip_ext, (2, 4, 8, 2, d), dtype, 1500, 3, 1504, [5000, 900], 64, 1024)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_large_scores_scales_and_magnitudes(hip_ext, dtype):
    for shape in ((1, 100, 300, 2, 2, 64), (65, 62, 62, 4, 4, 64)):
        rule = dict(left=80, right=30, sinks=2, buckets=16, distance=50)
        check_attention(hip_ext, shape, dtype, **rule, edit=lambda q, k, v, do: (q * 16, k, v, do))
        check_attention(hip_ext, shape, dtype, **rule, scale=0.37)
        for fv, fo in ((1.0, 1e-5), (300.0, 1.0), (30.0, 300.0), (1e-3, 1e-4)):
            check_attention(hip_ext, shape, dtype, **rule, edit=lambda q, k, v, do: (q, k, v * fv, do * fo))


# ---------------------------------------------------------------------- GPU: layouts, far offsets


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_views_are_read_in_place(hip_ext, dtype):
    b, n, h, d = 2, 75, 4, 64
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(b, n, 3, h, d, generator=g).to(dtype).cuda()
    do = torch.randn(b, h, n, d, generator=g).to(dtype).cuda().transpose(1, 2)
    bias, plan = _bias(hip_ext, h, 8, 20, True, dtype)
    kw = dict(left=30, right=7, sinks=1, bias=bias, bias_plan=plan)
    q, k, v = qkv.unbind(2)
    dense = [t.contiguous() for t in (q, k, v)]
    want = _run(hip_ext, *dense, do.contiguous(), **kw)
    assert all(torch.equal(x, y) for x, y in zip(_run(hip_ext, q, k, v, do, **kw), want))
    kw["bias"] = torch.stack((bias, bias), dim=2)[..., 0]  # a strided table
    assert all(torch.equal(x, y) for x, y in zip(_run(hip_ext, q, k, v, do, **kw), want))
    one = [t[:1].expand(b, -1, -1, -1) for t in dense[1:]]
    for x, y in zip(_run(hip_ext, q, *one, do, **kw), _run(hip_ext, q, *[t.contiguous() for t in one], do, **kw)):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_strided_caches(hip_ext, dtype):
    """Caches side by side in one buffer, heads before slots, slots far apart; the elements between are left alone."""
    shape, left, sinks, ring, positions = (3, 2, 4, 2, 64), 9, 2, 13, [3, 400, -1]
    for make in (lambda t: torch.stack((t, t), dim=2).unbind(2)[0], lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda t: torch.cat((t, t), dim=1)[:, : t.shape[1]]):
        bases = []

        def edit(q, k, v, kc, vc):
            views = [make(t) for t in (kc, vc)]
            bases.extend(t._base if t._base is not None else t for t in views)
            return q, k, v, *views

        check_step(hip_ext, shape, dtype, left, sinks, ring, positions, 8, 6, edit=edit)
    q, k, v, kc, vc, pos = _step_case(shape, dtype, sinks + ring, positions)
    both = torch.stack((kc, vc), dim=1).contiguous()  # [B, 2, slots, Hk, D]
    wide = torch.zeros(3, 2, sinks + ring, 2, 128, dtype=dtype, device="cuda")
    wide[..., 64:] = 7
    wide[..., :64] = both
    want = hip_ext.local_attention_step(q, k, v, kc, vc, pos, left, sinks)
    got = hip_ext.local_attention_step(q, k, v, wide[:, 0, ..., :64], wide[:, 1, ..., :64], pos, left, sinks)
    assert torch.equal(got, want) and torch.equal(wide[:, 0, ..., :64], kc) and torch.equal(wide[:, 1, ..., :64], vc)
    assert bool((wide[..., 64:] == 7).all())


@pytest.mark.gpu
def test_offsets_past_32_bits(hip_ext):
    """Frames 2^26 elements apart: the last ones lie past 2^32 elements."""
    dtype, m, d = torch.bfloat16, 70, 64
    pitch = 1 << 26
    store = torch.empty((m - 1) * pitch + 2 * d, dtype=dtype, device="cuda")
    k, v = (store.as_strided((1, m, 1, d), (d, pitch, d, 1), storage_offset=i * d) for i in range(2))
    g = torch.Generator().manual_seed(3)
    for t in (k, v):
        t.copy_(torch.randn(1, m, 1, d, generator=g).to(dtype))
    q, do = (torch.randn(1, n, 2, d, generator=g).to(dtype).cuda() for n in (m, m))
    bias, plan = _bias(hip_ext, 2, 8, 20, True, torch.float32)
    kw = dict(left=40, right=3, bias=bias, bias_plan=plan)
    want = _run(hip_ext, q, k.contiguous(), v.contiguous(), do, **kw)
    assert all(torch.equal(x, y) for x, y in zip(_run(hip_ext, q, k, v, do, **kw), want))
    pos = torch.tensor([2 * m + 5], dtype=torch.int32, device="cuda")
    new = [torch.randn(1, 1, 1, d, generator=g).to(dtype).cuda() for _ in range(2)]
    kd, vd = k.contiguous(), v.contiguous()
    want = hip_ext.local_attention_step(q[:, :1], *new, kd, vd, pos, left=60, sinks=4)
    got = hip_ext.local_attention_step(q[:, :1], *new, k, v, pos, left=60, sinks=4)
    assert torch.equal(got, want) and torch.equal(k, kd) and torch.equal(v, vd)


# ---------------------------------------------------------------------- GPU: graphs, streams, repeats, guards


def _mixed_call(ext, q, k, v, do, kw, step):
    return [*_run(ext, q, k, v, do, **kw), ext.local_attention_step(*step, left=20, sinks=3, bias=kw["bias"], bias_plan=kw["bias_plan"])]


def _mixed_inputs(ext, dtype, seed=1):
    q, k, v, do, km, kl = _inputs((2, 200, 200, 4, 2, 64), dtype, "both", seed=seed)
    bias, plan = _bias(ext, 4, 16, 48, True, torch.float32)
    kw = dict(left=60, right=20, sinks=2, bias=bias, bias_plan=plan, key_mask=km, key_lengths=kl)
    return q, k, v, do, kw, list(_step_case((3, 1, 4, 2, 64), dtype, 30, [5, 70, -1], seed))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_captured_replays_with_new_values(hip_ext, dtype):
    """Forward, backward and a step in one captured graph: replays take the tensors' values of the moment (lengths,
    positions, the bias), with eager work and synchronisations between them; two graphs do not disturb each other."""
    q, k, v, do, kw, step = _mixed_inputs(hip_ext, dtype)
    _mixed_call(hip_ext, q, k, v, do, kw, step)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            held = _mixed_call(hip_ext, q, k, v, do, kw, step)
        graphs.append((graph, held))
    gen = torch.Generator().manual_seed(5)
    for i in range(4):
        kw["key_lengths"].copy_(torch.randint(0, 201, (2,), generator=gen, dtype=torch.int32))
        kw["bias"].copy_(torch.randn(16, 4, generator=gen))
        step[5].copy_(torch.tensor([6 + i, 90 * i, -1 if i % 2 else 44], dtype=torch.int32))
        caches = [t.clone() for t in step[3:5]]
        graph, held = graphs[i % 2]
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        got = [t.clone() for t in (*held, *step[3:5])]
        want = _mixed_call(hip_ext, q, k, v, do, kw, [*step[:3], *caches, step[5]])
        assert all(torch.equal(x, y) for x, y in zip(got, [*want, *caches]))
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_streams_and_repeated_calls(hip_ext, dtype):
    """The same bits on every call, on another stream, and from calls that overlap on two streams."""
    q, k, v, do, kw, step = _mixed_inputs(hip_ext, dtype)
    caches = [t.clone() for t in step[3:5]]
    want = _mixed_call(hip_ext, q, k, v, do, kw, step)
    for _ in range(3):
        again = _mixed_call(hip_ext, q, k, v, do, kw, [*step[:3], *[t.clone() for t in caches], step[5]])
        assert all(torch.equal(x, y) for x, y in zip(want, again))
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(3):
        for s, r in zip(streams, results):
            with torch.cuda.stream(s):
                r.append(_mixed_call(hip_ext, q, k, v, do, kw, [*step[:3], *[t.clone() for t in caches], step[5]]))
    torch.cuda.synchronize()
    for r in results:
        for again in r:
            assert all(torch.equal(x, y) for x, y in zip(want, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_no_write_outside_the_outputs(hip_ext, monkeypatch, dtype):
    guard = _GuardedTorch(torch)
    monkeypatch.setattr(ext_mod, "torch", guard)
    bias, plan = {}, {}
    for shape, rule in (((2, 70, 70, 4, 2, 64), (20, 5, 3)), ((1, 333, 333, 3, 1, 40), (40, 0, 70)), ((130, 62, 61, 2, 2, 64), (None, None, 0)),
                        ((1, 130, 700, 2, 2, 128), (100, 9, 4)), ((1, 1, 1, 1, 1, 8), (0, 0, 0)), ((2, 3, 1500, 4, 2, 32), (None, 0, 0))):
        q, k, v, do, km, kl = _inputs(shape, dtype, "both" if shape[0] > 1 else "none")
        plan = hip_ext.relative_bias_plan(16, 48, "cuda")
        bias = torch.randn(16, shape[3], device="cuda")
        for b in (None, bias):
            _run(hip_ext, q, k, v, do, left=rule[0], right=rule[1], sinks=rule[2], key_mask=km, key_lengths=kl, bias=b, bias_plan=plan)
            assert not guard.damaged(), (shape, dtype)
    for shape, left, sinks in (((3, 2, 4, 2, 64), 20, 3), ((1, 1, 2, 2, 128), 4000, 8), ((2, 5, 6, 1, 40), 9, 0)):
        q, k, v, _, _, pos = _step_case(shape, dtype, 1, [50, 3, -1][: shape[0]])
        caches = [guard.empty((shape[0], left + sinks + shape[1], shape[3], shape[4]), dtype=dtype, device="cuda") for _ in range(2)]
        for c in caches:
            c.fill_(0.5)
        hip_ext.local_attention_step(q, k, v, *caches, pos, left, sinks, bias=torch.randn(16, shape[2], device="cuda"), bias_plan=plan)
        assert not guard.damaged(), (shape, dtype)


@pytest.mark.gpu
def test_refusals(hip_ext):
    q, k, v, do, _, _ = _inputs((2, 9, 30, 4, 2, 64), torch.bfloat16)
    plan = hip_ext.relative_bias_plan(8, 10, "cuda")
    bias = torch.zeros(8, 4, device="cuda")
    fwd = hip_ext.local_attention_forward
    for kw in (dict(left=-1), dict(right=-1), dict(left=2**29 + 1), dict(sinks=-1), dict(bias=bias), dict(bias=bias[:7], bias_plan=plan),
               dict(bias=bias[:, :3], bias_plan=plan), dict(bias=bias.half(), bias_plan=plan), dict(bias=bias.cpu(), bias_plan=plan),
               dict(bias=bias, bias_plan=hip_ext.relative_bias_plan(8, 10, "cpu")), dict(bias=bias, bias_plan=plan, scale=2.0**30),
               dict(query_starts=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(query_starts=torch.zeros(3, dtype=torch.int32, device="cuda")),
               dict(key_mask=torch.ones(2, 29, dtype=torch.bool, device="cuda")), dict(scale=0.0),
               dict(key_lengths=torch.ones(2, dtype=torch.int64, device="cuda"))):
        if kw.get("left") == -1 or kw.get("right") == -1:
            kw = {n: -2 for n in kw}
        with pytest.raises(RuntimeError):
            fwd(q, k, v, **kw)
    for args in ((q.cpu(), k, v), (q, k.half(), v), (q, k[:1], v[:1]), (q, k[..., :32], v), (q[..., :60], k[..., :60], v[..., :60]), (q, k[:, :, :0], v[:, :, :0])):
        with pytest.raises(RuntimeError):
            fwd(*args)
    out, lse = fwd(q, k, v, need_lse=True)
    for bad in ((do[:, :8], out, lse), (do, out.float(), lse), (do, out, lse[:, :3]), (do, out, lse.double())):
        with pytest.raises(RuntimeError):
            hip_ext.local_attention_backward(bad[0], q, k, v, *bad[1:])
    sq, sk, sv, kc, vc, pos = _step_case((2, 2, 4, 2, 64), torch.bfloat16, 20, [0, 0])
    step = hip_ext.local_attention_step
    for args, kw in (((sq, sk, sv, kc, vc, pos), dict(left=19)), ((sq, sk, sv, kc, vc, pos), dict(left=5, sinks=14)),
                     ((sq, sk, sv, kc, vc, pos), dict(left=-1)), ((sq, sk, sv, kc, vc, pos.long()), dict(left=5)),
                     ((sq, sk, sv, kc, vc, pos[:1]), dict(left=5)), ((sq, sk, sv, kc, vc.float(), pos), dict(left=5)),
                     ((sq, sk, sv, kc, vc[:, :19], pos), dict(left=5)), ((sq, sk, sv, kc[:1].expand(2, -1, -1, -1), vc, pos), dict(left=5)),
                     ((sq, sk, sv, kc.transpose(1, 3).contiguous().transpose(1, 3), vc, pos), dict(left=5)),
                     ((sq, sk[:, :1], sv[:, :1], kc, vc, pos), dict(left=5)), ((sq, sk, sv, kc[..., :60], vc[..., :60], pos), dict(left=5)),
                     ((sq, sk, sv, kc, vc, pos), dict(left=5, bias=bias))):
        with pytest.raises(RuntimeError):
            step(*args, **kw)


# ---------------------------------------------------------------------- GPU: used together


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("n", [1, 3])
def test_a_stream_taken_frame_by_frame(hip_ext, dtype, n):
    """Two streams from their first frame on, ``n`` frames a step through caches that wrap several times, against the
    whole sequence at once; both against 64 bits."""
    b, frames, h, hk, d, left, sinks = 2, 120, 4, 2, 64, 17, 3
    q, k, v, _, _, _ = _inputs((b, frames, frames, h, hk, d), dtype, seed=7)
    bias, plan = _bias(hip_ext, h, 8, 12, False, torch.float32)
    kw = dict(left=left, sinks=sinks, bias=bias, bias_plan=plan)
    kc, vc = (torch.full((b, sinks + left + n, hk, d), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    pos = torch.zeros(b, dtype=torch.int32, device="cuda")
    parts = []
    for t in range(0, frames, n):
        parts.append(hip_ext.local_attention_step(q[:, t:t + n], k[:, t:t + n], v[:, t:t + n], kc, vc, pos, **kw))
        pos += n
    got = torch.cat(parts, dim=1)
    ref = bars.reference(dt_name(dtype), *map(to_np, (q, k, v)), None, "f32", left, 0, sinks, to_np(bias), plan.bucket_of.cpu().numpy())
    bars.check(got, ref["out"], ("steps", dtype))
    bars.check(hip_ext.local_attention_forward(q, k, v, right=0, **kw)[0], ref["out"], ("whole", dtype))


@pytest.mark.gpu
def test_the_differentiable_function(hip_ext):
    """A block of projections, local attention with a learned bias and a residual, in fp32, against autograd of the
    formula in 64 bits.  Bar: relative L2 of 3e-6 (two products and the attention, each within sqrt(K) 2^-24 of its
    sums, K up to 200: 1e-6 each, and what enters one carries the last one's)."""
    b, n, h, d, dim, left, right, sinks = 2, 90, 4, 32, 64, 25, 6, 2
    g = torch.Generator().manual_seed(0)
    x, go = (torch.randn(b, n, dim, generator=g, dtype=torch.float64) for _ in range(2))
    wqkv = torch.randn(3 * h * d, dim, generator=g, dtype=torch.float64) / dim**0.5
    wo = torch.randn(dim, h * d, generator=g, dtype=torch.float64) / (h * d) ** 0.5
    table = torch.randn(16, h, generator=g, dtype=torch.float64) * 0.5
    plan = hip_ext.relative_bias_plan(16, 40, "cuda")
    of = plan.bucket_of.cpu().long()

    def formula(q, k, v, table):
        delta = torch.arange(n)[None, :] - torch.arange(n)[:, None]
        s = torch.einsum("bnhd,bmhd->bhnm", q, k) * d**-0.5 + table[of[delta.clamp(-40, 40) + 40]].permute(2, 0, 1)
        seen = (delta <= right) & ((delta >= -left) | (torch.arange(n) < sinks))
        return torch.einsum("bhnm,bmhd->bnhd", torch.softmax(s.masked_fill(~seen, -torch.inf), dim=-1), v)

    def run(x, wqkv, wo, table, go, attend):
        leaves = [t.detach().clone().requires_grad_() for t in (x, wqkv, wo, table)]
        q, k, v = torch.nn.functional.linear(leaves[0], leaves[1]).view(b, n, 3, h, d).unbind(2)
        out = torch.nn.functional.linear(attend(q, k, v, leaves[3]).reshape(b, n, -1), leaves[2]) + leaves[0]
        return [out.detach(), *torch.autograd.grad(out, leaves, go)]

    want = run(x, wqkv, wo, table, go, formula)
    got = run(*(t.float().cuda() for t in (x, wqkv, wo, table, go)),
              lambda q, k, v, t: fr.local_attention(q, k, v, left=left, right=right, sinks=sinks, bias=t, bias_plan=plan))
    for a, r in zip(got, want):
        assert float((a.double().cpu() - r).norm()) <= 3e-6 * float(r.norm())
    # what needs no gradient gets none; a second derivative is refused; a bias alone learns
    q = torch.randn(1, 20, 2, 32, device="cuda")
    t = torch.zeros(16, 2, device="cuda", requires_grad=True)
    out = fr.local_attention(q, q, q, left=4, bias=t, bias_plan=plan)
    (gt,) = torch.autograd.grad(out.square().sum(), t, create_graph=True)
    assert gt.shape == t.shape and bool((gt != 0).any())
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gt.sum(), t)
    with torch.no_grad():
        assert not fr.local_attention(q, q, q, left=4, bias=t, bias_plan=plan).requires_grad
    # no bias, and under autocast: the tensors' own type
    ql = q.bfloat16().requires_grad_()
    (gq,) = torch.autograd.grad(fr.local_attention(ql, ql, ql, left=4, sinks=1).float().sum(), ql)
    assert gq.dtype == torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_without_limits_it_is_cross_attention(hip_ext, dtype):
    q, k, v, do, km, kl = _inputs((3, 100, 230, 4, 2, 64), dtype, "both", seed=2)
    results = _run(hip_ext, q, k, v, do, key_mask=km, key_lengths=kl)
    out, lse = hip_ext.cross_attention_forward(q, k, v, km, kl, need_lse=True)
    other = [out, lse, *hip_ext.cross_attention_backward(do, q, k, v, out, lse, km, kl)]
    ref = bars.reference(dt_name(dtype), *map(to_np, (q, k, v, do)), key_mask=km.cpu().numpy(), key_lengths=kl.cpu().numpy())
    for name, x, y in zip(("out", "lse", "dq", "dk", "dv"), results, other):
        bars.check(x, ref[name], (name, "local"))
        bars.check(y, ref[name], (name, "cross"))
