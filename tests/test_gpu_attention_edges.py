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


# ---------------------------------------------------------------------- groups that do not divide a tile


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("shape", [
    (2, 129, 65, 6, 2, 24),   # three heads a key head: two kernels
    (1, 90, 300, 3, 1, 64),
    (2, 47, 50, 10, 2, 32),   # five, few keys
    (1, 150, 130, 6, 1, 128),
    (2, 1, 1500, 6, 2, 64),   # keys split
    (1, 700, 33, 3, 1, 40),   # rows split
])
def test_groups_that_do_not_divide_a_tile(hip_ext, dtype, p, shape):
    q, k, v, do = _inputs(shape, dtype, seed=5)
    kl = torch.tensor([shape[2], max(shape[2] - 30, 2)][:shape[0]], dtype=torch.int32, device="cuda")
    kw = dict(key_lengths=kl, dropout_p=p, rng=_rng() if p else None)
    results = _run(hip_ext, q, k, v, do, **kw)
    ref = bars.reference(dt_name(dtype), *(to_np(t) for t in (q, k, v, do)), None, kl.cpu().numpy(), None, p, _SEED, _OFFSET)
    for name, t in zip(_NAMES, results):
        bars.check(t, ref[name], (name, shape, dtype, p))


# ---------------------------------------------------------------------- the numbering's kinds


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
@pytest.mark.parametrize("b,hk", [(65, 1), (50, 2), (171, 3), (72, 8), (683, 3), (512, 4)])
@pytest.mark.parametrize("n,m", [(150, 150), (150, 40), (9, 70)])
def test_pairs_of_every_numbering(hip_ext, dtype, b, hk, n, m):
    """65 to 2049 pairs, padded and not, one by one and by eights, with several tiles each: the first and the last batch
    rows, and those around the numbering's steps, against 64 bits; all of them against a call of each half, of other
    numberings (which may split a long axis, and then rounds its sums elsewhere)."""
    q, k, v, do = _inputs((b, n, m, hk, hk, 16), dtype, seed=b)
    results = _run(hip_ext, q, k, v, do)
    rows = sorted({0, 1, 64 // hk, b // 2, b - 1})
    at = torch.tensor(rows, device="cuda")
    ref = bars.reference(dt_name(dtype), *(to_np(t[at]) for t in (q, k, v, do)))
    for name, t in zip(_NAMES, results):
        bars.check(t[at], ref[name], (name, b, hk, n, m))
    half = b // 2
    for part in (slice(0, half), slice(half, b)):
        again = _run(hip_ext, *(t[part] for t in (q, k, v, do)))
        for name, x, y in zip(_NAMES, results, again):
            bar = max(8 * torch.finfo(dtype).eps, 1e-5) * max(1.0, float(y.abs().max()))
            assert float((x[part].double() - y.double()).abs().max()) <= bar, name


# ---------------------------------------------------------------------- fp16's powers of two, few keys


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("factors", [(1e-5, 1.0), (1.0, 300.0), (300.0, 30.0), (1e-4, 1e-3)])
@pytest.mark.parametrize("shape", [(1, 300, 50, 2, 2, 64), (2, 130, 64, 3, 1, 32), (1, 200, 9, 2, 2, 128)])
def test_fp16_gradients_of_any_size_over_few_keys(hip_ext, p, factors, shape):
    q, k, v, do = _inputs(shape, torch.float16, seed=4)
    v, do = v * factors[1], do * factors[0]
    kw = dict(dropout_p=p, rng=_rng() if p else None)
    ref = bars.reference("f16", *(to_np(t) for t in (q, k, v, do)), None, None, None, p, _SEED, _OFFSET)
    for name, t in zip(_NAMES, _run(hip_ext, q, k, v, do, **kw)):
        bars.check(t, ref[name], (name, shape, factors, p))


_PROFILES = {
    # a power of ten for each row tile of 64; None: no gradient
    "rising": (-6, -4, -2, 0, 2), "falling": (2, 0, -2, -4, -6), "zeros first": (None, None, -3, 1, -5),
    "zeros between": (-4, None, 1, None, -2), "zeros last": (1, -4, None, None, None), "one": (None, None, -5, None, None),
    "none": (None,) * 5,
}


@pytest.mark.gpu
@pytest.mark.parametrize("profile", list(_PROFILES))
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_fp16_row_tiles_of_different_magnitudes(hip_ext, profile, d, p):
    """dK is summed at a power of two that falls from row tile to row tile (512 pairs: one block takes all five tiles of
    its pair); each tile's own gradients keep their digits."""
    b, n, m, h = 64, 300, 30, 8
    g = torch.Generator(device="cuda").manual_seed(d)
    q, do = (torch.randn(b, n, h, d, generator=g, device="cuda") for _ in range(2))
    k, v = (torch.randn(b, m, h, d, generator=g, device="cuda").half() for _ in range(2))
    for tile, power in enumerate(_PROFILES[profile]):
        do[:, 64 * tile:64 * tile + 64] *= 0.0 if power is None else 10.0**power
    q, do = q.half(), do.half()
    kw = dict(dropout_p=p, rng=_rng() if p else None)
    results = _run(hip_ext, q, k, v, do, **kw)
    if profile == "none":
        assert all(bool((t == 0).all()) for t in results[2:])
    one = slice(0, 1)  # its dropout's numbers are the first ones of the whole call's
    ref = bars.reference("f16", *(to_np(t[one]) for t in (q, k, v, do)), None, None, None, p, _SEED, _OFFSET)
    for name, t in zip(_NAMES, results):
        bars.check(t[one], ref[name], (name, profile, d, p))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [200, 40])
def test_fp16_gradients_next_to_values_that_nearly_overflow(hip_ext, m):
    """Values of 3e4, whose products with dO are far above fp16's range: what fp16 can hold of the gradients is right."""
    q, k, v, do = _inputs((1, 64, m, 2, 2, 64), torch.float16)
    v, do = torch.full_like(v, 3e4), (torch.full_like(do, 0.5) * (1 + torch.arange(64, device="cuda") % 2)).half()
    v[:, ::2] *= -1
    results = _run(hip_ext, q, k, v, do)
    ref = bars.reference("f16", *(to_np(t) for t in (q, k, v, do)))
    for name, t in zip(_NAMES, results):
        want, bar = ref[name]
        fits = np.abs(want) + bar < 6.5e4
        got = to_np(t)
        assert fits.any() and np.all(np.abs(got - want)[fits] <= bar[fits]), (name, m)
        assert np.all(np.isinf(got)[np.abs(want) - bar > 65536]) or not (np.abs(want) - bar > 65536).any()


# ---------------------------------------------------------------------- drawn seeds in a captured graph


@pytest.mark.gpu
def test_a_captured_graph_draws_new_masks_on_every_replay(hip_ext):
    """The seed and offset come from torch's generator inside the graph: each replay has masks of its own, of the
    probability asked for, the backward's are the forward's, and eager calls between the replays change nothing."""
    from pymsst_amd import fused_roformer as fr

    x = torch.ones(64, 1000, device="cuda")
    q, k, v, _ = _inputs((1, 70, 90, 2, 2, 64), torch.float32)

    def step():
        rng = fr.draw_rng(x.device)
        y = hip_ext.dropout_forward(x, 0.25, rng)
        dx = hip_ext.dropout_backward(x, 0.25, rng)
        return rng, y, dx, hip_ext.cross_attention_forward(q, k, v, dropout_p=0.25, rng=rng)[0]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    seen = []
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        rng, y, dx, out = (t.clone() for t in held)
        assert torch.equal(y, dx) and abs(float((y == 0).double().mean()) - 0.25) < 0.02  # deviation 0.0017
        assert torch.equal(y, hip_ext.dropout_forward(x, 0.25, rng))
        assert torch.equal(out, hip_ext.cross_attention_forward(q, k, v, dropout_p=0.25, rng=rng)[0])
        seen.append(y)
        step()
    for i in range(4):
        for j in range(i):
            assert not torch.equal(seen[i], seen[j])
