"""Cross attention and dropout as they are used together: the differentiable functions, a conditioned block of both,
and the model patched onto them."""

from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

from pymsst_amd import fused_roformer as fr
from pymsst_amd.core import transformer
from pymsst_amd.workloads import WORKLOADS, workload_batch

_FLAGS = (fr.EXPERIMENTAL_FUSED_ATTENTION_ENV, fr.EXPERIMENTAL_FUSED_DROPOUT_ENV)


@pytest.fixture
def flags(monkeypatch):
    for name in _FLAGS:
        monkeypatch.setenv(name, "1")
    monkeypatch.setenv(fr.CORE_GROUPED_TRAIN_ENV, "1")
    yield
    fr.restore_stock_implementations()


# ---------------------------------------------------------------------- CPU


def test_patches_leave_the_cpu_model_alone_and_are_undone(monkeypatch):
    """With the flags, a CPU model computes what the stock one does (dropout masks included: both go to torch);
    without them, or with an extension that lacks the ops, nothing is patched."""

    class Ops:
        cross_attention_forward = cross_attention_backward = dropout_forward = dropout_backward = None

    stock = (transformer._sdpa, transformer.FeedForward.forward, transformer.Transformer.forward)
    torch.manual_seed(0)
    block = transformer.Transformer(dim=16, depth=1, dim_head=8, heads=2, attn_dropout=0.2, ff_dropout=0.3).train()
    x = torch.randn(2, 5, 16)

    def run():
        torch.manual_seed(1)
        return block(x)

    want = run()
    assert not fr.apply_roformer_fused_training_backend(block, "hip", extension=Ops()).patched_attention
    assert (transformer._sdpa, transformer.FeedForward.forward, transformer.Transformer.forward) == stock
    for name in _FLAGS:
        monkeypatch.setenv(name, "1")
    try:
        assert not fr.apply_roformer_fused_training_backend(block, "hip", extension=object()).patched_dropout
        status = fr.apply_roformer_fused_training_backend(block, "hip", extension=Ops())
        assert status.patched_attention and status.patched_dropout and status.active == "cuda_ext"
        assert transformer._sdpa is not stock[0]
        again = fr.apply_roformer_fused_training_backend(block, "hip", extension=Ops())
        assert again.patched_attention and again.patched_dropout
        assert torch.equal(run(), want)
        assert block.layers[0][0].to_out[1].p == 0.2 and block.layers[0][1].net[5].p == 0.3
    finally:
        fr.restore_stock_implementations()
    assert (transformer._sdpa, transformer.FeedForward.forward, transformer.Transformer.forward) == stock


# ---------------------------------------------------------------------- GPU


def _weights(dim, ctx_dim, heads, kv_heads, d, seed):
    g = torch.Generator().manual_seed(seed)
    shapes = dict(q=(heads * d, dim), k=(kv_heads * d, ctx_dim), v=(kv_heads * d, ctx_dim), o=(dim, heads * d),
                  up=(4 * dim, dim), down=(dim, 4 * dim))
    return {n: (torch.randn(s, generator=g, dtype=torch.float64) / s[1] ** 0.5) for n, s in shapes.items()}


def _block(x, ctx, w, heads, kv_heads, d, attend, drop, gelu_drop):
    """Queries from one stream over another's frames, output dropout into the residual, then a feed-forward."""
    b, n, _ = x.shape
    q = F.linear(x, w["q"]).reshape(b, n, heads, d)
    k, v = (F.linear(ctx, w[s]).reshape(b, ctx.shape[1], kv_heads, d) for s in ("k", "v"))
    x = drop(F.linear(attend(q, k, v).reshape(b, n, -1), w["o"]), x, 1)
    return drop(F.linear(gelu_drop(F.linear(x, w["up"])), w["down"]), x, 3)


@pytest.mark.gpu
def test_a_conditioned_block_and_its_gradients(hip_ext):
    """Projections, cross attention with ragged lengths, shared heads and dropped weights, dropout into the residual,
    GELU and dropout, all in one autograd graph in fp32, against the same block in 64 bits with the same masks.
    Bar: relative L2 of 3e-6 (six products deep, each within sqrt(K) 2^-24 of its sum, K up to 256: 1e-6 each, and
    what enters one carries the last one's)."""
    b, n, m, heads, kv_heads, d, dim, ctx_dim, p = 3, 37, 70, 4, 2, 32, 64, 48, 0.2
    g = torch.Generator().manual_seed(0)
    x, ctx, go = (torch.randn(b, s, c, generator=g, dtype=torch.float64) for s, c in ((n, dim), (m, ctx_dim), (n, dim)))
    lengths = torch.tensor([m, 23, 0], dtype=torch.int32)
    w64 = _weights(dim, ctx_dim, heads, kv_heads, d, 1)
    rngs = [torch.tensor([77, i], device="cuda") for i in range(4)]

    def keep(shape, i):
        return hip_ext.dropout_forward(torch.ones(shape, device="cuda"), p, rngs[i]).double().cpu()

    def ref_attend(q, k, v):
        k, v = (t.repeat_interleave(heads // kv_heads, dim=2) for t in (k, v))
        s = torch.einsum("bnhd,bmhd->bhnm", q, k) * d**-0.5
        seen = torch.arange(m)[None] < lengths[:, None]
        s = torch.where(seen[:, None, None], s, -1e30)
        wt = torch.softmax(s, dim=-1) * seen[:, None, None]
        return torch.einsum("bhnm,bmhd->bnhd", wt * keep((b, heads, n, (m + 7) // 8 * 8), 0)[..., :m], v)

    def run(x, ctx, w, go, attend, drop, gelu_drop):
        leaves = [t.detach().clone().requires_grad_() for t in (x, ctx, *w.values())]
        out = _block(leaves[0], leaves[1], dict(zip(w, leaves[2:])), heads, kv_heads, d, attend, drop, gelu_drop)
        return [out.detach(), *torch.autograd.grad(out, leaves, go)]

    want = run(x, ctx, w64, go, ref_attend, lambda t, r, i: t * keep(t.shape, i) + r,
               lambda t: F.gelu(t) * keep(t.shape, 2))
    cuda = lambda t: t.float().cuda()  # noqa: E731
    got = run(cuda(x), cuda(ctx), {k: cuda(v) for k, v in w64.items()}, cuda(go),
              lambda q, k, v: fr.cross_attention(q, k, v, key_lengths=lengths.cuda(), dropout_p=p, rng=rngs[0]),
              lambda t, r, i: fr.dropout(t, p, residual=r, rng=rngs[i]),
              lambda t: fr.dropout(t, p, activation="gelu", rng=rngs[2]))
    for a, r in zip(got, want):
        a = a.double().cpu()
        assert float((a - r).norm()) <= 3e-6 * float(r.norm()), float((a - r).norm() / r.norm())


@pytest.mark.gpu
def test_generator_seeds_are_drawn_and_repeated(hip_ext):
    """No rng given: torch's generator decides; the same seed repeats, another call does not; no gradient is formed
    for what needs none; a second derivative is refused."""
    q = torch.randn(2, 9, 2, 32, device="cuda", requires_grad=True)
    k, v = (torch.randn(2, 30, 2, 32, device="cuda") for _ in range(2))

    def call(seed=None):
        if seed is not None:
            torch.manual_seed(seed)
        return fr.cross_attention(q, k, v, dropout_p=0.5), fr.dropout(q, 0.5, activation="gelu")

    first, again, other = call(3), call(3), call()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert not any(torch.equal(a, b) for a, b in zip(first, other))
    (gq,) = torch.autograd.grad(first[0].sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gq.sum(), q)
    with torch.no_grad():
        assert not fr.cross_attention(q, k, v).requires_grad
    # shared by the batch: the gradient of an expanded key is the sum
    ke = k[:1].clone().requires_grad_()
    out = fr.cross_attention(q, ke.expand(2, -1, -1, -1), v)
    (ge,) = torch.autograd.grad(out.sum(), ke)
    kd = k[:1].repeat(2, 1, 1, 1).requires_grad_()
    (gd,) = torch.autograd.grad(fr.cross_attention(q, kd, v).sum(), kd)
    assert torch.equal(ge, gd.sum(dim=0, keepdim=True))


def _loss_grads(model, mixture, target, amp, seed=11):
    torch.manual_seed(seed)
    with torch.autocast("cuda", dtype=amp, enabled=amp is not None):
        loss = model(mixture, target=target)
    loss = loss[0] if isinstance(loss, tuple) else loss
    loss.backward()
    grads = {n: p.grad.detach().float().clone() for n, p in model.named_parameters() if p.grad is not None}
    model.zero_grad(set_to_none=True)
    return float(loss.detach()), grads


@pytest.mark.gpu
@pytest.mark.parametrize("full", [False, True])
@pytest.mark.parametrize("amp", [None, torch.bfloat16])
def test_patched_model_without_dropout_matches_stock(monkeypatch, flags, hip_ext, amp, full):
    """Attention on the kernels in place of SDPA, alone and with the whole ``hip_full`` preset: loss and gradients of
    the tiny model against the stock modules in fp32.  fp32: 1e-4 relative L2 of every gradient (the model tests').
    bf16: the kernels round where SDPA's do (scores in fp32, weights, dS and results once each), so the gradients
    together are as far from the fp32 model's as the stock bf16 model's are, with other roundings of the same number: two such errors
    of many independent roundings have norms of one size, and a factor of 2 between them is allowed (3 where the
    preset rounds at other places too)."""
    wl = WORKLOADS["bsr_tiny"]
    target, mixture = (t.cuda() for t in workload_batch(wl, seed=3)[:2])
    model = wl.build_model("cuda", seed=4).train()
    fr.restore_stock_implementations()
    ref_loss, ref = _loss_grads(model, mixture, target, None)
    low = _loss_grads(model, mixture, target, amp)[1] if amp is not None else None
    if full:
        for key, value in fr.RUNTIME_PRESETS["hip_full"].items():
            monkeypatch.setenv(key, value)
    status = fr.apply_roformer_fused_training_backend(model, "hip", extension=hip_ext,
                                                      rms_norm_mode="fast" if full else None)
    assert status.patched_attention and status.patched_dropout
    calls = []
    real = hip_ext.cross_attention_backward
    monkeypatch.setattr(hip_ext, "cross_attention_backward", lambda *a, **k: calls.append(1) or real(*a, **k),
                        raising=False)
    loss, grads = _loss_grads(model, mixture, target, amp)
    assert len(calls) == 2  # one attention along time, one along the bands
    assert abs(loss - ref_loss) <= (1e-5 if amp is None else 2e-2) * abs(ref_loss)
    if amp is None:
        for name, g in grads.items():
            assert float((g - ref[name]).norm()) <= 1e-4 * float(ref[name].norm()) + 1e-7, name
        return

    def off(gs):  # over all gradients, each in units of its own norm (a single band's gamma has 8 elements)
        return sum((float((gs[n] - ref[n]).norm()) / max(float(ref[n].norm()), 1e-7)) ** 2 for n in ref) ** 0.5

    assert off(grads) <= (3 if full else 2) * off(low), (off(grads), off(low))


@pytest.mark.gpu
@pytest.mark.parametrize("amp", [None, torch.bfloat16])
def test_patched_model_with_dropout(flags, hip_ext, amp):
    """attn_dropout and ff_dropout on the kernels: a seed repeats its loss and gradients bit for bit, another does not,
    activation checkpointing draws the same masks again, and evaluation drops nothing."""
    wl = WORKLOADS["bsr_tiny"]
    target, mixture = (t.cuda() for t in workload_batch(wl, seed=3)[:2])
    wl = copy.deepcopy(wl)
    wl.model.update(attn_dropout=0.2, ff_dropout=0.3)
    model = wl.build_model("cuda", seed=4).train()
    fr.restore_stock_implementations()
    model.eval()
    with torch.no_grad():
        want = model(mixture)
    model.train()
    status = fr.apply_roformer_fused_training_backend(model, "hip", extension=hip_ext)
    assert status.patched_attention and status.patched_dropout
    loss, grads = _loss_grads(model, mixture, target, amp)
    again, same = _loss_grads(model, mixture, target, amp)
    other, _ = _loss_grads(model, mixture, target, amp, seed=12)
    assert loss == again and all(torch.equal(grads[n], same[n]) for n in grads)
    assert loss != other
    model.checkpoint_blocks = True
    ckpt, cg = _loss_grads(model, mixture, target, amp)
    assert ckpt == loss and all(torch.equal(grads[n], cg[n]) for n in grads)
    model.eval()
    with torch.no_grad():
        got = model(mixture)
    assert float((got - want).norm()) <= 1e-5 * float(want.norm())


@pytest.mark.gpu
def test_dropout_modules_keep_their_own_mode(flags, hip_ext):
    """Dropout modules set to evaluation inside a training model drop nothing, and ones left in training inside an
    evaluated model (samples of its predictions) do: the mode is the module's, as in the stock blocks."""
    wl = copy.deepcopy(WORKLOADS["bsr_tiny"])
    _, mixture = (t.cuda() for t in workload_batch(wl, seed=3)[:2])
    wl.model.update(attn_dropout=0.0, ff_dropout=0.3)
    model = wl.build_model("cuda", seed=4).eval()
    status = fr.apply_roformer_fused_training_backend(model, "hip", extension=hip_ext)
    assert status.patched_dropout
    drops = [m for m in model.modules() if isinstance(m, torch.nn.Dropout)]
    with torch.no_grad():
        want = model(mixture)
        model.train()
        for m in drops:
            m.eval()
        assert float((model(mixture) - want).norm()) <= 1e-5 * float(want.norm())
        model.eval()
        for m in drops:
            m.train()
        runs = []
        for seed in (1, 1, 2):
            torch.manual_seed(seed)
            runs.append(model(mixture))
    assert torch.equal(runs[0], runs[1]) and not torch.equal(runs[0], runs[2])
    assert float((runs[0] - want).norm()) > 1e-3 * float(want.norm())
