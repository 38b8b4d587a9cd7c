"""The blocks patched onto the dropout without stored masks, as programs use modules: called from several threads,
with other modules in a dropout's place, with hooks, and inside torch's function transforms."""

from __future__ import annotations

import threading

import pytest
import torch
from torch import nn

from pymsst_amd import fused_roformer as fr
from pymsst_amd.core import transformer

@pytest.fixture
def patched(monkeypatch, hip_ext):
    def patch(block, gates=False, attention=True):
        monkeypatch.setenv(fr.EXPERIMENTAL_FUSED_DROPOUT_ENV, "1")
        if attention:
            monkeypatch.setenv(fr.EXPERIMENTAL_FUSED_ATTENTION_ENV, "1")
        if gates:
            monkeypatch.setenv(fr.EXPERIMENTAL_ATTENTION_GATES_ENV, "1")
        status = fr.apply_roformer_fused_training_backend(block, "hip", extension=hip_ext)
        assert status.patched_dropout
        assert status.patched_attention == attention and status.patched_attention_gates == gates
        return block

    yield patch
    fr.restore_stock_implementations()


def _block(attn_dropout=0.5, ff_dropout=0.5, depth=1):
    torch.manual_seed(0)
    return transformer.Transformer(dim=64, depth=depth, dim_head=32, heads=2, attn_dropout=attn_dropout,
                                   ff_dropout=ff_dropout, norm_output=False).cuda().train()


# ---------------------------------------------------------------------- modules stay as they are


@pytest.mark.gpu
@pytest.mark.parametrize("gates", [False, True])
def test_modules_are_not_changed_during_a_forward(patched, gates):
    """What another caller of the same modules reads while a forward runs: every probability as it was set."""
    block = patched(_block(0.25, 0.5, depth=2), gates)
    drops = [m for m in block.modules() if isinstance(m, nn.Dropout)]
    want, seen = [m.p for m in drops], []
    for m in block.modules():
        if isinstance(m, nn.Linear):
            m.register_forward_hook(lambda *_: seen.append([d.p for d in drops]))
    block(torch.randn(3, 40, 64, device="cuda")).sum().backward()
    assert len(seen) == 2 * (4 if gates else 5) and all(s == want for s in seen)  # the gates' Linear is in their op


@pytest.mark.gpu
@pytest.mark.parametrize("part", ["attention", "feed_forward"])
def test_two_threads_that_meet_inside_a_block_both_drop(patched, part):
    """Both threads are held inside the block at the same time: each result has the share of dropped elements."""
    block = patched(_block())
    attn, ff = block.layers[0]
    with torch.no_grad():  # the other block's part of the sum is 0
        (ff.net[4] if part == "attention" else attn.to_out[0]).weight.zero_()
        ff.net[4].bias.zero_()
    inside = attn.to_qkv if part == "attention" else ff.net[1]
    meet = threading.Barrier(2)

    def hold(*_):
        meet.wait(timeout=60)

    inside.register_forward_hook(hold)
    x = torch.randn(4, 300, 64, device="cuda")
    got, errors = [], []

    def run():
        try:
            with torch.no_grad():
                got.append(block(x))
        except Exception as e:  # shown by the assertion below
            errors.append(e)
            meet.abort()

    threads = [threading.Thread(target=run) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(got) == 2
    for y in got:  # 76800 elements, a standard deviation of 0.002
        assert abs(float((y == x).double().mean()) - 0.5) < 0.02


# ---------------------------------------------------------------------- other modules in a dropout's place


class _Flipped(nn.Dropout):
    """A dropout of another kind: it turns its input's sign, and has a p."""

    def forward(self, x):
        return -x


class _Bare(nn.Module):
    def forward(self, x):
        return 2 * x


class _OwnForward(transformer.Attention):
    def forward(self, x):
        return self.to_out(self.gated_heads(x)) * 3


class _OwnFeedForward(transformer.FeedForward):
    def forward(self, x):
        return self.net(x) * 3


def _replace(block, case):
    """Puts the case's modules into the block; what is left of nn.Dropout has p = 0, so that no mask is drawn."""
    attn, ff = block.layers[0]
    attn.dropout = 0.0  # of the weights
    for m in block.modules():
        if isinstance(m, nn.Dropout):
            m.p = 0.0
    if case == "identity":
        attn.to_out[1] = ff.net[3] = ff.net[5] = nn.Identity()
    elif case == "subclass":
        attn.to_out[1], ff.net[3], ff.net[5] = (_Flipped(0.5) for _ in range(3))
    elif case == "alpha":
        attn.to_out[1], ff.net[3], ff.net[5] = (nn.AlphaDropout(0.0) for _ in range(3))
    elif case == "shorter":
        attn.to_out, ff.net = attn.to_out[:1], nn.Sequential(*list(ff.net)[:3], ff.net[4])
    elif case == "longer":
        attn.to_out.append(_Bare())
        ff.net.append(_Bare())
    elif case == "no sequence":
        attn.to_out, ff.net = attn.to_out[0], nn.Sequential(ff.net[:3], ff.net[4], _Bare())
    elif case == "own forward":
        for m, kind in ((attn, _OwnForward), (ff, _OwnFeedForward)):
            m.__class__ = kind
    elif case == "tanh gelu":
        ff.net[2] = nn.GELU(approximate="tanh")
    elif case == "gelu subclass":
        ff.net[2] = type("Twice", (nn.GELU,), {"forward": lambda self, x: 2 * x})()
    return block


@pytest.mark.gpu
@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("case", ["identity", "subclass", "alpha", "shorter", "longer", "no sequence", "own forward",
                                  "tanh gelu", "gelu subclass"])
def test_other_modules_in_a_dropouts_place_are_called(patched, case, training):
    """They run as they do in the stock block, and no nn.Dropout is taken for granted: the same modules give the same
    values and gradients, but for the order in which SDPA's backward sums."""
    x = torch.randn(2, 30, 64, device="cuda")
    block = _replace(_block(), case).train(training)

    def run():
        inp = x.clone().requires_grad_()
        out = block(inp)
        return [out.detach(), *torch.autograd.grad(out.square().sum(), [inp, *block.parameters()])]

    fr.restore_stock_implementations()
    want = run()
    patched(block, attention=False)
    for a, b in zip(run(), want):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)


@pytest.mark.gpu
def test_blocks_that_own_a_forward_drop_in_it(patched):
    """Their own forward runs once, its dropout included, with nothing dropped again in the residual sum."""
    block = patched(_block())
    attn, ff = block.layers[0]
    with torch.no_grad():
        ff.net[4].weight.zero_()
        ff.net[4].bias.zero_()
    attn.__class__ = _OwnForward
    x = torch.randn(4, 300, 64, device="cuda")
    with torch.no_grad():
        assert abs(float((block(x) == x).double().mean()) - 0.5) < 0.02


def test_another_programs_forward_is_left_alone(monkeypatch):
    class Ops:
        dropout_forward = dropout_backward = None

    def own(self, x):
        return x

    monkeypatch.setenv(fr.EXPERIMENTAL_FUSED_DROPOUT_ENV, "1")
    monkeypatch.setattr(transformer.FeedForward, "forward", own)
    block = transformer.Transformer(dim=16, depth=1, dim_head=8, heads=2, ff_dropout=0.3)
    assert not fr.apply_roformer_fused_training_backend(block, "hip", extension=Ops()).patched_dropout
    assert transformer.FeedForward.forward is own


# ---------------------------------------------------------------------- hooks


def _parts(block):
    attn, ff = block.layers[0]
    return {"attention": attn, "attention chain": attn.to_out, "attention dropout": attn.to_out[1], "feed-forward": ff,
            "feed-forward chain": ff.net, "gelu": ff.net[2], "hidden dropout": ff.net[3], "last dropout": ff.net[5]}


@pytest.mark.gpu
@pytest.mark.parametrize("part", ["attention", "attention chain", "attention dropout", "feed-forward",
                                  "feed-forward chain", "gelu", "hidden dropout", "last dropout"])
@pytest.mark.parametrize("kind", ["forward", "pre", "backward", "backward pre", "instance", "global"])
def test_hooks_run_and_see_what_they_see_in_the_stock_block(patched, part, kind):
    """Every module of the chain that a fused op stands for is called where something hangs on its call; a forward
    hook on a dropout, or on what ends in one, sees the dropped output."""
    block = patched(_block())
    module, seen = _parts(block)[part], []
    note = lambda *a: seen.append(a)  # noqa: E731
    handle = None
    if kind == "forward":
        module.register_forward_hook(note)
    elif kind == "pre":
        module.register_forward_pre_hook(note)
    elif kind == "backward":
        module.register_full_backward_hook(note)
    elif kind == "backward pre":
        module.register_full_backward_pre_hook(note)
    elif kind == "instance":
        stock = module.forward
        module.forward = lambda *a: (seen.append(a), stock(*a))[1]
    else:
        handle = nn.modules.module.register_module_forward_hook(
            lambda m, i, o: seen.append((m, i, o)) if m is module else None)
    try:
        x = torch.randn(2, 100, 64, device="cuda", requires_grad=True)
        block(x).sum().backward()
    finally:
        if handle is not None:
            handle.remove()
    assert len(seen) == 1
    if kind in ("forward", "global") and part != "gelu":
        assert abs(float((seen[0][2] == 0).double().mean()) - 0.5) < 0.05  # 12800 elements or more
    seen.clear()
    if kind == "global":  # and without it the fused ops are back
        block(x).sum().backward()
        assert not seen


# ---------------------------------------------------------------------- function transforms


def _transforms():
    def vmap(f, x):
        return torch.func.vmap(f)(x[:, None])[:, 0]

    def grad(f, x):
        return torch.func.grad(lambda t: f(t).square().sum())(x)

    def per_sample_grads(f, x):
        return torch.func.vmap(torch.func.grad(lambda t: f(t[None]).square().sum()))(x)

    def jvp(f, x):
        return torch.func.jvp(f, (x,), (torch.ones_like(x),))[1]

    def forward_mode(f, x):
        with torch.autograd.forward_ad.dual_level():
            out = f(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
            return torch.autograd.forward_ad.unpack_dual(out).tangent

    return {f.__name__: f for f in (vmap, grad, per_sample_grads, jvp, forward_mode)}


def _outcome(f):
    try:
        return f()
    except Exception as e:  # what the stock modules cannot do either
        return type(e)


@pytest.mark.gpu
@pytest.mark.parametrize("transform", list(_transforms()))
def test_function_transforms_of_the_patched_block(patched, transform):
    """They give what they give for the stock block (or fail as they do there); fp32, without dropped elements."""
    f, block = _transforms()[transform], _block().eval()
    x = torch.randn(3, 20, 64, device="cuda")
    fr.restore_stock_implementations()
    want = _outcome(lambda: f(block, x))
    patched(block)
    got = _outcome(lambda: f(block, x))
    assert isinstance(got, torch.Tensor) == isinstance(want, torch.Tensor), (got, want)
    if isinstance(want, torch.Tensor):
        assert float((got - want).detach().norm()) <= 1e-5 * float(want.detach().norm())
    else:
        assert got is want
    assert transform not in ("vmap", "grad") or isinstance(want, torch.Tensor)


@pytest.mark.gpu
def test_vmap_of_the_training_block_drops(patched):
    block = patched(_block())
    attn, ff = block.layers[0]
    with torch.no_grad():
        attn.to_out[0].weight.zero_()
        x = torch.randn(4, 1, 300, 64, device="cuda")
        y = torch.func.vmap(block, randomness="different")(x)
    assert abs(float((y == x).double().mean()) - 0.5) < 0.02


# ---------------------------------------------------------------------- shapes


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [
    ((2, 4, 30, 32), (2, 4, 50, 32), (2, 4, 50, 64)),  # values of another head dimension
    ((2, 4, 30, 32), (1, 4, 50, 32), (1, 4, 50, 32)),  # a batch that is broadcast
    ((2, 4, 30, 32), (2, 1, 50, 32), (2, 1, 50, 32)),  # heads that are
    ((4, 30, 32), (4, 50, 32), (4, 50, 32)),           # no heads
    ((2, 4, 30, 36), (2, 4, 50, 36), (2, 4, 50, 36)),  # no multiple of 8
    ((2, 4, 30, 32), (2, 4, 50, 32), (2, 4, 50, 32)),  # the kernels'
])
def test_what_the_kernels_do_not_take_goes_to_sdpa(patched, shapes):
    q, k, v = (torch.randn(s, device="cuda") for s in shapes)
    fr.restore_stock_implementations()
    want = _outcome(lambda: transformer._sdpa(q, k, v, 0.0))
    patched(_block())
    got = _outcome(lambda: transformer._sdpa(q, k, v, 0.0))
    assert isinstance(want, torch.Tensor) and got.shape == want.shape
    assert float((got - want).norm()) <= 1e-6 * float(want.norm())  # fp32, sums of 50 terms
