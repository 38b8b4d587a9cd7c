"""The blocks patched onto the dropout without stored masks, as programs use modules: called from several threads,
with other modules in a dropout's place, with hooks, and inside torch's function transforms."""

from __future__ import annotations

import threading

import pytest
import torch
from torch import nn

from pymsst_amd import fused_roformer as fr
from pymsst_amd.core import transformer

_FLAGS = (fr.EXPERIMENTAL_FUSED_ATTENTION_ENV, fr.EXPERIMENTAL_FUSED_DROPOUT_ENV)


@pytest.fixture
def patched(monkeypatch, hip_ext):
    for name in _FLAGS:
        monkeypatch.setenv(name, "1")

    def patch(block, gates=False):
        if gates:
            monkeypatch.setenv(fr.EXPERIMENTAL_ATTENTION_GATES_ENV, "1")
        status = fr.apply_roformer_fused_training_backend(block, "hip", extension=hip_ext)
        assert status.patched_attention and status.patched_dropout and status.patched_attention_gates == gates
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
