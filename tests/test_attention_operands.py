"""Which views the cross attention reads in place, on the CPU: the strides that reach the C entry are whole 16 bytes,
whatever an axis of one element carries."""

from __future__ import annotations

import pytest
import torch

from pymsst_amd.extension import HipFusedExtension

_F = [torch.float32, torch.bfloat16, torch.float16]


def _single_axis_views(dtype):
    """(name, tensor [B, N, H, D]): views that torch calls contiguous though a stride is no whole 16 bytes."""
    x = torch.arange(2 * 5 * 4 * 64 + 64, dtype=torch.float32).to(dtype)
    conv = x[:2 * 256].view(2, 256, 1).view(2, 4, 64, 1).permute(0, 3, 1, 2)
    head = x[:2 * 5 * 64].view(2, 5, 64, 1).transpose(2, 3)
    batch = x[:5 * 4 * 64].as_strided((1, 5, 4, 64), (1, 256, 64, 1))
    row = x[:1283].as_strided((1, 5, 4, 64), (1283, 256, 64, 1))
    token = x.as_strided((2, 1, 4, 64), (256, 67, 64, 1))
    one = x[:64].as_strided((1, 1, 1, 64), (3, 1, 7, 1))
    return [("one frame", conv), ("one head", head), ("batch of one", batch), ("odd batch pitch", row),
            ("odd frame pitch", token), ("one row", one)]


def _view(operand, strides, t):
    """The tensor that the C entry would read."""
    return operand.as_strided(t.shape, list(strides) + [1])


@pytest.mark.parametrize("dtype", _F)
def test_axes_of_one_element_have_no_stride_of_their_own(dtype):
    ext = HipFusedExtension()
    unit = 16 // torch.empty(0, dtype=dtype).element_size()
    for name, t in _single_axis_views(dtype):
        assert t.is_contiguous(), name  # so .contiguous() would not change it
        got, strides = ext._attention_operand(t)
        assert all(s % unit == 0 for s in strides), (name, list(strides))
        assert got.data_ptr() % 16 == 0
        assert got.data_ptr() == t.data_ptr() or t.data_ptr() % 16  # read in place
        assert torch.equal(_view(got, strides, t), t), name


@pytest.mark.parametrize("dtype", _F)
def test_other_views_are_read_in_place_or_copied(dtype):
    ext = HipFusedExtension()
    unit = 16 // torch.empty(0, dtype=dtype).element_size()
    x = torch.arange(2 * 7 * 3 * 4 * 64 + 8).float().to(dtype)
    fused = x[:-8].view(2, 7, 3, 4, 64)
    for t, in_place in ((fused.unbind(2)[1], True), (fused[:, :, 0].transpose(1, 2), True),
                        (fused[:1, :, 2].expand(3, -1, -1, -1), True), (fused[:, :, 0, :, 1:41], False),
                        (fused[:, :, 1].transpose(2, 3)[..., :3].transpose(2, 3), True),
                        (x[:2 * 4 * 64 * 8].view(2, 4, 64, 8).permute(0, 3, 1, 2), False), (x[3:3 + 2 * 7 * 64].view(2, 7, 1, 64), False),
                        (x[:64 * 67].view(64, 67)[None, :, None, :64], False), (x[:1].expand(2, 3, 4, 64), False)):
        got, strides = ext._attention_operand(t)
        assert (got.data_ptr() == t.data_ptr()) == in_place, t.stride()
        assert all(s % unit == 0 for s in strides) and got.data_ptr() % 16 == 0
        assert torch.equal(_view(got, strides, t), t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_views_with_single_axes_on_the_gpu(hip_ext, dtype):
    """Forward and backward over each, as queries and as keys and values, give the bits of dense copies; and so does
    the gradient that autograd hands a one-head attention's output."""
    for name, t in _single_axis_views(dtype):
        t = torch.randn(t.untyped_storage().nbytes() // t.element_size(),
                        device="cuda").to(dtype).as_strided(t.shape, t.stride(), t.storage_offset())
        dense = torch.empty(t.shape, dtype=dtype, device="cuda").copy_(t)
        kv = torch.randn(t.shape[0], 70, t.shape[2], t.shape[3], device="cuda").to(dtype)
        for q, k, q2, k2 in ((t, kv, dense, kv), (kv, t, kv, dense)):
            out, lse = hip_ext.cross_attention_forward(q, k, k, need_lse=True)
            want, wlse = hip_ext.cross_attention_forward(q2, k2, k2, need_lse=True)
            assert torch.equal(out, want) and torch.equal(lse, wlse), name
            go = t if q is t else kv
            go2 = dense if q is t else kv
            for x, y in zip(hip_ext.cross_attention_backward(go, q, k, k, out, lse),
                            hip_ext.cross_attention_backward(go2, q2, k2, k2, want, wlse)):
                assert torch.equal(x, y), name
    from pymsst_amd import fused_roformer as fr

    for b in (1, 2):
        q = torch.randn(b, 5, 1, 64, device="cuda", dtype=torch.float32).to(dtype).requires_grad_()
        k = torch.randn(b, 9, 1, 64, device="cuda", dtype=torch.float32).to(dtype)
        w = torch.randn(64, 24, device="cuda").to(dtype)
        out = fr.cross_attention(q, k, k)
        # the product leaves a one-head gradient with whatever stride its single head has
        (g,) = torch.autograd.grad(torch.matmul(out.transpose(2, 3).squeeze(-1), w).float().sum(), q)
        out2 = fr.cross_attention(q, k, k)
        go = torch.matmul(torch.ones(b, 5, 24, device="cuda", dtype=dtype), w.t().contiguous())[:, :, None].contiguous()
        (want,) = torch.autograd.grad(out2, q, go)
        assert torch.equal(g, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", _F)
def test_a_saved_output_between_16_bytes_is_copied(hip_ext, dtype):
    """A forward's output and log-sums kept in a buffer of the caller's own, at any offset and stride."""
    q, do = (torch.randn(2, 37, 4, 64, device="cuda").to(dtype) for _ in range(2))
    k = torch.randn(2, 90, 2, 64, device="cuda").to(dtype)
    out, lse = hip_ext.cross_attention_forward(q, k, k, need_lse=True)
    want = hip_ext.cross_attention_backward(do, q, k, k, out, lse)
    flat = torch.empty(out.numel() + 1, dtype=dtype, device="cuda")
    kept = flat[1:].view(out.shape).copy_(out)
    wide = torch.empty(2, 37, 4, 65, dtype=dtype, device="cuda")
    strided = wide[..., 1:].copy_(out)
    sums = torch.empty(2, 37, 4, device="cuda").transpose(1, 2).copy_(lse)
    for o in (kept, strided):
        for x, y in zip(hip_ext.cross_attention_backward(do, q, k, k, o, sums), want):
            assert torch.equal(x, y)
