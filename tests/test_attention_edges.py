"""Calls of the attention operators at the edges of their arguments, on the CPU."""

import importlib
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import bitscom_b200 as bitscom
from bitscom_b200 import _ext
from bitscom_b200.models import GPT2, GPT2Config


def test_caps_and_scales_outside_fp32_are_refused():
    q, k, v = torch.randn(1, 2, 4, 8), torch.randn(1, 2, 4, 8), torch.randn(1, 2, 4, 8)
    inf = float("inf")
    for bad in (inf, -inf, float("nan"), 0.0, 1e-40, 1e-50, 1e39, 1e300):
        with pytest.raises(ValueError):
            bitscom.attention(q, k, v, softcap=bad)
        with pytest.raises(ValueError):
            bitscom.attention(q, k, v, scale=bad)
    for cap in (1e-12, 1e30):
        assert torch.isfinite(bitscom.attention(q, k, v, softcap=cap)).all()


@pytest.mark.parametrize("options", [dict(rotary=True), dict(distance_bias=True)], ids=str)
def test_inference_mode_leaves_no_inference_tensors(options):
    """What the model and a mask keep from a call in inference mode can be saved for a backward pass."""
    model = GPT2(GPT2Config(vocab_size=61, n_positions=32, n_embd=32, n_layer=1, n_head=4, **options))
    idx, ids = torch.randint(0, 61, (1, 9)), torch.zeros(1, 9, dtype=torch.int32)
    with torch.inference_mode():
        model(idx, documents=ids)
        mask = bitscom.attention_mask(ids.clone(), torch.tensor([3]))
    kept = list(model.blocks[0].attn._constants.values()) + [mask.documents, mask.prefix]
    assert len(kept) == 3 and not any(t.is_inference() for t in kept)
    model(idx, documents=ids).sum().backward()


def test_wrong_ranks_are_refused_with_masks():
    q, k, ids = torch.randn(2, 4, 6, 8), torch.randn(2, 2, 6, 8), torch.zeros(2, 6, dtype=torch.int32)
    for kw in ({}, {"documents": ids}, {"mask": bitscom.attention_mask(ids)}, {"prefix": ids[:, 0]}):
        for args in ((q[0], k, k), (q[0, 0], k, k), (q, k[0, 0], k), (q, k, k[0, 0])):
            with pytest.raises(ValueError, match="batch, heads, length"):
                bitscom.attention(*args, **kw)


def test_modules_can_be_reloaded():
    for name in ("attention", "rotary"):
        importlib.reload(sys.modules[f"bitscom_b200.ops.{name}"])


@pytest.mark.skipif(not _ext.available(), reason="the native extension is not built")
@pytest.mark.parametrize("dtype,d", [(torch.half, 64), (torch.half, 100), (torch.float32, 64)], ids=str)
def test_fake_tensors_have_the_layout_of_results(dtype, d):
    """Shapes, types and strides that a trace sees of each operator, without a GPU."""
    ops = torch.ops.bitscom_b200
    with FakeTensorMode():
        q, k, v = (torch.empty(2, s, h, d, device="cuda", dtype=dtype).transpose(1, 2)
                   for s, h in ((5, 4), (9, 2), (9, 2)))
        mask = bitscom.attention_mask(torch.empty(2, 9, device="cuda", dtype=torch.int32), q_len=5)
        assert mask.plan.shape == (2 * (128 * 2 + 8 + 4),) and mask.plan.dtype == torch.int32
        args = (mask.plan, None, True, 0.125, 3.0)
        out, sums, low = ops.attention_forward_sums(q, k, v, *args)
        kept = dtype == torch.half and d == 64
        assert sums.shape == (2, 4, 5) and sums.dtype == torch.float32
        assert low.dtype == dtype and low.shape == (q.shape if kept else (0,))
        grads = ops.attention_backward(out, q, k, v, out, sums, low, *args)
        for x, y in zip((q, q, k, v), (out, *grads)):
            assert y.shape == x.shape and y.dtype == x.dtype and y.transpose(1, 2).is_contiguous()
        graph = bitscom.attention(q.requires_grad_(True), k, v, mask=mask, softcap=3.0)
        assert graph.requires_grad and graph.shape == q.shape and graph.transpose(1, 2).is_contiguous()
        x, y = (t.detach().transpose(1, 2)[:, :5] for t in (q, k))
        rest = (torch.empty(d // 2, device="cuda", dtype=torch.double), None, None, None, 1e-6, False)
        for a, b in zip(bitscom.qk_norm_rotary(x, y, rest[0]), (x, y)):
            assert a.shape == b.shape and a.dtype == dtype and a.is_contiguous()
        for want in (True, False):
            dx, dy, gains = ops.rotary_backward(x, y, x, y, *rest, want)
            assert dx.shape == x.shape and dy.shape == y.shape and dx.is_contiguous() and dx.dtype == dtype
            assert gains.shape == ((2, d) if want else (0,)) and gains.dtype == torch.float32
