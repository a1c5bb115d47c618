"""Calls of the attention operators at the edges of their arguments, on the CPU."""

import pytest
import torch

import bitscom_b200 as bitscom
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
