"""Calls of the attention operators at the edges of their arguments, on the CPU."""

import pytest
import torch

import bitscom_b200 as bitscom


def test_caps_and_scales_outside_fp32_are_refused():
    q, k, v = torch.randn(1, 2, 4, 8), torch.randn(1, 2, 4, 8), torch.randn(1, 2, 4, 8)
    inf = float("inf")
    for bad in (inf, -inf, float("nan"), 0.0, 1e-40, 1e-50, 1e39, 1e300):
        with pytest.raises(ValueError):
            bitscom.attention(q, k, v, softcap=bad)
        with pytest.raises(ValueError):
            bitscom.attention(q, k, v, scale=bad)
    for cap in (1e-30, 1e30):
        assert torch.isfinite(bitscom.attention(q, k, v, softcap=cap)).all()
