"""Norm of queries and keys for each head, with the position rotation in the
same pass, forward and backward.

``qk_norm_rotary`` prepares the queries and keys of an attention block: every
head vector is divided by its root mean square, scaled by a gain, and its
first values are rotated in pairs by angles ``position * frequency``.  CUDA
tensors run ``csrc/kernels/qk_norm_rotary.cu`` (one read and one write of each
head); CPU tensors use the torch code below.  Angles are formed in 64 bits on
both, so far positions lose nothing.  No counterpart in the reference.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _ext


def rotary_frequencies(rotated: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """float64 ``base ** (-2 i / rotated)`` for the ``rotated / 2`` pairs of a head."""
    if rotated < 2 or rotated % 2:
        raise ValueError(f"rotated must be a positive even number, got {rotated}")
    return base ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device=device) / rotated)


def qk_norm_rotary(
    q: torch.Tensor,
    k: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Normalised and rotated ``(q, k)``, contiguous, in their dtype.

    Args:
        q, k: ``[batch, length, heads, head size]`` and ``[batch, length, key
            heads, head size]`` (views of a joint projection are fine);
            float32, bfloat16 or float16; head size 1 to 256.
        frequencies: ``[rotated / 2]`` floating point (float64 is used as it is),
            see :func:`rotary_frequencies`; ``2 * len(frequencies)`` values of
            each head are rotated, the rest is only normalised.
        q_weight, k_weight: ``[head size]`` gains, None for ones.
        positions: int32 or int64 ``[length]`` or ``[batch, length]``; default
            0, 1, 2, ...
        eps: added to the mean square.
        interleaved: pairs are neighbours (2 i, 2 i + 1) in place of
            (i, i + rotated / 2).

    Arithmetic is float32 with one rounding at the end.  Gradients reach q, k
    and the gains (summed in a fixed order), not frequencies or positions; on CUDA
    a forward-mode tangent is refused.
    """
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise ValueError("qk_norm_rotary does not differentiate frequencies: detach them")
    if not _ext.use_cuda_kernels(q):
        return _qk_norm_rotary_cpu(q, k, frequencies, q_weight, k_weight, positions, eps, interleaved)
    return _ext.operator("rotary_forward")(q, k, frequencies, q_weight, k_weight, positions, eps, interleaved)


def _qk_norm_rotary_cpu(q, k, freq, wq, wk, positions, eps, interleaved):
    floats = (torch.float32, torch.bfloat16, torch.float16)
    if q.dtype not in floats or k.dtype != q.dtype:
        raise TypeError(f"q and k must have one dtype of {floats}, got {q.dtype} and {k.dtype}")
    if not freq.is_floating_point():
        raise TypeError("frequencies must be floating point")
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must be [batch, length, heads, head size], "
                         "alike but for the heads")
    b, s, _, d = q.shape
    if not 1 <= d <= 256:
        raise ValueError(f"head size must be 1 to 256, got {d}")
    if freq.dim() != 1 or 2 * freq.shape[0] > d:
        raise ValueError(f"frequencies must be a vector of at most {d // 2} values, got {tuple(freq.shape)}")
    for name, w in (("q_weight", wq), ("k_weight", wk)):
        if w is not None and not w.dtype in floats:
            raise TypeError(f"{name} must be floating point")
        if w is not None and w.shape != (d,):
            raise ValueError(f"{name} must be [{d}], got {tuple(w.shape)}")
    if positions is None:
        positions = torch.arange(s)
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if positions.shape not in ((s,), (b, s)):
        raise ValueError(f"positions must be [{s}] or [{b}, {s}], got {tuple(positions.shape)}")
    angle = positions.double()[..., None, None] * freq.double()
    cos, sin = angle.cos().float(), angle.sin().float()
    r = 2 * freq.shape[0]

    def one(x, w):
        xf = x.float()
        y = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * w.float()
        if interleaved:
            a, c = y[..., 0:r:2], y[..., 1:r:2]
            z = torch.stack((a * cos - c * sin, c * cos + a * sin), -1).flatten(-2)
        else:
            a, c = y[..., : r // 2], y[..., r // 2 : r]
            z = torch.cat((a * cos - c * sin, c * cos + a * sin), -1)
        return torch.cat((z, y[..., r:]), -1).to(x.dtype)

    return one(q, wq), one(k, wk)


if _ext.available():  # what tracing with fake tensors sees

    @torch.library.register_fake("bitscom_b200::rotary_forward", allow_override=True)
    def _(q, k, frequencies, q_weight, k_weight, positions, eps, interleaved):
        return q.new_empty(q.shape), k.new_empty(k.shape)

    @torch.library.register_fake("bitscom_b200::rotary_backward", allow_override=True)
    def _(grad_q, grad_k, q, k, frequencies, q_weight, k_weight, positions, eps, interleaved, want_gains):
        gains = q.new_empty((2, q.shape[3]) if want_gains else (0,), dtype=torch.float32)
        return q.new_empty(q.shape), k.new_empty(k.shape), gains


__all__ = ["qk_norm_rotary", "rotary_frequencies"]
