"""Masked attention for GPT-style models: packed documents, prefixes, capped
scores and a distance bias, forward and backward.

``F.scaled_dot_product_attention(is_causal=True)`` sees a row of tokens as one
document.  :func:`attention` takes what packed training rows and prompts need
on top, without a mask tensor of length x length anywhere:

* ``documents``: ids of the key tokens; a run of equal ids is a document, and
  tokens see their own document only.  A negative id is padding: it sees
  nothing (its output is zero) and nothing sees it;
* ``prefix``: the first ``prefix[b]`` keys are visible to every token of their
  document (prefix language models), beside the causal ones;
* ``softcap``: scores become ``softcap * tanh(score / softcap)``;
* ``slopes``: ``slopes[h] * |distance|`` is subtracted from head h's scores.

CUDA tensors run the kernels of ``csrc/kernels/attention_*.cu``; CPU tensors use
the torch code below.  The reference has no attention of its own (its
benchmarks call Hugging Face models).
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _ext

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_INTS = (torch.int32, torch.int64)


class AttentionMask:
    """Which keys each query sees, built once by :func:`attention_mask` and
    shared by all layers of a model (and by the backward pass)."""

    __slots__ = ("causal", "batch", "q_len", "k_len", "plan", "documents", "prefix")

    def __init__(self, causal, batch, q_len, k_len, plan, documents, prefix):
        self.causal, self.batch, self.q_len, self.k_len = causal, batch, q_len, k_len
        self.plan, self.documents, self.prefix = plan, documents, prefix

    def __repr__(self) -> str:
        return f"AttentionMask(batch={self.batch}, q_len={self.q_len}, k_len={self.k_len}, causal={self.causal})"

    def visible(self) -> torch.Tensor:
        """[batch, q_len, k_len] truth values (CPU masks only: for tests and the torch path)."""
        if self.plan is not None:
            raise ValueError("visible() is for masks of CPU tensors")
        return _visible(self.causal, self.batch, self.q_len, self.k_len, self.documents, self.prefix)


def attention_mask(
    documents: Optional[torch.Tensor] = None,
    prefix: Optional[torch.Tensor] = None,
    *,
    causal: bool = True,
    q_len: Optional[int] = None,
    k_len: Optional[int] = None,
) -> AttentionMask:
    """Mask of :func:`attention` from document ids ``[batch, k_len]`` and / or
    prefix lengths ``[batch]`` (int32 or int64).

    ``k_len`` is taken from ``documents`` where given; ``q_len`` defaults to
    it, otherwise the queries are the last ``q_len`` positions.  On CUDA one
    kernel finds each row's interval of visible keys; later changes of
    ``documents`` or ``prefix`` do not reach the mask.
    """
    if documents is None and prefix is None:
        raise ValueError("attention_mask needs documents or prefix (without either, pass causal= to attention)")
    if documents is not None:
        if documents.dim() != 2:
            raise ValueError(f"documents must be [batch, key length], got {tuple(documents.shape)}")
        if k_len is not None and k_len != documents.shape[1]:
            raise ValueError(f"documents cover {documents.shape[1]} keys, k_len is {k_len}")
        k_len = documents.shape[1]
    if prefix is not None:
        if not causal:
            raise ValueError("a prefix needs a causal mask")
        if prefix.dim() != 1 or (documents is not None and prefix.shape[0] != documents.shape[0]):
            raise ValueError(f"prefix must hold one length for each batch entry, got {tuple(prefix.shape)}")
        if documents is not None and prefix.device != documents.device:
            raise ValueError("documents and prefix must be on one device")
    if k_len is None:
        raise ValueError("k_len is needed without documents")
    q_len = k_len if q_len is None else q_len
    if q_len < 0 or k_len < 0:
        raise ValueError("lengths must not be negative")
    like = documents if documents is not None else prefix
    batch = like.shape[0]
    for name, t in (("documents", documents), ("prefix", prefix)):
        if t is not None and t.dtype not in _INTS:
            raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    if _ext.use_cuda_kernels(like):
        plan = _ext.operator("attention_plan")(documents, prefix, causal, batch, q_len, k_len)
        return AttentionMask(causal, batch, q_len, k_len, plan, None, None)
    with torch.inference_mode(False):  # a mask made in inference mode serves training too
        return AttentionMask(causal, batch, q_len, k_len, None, None if documents is None else documents.clone(),
                             None if prefix is None else prefix.clone())


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    causal: bool = True,
    documents: Optional[torch.Tensor] = None,
    prefix: Optional[torch.Tensor] = None,
    mask: Optional[AttentionMask] = None,
    softcap: Optional[float] = None,
    slopes: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """``softmax(scores) v`` over each query's visible keys.

    Args:
        q: ``[batch, heads, q_len, head size]``; k, v: ``[batch, key heads, k_len,
            head size]`` with ``heads`` a multiple of ``key heads`` (consecutive
            query heads share one).  float32, bfloat16 or float16, any strides;
            head size 1 to 256.
        causal: a query sees keys up to its own position.  The queries are the
            last ``q_len`` of the ``k_len`` positions.
        documents, prefix: see the module's description and
            :func:`attention_mask`, which builds them into a ``mask`` once for
            several calls; ``mask`` replaces ``causal``, ``documents``, ``prefix``.
        softcap: cap of the scores (1e-12 to 1e30), None for none.
        slopes: ``[heads]`` distance slopes (not differentiated).
        scale: factor of ``q.k`` (1e-30 to 1e30), default ``head size ** -0.5``.

    Returns ``[batch, heads, q_len, head size]`` in q's dtype (stored
    ``[batch, q_len, heads, head size]``).  Rows that see no key are zero, with
    zero gradients.  Keys that no query may see because they are padding are
    never touched by the arithmetic, whatever they hold; a NaN or infinity in
    any other key can reach every query whose tile of 128 keys holds it.
    Gradients are by the backward pass, once; on CUDA a forward-mode tangent is refused.
    float16 and bfloat16 round the probabilities and score gradients to that
    type for the products (in float16 score gradients below 6e-5 lose bits: scale
    the loss); all sums are float32.  Under autocast float32 inputs
    are cast like those of torch's own attention.
    """
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k and v must be [batch, heads, length, head size]")
    if softcap is not None and not 1e-12 <= softcap <= 1e30:
        raise ValueError(f"softcap must be positive, from 1e-12 to 1e30, got {softcap}")
    if scale is not None and not 1e-30 <= scale <= 1e30:
        raise ValueError(f"scale must be positive, from 1e-30 to 1e30, got {scale}")
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError("attention does not differentiate slopes: detach them")
    if torch.is_autocast_enabled(q.device.type):
        dt = torch.get_autocast_dtype(q.device.type)
        q, k, v = (t.to(dt) if t.dtype == torch.float32 else t for t in (q, k, v))
    if mask is not None:
        if documents is not None or prefix is not None:
            raise ValueError("pass documents and prefix to attention_mask, or to attention without a mask")
        causal = mask.causal
    elif documents is not None or prefix is not None:
        mask = attention_mask(documents, prefix, causal=causal, q_len=q.shape[2], k_len=k.shape[2])
    if mask is not None and (mask.batch, mask.q_len, mask.k_len) != (q.shape[0], q.shape[2], k.shape[2]):
        raise ValueError(f"{mask} does not fit q {tuple(q.shape)} and k {tuple(k.shape)}")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    cap = 0.0 if softcap is None else float(softcap)
    if not _ext.use_cuda_kernels(q):
        return _attention_cpu(q, k, v, mask, causal, slopes, scale, cap)
    if mask is not None and mask.plan is None:
        raise ValueError("the mask was built from CPU tensors, q is on " + str(q.device))
    plan = None if mask is None else mask.plan
    return _ext.operator("attention_forward")(q, k, v, plan, slopes, causal, scale, cap)


def _visible(causal, batch, q_len, k_len, documents, prefix) -> torch.Tensor:
    pos = torch.arange(q_len) + (k_len - q_len)
    key = torch.arange(k_len)
    seen = torch.ones(batch, q_len, k_len, dtype=torch.bool)
    if causal:
        seen &= key <= pos[:, None]
        if prefix is not None:
            seen |= (key < prefix[:, None])[:, None, :]
    if documents is not None:
        # A run of equal ids is one document: number the runs.
        change = torch.ones_like(documents, dtype=torch.int64)
        change[:, 1:] = (documents[:, 1:] != documents[:, :-1]).long()
        run = change.cumsum(1).masked_fill(documents < 0, -1)
        mine = torch.full((batch, q_len), -1, dtype=torch.int64)
        inside = pos >= 0
        mine[:, inside] = run[:, pos[inside]]
        seen &= (mine[:, :, None] == run[:, None, :]) & (mine >= 0)[:, :, None]
    return seen


def _attention_cpu(q, k, v, mask, causal, slopes, scale, cap):
    if q.dtype not in _FLOATS or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must have one dtype of {_FLOATS}, got {q.dtype}, {k.dtype} and {v.dtype}")
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"shapes do not fit: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    b, h, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    if hk == 0 or h % hk:
        raise ValueError(f"{h} query heads are not a multiple of {hk} key heads")
    if not 1 <= d <= 256:
        raise ValueError(f"head size must be 1 to 256, got {d}")
    if slopes is not None and slopes.dtype != torch.float32:
        raise TypeError("slopes must be float32")
    if slopes is not None and slopes.shape != (h,):
        raise ValueError(f"slopes must be one value for each of the {h} query heads")
    if mask is not None and mask.plan is not None:
        raise ValueError("the mask was built from CUDA tensors, q is on the CPU")
    if mask is not None:
        seen = mask.visible()
    else:
        seen = _visible(causal, 1, sq, sk, None, None)
    seen = seen[:, None, None]  # [batch, key head, group, query, key]
    qf = q.float().reshape(b, hk, h // hk, sq, d)
    dead = torch.zeros(1, 1, sk, 1, dtype=torch.bool)
    if mask is not None and mask.documents is not None:
        dead = (mask.documents < 0)[:, None, :, None]
    kf, vf = (x.float().masked_fill(dead, 0.0)[:, :, None] for x in (k, v))
    none = ~seen.any(-1, keepdim=True)
    s = (qf.masked_fill(none, 0.0) @ kf.transpose(-1, -2)) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        far = (torch.arange(sk - sq, sk)[:, None] - torch.arange(sk)[None, :]).abs().float()
        s = s - slopes.view(1, hk, h // hk, 1, 1) * far
    s = torch.where(none, torch.zeros_like(s), s.masked_fill(~seen, -math.inf))
    p = torch.softmax(s, -1).masked_fill(none, 0.0) if sk else s
    out = (p @ vf).reshape(b, h, sq, d)
    return out.transpose(1, 2).to(q.dtype).contiguous().transpose(1, 2)


if _ext.available():  # what tracing with fake tensors sees: the layouts of csrc/ops/attention_ops.cpp

    def _tokens_first(t):
        return t.new_empty((t.shape[0], t.shape[2], t.shape[1], t.shape[3])).transpose(1, 2)

    @torch.library.register_fake("bitscom_b200::attention_plan", allow_override=True)
    def _(documents, prefix, causal, batch, q_len, k_len):
        like = documents if documents is not None else prefix
        q_tiles, k_tiles = (q_len + 127) // 128, (k_len + 127) // 128
        return like.new_empty(batch * (q_tiles * (2 * 128 + 8) + k_tiles * 4), dtype=torch.int32)

    @torch.library.register_fake("bitscom_b200::attention_forward", allow_override=True)
    def _(q, k, v, plan, slopes, causal, scale, cap):
        return _tokens_first(q)

    @torch.library.register_fake("bitscom_b200::attention_forward_sums", allow_override=True)
    def _(q, k, v, plan, slopes, causal, scale, cap):
        tensor_cores = q.dtype != torch.float32 and q.shape[3] % 8 == 0 and q.shape[3] <= 128
        sums = q.new_empty(q.shape[:3], dtype=torch.float32)
        return _tokens_first(q), sums, _tokens_first(q) if tensor_cores else q.new_empty(0)

    @torch.library.register_fake("bitscom_b200::attention_backward", allow_override=True)
    def _(grad, q, k, v, out, sums, low, plan, slopes, causal, scale, cap):
        return _tokens_first(q), _tokens_first(k), _tokens_first(v)


__all__ = ["AttentionMask", "attention", "attention_mask"]
