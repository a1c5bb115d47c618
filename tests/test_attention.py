"""Attention operators on the CPU: torch forms against the 64-bit oracle, masks,
refusals, and the GPT-2 options that use them."""

import pytest
import torch
import torch.nn.functional as F

import bitscom_b200 as bitscom
from bitscom_b200.models import GPT2, GPT2Config

from .attention_oracle import check, reference, rotary_reference, visible


def _qkv(b, h, hk, sq, sk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(b, n, s, d, generator=g).to(dtype) for n, s in ((h, sq), (hk, sk), (hk, sk), (h, sq)))
    return [x.requires_grad_(True) for x in (q, k, v)] + [do]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 8), (2, 4, 2, 9, 13, 16), (1, 2, 1, 12, 5, 6)], ids=str)
def test_cpu_form_matches_64_bits(shape, dtype):
    b, h, hk, sq, sk, d = shape
    q, k, v, do = _qkv(*shape, dtype)
    ids = (torch.arange(sk) // 4).repeat(b, 1)
    ids[:, -1:] = -1 if sk > 1 else 0
    for causal, docs, prefix in ((True, None, None), (False, None, None), (True, ids, None), (False, ids, None),
                                 (True, ids, torch.full((b,), 3))):
        slopes = 0.5 ** torch.arange(1, h + 1, dtype=torch.float32)
        out = bitscom.attention(q, k, v, causal=causal, documents=docs, prefix=prefix, softcap=3.0, slopes=slopes)
        grads = torch.autograd.grad(out, (q, k, v), do)
        vals, bounds = reference(q, k, v, do, seen=visible(b, sq, sk, causal, docs, prefix), softcap=3.0, slopes=slopes)
        check({"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}, vals, bounds)


def test_cpu_padding_may_hold_anything():
    q, k, v, do = _qkv(1, 2, 2, 8, 8, 4, torch.float32)
    ids = torch.tensor([[0, 0, 0, 1, 1, -1, -1, -1]])
    want = bitscom.attention(q, k, v, documents=ids)
    bad = [x.detach().clone() for x in (q, k, v)]
    for x in bad:
        x[:, :, 5:] = float("nan")
    got = bitscom.attention(*bad, documents=ids)
    assert torch.equal(got, want) and (got[:, :, 5:] == 0).all()


def test_mask_visible_matches_its_definition():
    ids = torch.tensor([[3, 3, 3, 5, 5, -1, -1, 3], [0, 1, 1, 1, 2, 2, 2, 2]])
    prefix = torch.tensor([2, 3])
    for causal, p in ((True, None), (False, None), (True, prefix)):
        mask = bitscom.attention_mask(ids, p, causal=causal, q_len=6)
        assert torch.equal(mask.visible(), visible(2, 6, 8, causal, ids, p))
    mask = bitscom.attention_mask(prefix=prefix, q_len=4, k_len=9)
    assert torch.equal(mask.visible(), visible(2, 4, 9, True, None, prefix))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_cpu_rotary_matches_64_bits(dtype, interleaved):
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(2, 5, 3, 12, generator=g).to(dtype), torch.randn(2, 5, 1, 12, generator=g).to(dtype)
    w = 1 + 0.1 * torch.randn(12, generator=g)
    freq = bitscom.rotary_frequencies(8)
    pos = torch.arange(5) + 1_000_000
    oq, ok = bitscom.qk_norm_rotary(q, k, freq, q_weight=w, positions=pos, interleaved=interleaved)
    for got, x, wt in ((oq, q, w), (ok, k, None)):
        want, _, _ = rotary_reference(x, wt, freq, pos, 1e-6, interleaved)
        u = torch.finfo(dtype).eps / 2
        assert got.dtype == dtype
        # one rounding, and fp32 products of values below 4 before it
        assert ((got.double() - want).abs() <= u * want.abs() + 32 * 2.0 ** -24 * 4).all()


def test_rotary_gradients_on_the_cpu():
    q, k = torch.randn(1, 3, 2, 8, requires_grad=True), torch.randn(1, 3, 1, 8)
    w = torch.ones(8, requires_grad=True)
    freq = bitscom.rotary_frequencies(4)
    out = bitscom.qk_norm_rotary(q, k, freq, q_weight=w)[0]
    g = torch.randn_like(out)
    dq, dw = torch.autograd.grad(out, (q, w), g)
    _, wq, ww = rotary_reference(q, w, freq, torch.arange(3), 1e-6, False, g)
    assert torch.allclose(dq.double(), wq, atol=1e-5) and torch.allclose(dw.double(), ww, atol=1e-5)


def test_refusals_on_the_cpu():
    q, k, v = torch.randn(2, 4, 6, 8), torch.randn(2, 2, 6, 8), torch.randn(2, 2, 6, 8)
    a, m = bitscom.attention, bitscom.attention_mask
    ids = torch.zeros(2, 6, dtype=torch.int32)
    bad = [
        (ValueError, lambda: a(q[0], k, v)),
        (ValueError, lambda: a(q, k, v[:, :, :3])),
        (ValueError, lambda: a(q[:, :3], k, v)),
        (TypeError, lambda: a(q, k.half(), v)),
        (TypeError, lambda: a(q.double(), k.double(), v.double())),
        (ValueError, lambda: a(*[torch.zeros(1, 1, 2, 257)] * 3)),
        (ValueError, lambda: a(q, k, v, softcap=-1.0)),
        (ValueError, lambda: a(q, k, v, scale=0.0)),
        (ValueError, lambda: a(q, k, v, slopes=torch.ones(2))),
        (TypeError, lambda: a(q, k, v, slopes=torch.ones(4).half())),
        (ValueError, lambda: a(q, k, v, slopes=torch.ones(4, requires_grad=True))),
        (ValueError, lambda: a(q, k, v, documents=ids[:, :5])),
        (ValueError, lambda: a(q, k, v, documents=ids[:1])),
        (TypeError, lambda: a(q, k, v, documents=ids.float())),
        (ValueError, lambda: a(q, k, v, causal=False, prefix=torch.zeros(2, dtype=torch.int32))),
        (ValueError, lambda: a(q, k, v, prefix=torch.zeros(1, dtype=torch.int32))),
        (ValueError, lambda: a(q, k, v, mask=m(ids), documents=ids)),
        (ValueError, lambda: a(q[:, :, :3], k, v, mask=m(ids))),
        (ValueError, lambda: m()),
        (ValueError, lambda: m(ids[0])),
        (ValueError, lambda: m(ids, k_len=7)),
        (ValueError, lambda: m(prefix=torch.zeros(2, dtype=torch.int32))),
        (ValueError, lambda: m(ids, q_len=-1)),
        (ValueError, lambda: bitscom.rotary_frequencies(7)),
        (ValueError, lambda: bitscom.rotary_frequencies(0)),
    ]
    freq = bitscom.rotary_frequencies(8)
    x, y = torch.randn(2, 5, 4, 8), torch.randn(2, 5, 2, 8)
    f = bitscom.qk_norm_rotary
    bad += [
        (ValueError, lambda: f(x[0], y, freq)),
        (ValueError, lambda: f(x, y[:, :4], freq)),
        (TypeError, lambda: f(x, y.half(), freq)),
        (TypeError, lambda: f(x, y, freq.long())),
        (ValueError, lambda: f(x, y, bitscom.rotary_frequencies(10))),
        (ValueError, lambda: f(x, y, freq, q_weight=torch.ones(4))),
        (TypeError, lambda: f(x, y, freq, positions=torch.zeros(5))),
        (ValueError, lambda: f(x, y, freq, positions=torch.zeros(4, dtype=torch.int64))),
        (ValueError, lambda: f(x, y, freq.clone().requires_grad_(True))),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def _tiny(**kw):
    torch.manual_seed(0)
    return GPT2(GPT2Config(vocab_size=61, n_positions=32, n_embd=32, n_layer=2, n_head=4, **kw))


def test_gpt2_without_options_is_unchanged():
    """The plain model has the parameters it had and attends through torch's own attention."""
    model = _tiny()
    names = [n for n, _ in model.named_parameters()]
    assert len(names) == 2 + 2 * 12 + 2 and not any("gain" in n for n in names)
    idx = torch.randint(0, 61, (2, 20))
    x = model.wte(idx) + model.wpe(torch.arange(20))
    for blk in model.blocks:
        q, k, v = (z.view(2, 20, 4, 8).transpose(1, 2) for z in blk.attn.qkv(blk.ln1(x)).split(32, dim=2))
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        x = x + blk.attn.proj(y.transpose(1, 2).reshape(2, 20, 32))
        x = x + blk.out(F.gelu(blk.fc(blk.ln2(x)), approximate="tanh"))
    assert torch.equal(model(idx), F.linear(model.ln_f(x), model.wte.weight))


@pytest.mark.parametrize("options", [{}, {"rotary": True}, {"rotary": True, "softcap": 4.0},
                                     {"distance_bias": True, "softcap": 4.0}], ids=str)
def test_packed_documents_are_as_if_alone(options):
    """Logits and gradients of two documents packed into a row are those of the two rows apart."""
    model = _tiny(**options)
    a, b = torch.randint(0, 61, (1, 9)), torch.randint(0, 61, (1, 14))
    row = torch.cat([a, b, torch.zeros(1, 4, dtype=torch.int64)], 1)
    ids = torch.tensor([[0] * 9 + [1] * 14 + [-1] * 4])
    packed = model(row, documents=ids)
    alone = [model(a), model(b)]
    for x, y in ((packed[:, :9], alone[0]), (packed[:, 9:23], alone[1])):
        assert torch.allclose(x, y, atol=1e-5)
    params = list(model.parameters())
    g1 = torch.autograd.grad(packed[:, :23].square().sum(), params)
    g2 = torch.autograd.grad(alone[0].square().sum() + alone[1].square().sum(), params)
    for x, y in zip(g1, g2):
        assert torch.allclose(x, y, atol=1e-4 * float(y.abs().max()) + 1e-6)


def test_prefix_tokens_see_each_other():
    model = _tiny(rotary=True)
    idx = torch.randint(0, 61, (1, 12))
    changed = idx.clone()
    changed[0, 4] = (changed[0, 4] + 1) % 61
    p = torch.tensor([6])
    assert not torch.allclose(model(idx, prefix=p)[0, 0], model(changed, prefix=p)[0, 0])
    assert torch.allclose(model(idx)[0, :4], model(changed)[0, :4])


def test_frequencies_survive_a_cast():
    model = _tiny(rotary=True).bfloat16()
    model(torch.randint(0, 61, (1, 4)))
    freq = model.blocks[0].attn._constant("frequencies", torch.device("cpu"))
    assert freq.dtype == torch.float64 and torch.equal(freq, bitscom.rotary_frequencies(8))
