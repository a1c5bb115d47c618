"""The attention operators at the edges of their range: waits that run out, what
other kernels leave in shared memory, extreme caps, derivatives and traces.
Needs a CUDA device."""

import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch.fx.experimental.proxy_tensor import make_fx

import bitscom_b200 as bitscom
from bitscom_b200 import _ext
from bitscom_b200.models import gpt2_small_test

from .attention_oracle import check, reference, visible

pytestmark = pytest.mark.gpu


def _qkv(b, h, hk, sq, sk, d, dtype, seed=0, grad=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, do = (torch.randn(b, s, n, d, generator=g, device="cuda").to(dtype).transpose(1, 2)
                   for n, s in ((h, sq), (hk, sk), (hk, sk), (h, sq)))
    if grad:
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    return q, k, v, do


@pytest.fixture
def wait_limit(cuda):
    """Sets the limit of the kernels' waits; puts it back and clears the status."""
    before = _ext._C.attention_wait_limit(1 << 33)
    yield _ext._C.attention_wait_limit
    _ext._C.attention_wait_limit(before)
    _ext._C.attention_status(True)


# Copies that the block has no stage for, that it has, key splits with shared heads; both widths.
@pytest.mark.parametrize("limit", [0, 2000])
@pytest.mark.parametrize("shape", [(1, 2, 2, 100, 100, 64), (2, 4, 2, 700, 700, 64), (1, 4, 2, 300, 900, 128),
                                   (1, 4, 1, 1, 5000, 128), (1, 4, 4, 1, 5000, 64)], ids=str)
def test_waits_that_run_out(wait_limit, shape, limit):
    """A kernel whose waits run out leaves NaN and raises the status, and the next call is right again.

    With limit 0 the scores are never reported: the arithmetic warps give up, with copies and products
    under way.  With a limit of the length of a few tiles some waits may run out: a value is then right or NaN.
    """
    q, k, v, do = _qkv(*shape, torch.bfloat16, grad=True)
    out = bitscom.attention(q, k, v)
    want = torch.autograd.grad(out, (q, k, v), do)
    for _ in range(3):
        out_now = bitscom.attention(q, k, v)
        wait_limit(limit)
        got = [bitscom.attention(q.detach(), k, v), *torch.autograd.grad(out_now, (q, k, v), do)]
        torch.cuda.synchronize()
        wait_limit(1 << 33)
        status = _ext._C.attention_status(True)
        if limit == 0:
            assert status == 1 and all(torch.isnan(x).all() for x in got)
        else:
            assert all(((x == y) | torch.isnan(x)).all() for x, y in zip(got, (out, *want)))
            assert status == 1 or not any(torch.isnan(x).any() for x in got)
        again = bitscom.attention(q, k, v)
        grads = torch.autograd.grad(again, (q, k, v), do)
        assert torch.equal(again, out) and all(torch.equal(x, y) for x, y in zip(grads, want))
        assert _ext._C.attention_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_shared_memory_of_another_call_does_not_show(cuda, dtype):
    """Shared heads packed into one tile: rows of the tile that are no query's hold what the last kernel left unless
    they are cleared.  With scores far above the cap there, a warp's choice of the tanh would change with them."""
    q, k, v, _ = _qkv(2, 8, 2, 3, 900, 128, dtype)
    other = _qkv(2, 16, 16, 1300, 300, 128, dtype, seed=1)
    outs = []
    for scale in (0.0, 40.0, 0.0):
        bitscom.attention(other[0] * scale, other[1], other[2], causal=False, softcap=30.0)
        outs.append(bitscom.attention(q * 0.5, k, v, softcap=30.0))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("cap", [1e-3, 1e-5, 1e-8, 1e-12])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64)], ids=str)
def test_caps_far_below_the_scores(cuda, dtype, d, cap):
    """Scores of +-cap: nearly even weights, and no gradient through the scores but where one is near zero."""
    for causal, ids in ((True, None), (True, torch.arange(200).div(70, rounding_mode="floor").repeat(2, 1))):
        q, k, v, do = _qkv(2, 4, 2, 200, 200, d, dtype, grad=True)
        out = bitscom.attention(q, k, v, causal=causal, documents=None if ids is None else ids.cuda(), softcap=cap)
        grads = torch.autograd.grad(out, (q, k, v), do)
        vals, bounds = reference(q, k, v, do, seen=visible(2, 200, 200, causal, ids), softcap=cap)
        # The gradient's factor 1 - tanh^2 of a score x is a step at x = 0, as wide as the cap: where the fp32 score's
        # rounding (below 2 d sum|q||k| 2^-24) can cross it, all of ds is open.
        check({"out": out, "dv": grads[2]}, vals, bounds)
        assert all(torch.isfinite(x).all() for x in grads[:2])


def test_caps_far_above_the_scores(cuda):
    """A cap that no score comes near changes nothing beyond rounding, up to the largest accepted."""
    q, k, v, do = _qkv(1, 4, 2, 200, 200, 64, torch.float16, grad=True)
    vals, bounds = reference(q, k, v, do, seen=visible(1, 200, 200, True))
    for cap in (1e6, 1e12, 1e25, 1e30):
        out = bitscom.attention(q, k, v, softcap=cap)
        grads = torch.autograd.grad(out, (q, k, v), do)
        check(dict(zip(("out", "dq", "dk", "dv"), (out, *grads))), vals, bounds)


def test_forward_mode_is_refused(cuda):
    """The operators have no forward-mode derivative: a dual input is refused, never taken as a constant."""
    q, k, v, t = _qkv(1, 2, 2, 20, 20, 64, torch.float16)
    freq = bitscom.rotary_frequencies(64, device="cuda")
    gain = torch.ones(64, device="cuda")
    slopes = torch.ones(2, device="cuda")
    with fwad.dual_level():
        dual = fwad.make_dual(q, t)
        bad = [
            lambda: bitscom.attention(dual, k, v),
            lambda: bitscom.attention(q, fwad.make_dual(k, t), v),
            lambda: bitscom.attention(q, k, fwad.make_dual(v, t), softcap=3.0),
            lambda: bitscom.attention(q, k, v, slopes=fwad.make_dual(slopes, slopes)),
            lambda: bitscom.attention(dual, k.detach().requires_grad_(True), v),
            lambda: bitscom.qk_norm_rotary(dual, k, freq),
            lambda: bitscom.qk_norm_rotary(q, fwad.make_dual(k, t), freq),
            lambda: bitscom.qk_norm_rotary(q, k, fwad.make_dual(freq, freq)),
            lambda: bitscom.qk_norm_rotary(q, k, freq, q_weight=fwad.make_dual(gain, gain)),
            lambda: bitscom.qk_norm_rotary(q, k, freq, k_weight=fwad.make_dual(gain, gain)),
        ]
        for call in bad:
            with torch.no_grad():
                with pytest.raises((NotImplementedError, ValueError)):
                    call()
            with pytest.raises((NotImplementedError, ValueError)):
                call()
        assert fwad.unpack_dual(bitscom.attention(q, k, v)).tangent is None
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda x: bitscom.attention(x, k, v), (q,), (t,))


@pytest.mark.parametrize("options", [dict(rotary=True), dict(distance_bias=True)], ids=str)
def test_training_after_inference_mode(cuda, options):
    """A first forward pass in inference mode leaves nothing behind that a training step cannot use."""
    torch.manual_seed(0)
    model = gpt2_small_test(vocab_size=64, n_positions=40, **options).cuda()
    idx = torch.randint(0, 64, (1, 30), device="cuda")
    ids = torch.zeros(1, 30, dtype=torch.int32, device="cuda")
    with torch.inference_mode():
        want = model(idx, documents=ids)
        mask = bitscom.attention_mask(ids.clone())
    out = model(idx, documents=ids)
    assert torch.equal(out, want)
    out.square().mean().backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
    q, k, v, do = _qkv(1, 2, 2, 30, 30, 64, torch.float16, grad=True)
    torch.autograd.grad(bitscom.attention(q, k, v, mask=mask), (q, k, v), do)


def test_slopes_of_any_stride(cuda):
    q, k, v, do = _qkv(1, 4, 2, 130, 130, 64, torch.float16, grad=True)
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    wide = torch.full((4, 3), 9.0, device="cuda")
    wide[:, 1] = slopes
    want = bitscom.attention(q, k, v, slopes=slopes)
    grads = torch.autograd.grad(want, (q, k, v), do)
    for given in (wide[:, 1], slopes.flip(0).contiguous().flip(0)):
        got = bitscom.attention(q, k, v, slopes=given)
        assert torch.equal(got, want)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, (q, k, v), do), grads))
    same = bitscom.attention(q, k, v, slopes=slopes[:1].expand(4))
    assert torch.equal(same, bitscom.attention(q, k, v, slopes=torch.full((4,), 0.5, device="cuda")))


def _traced_calls():
    freq = bitscom.rotary_frequencies(64, device="cuda")
    slopes = torch.tensor([0.5, 0.25], device="cuda")
    gain = torch.linspace(0.5, 1.5, 64, device="cuda")
    ids = torch.zeros(1, 150, dtype=torch.int32, device="cuda")
    ids[:, 70:] = 1
    return [
        lambda q, k, v: bitscom.attention(q, k, v, softcap=5.0, slopes=slopes),
        lambda q, k, v: bitscom.attention(q, k, v, documents=ids),
        lambda q, k, v: bitscom.qk_norm_rotary(q.transpose(1, 2), k.transpose(1, 2), freq, q_weight=gain)[0],
    ]


@pytest.mark.parametrize("which", range(3))
def test_traces_hold_the_kernels(cuda, which):
    """A trace replayed on other inputs computes them: torch.jit.trace, and make_fx without and with a backward pass."""
    f = _traced_calls()[which]
    a, b = (_qkv(1, 2, 2, 150, 150, 64, torch.float16, seed=s) for s in (0, 1))

    def with_grads(q, k, v, do):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = f(*leaves)
        g = torch.autograd.grad(out, leaves, do if out.shape == do.shape else do.transpose(1, 2), allow_unused=True)
        return (out.detach(), *(x for x in g if x is not None))

    traced = torch.jit.trace(f, a[:3], check_trace=False)
    torch.cuda.empty_cache()
    assert torch.equal(traced(*b[:3]), f(*b[:3]))
    graph = make_fx(f)(*a[:3])
    assert torch.equal(graph(*b[:3]), f(*b[:3]))
    for mode in ("real", "fake"):
        graph = make_fx(with_grads, tracing_mode=mode, _allow_non_fake_inputs=True)(*a)
        assert all(torch.equal(x, y) for x, y in zip(graph(*b), with_grads(*b)))


@pytest.mark.parametrize("options", [dict(rotary=True, softcap=5.0), dict(distance_bias=True)], ids=str)
def test_compiled_in_one_graph(cuda, options):
    torch.manual_seed(0)
    model = gpt2_small_test(vocab_size=64, n_positions=200, **options).cuda()
    idx = torch.randint(0, 64, (2, 150), device="cuda")
    ids = torch.arange(150, device="cuda").div(60, rounding_mode="floor").repeat(2, 1)

    def run(m):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out = m(idx, documents=ids)
        return [out.detach(), *torch.autograd.grad(out.float().square().mean(), list(model.parameters()))]

    want = run(model)
    torch._dynamo.reset()
    got = run(torch.compile(model, backend="aot_eager", fullgraph=True))
    # The same kernels on the same tensors; torch's embedding gradient adds with atomics.
    assert torch.equal(got[0], want[0])
    assert all(float((x - y).norm()) <= 1e-5 * float(y.norm()) for x, y in zip(got, want))


def test_function_transforms(cuda):
    """vmap runs the operators entry by entry; derivatives by transforms are refused."""
    q, k, v, _ = _qkv(3, 2, 2, 40, 40, 64, torch.float16)
    freq = bitscom.rotary_frequencies(64, device="cuda")
    each = [x[:, None] for x in (q, k, v)]
    assert torch.equal(torch.vmap(bitscom.attention)(*each)[:, 0], bitscom.attention(q, k, v))
    got = torch.vmap(lambda a, b: bitscom.qk_norm_rotary(a, b, freq))(*each[:2])
    assert all(torch.equal(x[:, 0], y) for x, y in zip(got, bitscom.qk_norm_rotary(q, k, freq)))
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda x: bitscom.attention(x, k, v).float().sum())(q)
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda x: bitscom.qk_norm_rotary(x, k, freq)[0].float().sum())(q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_score_gradients_do_not_see_the_outputs_rounding(cuda, dtype, d):
    """delta = do.o takes o as it was before its rounding.

    Queries of zero make every weight 1/16, which no type rounds, and values near 8 make o.do large beside
    do.(v - o), so that half a step of o in delta would show.  Left are: ds rounded once, o kept in two values of
    the type (a half step of a half step), and fp32 sums of d and 16 terms, at most (2 * 16 + d + 16) roundings of 2^-24
    of sum |do| |v|.  Each goes into dq with weight |k|, and dq is rounded once.
    """
    u, sk = torch.finfo(dtype).eps / 2, 16
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.zeros(1, 2, 200, d, device="cuda", dtype=dtype, requires_grad=True)
    k, v = ((m + f * torch.randn(1, 2, sk, d, generator=g, device="cuda")).to(dtype) for m, f in ((1, 0.1), (8, 0.25)))
    do = torch.randn(1, 2, 200, d, generator=g, device="cuda").to(dtype)
    (dq,) = torch.autograd.grad(bitscom.attention(q, k, v, causal=False), q, do)
    kd, vd, dod = (x.double() for x in (k, v, do))
    o = vd.mean(2, keepdim=True)
    ds = (dod @ (vd - o).transpose(-1, -2)) / sk
    want = ds @ kd * d ** -0.5
    ado = (dod.abs() @ vd.abs().transpose(-1, -2)) / sk
    e = 2.0 ** -24 * (2 * sk + d + 16)
    step = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half of fp16's smallest step
    bound = ((u + e) * ds.abs() + (u * u + e) * ado + step) @ kd.abs() * d ** -0.5 + u * want.abs() + step
    assert ((dq.double() - want).abs() <= 1.05 * bound).all()
    # A delta from the rounded output is beyond it: the test can tell.
    off = ((o.to(dtype).double() - o) * dod).sum(-1, keepdim=True) / sk
    assert ((off * kd.sum(2, keepdim=True) * d ** -0.5).abs() > 1.05 * bound).any()


@pytest.mark.parametrize("sq,sk", [(1, 300), (3, 2600), (17, 1100)])
@pytest.mark.parametrize("heads", [(8, 2), (6, 6)], ids=str)
def test_few_queries_over_packed_documents(cuda, heads, sq, sk):
    """Shared heads in one tile and key splits, with documents, padding on the left and prefixes."""
    ids = torch.zeros(2, sk, dtype=torch.int32)
    ids[0, : sk // 3] = -1
    ids[1, sk - 2 :] = 4  # the last queries are alone, the first of 17 see the long document
    for d, dtype, cap in ((64, torch.bfloat16, None), (128, torch.float16, 20.0), (128, torch.bfloat16, None)):
        q, k, v, do = _qkv(2, *heads, sq, sk, d, dtype, seed=sk)
        for prefix in (None, torch.tensor([sk // 2, sk])):
            out = bitscom.attention(q, k, v, documents=ids.cuda(), prefix=None if prefix is None else prefix.cuda(), softcap=cap)
            vals, bounds = reference(q, k, v, do, seen=visible(2, sq, sk, True, ids, prefix), softcap=cap)
            check({"out": out}, vals, bounds)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=str)
def test_saved_tensors_may_come_back_elsewhere(cuda, dtype):
    """Hooks that hand saved tensors back with other strides, or off their alignment, change nothing."""
    q, k, v, do = _qkv(2, 4, 2, 150, 150, 64, dtype, grad=True)
    ids = torch.arange(150, device="cuda").div(60, rounding_mode="floor").int().repeat(2, 1)
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    out = bitscom.attention(q, k, v, documents=ids, slopes=slopes)
    want = torch.autograd.grad(out, (q, k, v), do)

    def moved(t):  # one element further in memory
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)

    def reordered(t):  # dimensions in the reverse order, the last one too
        return t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim())))

    count = [0]

    def in_turn(t):
        count[0] += 1
        return (moved, reordered, torch.clone)[count[0] % 3](t)

    for unpack in (moved, reordered, in_turn, in_turn):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            out = bitscom.attention(q, k, v, documents=ids, slopes=slopes)
        assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(out, (q, k, v), do), want))
