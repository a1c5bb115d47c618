"""Attention operators on the GPU against the 64-bit oracle, with bounds that
count roundings (attention_oracle.py).  Needs a CUDA device."""

import pytest
import torch

import bitscom_b200 as bitscom
from bitscom_b200 import _ext

from .attention_oracle import check, reference, rotary_reference, visible

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _tensors(b, h, hk, sq, sk, d, dtype, seed=0, scale=1.0, grad=True):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def new(heads, s, f=1.0):
        return (torch.randn(b, s, heads, d, generator=g, device="cuda") * f).to(dtype).transpose(1, 2)

    q, k, v, do = new(h, sq, scale), new(hk, sk, scale), new(hk, sk), new(h, sq)
    if grad:
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    return q, k, v, do


def _documents(b, sk, n, pad, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.zeros(b, sk, dtype=torch.int32)
    for i in range(b):
        cuts = torch.sort(torch.randint(0, sk, (n - 1,), generator=g))[0].tolist()
        for m, c in enumerate(cuts):
            ids[i, c:] = m + 1
        if pad:
            ids[i, sk - max(1, sk // 5):] = -1
            ids[i, sk // 3 : sk // 3 + 3] = -7
    return ids


def _mask_args(kind, b, sk, seed=0):
    """(causal, documents, prefix) of a named mask."""
    docs = prefix = None
    if "docs" in kind:
        docs = _documents(b, sk, 4, "pad" in kind, seed)
    if "prefix" in kind:
        prefix = torch.tensor([(37 * (i + 1)) % (sk + 1) for i in range(b)], dtype=torch.int64)
    return "full" not in kind, docs, prefix


def _run(q, k, v, do, causal, docs, prefix, **kw):
    out = bitscom.attention(q, k, v, causal=causal, documents=None if docs is None else docs.cuda(),
                            prefix=None if prefix is None else prefix.cuda(), **kw)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    assert out.dtype == dq.dtype == dk.dtype == dv.dtype == q.dtype
    assert out.shape == dq.shape == q.shape and dk.shape == dv.shape == k.shape
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _compare(shape, dtype, kind, softcap=None, slopes=None, scale=1.0, seed=0):
    b, h, hk, sq, sk, d = shape
    q, k, v, do = _tensors(*shape, dtype, seed, scale)
    causal, docs, prefix = _mask_args(kind, b, sk, seed)
    sl = None if not slopes else 0.5 ** torch.arange(1, h + 1, device="cuda", dtype=torch.float32)
    got = _run(q, k, v, do, causal, docs, prefix, softcap=softcap, slopes=sl)
    vals, bounds = reference(q, k, v, do, seen=visible(b, sq, sk, causal, docs, prefix), softcap=softcap, slopes=sl)
    check(got, vals, bounds)


SHAPES = [
    (1, 1, 1, 1, 1, 8),          # one token, one key
    (2, 4, 2, 1, 5, 64),         # fewer keys than a tile
    (2, 4, 4, 127, 127, 64),     # a tile less one
    (1, 4, 4, 129, 129, 64),     # a tile and one
    (2, 6, 2, 77, 203, 80),      # a chunk over a longer cache, width between the tiles
    (1, 2, 1, 256, 256, 128),
    (1, 2, 2, 300, 17, 64),      # more queries than keys: rows that see nothing under a causal mask
    (3, 3, 1, 130, 1000, 40),
    (1, 8, 2, 515, 515, 96),
    (1, 2, 2, 70, 70, 256),      # wider than the tensor-core tiles
    (2, 2, 1, 65, 190, 36),      # width that is not a multiple of 8
]
MASKS = ["causal", "full", "docs causal", "docs pad causal", "docs pad full", "prefix causal", "docs pad prefix causal"]


@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_matches_64_bits(cuda, shape, kind):
    _compare(shape, torch.bfloat16, kind)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("scores", ["plain", "capped", "distance", "both"])
@pytest.mark.parametrize("shape", [(2, 4, 2, 193, 193, 64), (1, 4, 1, 140, 300, 128)], ids=str)
def test_scores_and_types(cuda, shape, scores, dtype):
    _compare(shape, dtype, "docs causal", softcap=5.0 if scores in ("capped", "both") else None,
             slopes=scores in ("distance", "both"), scale=2.0, seed=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_distance_counts_both_ways(cuda, dtype):
    _compare((1, 4, 4, 150, 260, 64), dtype, "full", slopes=True, seed=5)
    _compare((1, 4, 4, 150, 260, 64), dtype, "prefix causal", slopes=True, softcap=3.0, seed=6)


@pytest.mark.parametrize("d", [8, 16, 24, 48, 56, 64, 72, 104, 112, 120, 128])
def test_head_sizes(cuda, d):
    _compare((1, 2, 1, 150, 150, d), torch.float16, "causal", seed=d)


@pytest.mark.parametrize("sq,sk", [(1, 1), (1, 2), (1, 64), (1, 127), (1, 128), (1, 129), (1, 4097), (2, 9000), (3, 1025),
                                   (5, 640), (17, 2500), (128, 3000), (129, 2049)])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (7, 1)], ids=str)
def test_few_queries_over_many_keys(cuda, heads, sq, sk):
    h, hk = heads
    for d, dtype, cap in ((64, torch.bfloat16, None), (128, torch.float16, 20.0)):
        q, k, v, do = _tensors(2, h, hk, sq, sk, d, dtype, seed=sk, grad=False)
        sl = 0.5 ** torch.arange(1, h + 1, device="cuda", dtype=torch.float32)
        for slopes in (None, sl):
            out = bitscom.attention(q, k, v, softcap=cap, slopes=slopes)
            vals, bounds = reference(q, k, v, do, seen=visible(1, sq, sk, True), softcap=cap, slopes=slopes)
            check({"out": out}, vals, bounds)


def test_documents_across_many_tiles(cuda):
    """Documents that span, start and end on tiles; one id used twice is two documents."""
    b, s = 2, 1200
    ids = torch.zeros(b, s, dtype=torch.int64)
    for i, (a, e) in enumerate([(0, 128), (128, 256), (256, 900), (900, 901), (901, 1100), (1100, 1200)]):
        ids[0, a:e] = i % 2
    ids[1, 640:] = 5
    q, k, v, do = _tensors(b, 2, 2, s, s, 64, torch.float16)
    for causal in (True, False):
        got = _run(q, k, v, do, causal, ids, None)
        vals, bounds = reference(q, k, v, do, seen=visible(b, s, s, causal, ids))
        check(got, vals, bounds)


def test_large_scores(cuda):
    """Scores of hundreds, where a softmax without its running maximum overflows."""
    _compare((1, 2, 2, 200, 200, 64), torch.bfloat16, "causal", scale=12.0)
    _compare((1, 2, 2, 200, 200, 128), torch.float16, "causal", scale=9.0, softcap=30.0)


def test_rising_scores_rescale_the_output(cuda):
    """Later keys score higher by far: the running maximum moves in every tile."""
    q, k, v, do = _tensors(1, 2, 2, 130, 700, 64, torch.float16, grad=False)
    q = q.abs()
    k = (torch.linspace(-12, 12, 700, device="cuda")[None, None, :, None] + 0.1 * k.float()).half()
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    for causal in (True, False):
        got = _run(q, k, v, do, causal, None, None)
        vals, bounds = reference(q, k, v, do, seen=visible(1, 130, 700, causal))
        check(got, vals, bounds)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64)], ids=str)
def test_padding_may_hold_anything(cuda, dtype, d):
    """NaN and infinities where documents < 0: in keys, values, queries and output gradients."""
    shape = (2, 4, 2, 300, 300, d)
    q, k, v, do = _tensors(*shape, dtype)
    ids = _documents(2, 300, 3, True)
    vals, bounds = reference(q, k, v, do, seen=visible(2, 300, 300, True, ids))
    bad = (ids < 0).cuda()
    qs, ks, vs, dos = (x.detach().clone() for x in (q, k, v, do))
    for x, val in ((qs, float("nan")), (ks, float("inf")), (vs, float("nan")), (dos, float("-inf"))):
        x.transpose(1, 2)[bad] = val
    qs, ks, vs = (x.requires_grad_(True) for x in (qs, ks, vs))
    got = _run(qs, ks, vs, dos, True, ids, None)
    check(got, vals, bounds)
    for name in ("out", "dq", "dk", "dv"):
        assert (got[name].transpose(1, 2)[bad] == 0).all(), name


def test_rows_without_keys_are_zero(cuda):
    """More queries than keys under a causal mask, whatever the queries hold."""
    q, k, v, do = _tensors(1, 2, 2, 200, 60, 64, torch.bfloat16, grad=False)
    vals, bounds = reference(q, k, v, do, seen=visible(1, 200, 60, True))
    q[:, :, :140] = float("nan")
    do[:, :, :140] = float("inf")
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    got = _run(q, k, v, do, True, None, None)
    assert (got["out"][:, :, :140] == 0).all() and (got["dq"][:, :, :140] == 0).all()
    check(got, vals, bounds)


def test_all_padding(cuda):
    q, k, v, do = _tensors(1, 2, 2, 70, 70, 64, torch.float16)
    got = _run(q, k, v, do, True, torch.full((1, 70), -1), None)
    for x in got.values():
        assert (x == 0).all()


@pytest.mark.parametrize("sq,sk,b", [(0, 5, 1), (5, 0, 1), (0, 0, 1), (3, 3, 0)])
def test_empty_tensors(cuda, sq, sk, b):
    q, k, v, do = _tensors(b, 2, 1, sq, sk, 64, torch.bfloat16)
    for kw in ({}, {"documents": torch.zeros(b, sk, dtype=torch.int32, device="cuda")}):
        out = bitscom.attention(q, k, v, **kw)
        grads = torch.autograd.grad(out, (q, k, v), do)
        assert out.shape == q.shape and (out == 0).all()
        assert all((x == 0).all() for x in grads)


def test_strides(cuda):
    """Views of a joint projection, head-major copies, shared heads by expand, a reversed order of dimensions, odd
    offsets and gradients without strides give the bits of contiguous tensors."""
    b, h, s, d = 2, 4, 150, 64
    joint = torch.randn(b, s, 3 * h * d, device="cuda").half()
    views = [x.view(b, s, h, d).transpose(1, 2) for x in joint.split(h * d, dim=2)]
    want = bitscom.attention(*[x.contiguous() for x in views])
    assert torch.equal(bitscom.attention(*views), want)
    last = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in views]
    assert last[0].stride(3) != 1 and torch.equal(bitscom.attention(*last), want)
    for pad in (1, 4, 8):  # rows that start off 16-byte boundaries, and a row pitch that is none
        wide = [torch.zeros(b, h, s, d + 2 * pad, device="cuda", dtype=torch.half) for _ in range(3)]
        for w, x in zip(wide, views):
            w[..., pad : pad + d] = x
        assert torch.equal(bitscom.attention(*[w[..., pad : pad + d] for w in wide]), want)
    one = [views[0], *(x[:, :1].expand(b, h, s, d) for x in views[1:])]
    assert torch.equal(bitscom.attention(*one), bitscom.attention(*[x.contiguous() for x in one]))
    batch = [x[:1].expand(b, h, s, d) for x in views]
    assert torch.equal(bitscom.attention(*batch)[0], bitscom.attention(*[x[:1] for x in views])[0])
    leaves = [x.detach().requires_grad_(True) for x in views]
    a = torch.autograd.grad(bitscom.attention(*leaves).sum(), leaves)
    c = torch.autograd.grad(bitscom.attention(*leaves), leaves, torch.ones_like(want))
    assert all(torch.equal(x, y) for x, y in zip(a, c))


def test_same_bits_every_time(cuda):
    q, k, v, do = _tensors(2, 8, 2, 700, 700, 64, torch.bfloat16)
    ids = _documents(2, 700, 5, True)
    a, c = (_run(q, k, v, do, True, ids, None, softcap=9.0) for _ in range(2))
    assert all(torch.equal(a[n], c[n]) for n in a)


def test_batch_entries_are_independent(cuda):
    q, k, v, do = _tensors(3, 4, 2, 333, 333, 64, torch.float16)
    all3 = _run(q, k, v, do, True, None, None)
    for i in range(3):
        leaves = [x[i : i + 1].detach().requires_grad_(True) for x in (q, k, v)]
        one = _run(*leaves, do[i : i + 1], True, None, None)
        assert all(torch.equal(one[n][0], all3[n][i]) for n in one)


def test_mask_is_reused(cuda):
    q, k, v, do = _tensors(2, 4, 4, 260, 260, 64, torch.float16)
    ids = _documents(2, 260, 4, True).cuda()
    want = bitscom.attention(q, k, v, documents=ids)
    mask = bitscom.attention_mask(ids)
    ids.zero_()  # the mask keeps what it was built from
    assert torch.equal(bitscom.attention(q, k, v, mask=mask), want)
    assert torch.equal(bitscom.attention(q, k, v, mask=mask), want)


def test_mask_of_long_documents(cuda):
    """Runs that reach over many tiles on both sides, strided and 64-bit ids."""
    for s in (513, 5000):
        wide = torch.zeros(1, 2 * s, dtype=torch.int64, device="cuda")
        ids = wide[:, ::2]
        ids[:, s - 3 :] = 4
        q, k, v, do = _tensors(1, 1, 1, s, s, 64, torch.float16)
        for causal in (True, False):
            got = _run(q, k, v, do, causal, ids, None)
            vals, bounds = reference(q, k, v, do, seen=visible(1, s, s, causal, ids.cpu()))
            check(got, vals, bounds)


def test_runs_on_the_current_stream(cuda):
    q, k, v, do = _tensors(2, 4, 4, 400, 400, 64, torch.bfloat16)
    ids = _documents(2, 400, 3, False)
    want = _run(q, k, v, do, True, ids, None)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s in streams:  # two calls at once
        with torch.cuda.stream(s):
            got.append(_run(q, k, v, do, True, ids, None))
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(one[n], want[n]) for n in want)


@pytest.mark.parametrize("shape", [(2, 4, 2, 300, 300, 64), (1, 4, 1, 1, 5000, 128)], ids=str)
def test_captured_and_replayed(cuda, shape):
    """Two graphs of one call replayed in turn on changing inputs, forward and backward."""
    q, k, v, do = _tensors(*shape, torch.bfloat16)
    ids = torch.zeros(shape[0], shape[4], dtype=torch.int32, device="cuda")
    ids[:, shape[4] // 2 :] = 1

    def step():
        out = bitscom.attention(q, k, v, documents=ids, softcap=11.0)
        return (out, *torch.autograd.grad(out, (q, k, v), do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (1, 2):
        fresh = _tensors(*shape, torch.bfloat16, seed=seed, grad=False)
        with torch.no_grad():
            for x, y in zip((q, k, v, do), fresh):
                x.copy_(y)
        for g in graphs:
            g.replay()
        want = step()
        torch.cuda.synchronize()
        for got in outs:
            assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_gradients_against_differences(cuda):
    """fp32: directional derivatives by central differences, error h^2 and rounding 2^-24 / h balanced at h = 2^-8."""
    q, k, v, do = _tensors(1, 4, 2, 90, 90, 32, torch.float32)
    sl = torch.tensor([0.3, 0.1, 0.03, 0.01], device="cuda")
    kw = dict(documents=_documents(1, 90, 3, True).cuda(), softcap=2.0, slopes=sl)
    out = bitscom.attention(q, k, v, **kw)
    grads = torch.autograd.grad(out, (q, k, v), do)
    h = 2.0 ** -8
    for i, x in enumerate((q, k, v)):
        way = torch.randn_like(x)
        way /= way.norm()
        args = [t.detach() for t in (q, k, v)]

        def loss(f):
            moved = [t + f * way if j == i else t for j, t in enumerate(args)]
            return (bitscom.attention(*moved, **kw).double() * do.double()).sum()

        slope = float((loss(h) - loss(-h)) / (2 * h))
        # The third derivative along a unit vector is below 10 |do|; out carries about 2^-22 |do| |out|.
        norm = float(do.norm())
        assert abs(slope - float((grads[i].double() * way.double()).sum())) < norm * (10 * h * h + 2.0 ** -18 / h)


def test_only_some_gradients(cuda):
    q, k, v, do = _tensors(1, 2, 2, 100, 100, 64, torch.float16)
    full = _run(q, k, v, do, True, None, None)
    for keep, name in ((0, "dq"), (1, "dk"), (2, "dv")):
        leaves = [x.detach().requires_grad_(i == keep) for i, x in enumerate((q, k, v))]
        (got,) = torch.autograd.grad(bitscom.attention(*leaves), [leaves[keep]], do)
        assert torch.equal(got, full[name])
    with torch.no_grad():
        assert torch.equal(bitscom.attention(q, k, v), full["out"])


def test_autocast_and_wide_gradient(cuda):
    q, k, v, do = _tensors(1, 2, 2, 64, 64, 64, torch.float32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = bitscom.attention(q, k, v)
    assert out.dtype == torch.bfloat16
    (out.float() * do).sum().backward()
    assert q.grad.dtype == torch.float32
    assert torch.equal(out, bitscom.attention(q.bfloat16(), k.bfloat16(), v.bfloat16()))


def test_double_backward_is_refused(cuda):
    q, k, v, do = _tensors(1, 1, 1, 8, 8, 64, torch.float32)
    (dq,) = torch.autograd.grad(bitscom.attention(q, k, v).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.sum().backward()


def test_refusals(cuda):
    q, k, v, _ = _tensors(2, 4, 2, 10, 10, 64, torch.float16, grad=False)
    bad = [
        (ValueError, lambda: bitscom.attention(q[0], k, v)),
        (ValueError, lambda: bitscom.attention(q, k, v[:, :, :5])),
        (ValueError, lambda: bitscom.attention(q[:, :3], k, v)),
        (ValueError, lambda: bitscom.attention(q[:1], k, v)),
        (ValueError, lambda: bitscom.attention(q, k.cpu(), v)),
        (ValueError, lambda: bitscom.attention(q[..., :32], k, v)),
        (TypeError, lambda: bitscom.attention(q, k.float(), v)),
        (TypeError, lambda: bitscom.attention(q.double(), k.double(), v.double())),
        (ValueError, lambda: bitscom.attention(*[torch.zeros(1, 1, 4, 257, device="cuda")] * 3)),
        (ValueError, lambda: bitscom.attention(q, k, v, softcap=0.0)),
        (ValueError, lambda: bitscom.attention(q, k, v, softcap=float("nan"))),
        (ValueError, lambda: bitscom.attention(q, k, v, slopes=torch.ones(3, device="cuda"))),
        (ValueError, lambda: bitscom.attention(q, k, v, slopes=torch.ones(4))),
        (TypeError, lambda: bitscom.attention(q, k, v, slopes=torch.ones(4, device="cuda").half())),
        (ValueError, lambda: bitscom.attention(q, k, v, slopes=torch.ones(4, device="cuda", requires_grad=True))),
        (ValueError, lambda: bitscom.attention(q, k, v, documents=torch.zeros(2, 9, dtype=torch.int32, device="cuda"))),
        (ValueError, lambda: bitscom.attention(q, k, v, documents=torch.zeros(1, 10, dtype=torch.int32, device="cuda"))),
        (ValueError, lambda: bitscom.attention(q, k, v, documents=torch.zeros(2, 10, dtype=torch.int32))),
        (TypeError, lambda: bitscom.attention(q, k, v, documents=torch.zeros(2, 10, device="cuda"))),
        (ValueError, lambda: bitscom.attention(q, k, v, causal=False, prefix=torch.zeros(2, dtype=torch.int32, device="cuda"))),
        (ValueError, lambda: bitscom.attention(q, k, v, prefix=torch.zeros(3, dtype=torch.int32, device="cuda"))),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    mask = bitscom.attention_mask(torch.zeros(2, 10, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        bitscom.attention(q[:, :, :5], k, v, mask=mask)
    with pytest.raises(ValueError):
        bitscom.attention(q, k, v, mask=mask, documents=torch.zeros(2, 10, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        bitscom.attention(q.cpu(), k.cpu(), v.cpu(), mask=mask)
    assert torch.isfinite(bitscom.attention(q, k, v)).all()  # nothing was left broken


# --- norm and rotation -----------------------------------------------------------------------------------------------


def _rotary_case(b, s, h, hk, d, r, dtype, *, interleaved=False, start=0, weights=True, seed=0, positions="rows"):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dt=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    joint = randn(b, s, (h + 2 * hk) * d, dt=dtype)
    q = joint[..., : h * d].view(b, s, h, d).detach().requires_grad_(True)
    k = joint[..., h * d : (h + hk) * d].view(b, s, hk, d).detach().requires_grad_(True)
    wq = wk = None
    if weights:
        wq, wk = ((1 + 0.2 * randn(d)).requires_grad_(True) for _ in range(2))
    pos = torch.arange(s, device="cuda") + start
    if positions == "rows":
        pos = torch.stack([pos + 3 * i for i in range(b)]) if b else pos.view(1, s)[:0]
    freq = bitscom.rotary_frequencies(r, device="cuda") if r else torch.empty(0, dtype=torch.float64, device="cuda")
    gq, gk = randn(b, s, h, d, dt=dtype), randn(b, s, hk, d, dt=dtype)
    oq, ok = bitscom.qk_norm_rotary(q, k, freq, q_weight=wq, k_weight=wk, positions=pos, eps=1e-5, interleaved=interleaved)
    leaves = [q, k] + ([wq, wk] if weights else [])
    grads = torch.autograd.grad((oq, ok), leaves, (gq, gk))
    u = torch.finfo(dtype).eps / 2
    for x, w, y, dy, dx, dw in ((q, wq, oq, gq, grads[0], grads[2] if weights else None),
                                (k, wk, ok, gk, grads[1], grads[3] if weights else None)):
        assert y.dtype == dx.dtype == dtype and y.is_contiguous() and y.shape == x.shape
        wy, wdx, wdw = rotary_reference(x, w, freq, pos, 1e-5, interleaved, dy)
        # y: at most three fp32 products and a sum per value of size |pair|, the norm over d terms, then one rounding.
        f32 = 2.0 ** -24
        size = wy.abs().amax(-1, keepdim=True) * 2
        assert ((y.double() - wy).abs() <= u * wy.abs() + (d + 16) * f32 * size + torch.finfo(dtype).tiny).all()
        rs = torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-5)
        wmax = 1.0 if w is None else float(w.detach().abs().max())
        size = rs * wmax * (dy.double().norm(dim=-1, keepdim=True) * (2 + x.double().abs() * rs))
        assert ((dx.double() - wdx).abs() <= u * wdx.abs() + (d + 16) * f32 * size + torch.finfo(dtype).tiny).all()
        if w is not None:
            n = (x.double().abs() * rs).flatten(0, 2)
            pair = dy.double().norm(dim=-1, keepdim=True).expand(dy.shape).flatten(0, 2)
            terms = b * s * x.shape[2]
            # Sums of `terms` products in fp32; partial sums of about 64 to 600 bound the growth far below `terms`.
            bound = f32 * (n * pair).sum(0) * (min(terms, 1200) + d)
            assert dw.dtype == w.dtype and ((dw.double() - wdw).abs() <= bound + 1e-30).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", [
    (1, 1, 1, 1, 64, 64), (2, 7, 4, 2, 64, 32), (3, 50, 3, 1, 80, 40), (1, 129, 6, 2, 128, 128), (2, 33, 2, 2, 40, 20),
    (1, 17, 2, 1, 256, 256), (1, 9, 2, 1, 256, 100), (2, 5, 3, 3, 6, 2), (1, 40, 4, 4, 96, 0), (1, 3, 1, 1, 1, 0),
    (1, 600, 12, 4, 64, 64), (2, 31, 1, 1, 30, 30)], ids=str)
def test_rotary_matches_64_bits(cuda, case, dtype):
    for interleaved in (False, True):
        _rotary_case(*case, dtype, interleaved=interleaved, seed=case[1])


def test_rotary_far_positions_and_options(cuda):
    _rotary_case(1, 300, 4, 2, 128, 128, torch.float32, start=1_000_003)
    _rotary_case(1, 20, 4, 2, 64, 64, torch.float32, start=2**31 - 30)
    _rotary_case(1, 20, 4, 2, 64, 64, torch.float32, start=-50)
    _rotary_case(2, 60, 4, 2, 64, 64, torch.bfloat16, weights=False)
    _rotary_case(2, 60, 4, 2, 64, 64, torch.bfloat16, positions="shared")


def test_rotary_defaults_and_strides(cuda):
    q = torch.randn(2, 21, 3, 64, device="cuda")
    k = torch.randn(2, 21, 1, 64, device="cuda")
    freq = bitscom.rotary_frequencies(64, device="cuda")
    want = bitscom.qk_norm_rotary(q, k, freq)
    pos = torch.arange(21, device="cuda", dtype=torch.int32)
    for p in (pos, pos.long(), pos.expand(2, 21), torch.stack([pos, pos], 1).reshape(-1)[::2]):
        got = bitscom.qk_norm_rotary(q, k, freq, positions=p)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    odd = torch.empty(2 * 21 * 3 * 64 + 1, device="cuda")[1:].view(2, 21, 3, 64).copy_(q)
    got = bitscom.qk_norm_rotary(odd, k.transpose(2, 3).contiguous().transpose(2, 3), freq)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(bitscom.qk_norm_rotary(heads_first, k, freq)[0], want[0])


def test_rotary_same_bits_streams_and_graphs(cuda):
    q = torch.randn(2, 500, 8, 64, device="cuda").bfloat16().requires_grad_(True)
    k = torch.randn(2, 500, 2, 64, device="cuda").bfloat16().requires_grad_(True)
    w = torch.rand(64, device="cuda").add(0.5).requires_grad_(True)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    freq = bitscom.rotary_frequencies(64, device="cuda")

    def step():  # detached: torch refuses to capture a backward pass while an eager graph of its leaves lives
        out = bitscom.qk_norm_rotary(q, k, freq, q_weight=w, k_weight=w)
        return (*(x.detach() for x in out), *torch.autograd.grad(out, (q, k, w), (gq, gk)))

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rotary_empty_and_refusals(cuda):
    freq = bitscom.rotary_frequencies(64, device="cuda")
    q, k = torch.zeros(1, 0, 4, 64, device="cuda", requires_grad=True), torch.zeros(1, 0, 2, 64, device="cuda")
    w = torch.ones(64, device="cuda", requires_grad=True)
    out = bitscom.qk_norm_rotary(q, k, freq, q_weight=w)
    assert out[0].shape == q.shape
    assert (torch.autograd.grad(out[0].sum(), w)[0] == 0).all()
    q, k = torch.randn(2, 5, 4, 64, device="cuda"), torch.randn(2, 5, 2, 64, device="cuda")
    f = bitscom.qk_norm_rotary
    bad = [
        (ValueError, lambda: f(q[0], k, freq)),
        (ValueError, lambda: f(q, k[:, :4], freq)),
        (ValueError, lambda: f(q, k[..., :32], freq)),
        (TypeError, lambda: f(q, k.half(), freq)),
        (TypeError, lambda: f(q.double(), k.double(), freq)),
        (ValueError, lambda: f(q, k.cpu(), freq)),
        (ValueError, lambda: f(q, k, freq.cpu())),
        (TypeError, lambda: f(q, k, freq.long())),
        (ValueError, lambda: f(q, k, bitscom.rotary_frequencies(66, device="cuda"))),
        (ValueError, lambda: f(q, k, freq.clone().requires_grad_(True))),
        (ValueError, lambda: f(q, k, freq, q_weight=torch.ones(32, device="cuda"))),
        (TypeError, lambda: f(q, k, freq, q_weight=torch.ones(64, device="cuda", dtype=torch.int32))),
        (ValueError, lambda: f(q, k, freq, positions=torch.zeros(4, dtype=torch.int32, device="cuda"))),
        (ValueError, lambda: f(q, k, freq, positions=torch.zeros(1, 5, dtype=torch.int32, device="cuda"))),
        (TypeError, lambda: f(q, k, freq, positions=torch.zeros(5, device="cuda"))),
        (ValueError, lambda: f(*[torch.zeros(1, 1, 1, 257, device="cuda")] * 2, freq)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_extension_runs_the_operators(cuda):
    assert _ext.available() and hasattr(_ext._C, "attention_forward")


def test_no_wait_ran_out(cuda):
    """Every wait of the tensor-core kernels is bounded; none of this file's calls reached the bound."""
    torch.cuda.synchronize()
    assert _ext._C.attention_status() == 0
