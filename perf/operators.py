"""What the attention operators are measured on.

Two operators of a GPT-style attention block: ``attention`` (score cap, distance
bias, documents packed into rows, prefix masks; both directions and the form for
a few queries over a long cache) and ``qk_norm_rotary`` (norm of every query and
key head with the position rotation in the same pass; both directions).

A case is a dict of plain values; ``prepare`` makes its inputs from a seed,
``run`` computes it (in elementary torch operations, or through bitscom_b200
where ``own`` is true), ``exact`` computes it in 64 bits.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _attention(name, dtype, batch, heads, kv_heads, q_len, k_len, dim, *, causal=True, documents=0, padded=False,
               prefix=False, cap=0.0, bias=False, backward=False):
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "q_len": q_len, "k_len": k_len, "dim": dim, "causal": causal, "documents": documents, "padded": padded,
            "prefix": prefix, "cap": cap, "bias": bias, "backward": backward}


def _rotary(name, dtype, batch, seq, heads, kv_heads, dim, rotated, *, start=0, interleaved=False, backward=False):
    return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "seq": seq, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rotated": rotated, "start": start, "interleaved": interleaved,
            "backward": backward}


def listed():
    return [
        # The next token of one short answer, in the width of the small GPT-2: latency alone counts.
        _attention("one token, short cache", "bf16", 1, 4, 4, 1, 129, 64),
        # The next tokens of eight long answers with shared key heads: the cache is read once.
        _attention("one token, long cache", "fp16", 8, 16, 4, 1, 32768, 128, cap=30.0),
        # One layer of a GPT-2 medium training step on rows of packed documents.
        _attention("packed documents, training", "bf16", 8, 16, 16, 1024, 1024, 64, documents=5, padded=True,
                   backward=True),
        # One layer of the small GPT-2 on prompts that see themselves whole; an odd length.
        _attention("prefix, odd length, training", "fp16", 4, 4, 4, 509, 509, 64, prefix=True, backward=True),
        # A long row, capped scores, shared key heads: the largest work.
        _attention("capped, long row, training", "bf16", 1, 16, 4, 8192, 8192, 128, cap=50.0, backward=True),
        # Reading prompts with a distance bias in place of learned positions.
        _attention("distance bias, prompt", "fp16", 2, 16, 16, 4096, 4096, 64, bias=True),
        # Ragged everything: a chunk of queries over a longer cache, a head width between the tiles.
        _attention("ragged chunk, training", "bf16", 2, 6, 2, 777, 1531, 80, cap=20.0, bias=True, documents=3,
                   backward=True),
        # The same eight answers' queries and keys of the next token.
        _rotary("norm and rotation, one token", "bf16", 8, 1, 16, 4, 128, 128, start=32767),
        # One layer of a GPT-2 medium training step, queries and keys inside the joint projection.
        _rotary("norm and rotation, training", "bf16", 8, 1024, 16, 16, 64, 64, backward=True),
        # A long row far from the first position, where an angle in 32 bits would be lost.
        _rotary("norm and rotation, far positions", "fp16", 1, 131072, 16, 4, 128, 128, start=1000003),
        # Full precision, odd sizes, half of each head rotated in neighbouring pairs.
        _rotary("norm and rotation, odd, training", "fp32", 3, 1237, 6, 2, 80, 40, interleaved=True, backward=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.35:
        dim = 8 * rng.randint(4, 16)
        rotated = dim if rng.random() < 0.6 else max(8, dim // 2 // 2 * 2)
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4])
        seq = 1 if rng.random() < 0.2 else _log_int(rng, 2, 16384)
        return {k: v for k, v in _rotary("", rng.choice(["bf16", "fp16", "fp32"]), rng.randint(1, 4), seq, heads, kv, dim,
                                         rotated, start=rng.choice([0, 17, 70001, 1000003]),
                                         interleaved=rng.random() < 0.3, backward=rng.random() < 0.5).items()
                if k != "name"}
    dim = rng.choice([64, 64, 128, 8 * rng.randint(4, 16)])
    kv = rng.choice([1, 2, 4])
    heads = kv * rng.choice([1, 2, 4])
    backward = rng.random() < 0.6
    few = not backward and rng.random() < 0.5
    k_len = _log_int(rng, 1000, 40000) if few else _log_int(rng, 16, 3000)
    q_len = rng.choice([1, 1, 2, 5]) if few else (k_len if rng.random() < 0.6 else rng.randint(1, k_len))
    batch = rng.randint(1, 6)
    causal = rng.random() < 0.75
    documents = rng.randint(2, 9) if not few and rng.random() < 0.4 else 0
    return {k: v for k, v in _attention("", rng.choice(["bf16", "fp16"]), batch, heads, kv, q_len, k_len, dim,
                                        causal=causal, documents=documents,
                                        padded=documents > 0 and rng.random() < 0.5,
                                        prefix=causal and not few and rng.random() < 0.3,
                                        cap=rng.choice([0.0, 0.0, 15.0, 50.0]), bias=rng.random() < 0.3,
                                        backward=backward).items() if k != "name"}


# --- inputs ----------------------------------------------------------------------------------------------------------


def _lengths(case):
    """Document lengths of a row (summing to k_len, the last being padding if `padded`), from the case alone: a seed
    at most orders them, so every seed has the same number of visible pairs."""
    n = min(case["documents"], case["k_len"])
    rng = random.Random(case["k_len"] * 31 + n)
    w = [math.exp(rng.uniform(0.0, 3.0)) for _ in range(n)]
    lens = [max(1, int(case["k_len"] * x / sum(w))) for x in w]
    lens[lens.index(max(lens))] += case["k_len"] - sum(lens)
    return lens


def _prefixes(case):
    rng = random.Random(case["k_len"] * 17 + case["batch"])
    return [rng.randint(0, case["k_len"]) for _ in range(case["batch"])]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    dt = DTYPES[case["dtype"]]
    d, h, hk, b = case["dim"], case["heads"], case["kv_heads"], case["batch"]

    def randn(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * scale).to(dtype)

    st = {"case": dict(case)}
    if case["op"] == "rotary":
        s = case["seq"]
        # Queries and keys as the joint projection [q | k | v] leaves them: strided views of one buffer.
        joint = randn(b, s, (h + 2 * hk) * d)
        st["q"] = joint[..., : h * d].view(b, s, h, d)
        st["k"] = joint[..., h * d : (h + hk) * d].view(b, s, hk, d)
        st["wq"] = 1.0 + randn(d, dtype=torch.float32, scale=0.1)
        st["wk"] = 1.0 + randn(d, dtype=torch.float32, scale=0.1)
        st["positions"] = torch.arange(s, device=DEVICE).view(1, s).expand(b, s).contiguous() + case["start"]
        r = case["rotated"]
        st["freq"] = 10000.0 ** (-torch.arange(0, r, 2, device=DEVICE, dtype=torch.float64) / r)
        if case["backward"]:
            for n in ("q", "k", "wq", "wk"):
                st[n] = st[n].detach().requires_grad_(True)
            st["dq"], st["dk"] = randn(b, s, h, d), randn(b, s, hk, d)
        return st
    sq, sk = case["q_len"], case["k_len"]
    st["q"] = randn(b, sq, h, d, scale=1.5).transpose(1, 2)
    st["k"] = randn(b, sk, hk, d, scale=1.5).transpose(1, 2)
    st["v"] = randn(b, sk, hk, d).transpose(1, 2)
    st["documents"] = st["prefix"] = st["slopes"] = None
    if case["documents"]:
        rows = []
        for _ in range(b):
            lens = _lengths(case)
            pad = lens.pop() if case["padded"] else 0
            if case["q_len"] == case["k_len"] and not case["prefix"]:
                rng.shuffle(lens)
            rows.append([i for i, n in enumerate(lens) for _ in range(n)] + [-1] * pad)
        st["documents"] = torch.tensor(rows, dtype=torch.int32, device=DEVICE)
    if case["prefix"]:
        p = _prefixes(case)
        rng.shuffle(p)
        st["prefix"] = torch.tensor(p, dtype=torch.int32, device=DEVICE)
    if case["bias"]:
        st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, h + 1, device=DEVICE, dtype=torch.float32) / h)
    if case["backward"]:
        for n in ("q", "k", "v"):
            st[n] = st[n].detach().requires_grad_(True)
        st["do"] = randn(b, sq, h, d).transpose(1, 2)
    return st


# --- one pass --------------------------------------------------------------------------------------------------------


def run(state):
    return _run_rotary(state) if state["case"]["op"] == "rotary" else _run_attention(state)


def _run_attention(st):
    c = st["case"]
    if own:
        import bitscom_b200 as bitscom

        out = bitscom.attention(st["q"], st["k"], st["v"], causal=c["causal"], documents=st["documents"],
                                prefix=st["prefix"], softcap=c["cap"] or None, slopes=st["slopes"])
        if not c["backward"]:
            return out
        return (out, *torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["do"]))
    with torch.no_grad():
        return _plain_attention(st, c)


def _visible(st, c):
    """[batch or 1, q_len, k_len] truth values: which key each query sees."""
    dev = st["q"].device
    pos = torch.arange(c["q_len"], device=dev) + (c["k_len"] - c["q_len"])
    key = torch.arange(c["k_len"], device=dev)
    seen = torch.ones(1, c["q_len"], c["k_len"], dtype=torch.bool, device=dev)
    if c["causal"]:
        seen = (key[None, :] <= pos[:, None])[None]
        if st["prefix"] is not None:
            seen = seen | (key < st["prefix"][:, None])[:, None, :]
    if st["documents"] is not None:
        ids = st["documents"]
        mine = ids[:, pos]
        seen = seen & (mine[:, :, None] == ids[:, None, :]) & (mine >= 0)[:, :, None]
    return seen


def _plain_attention(st, c):
    b, h, hk, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    sq, sk, dt = c["q_len"], c["k_len"], st["q"].dtype
    scale = d ** -0.5
    q = st["q"].float().reshape(b, hk, h // hk, sq, d)
    k, v = st["k"].float()[:, :, None], st["v"].float()[:, :, None]
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    t = None
    if c["cap"]:
        t = torch.tanh(s / c["cap"])
        s = t * c["cap"]
    if st["slopes"] is not None:
        pos = torch.arange(sq, device=q.device) + (sk - sq)
        far = (pos[:, None] - torch.arange(sk, device=q.device)[None, :]).abs().float()
        s = s - st["slopes"].view(1, hk, h // hk, 1, 1) * far
    seen = _visible(st, c)[:, None, None]
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p, v)
    out = o.reshape(b, h, sq, d).to(dt)
    if not c["backward"]:
        return out
    do = st["do"].float().reshape(b, hk, h // hk, sq, d)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    ds = p * (torch.matmul(do, v.transpose(-1, -2)) - (do * o).sum(-1, keepdim=True)) * scale
    if t is not None:
        ds = ds * (1.0 - t * t)
    dq = torch.matmul(ds, k).reshape(b, h, sq, d)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2)
    return out, dq.to(dt), dk.to(dt), dv.to(dt)


def _run_rotary(st):
    c = st["case"]
    if own:
        import bitscom_b200 as bitscom

        out = bitscom.qk_norm_rotary(st["q"], st["k"], st["freq"], q_weight=st["wq"], k_weight=st["wk"],
                                     positions=st["positions"], eps=EPS, interleaved=c["interleaved"])
        if not c["backward"]:
            return out
        grads = torch.autograd.grad(out, (st["q"], st["k"], st["wq"], st["wk"]), (st["dq"], st["dk"]))
        return (*out, *grads)
    with torch.no_grad():
        angle = st["positions"].double()[..., None, None] * st["freq"]
        cos, sin = angle.cos().float(), angle.sin().float()
        q = _plain_rotary(st["q"], st["wq"], cos, sin, c, st.get("dq"))
        k = _plain_rotary(st["k"], st["wk"], cos, sin, c, st.get("dk"))
        return tuple(x for pair in zip(q, k) for x in pair)


def _turn(x, cos, sin, c):
    """Rotates the first `rotated` values of the last axis: pairs (i, i + half), or neighbours where interleaved."""
    r = c["rotated"]
    y = x[..., :r].unflatten(-1, (-1, 2) if c["interleaved"] else (2, -1))
    axis = -1 if c["interleaved"] else -2
    a, b = y.unbind(axis)
    y = torch.stack((a * cos - b * sin, b * cos + a * sin), axis).flatten(-2)
    return torch.cat((y, x[..., r:]), -1)


def _plain_rotary(x, w, cos, sin, c, dy):
    xf = x.float()
    n = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS)
    out = (_turn(n * w, cos, sin, c).to(x.dtype),)
    if dy is None:
        return out
    g = _turn(dy.float(), cos, -sin, c)
    dw = (g * n).sum((0, 1, 2))
    gw = g * w
    dx = torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS) * (gw - n * (gw * n).mean(-1, keepdim=True))
    return (*out, dx.to(x.dtype), dw)


# --- the definition in 64 bits ---------------------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_rotary(st, case) if case["op"] == "rotary" else _exact_attention(st, case)


def _exact_attention(st, c):
    """Head by head from log-softmax, the gradients by differentiation."""
    b, h, sq, sk, d = c["batch"], c["heads"], c["q_len"], c["k_len"], c["dim"]
    group = h // c["kv_heads"]
    out = torch.empty(b, h, sq, d, dtype=torch.float64, device=DEVICE)
    dq, dk, dv = (torch.zeros(st[n].shape, dtype=torch.float64, device=DEVICE) for n in ("q", "k", "v"))
    where = torch.arange(sk - sq, sk, device=DEVICE).view(sq, 1)
    keys = torch.arange(sk, device=DEVICE).view(1, sk)
    for i in range(b):
        hidden = torch.zeros(sq, sk, dtype=torch.bool, device=DEVICE)
        if c["causal"]:
            hidden |= keys > where
            if c["prefix"]:
                hidden &= keys >= int(st["prefix"][i])
        if c["documents"]:
            ids = st["documents"][i]
            own_id = ids[where.view(-1)].view(sq, 1)
            hidden |= (own_id != ids.view(1, sk)) | (own_id < 0)
        none = hidden.all(1, keepdim=True)
        for j in range(h):
            q, k, v = (st[n][i, m].detach().double().requires_grad_(c["backward"])
                       for n, m in (("q", j), ("k", j // group), ("v", j // group)))
            s = (q @ k.T) / math.sqrt(d)
            if c["cap"]:
                s = c["cap"] * torch.tanh(s / c["cap"])
            if c["bias"]:
                s = s - float(st["slopes"][j]) * (where - keys).abs()
            s = torch.where(none, torch.zeros_like(s), s.masked_fill(hidden & ~none, -math.inf))
            o = torch.log_softmax(s, -1).exp().masked_fill(none, 0.0) @ v
            out[i, j] = o.detach()
            if c["backward"]:
                a, e, f = torch.autograd.grad(o, (q, k, v), st["do"][i, j].double())
                dq[i, j] += a
                dk[i, j // group] += e
                dv[i, j // group] += f
    return (out, dq, dk, dv) if c["backward"] else out


def _exact_rotary(st, c):
    """Pairs as complex numbers, the gradients by differentiation."""
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), st["positions"].double()[..., None, None] * st["freq"])
    outs, grads = [], []
    for x, w, dy in (("q", "wq", "dq"), ("k", "wk", "dk")):
        xd, wd = (st[n].detach().double().requires_grad_(c["backward"]) for n in (x, w))
        y = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + EPS) * wd
        r = c["rotated"]
        if c["interleaved"]:
            z = torch.complex(y[..., 0:r:2], y[..., 1:r:2]) * turn
            z = torch.stack((z.real, z.imag), -1).flatten(-2)
        else:
            z = torch.complex(y[..., : r // 2], y[..., r // 2 : r]) * turn
            z = torch.cat((z.real, z.imag), -1)
        z = torch.cat((z, y[..., r:]), -1)
        outs.append(z.detach())
        if c["backward"]:
            grads.append(torch.autograd.grad(z, (xd, wd), st[dy].double()))
    if not c["backward"]:
        return tuple(outs)
    (dxq, dwq), (dxk, dwk) = grads
    return (*outs, dxq, dxk, dwq, dwk)


# --- what a pass cannot do without -----------------------------------------------------------------------------------


def _pairs(c):
    """Visible (query, key) pairs of one head over the whole batch."""
    sq, sk = c["q_len"], c["k_len"]
    total = 0
    prefixes = _prefixes(c) if c["prefix"] else [0] * c["batch"]
    lens = [sk]
    if c["documents"]:
        lens = _lengths(c)
        if c["padded"]:
            lens.pop()
    for p in prefixes:
        end = 0
        for n in lens:
            begin, end = end, end + n
            first = max(begin, sk - sq)
            count = max(0, end - first)
            if not c["causal"]:
                total += count * n
                continue
            # query at position i sees max(i + 1, min(prefix, end)) - begin keys
            free = max(first, min(p, end) - 1)
            inside = min(max(0, free - first), count)
            total += inside * (min(p, end) - begin)
            rest = count - inside
            a = first + inside + 1 - begin
            total += rest * a + rest * (rest - 1) // 2
    return total


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        n = b * case["seq"] * (h + hk) * d
        return {"bytes": n * size * (5 if case["backward"] else 2), "flops": n * (24 if case["backward"] else 8)}
    rows, keys = b * h * case["q_len"] * d, b * hk * case["k_len"] * d
    n = _pairs(case) * h * d
    if case["backward"]:
        return {"bytes": size * (4 * rows + 4 * keys), "flops": 14 * n}
    return {"bytes": size * (2 * rows + 2 * keys), "flops": 4 * n}
