"""64-bit oracle of the attention operators, with error bounds by arithmetic.

Bounds count roundings: u is half a step of the tensors' type (relative), 2^-24
that of the fp32 sums.  The kernels round the probabilities p and the score
gradients ds to the tensors' type before the second products, and each result
once at the end; everything else is fp32.  With P = p, A = P |v|:

  o:   u |o| + u A + e A                 (rounded result, rounded p, fp32 scores)
  dv:  u |dv| + u P^T|do| + e P^T|do|
  ds:  E = u |ds| + P (u sum|do||o| + e (|dp| + sum|do||o|)) f    (delta uses the rounded o)
  dq:  u |dq| + scale E |k|;   dk: u |dk| + scale E^T |q|

where e bounds the relative error that fp32 arithmetic leaves in p and in the sums.
float16 has a smallest step of 2^-24: p (held as 2^10 p / max p at least 2^-4) and ds also
move by half of it, which adds 2^-31 sum|v| to o, 2^-25 to p in dv and to ds.  In every type p is
an fp32 value, so one below 2^-126 (a score 88 under the row's log-sum) counts as zero: p moves by
up to 2^-126, ds by 2^-126 (|dp| + sum|do||o|), and both by 2^-126 where ds or p itself is below it.
"""

import math

import torch


def visible(b, sq, sk, causal, documents=None, prefix=None):
    """[b, sq, sk] truth values, entry by entry from the definition."""
    seen = torch.zeros(b, sq, sk, dtype=torch.bool)
    for n in range(b):
        run = [0] * sk
        if documents is not None:
            ids = documents[n].tolist()
            r = 0
            for j in range(sk):
                if j and ids[j] != ids[j - 1]:
                    r += 1
                run[j] = r if ids[j] >= 0 else -1
        run = torch.tensor(run, dtype=torch.int64)
        p = int(prefix[n]) if prefix is not None else 0
        key = torch.arange(sk)
        for i in range(sq):
            pos = i + sk - sq
            ok = torch.ones(sk, dtype=torch.bool)
            if causal:
                ok &= (key <= pos) | (key < p)
            if documents is not None:
                ok &= (run == run[pos]) & (run >= 0) if pos >= 0 else torch.zeros(sk, dtype=torch.bool)
            seen[n, i] = ok
    return seen


def reference(q, k, v, do, *, seen, softcap=None, slopes=None, scale=None):
    """({name: value}, {name: bound}) of out, dq, dk, dv in float64, on q's device."""
    dev = q.device
    b, h, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    g = h // hk
    u = torch.finfo(q.dtype).eps / 2
    scale = d ** -0.5 if scale is None else scale
    qd, dod = (x.detach().double().reshape(b, hk, g, sq, d) for x in (q, do))
    kd, vd = (x.detach().double()[:, :, None] for x in (k, v))
    seen = seen.to(dev)[:, None, None]
    s = qd @ kd.transpose(-1, -2) * scale
    f = torch.ones_like(s)
    if softcap:
        t = torch.tanh(s / softcap)
        s, f = softcap * t, 1 - t * t
    if slopes is not None:
        far = (torch.arange(sk - sq, sk, device=dev)[:, None] - torch.arange(sk, device=dev)).abs()
        s = s - slopes.double().view(1, hk, g, 1, 1) * far
    none = ~seen.any(-1, keepdim=True)
    s = torch.where(none, torch.zeros_like(s), s.masked_fill(~seen, -math.inf))
    p = torch.softmax(s, -1).masked_fill(none, 0.0) if sk else s
    o = p @ vd
    dp = dod @ vd.transpose(-1, -2)
    delta = (dod * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * f
    dq = ds @ kd * scale
    dk = (ds.transpose(-1, -2) @ qd).sum(2) * scale
    dv = (p.transpose(-1, -2) @ dod).sum(2)
    # fp32: products of d terms in the scores, the scores' own rounding, exp2 (2 steps), sums over up to sk (sq g) terms;
    # tanh by exp2 and a reciprocal: 4 steps of a value near one, times the cap.
    eps = 2.0 ** -24
    live = s[(p > 1e-7)] if sk else s
    size = float(live.abs().max()) if live.numel() else 0.0
    dots = float((qd.abs() @ kd.abs().transpose(-1, -2)).max()) * scale if q.numel() and k.numel() else 0.0
    e = eps * (2 * (d + 8) * dots + 8 * size + 16 + 2 * max(sk, sq * g)) + (softcap or 0.0) * 8 * eps
    ado = (dod.abs() * o.abs()).sum(-1, keepdim=True)
    A = p @ vd.abs()
    E = u * ds.abs() + p * f.abs() * (u * ado + e * (dp.abs() + ado)) + e * ds.abs()
    vals = {"out": o.reshape(b, h, sq, d), "dq": dq.reshape(b, h, sq, d), "dk": dk, "dv": dv}
    tiny = torch.finfo(q.dtype).tiny  # results below it lose relative precision
    step = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    least = 2.0 ** -126
    E = E + (step + least * (1 + dp.abs() + ado)) * (p > 0)
    A = A + (step / 64 + least) * ((p > 0).double() @ vd.abs()) / (u + e)
    padv = (p + (step + least) * (p > 0) / (u + e)).transpose(-1, -2) @ dod.abs()
    bounds = {
        "out": (u * o.abs() + (u + e) * A).reshape(b, h, sq, d) + tiny,
        "dq": (u * dq.abs() + scale * (E @ kd.abs())).reshape(b, h, sq, d) + tiny,
        "dk": u * dk.abs() + scale * (E.transpose(-1, -2) @ qd.abs()).sum(2) + tiny,
        "dv": u * dv.abs() + (u + e) * padv.sum(2) + tiny,
    }
    return vals, {n: x * 1.05 for n, x in bounds.items()}  # second-order terms


def check(got, vals, bounds):
    for name, x in got.items():
        err = (x.detach().double() - vals[name]).abs()
        over = err > bounds[name]
        assert torch.isfinite(x).all(), f"{name}: not finite"
        assert not over.any(), (
            f"{name}: {int(over.sum())} of {over.numel()} values beyond their bound, worst "
            f"{float((err / bounds[name]).max()):.3g} times at {torch.nonzero(over)[0].tolist()}")


def rotary_reference(x, w, freq, positions, eps, interleaved, g=None):
    """(y, dx, dw) in float64 of one tensor [b, s, h, d], each with its absolute-value companion for bounds."""
    xd = x.detach().double()
    wd = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    xd.requires_grad_(True)
    wd = wd.clone().requires_grad_(True)
    n = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + eps)
    y = n * wd
    r = 2 * freq.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), positions.double()[..., None, None] * freq.double())
    if interleaved:
        z = torch.complex(y[..., 0:r:2], y[..., 1:r:2]) * turn
        z = torch.stack((z.real, z.imag), -1).flatten(-2)
    else:
        z = torch.complex(y[..., : r // 2], y[..., r // 2 : r]) * turn
        z = torch.cat((z.real, z.imag), -1)
    z = torch.cat((z, y[..., r:]), -1)
    if g is None:
        return z.detach(), None, None
    dx, dw = torch.autograd.grad(z, (xd, wd), g.double())
    return z.detach(), dx, dw
