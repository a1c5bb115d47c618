"""The attention operators at the edges of their range: waits that run out, what
other kernels leave in shared memory, extreme caps, derivatives and traces.
Needs a CUDA device."""

import pytest
import torch

import bitscom_b200 as bitscom
from bitscom_b200 import _ext

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
