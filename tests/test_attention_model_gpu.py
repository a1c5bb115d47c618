"""The attention operators together, as the GPT-2 model runs them: norm and
rotation, then masked and capped attention, forward and backward, eager,
sharded and captured."""

import datetime
import os

import pytest
import torch
import torch.distributed as dist

from bitscom_b200.models import gpt2_small_test
from bitscom_b200.parallel.fsdp import LowBitShardedDP
from bitscom_b200.parallel.graphs import GraphedStep

pytestmark = pytest.mark.gpu


def _model(**kw):
    torch.manual_seed(0)
    return gpt2_small_test(vocab_size=512, n_positions=300, **kw)


def _batch(b=2, t=200, seed=0):
    g = torch.Generator().manual_seed(seed)
    tok = torch.randint(0, 512, (b, t + 1), generator=g)
    ids = torch.zeros(b, t, dtype=torch.int32)
    for i in range(b):
        for n, cut in enumerate(sorted(torch.randint(1, t, (3,), generator=g).tolist())):
            ids[i, cut:] = n + 1
    ids[0, t - 7 :] = -1
    target = tok[:, 1:].clone()
    target[ids < 0] = -100
    return tok[:, :-1].contiguous(), target, ids


OPTIONS = [dict(rotary=True), dict(rotary=True, softcap=5.0), dict(distance_bias=True, softcap=5.0), dict()]


def _grads(model, batch, prefix=None, autocast=False):
    dev = next(model.parameters()).device
    idx, target, ids = (x.to(dev) for x in batch)
    with torch.autocast(dev.type, dtype=torch.bfloat16, enabled=autocast):
        logits, loss = model(idx, target, documents=ids, prefix=None if prefix is None else prefix.to(dev))
    return logits, torch.autograd.grad(loss, list(model.parameters()))


@pytest.mark.parametrize("options", OPTIONS, ids=str)
def test_model_gradients(cuda, options):
    """fp32 on the GPU against the torch forms on the CPU; bf16 autocast against fp32."""
    model = _model(**options)
    batch, prefix = _batch(), torch.tensor([17, 60])
    _, want = _grads(model, batch, prefix)
    gpu = _model(**options).cuda()
    _, got = _grads(gpu, batch, prefix)
    _, low = _grads(gpu, batch, prefix, autocast=True)
    for w, x, y in zip(want, got, low):
        w, n = w.double(), float(w.double().norm())
        # About 60 fp32 operations in a row with sums of up to 1024 terms: well below 60 * 1024 * 2^-24.
        assert float((x.cpu().double() - w).norm()) < 60 * 1024 * 2.0 ** -24 * n + 1e-8
        # About 60 roundings to bf16 in a row (forward and backward of 4 layers), 2^-9 rms each, if all added up.
        assert float((y.cpu().double() - w).norm()) < 60 * 2.0 ** -9 * 1.5 * n + 1e-6


def test_sharded_training_on_packed_documents(cuda):
    if not dist.is_initialized():
        os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
        os.environ.setdefault("MASTER_PORT", "29657")
        dist.init_process_group("nccl", rank=0, world_size=1, timeout=datetime.timedelta(seconds=60))
    try:
        model = _model(rotary=True, softcap=20.0).cuda()
        sdp = LowBitShardedDP(model, lambda ps: torch.optim.AdamW(ps, lr=1e-3), rs_bits=8, ag_bits=8)
        idx, target, ids = (x.cuda() for x in _batch())
        before = sdp.flat_param.clone()
        for _ in range(2):
            with torch.autocast("cuda", dtype=torch.bfloat16):
                _, loss = sdp(idx, target, documents=ids)
            loss.backward()
            assert all(torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in model.parameters())
            sdp.step()
        assert torch.isfinite(sdp.flat_param).all() and not torch.equal(sdp.flat_param, before)
    finally:
        dist.destroy_process_group()


def test_captured_training_step(cuda):
    """A whole step captured once and replayed on other rows and other documents follows eager steps."""
    def build():
        model = _model(rotary=True, softcap=10.0).cuda()
        opt = torch.optim.SGD(model.parameters(), lr=0.05)

        def step(idx, target, ids):
            with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
                _, loss = model(idx, target, documents=ids)
            loss.backward()
            opt.step()
            opt.zero_grad(set_to_none=False)
            return loss.detach()

        return model, step

    batches = [[x.cuda() for x in _batch(seed=i)] for i in range(4)]
    eager, step = build()
    for _ in range(2):
        step(*batches[0])
    want = [step(*b).clone() for b in batches[1:]]
    graphed, step = build()
    captured = GraphedStep(step, batches[0], warmup=2)
    got = [captured(*b).clone() for b in batches[1:]]
    torch.cuda.synchronize()
    # The attention operators repeat bit for bit; torch's embedding gradient adds with atomics, whose order moves
    # fp32 sums of at most 400 terms by 400 * 2^-24 a step.
    for x, y in zip(got, want):
        assert abs(float(x) - float(y)) < 1e-3 * abs(float(y))
    for a, b in zip(eager.parameters(), graphed.parameters()):
        assert float((a - b).detach().norm()) < 1e-2 * float(a.detach().norm()) + 1e-6
