"""Gradients of fused projections (q/k/v and gate/up as one operand) in the data-parallel runtime on CPU."""

import pytest
import torch

from mvp_engine import ops
from mvp_engine.models.qwen3 import build_qwen3
from mvp_engine.parallel.fsdp import NativeFSDP

TINY = dict(vocab_size=256, hidden_size=128, intermediate_size=256, num_attention_heads=2, num_key_value_heads=1)


@pytest.mark.parametrize("ckpt", [False, True])
def test_runtime_gradients_are_the_plain_models(ckpt):
    x = torch.randint(0, 256, (2, 40), generator=torch.Generator().manual_seed(2))
    plain = build_qwen3("mvp/qwen3-tiny", seed=3, **TINY)
    (plain(input_ids=x, labels=x)["loss"].sum() / 78).backward()
    model = build_qwen3("mvp/qwen3-tiny", seed=3, **TINY)
    if ckpt:
        model.gradient_checkpointing_enable()
    fsdp = NativeFSDP(model, group=None, device=torch.device("cpu"), param_dtype=torch.float32)
    fsdp.train()
    for micro in range(1, 3):  # two micro-batches add up
        (fsdp(input_ids=x, labels=x)["loss"].sum() / 78).backward()
        got = {e.fqns[0]: u.grad[e.offset:e.offset + e.numel].view(e.shape) for u in fsdp.units for e in u.entries}
        for name, p in plain.named_parameters():
            assert float(got[name].norm()) > 0, name
            # the same 32-bit products over at most 256 terms, taken in another order
            err = float((got[name] - micro * p.grad).norm())
            assert err <= 256 * 2.0**-24 * 16 * micro * float(p.grad.norm()), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_adds_into_the_accumulator_of_an_untracked_weight(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 5, 8, generator=g).to(dtype).requires_grad_()
    w = torch.randn(6, 8, generator=g).to(dtype)
    w._mvp_grad_acc = torch.ones(6, 8)
    dy = torch.randn(3, 5, 6, generator=g).to(dtype)
    y = ops.linear(x, w)
    y.backward(dy)
    x64, d64 = x.detach().double().view(15, 8), dy.double().view(15, 6)
    half = torch.finfo(dtype).eps / 2
    assert bool(((w._mvp_grad_acc.double() - 1 - d64.t() @ x64).abs() <= 17 * 2.0**-24 * (1 + d64.t().abs() @ x64.abs())).all())
    for got, want, size in ((y.detach().view(15, 6), x64 @ w.double().t(), x64.abs() @ w.double().abs().t()),
                            (x.grad.view(15, 8), d64 @ w.double(), d64.abs() @ w.double().abs())):
        assert bool(((got.double() - want).abs() <= half * want.abs() + 10 * 2.0**-24 * size + half * 10 * 2.0**-24).all())
    with torch.no_grad():
        assert not ops.linear(x, w).requires_grad
