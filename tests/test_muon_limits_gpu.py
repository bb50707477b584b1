"""The edges of what is documented for the Newton-Schulz kernels on the GPU."""

import pytest
import torch

from mvp_engine import ops

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]


def rand(shape, seed=0):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("momentum", [0.0, 0.5, 0.9, 0.95, 0.99, 0.999])
def test_momentum_weight_is_rounded_once(momentum):
    """From a zero buffer: half a step for the weight 1 - momentum, half a step for the product."""
    p, g, m = rand((40, 72)), rand((40, 72), 1), torch.zeros(40, 72, device="cuda")
    ops.muon_step_(p, g, m, lr=0.01, momentum=momentum)
    want = (1 - momentum) * g.double()
    assert bool(((m.double() - want).abs() <= 2.0**-23 * want.abs()).all())


def test_launches_are_counted_by_steps_and_groups():
    from mvp_engine.ops import _ext

    def count(fn):
        _ext.start_counting()
        fn()
        return _ext.stop_counting()

    x = rand((70, 8, 24))  # two groups of at most 64
    zeros = lambda: [torch.zeros(8, 24, device="cuda") for _ in range(70)]  # noqa: E731
    assert count(lambda: ops.orthogonalize(x[:3])) == 17 and count(lambda: ops.orthogonalize(x[:3], steps=2)) == 8
    assert count(lambda: ops.orthogonalize(x)) == 34
    assert count(lambda: ops.muon_step_(zeros(), list(x), zeros(), lr=0.1, steps=3)) == 22
    a, w = rand((20, 256)).to(torch.bfloat16).requires_grad_(), rand((130, 256), 1).to(torch.bfloat16)
    w8 = ops.quantize_fp8(w, "tile", rows=True, columns=True)
    assert count(lambda: ops.linear_fp8(a, w)) == 3 and count(lambda: ops.linear_fp8(a, w, w8)) == 2
    assert count(lambda: ops.linear_fp8(a, w, w8).sum().backward()) == 4  # dx alone
    assert count(lambda: ops.linear_fp8(a, w.requires_grad_()).sum().backward()) == 6
