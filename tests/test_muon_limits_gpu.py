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
