"""The edges of what is documented for the Newton-Schulz kernels on the GPU.

FINE_TOL, of fp32 results with sides up to 256, the shorter up to 64.  X, A and B are kept to 22 bits there, and no product
drops more than lo lo.  What is left: sums of l / 16 partial sums in 32 bits (a step of 2^-23 each, in one direction if the
hardware cuts off), three passes of 16 x 2^-23 of A in five iterations at l = 256, 3e-5; and an error of 2^-21 of B X in the strong directions,
passed on to the weak ones at most 3.44^4 = 140 times, 7e-5 of the strongest singular value.  Three times the sum.
"""

import pytest
import torch

from mvp_engine import ops

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]


COEF = (3.4445, -4.7750, 2.0315)
NS_TOL = 3e-3  # documented
FINE_TOL = 3e-4


def ns64(u, steps, eps):
    a, b, c = COEF
    x = u.double()
    x = x / max(float(x.norm()), eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * s @ s) @ x
    return x.T if tall else x


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


@pytest.mark.parametrize("shape", [(1, 9), (8, 8), (40, 72), (130, 64), (800, 1030)])
@pytest.mark.parametrize("ratio", [3.0, 1.0, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 1e-8, 1e-10, 1e-13])
def test_norms_below_eps(shape, ratio):
    """X is rounded to a step of 2^-24 in units in which |X|_F = 1 is at most sqrt(2) sqrt(m n): half a step in every
    value of five X is sqrt(2) 2^-25 (a + .. + a^5) = 2.9e-5 of the result."""
    x = rand(shape, 7)
    x = x / x.norm() * 1e-4
    eps = float(x.double().norm()) / ratio
    want = ns64(x, 5, eps)
    for dtype, half in ((torch.float32, 2.0**-24), (torch.bfloat16, 2.0**-8)):
        got = ops.orthogonalize(x, eps=eps, out_dtype=dtype).double()
        off = float((got - want).norm())
        size = float(want.norm())
        if ratio >= 1e-4:
            assert off <= (NS_TOL + half) * size
        else:
            assert off <= 3e-5 + half * (size + 3e-5)


@pytest.mark.parametrize("steps", [1, 5, 7, 12, 20, 50, 100, 200])
@pytest.mark.parametrize("shape", [(192, 320), (1000, 333), (1024, 1536)])
def test_many_steps(shape, steps):
    """With these coefficients singular values keep moving within 0.7 to 1.2, and each step rounds them again."""
    x = rand(shape, 3)
    want = ns64(x, steps, 1e-7)
    off = float((ops.orthogonalize(x, steps=steps, out_dtype=torch.float32).double() - want).norm())
    assert off <= NS_TOL * max(1.0, steps / 5) ** 0.5 * float(want.norm())


SMALL = [(1, 1), (1, 9), (9, 1), (8, 8), (8, 16), (16, 8), (33, 70), (64, 64), (63, 65), (64, 256), (256, 64), (8, 250),
         (200, 3)]


@pytest.mark.parametrize("shape", SMALL)
@pytest.mark.parametrize("power", [0.0, -1.0, -4.0])
def test_small_fp32_results_keep_more(shape, power):
    x = rand((3, *shape), 5)
    if power:  # singular values that decay as k ** power
        u, d, v = torch.linalg.svd(x.double(), full_matrices=False)
        x = ((u * torch.arange(1, d.shape[-1] + 1, device="cuda").double() ** power) @ v).float()
    got = ops.orthogonalize(x, out_dtype=torch.float32).double()
    for i in range(3):
        want = ns64(x[i], 5, 1e-7)
        assert float((got[i] - want).norm()) <= FINE_TOL * float(want.norm())


@pytest.mark.parametrize("shape", SMALL)
def test_small_steps_keep_the_weights_bits(shape):
    n = 3
    p, g, m = ([rand(shape, 50 + 10 * k + i) * s for i in range(n)] for k, s in enumerate((0.02, 1e-3, 1e-3)))
    want = []
    for pi, gi, mi in zip(p, g, m):
        pi, gi, mi = pi.double(), gi.double(), mi.double()
        mi = mi + 0.05 * (gi - mi)
        move = 2e-4 * 0.2 * max(shape) ** 0.5 * ns64(gi + 0.95 * (mi - gi), 5, 1e-7)
        want.append((pi * (1 - 2e-4 * 0.1) - move, move))
    ops.muon_step_(p, g, m, lr=2e-4, weight_decay=0.1, adjust_lr="match_rms_adamw")
    for got, (w, move) in zip(p, want):
        assert float((got.double() - w).norm()) <= FINE_TOL * float(move.norm()) + 2.0**-23 * float(w.norm())


@pytest.mark.parametrize("shape", [(257, 257), (256, 769), (769, 256), (16, 3000), (3000, 16), (64, 4096), (300, 700), (65, 65),
                                   (64, 257), (257, 64), (65, 256), (8, 257), (65, 769)])
def test_fp32_results_beyond(shape):
    """A side beyond one of the two limits: the documented bound, and one matrix as in a stack."""
    x = rand((2, *shape), 9)
    got = ops.orthogonalize(x, out_dtype=torch.float32)
    for i in range(2):
        want = ns64(x[i], 5, 1e-7)
        assert float((got[i].double() - want).norm()) <= NS_TOL * float(want.norm())
        assert torch.equal(ops.orthogonalize(x[i], out_dtype=torch.float32), got[i])
