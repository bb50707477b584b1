"""Orthogonalised updates and the Muon step on the GPU against 64-bit formulas.

Tolerances.  An iteration rounds X, A and the off-diagonal part of B to fp16 once each, half a step being 2^-11 of the value.
For a 1 x n matrix A and B are one number: its X rounding enters A doubled and A's own once, 3 x 2^-11 at most, of which
|b + 2 c| x sigma^2 / p(sigma), at most 1 near sigma = 1 (0.71 / 0.70), stays: 1.5e-3 for the worst signs in one iteration.
Over five iterations signs and sizes differ (and for larger matrices averages do the rest): twice one iteration's
worst, 3e-3, is documented and used.  Rounding the result adds half a step of its type (bf16 2^-8, fp16 2^-11).
"""

import math

import pytest
import torch

from mvp_engine import ops
from mvp_engine.ops import _ext

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

COEF = (3.4445, -4.7750, 2.0315)
NS_TOL = 3e-3
HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def ns64(u, steps=5, coef=COEF, eps=1e-7):
    a, b, c = coef
    x = u.double()
    x = x / x.flatten(-2).norm(dim=-1)[..., None, None].clamp(min=eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * s @ s) @ x
    return x.mT if tall else x


def rel(got, want):
    return float((got.double() - want).norm() / want.norm())


def rand(shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def spectrum(m, n, power, seed=0):
    """A matrix whose singular values decay as k ** power."""
    s = min(m, n)
    u = torch.linalg.qr(rand((m, s), seed).double()).Q
    v = torch.linalg.qr(rand((n, s), seed + 1).double()).Q
    d = torch.arange(1, s + 1, device="cuda").double() ** power
    return ((u * d) @ v.mT).float()


@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (9, 1), (8, 8), (7, 13), (130, 64), (64, 130), (255, 257), (257, 255),
                                   (512, 512), (1000, 333), (333, 1000), (513, 1030)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_orthogonalize_shapes_and_types(shape, out_dtype):
    x = rand(shape, seed=shape[0] * 1009 + shape[1])
    got = ops.orthogonalize(x, out_dtype=out_dtype)
    _ext.check_status()
    assert got.dtype == out_dtype and got.shape == x.shape
    assert rel(got, ns64(x)) <= NS_TOL + HALF_STEP[out_dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_orthogonalize_input_types(dtype):
    x = rand((3, 100, 300), 5, dtype)
    assert rel(ops.orthogonalize(x), ns64(x)) <= NS_TOL + HALF_STEP[torch.bfloat16]


@pytest.mark.parametrize("power", [-0.5, -1.0, -2.0, -4.0])
@pytest.mark.parametrize("shape", [(256, 256), (200, 520), (520, 200)])
def test_orthogonalize_decaying_spectrum(power, shape):
    """Weak singular directions are amplified 485 times: they must not drown in rounding noise."""
    x = spectrum(*shape, power, seed=3)
    assert rel(ops.orthogonalize(x, out_dtype=torch.float32), ns64(x)) <= NS_TOL


@pytest.mark.parametrize("count", [1, 2, 5, 65, 130])
def test_orthogonalize_stacks(count):
    """Stacks longer than one launch takes; each matrix has its own norm."""
    x = rand((count, 40, 72), 11) * torch.logspace(-12, 12, count, device="cuda")[:, None, None]
    got = ops.orthogonalize(x, out_dtype=torch.float32)
    want = ns64(x, eps=1e-7)
    big = x.flatten(1).norm(dim=1) > 1e-7  # below eps the first X is small and underflows gradually
    for i in range(count):
        if big[i]:
            assert rel(got[i], want[i]) <= NS_TOL
    assert torch.isfinite(got).all()


def test_orthogonalize_several_leading_dimensions_and_strides():
    x = rand((2, 3, 96, 160), 2)
    got = ops.orthogonalize(x, out_dtype=torch.float32)
    assert got.shape == x.shape and rel(got, ns64(x)) <= NS_TOL
    y = rand((200, 130), 4)[::2, 1:120:3]
    assert rel(ops.orthogonalize(y, out_dtype=torch.float32), ns64(y)) <= NS_TOL
    t = rand((96, 200), 6).t()
    assert rel(ops.orthogonalize(t, out_dtype=torch.float32), ns64(t)) <= NS_TOL


@pytest.mark.parametrize("steps,coef", [(1, COEF), (2, COEF), (8, COEF), (10, (2.0, -1.5, 0.5)), (6, (1.5, -0.5, 0.0))])
def test_orthogonalize_steps_and_coefficients(steps, coef):
    x = rand((192, 320), 8)
    got = ops.orthogonalize(x, steps=steps, coefficients=coef, out_dtype=torch.float32)
    # rounding errors of `steps` iterations add up in squares
    assert rel(got, ns64(x, steps, coef)) <= NS_TOL * math.sqrt(max(1.0, steps / 5))


def test_orthogonalize_zero_nan_inf_and_extreme_values():
    x = rand((6, 50, 70), 1)
    x[1] = 0
    x[2, 3, 4] = float("nan")
    x[3, 49, 69] = float("inf")
    x[4] *= 1e37  # squares overflow fp32
    x[5] *= 1e-3
    got = ops.orthogonalize(x, out_dtype=torch.float32)
    for i in (0, 4, 5):
        assert rel(got[i], ns64(x[i])) <= NS_TOL
    assert torch.equal(got[1], torch.zeros_like(got[1]))
    assert torch.isnan(got[2]).all() and torch.isnan(got[3]).all()


def test_orthogonalize_empty():
    assert ops.orthogonalize(torch.empty(0, 5, 7, device="cuda")).shape == (0, 5, 7)
    assert ops.orthogonalize(torch.empty(3, 0, device="cuda")).shape == (3, 0)


def test_orthogonalize_same_bits_again_and_on_another_stream():
    x = rand((3, 300, 500), 21)
    a = ops.orthogonalize(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = ops.orthogonalize(x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, b)


def test_orthogonalize_captured_graphs():
    """Two graphs with workspaces of their own, replayed in turn on new inputs."""
    xs = [rand((2, 128, 256), 31), rand((300, 200), 32)]
    for x in xs:
        ops.orthogonalize(x)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.orthogonalize(x))
        graphs.append(g)
    for r in range(3):
        for i, x in enumerate(xs):
            x.copy_(rand(x.shape, 100 + 10 * r + i))
        for g in graphs:
            g.replay()
        for x, o in zip(xs, outs):
            assert rel(o, ns64(x)) <= NS_TOL + HALF_STEP[torch.bfloat16]


def step64(p, g, m, lr, momentum, nesterov, wd, adjust, scale=1.0):
    p, g, m = p.double(), g.double() * scale, m.double()
    m = m + (1 - momentum) * (g - m)
    u = g + momentum * (m - g) if nesterov else m
    rows, cols = p.shape
    ratio = 0.2 * math.sqrt(max(rows, cols)) if adjust == "match_rms_adamw" else math.sqrt(max(1, rows / cols))
    o = ns64(u)
    return p * (1 - lr * wd) - lr * ratio * o, m, lr * ratio * o


@pytest.mark.parametrize("shape", [(64, 64), (33, 70), (300, 129), (256, 512)])
@pytest.mark.parametrize("nesterov,adjust,clip", [(True, None, False), (False, "match_rms_adamw", True)])
def test_muon_step(shape, nesterov, adjust, clip):
    n = 3
    p, g, m = ([rand(shape, 50 + 10 * k + i) * s for i in range(n)] for k, s in enumerate((0.02, 1e-3, 1e-3)))
    shadow = [torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in range(n)]
    norm_sq = sum(x.square().sum() for x in g) if clip else None
    scale, max_norm = (0.5, 0.3 * float(norm_sq.sqrt())) if clip else (1.0, 0.0)
    factor = scale * min(1.0, max_norm / (float(norm_sq.sqrt()) * scale + 1e-6)) if clip else 1.0
    want = [step64(p[i], g[i], m[i], 0.02, 0.9, nesterov, 0.1, adjust, factor) for i in range(n)]
    before = [t.clone() for t in g]
    ops.muon_step_(p, g, m, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, adjust_lr=adjust,
                   grad_scale=scale, norm_sq=norm_sq, max_norm=max_norm, p_bf16=shadow)
    _ext.check_status()
    for i in range(n):
        wp, wm, delta = want[i]
        # fp32 rounding of the weights and the 0.3 % of the update
        assert float((p[i].double() - wp).norm()) <= NS_TOL * float(delta.norm()) + 2.0**-22 * float(wp.norm())
        assert rel(m[i], wm) <= 2.0**-21  # the scaled gradient, a difference, a product, a sum: four roundings
        assert torch.equal(shadow[i], p[i].to(torch.bfloat16))
        assert torch.equal(g[i], before[i])


def test_muon_step_single_matrix_unaligned_views():
    """Matrices at odd offsets of a flat buffer, as a shard lays them out; what lies around them stays."""
    flat = [torch.full((3 * 1100,), 7.0, device="cuda") for _ in range(3)]
    sh = torch.full((3 * 1100,), 7.0, device="cuda", dtype=torch.bfloat16)
    shape, off = (31, 33), 1101
    n = shape[0] * shape[1]
    views = [f[off:off + n].view(shape) for f in flat]
    for k, v in enumerate(views):
        v.copy_(rand(shape, 70 + k) * 0.01)
    want = step64(*[v.clone() for v in views], 0.01, 0.95, True, 0.0, None)
    ops.muon_step_(views[0], views[1], views[2], lr=0.01, weight_decay=0.0, p_bf16=sh[off:off + n].view(shape))
    assert float((views[0].double() - want[0]).norm()) <= NS_TOL * float(want[2].norm()) + 2.0**-22 * float(want[0].norm())
    for f in flat + [sh]:
        assert bool((f[:off] == 7.0).all()) and bool((f[off + n:] == 7.0).all())
    assert torch.equal(sh[off:off + n].view(shape), views[0].to(torch.bfloat16))


def test_muon_step_more_matrices_than_one_launch():
    n = 70
    p = [rand((24, 40), i) for i in range(n)]
    g = [rand((24, 40), 1000 + i) for i in range(n)]
    m = [torch.zeros(24, 40, device="cuda") for _ in range(n)]
    want = [step64(p[i], g[i], m[i], 0.1, 0.95, True, 0.1, None) for i in range(n)]
    ops.muon_step_(p, g, m, lr=0.1)
    for i in range(n):
        assert float((p[i].double() - want[i][0]).norm()) <= NS_TOL * float(want[i][2].norm()) + 2.0**-22 * float(want[i][0].norm())


def test_muon_step_nan_gradient_norm_reaches_the_weights():
    p, g, m = rand((16, 16)), rand((16, 16), 1), torch.zeros(16, 16, device="cuda")
    ops.muon_step_(p, g, m, lr=0.1, norm_sq=torch.tensor(float("nan"), device="cuda"), max_norm=1.0)
    assert torch.isnan(p).all()


def test_muon_step_refuses_on_the_gpu():
    p, g, m = rand((8, 8)), rand((8, 8), 1), torch.zeros(8, 8, device="cuda")
    with pytest.raises(ValueError):
        ops.muon_step_(p, g.cpu(), m, lr=0.1)
    with pytest.raises(ValueError):
        ops.muon_step_(p, g.to(torch.bfloat16), m, lr=0.1)
    with pytest.raises((ValueError, RuntimeError)):
        ops.muon_step_(p, g, m, lr=0.1, norm_sq=torch.ones(2, device="cuda"), max_norm=1.0)
    with pytest.raises(ValueError):
        ops.muon_step_([p, p], [g, g], [m, torch.zeros_like(m)], lr=0.1)
