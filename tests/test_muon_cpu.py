"""Orthogonalised updates on the CPU path: formulas, the agreement with torch's own Muon, and what is refused."""

import math

import pytest
import torch

from mvp_engine import ops
from mvp_engine.ops.muon import _check_iteration


def ns64(u, steps=5, coef=(3.4445, -4.7750, 2.0315), eps=1e-7):
    a, b, c = coef
    x = u.double() / max(float(u.double().norm()), eps)
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * s @ s) @ x
    return x


@pytest.mark.parametrize("shape", [(1, 1), (5, 9), (9, 5), (40, 40)])
def test_orthogonalize_formula(shape):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1))
    got = ops.orthogonalize(x, out_dtype=torch.float32)
    want = ns64(x) if shape[0] <= shape[1] else ns64(x.T).T
    # 32-bit products over at most 40 terms in five iterations, each passing an error on at most 3.44 times
    assert float((got.double() - want).norm() / want.norm()) <= 40 * 5 * 2.0**-24 * 3.44
    assert ops.orthogonalize(x).dtype == torch.bfloat16


def test_orthogonalize_brings_singular_values_near_one():
    s = torch.linalg.svdvals(ops.orthogonalize(torch.randn(30, 50, generator=torch.Generator().manual_seed(2)),
                                               out_dtype=torch.float32))
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


def test_orthogonalize_stack_zero_and_nan():
    x = torch.randn(3, 4, 6)
    x[1] = 0
    x[2, 0, 0] = float("nan")
    y = ops.orthogonalize(x, out_dtype=torch.float32)
    assert torch.isfinite(y[0]).all() and bool((y[1] == 0).all()) and torch.isnan(y[2]).all()


@pytest.mark.parametrize("nesterov,adjust", [(True, "original"), (False, "match_rms_adamw"), (True, None)])
def test_muon_step_matches_torch(nesterov, adjust):
    """Three steps against torch.optim.Muon, whose products run in bf16 (so only to a few percent of the update)."""
    g = torch.Generator().manual_seed(3)
    w0 = torch.randn(24, 36, generator=g) * 0.02
    p, m = w0.clone(), torch.zeros(24, 36)
    q = torch.nn.Parameter(w0.clone())
    opt = torch.optim.Muon([q], lr=0.02, weight_decay=0.1, momentum=0.9, nesterov=nesterov, adjust_lr_fn=adjust)
    moved = 0.0
    for _ in range(3):
        grad = torch.randn(24, 36, generator=g)
        q.grad = grad.clone()
        opt.step()
        before = p.clone()
        ops.muon_step_(p, grad, m, lr=0.02, weight_decay=0.1, momentum=0.9, nesterov=nesterov, adjust_lr=adjust)
        moved += float((p - before).norm())
    assert float((p - q).norm()) <= 0.05 * moved


def test_muon_step_scale_clip_and_shadow():
    g = torch.Generator().manual_seed(4)
    p, grad = torch.randn(6, 10, generator=g), torch.randn(6, 10, generator=g)
    m = torch.randn(6, 10, generator=g) * 0.1
    norm_sq = grad.square().sum()
    factor = 0.5 * min(1.0, 1.0 / (float(norm_sq.sqrt()) * 0.5 + 1e-6))
    p2, m2 = p.clone(), m.clone()
    shadow = torch.empty(6, 10, dtype=torch.bfloat16)
    ops.muon_step_(p, grad, m, lr=0.1, grad_scale=0.5, norm_sq=norm_sq, max_norm=1.0, p_bf16=shadow)
    ops.muon_step_(p2, grad * factor, m2, lr=0.1)
    torch.testing.assert_close(p, p2, rtol=1e-5, atol=1e-6)  # the factor enters in another order: a few roundings
    torch.testing.assert_close(m, m2, rtol=1e-5, atol=1e-7)
    assert torch.equal(shadow, p.to(torch.bfloat16))


def test_muon_step_nan_gradient_norm_reaches_the_weights():
    p = torch.ones(4, 4)
    ops.muon_step_(p, torch.ones(4, 4), torch.zeros(4, 4), lr=0.1, norm_sq=torch.tensor(float("nan")), max_norm=1.0)
    assert torch.isnan(p).all()


def test_lr_ratio():
    assert ops.muon_lr_ratio(100, 400) == 1.0 and ops.muon_lr_ratio(400, 100) == 2.0
    assert ops.muon_lr_ratio(400, 100, "match_rms_adamw") == pytest.approx(0.2 * 20)
    with pytest.raises(ValueError):
        ops.muon_lr_ratio(4, 4, "rms")


def test_refusals():
    x = torch.randn(4, 4)
    for bad in ({"steps": 0}, {"coefficients": (1.0, 2.0)}, {"coefficients": (3.4445, -4.775, 4.0)}, {"eps": 0.0},
                {"coefficients": (float("nan"), 1.0, 1.0)}, {"coefficients": (4.0, 0.0, 0.0)}):
        with pytest.raises(ValueError):
            ops.orthogonalize(x, **bad)
    with pytest.raises(ValueError):
        ops.orthogonalize(torch.randn(4))
    with pytest.raises(TypeError):
        ops.orthogonalize(torch.randn(4, 4, dtype=torch.float64))
    with pytest.raises(TypeError):
        ops.orthogonalize(x, out_dtype=torch.int32)
    z = lambda *s: torch.zeros(*s)  # noqa: E731
    for p, g, m in ((z(4), z(4), z(4)), (z(4, 4), z(4, 5), z(4, 4)), (z(4, 4), z(4, 4), z(4, 4).to(torch.bfloat16)),
                    ([z(4, 4)], [z(4, 4), z(4, 4)], [z(4, 4)]), ([z(4, 4), z(4, 5)], [z(4, 4), z(4, 5)], [z(4, 4), z(4, 5)]),
                    (z(4, 6).t(), z(6, 4), z(6, 4))):
        with pytest.raises(ValueError):
            ops.muon_step_(p, g, m, lr=0.1)
    w = z(4, 4)
    with pytest.raises(ValueError):
        ops.muon_step_([w, w], [x, x], [z(4, 4), z(4, 4)], lr=0.1)
    with pytest.raises(ValueError):
        ops.muon_step_(z(4, 4), w, w, lr=0.1)  # the momentum is updated while the gradient is still read
    with pytest.raises(ValueError):
        ops.muon_step_(z(4, 4), x, z(4, 4), lr=0.1, p_bf16=z(4, 4))
    with pytest.raises(ValueError):
        ops.muon_step_(z(4, 4), x, z(4, 4), lr=0.1, adjust_lr="none")
    ops.muon_step_([], [], [], lr=0.1)  # nothing to do


@pytest.mark.parametrize("coef", [(3.4445, -4.7750, 2.0315), (2.0, -1.5, 0.5), (1.5, -0.5, 0.0), (15 / 8, -10 / 8, 3 / 8)])
def test_accepted_coefficients_stay_in_range(coef):
    """The range check against a scan: singular values below 1.9 through every iteration."""
    _check_iteration(12, coef, 1e-7)
    s = torch.linspace(0, 1, 20001, dtype=torch.float64)
    for _ in range(12):
        t = s * s
        assert float((coef[1] * t + coef[2] * t * t).abs().max()) < 3.9
        s = s * (coef[0] + coef[1] * t + coef[2] * t * t)
        assert float(s.abs().max()) < 1.9
    assert math.isfinite(float(s.sum()))
