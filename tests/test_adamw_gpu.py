"""The fused AdamW step on slices of flat buffers, against the formula in 64 bits.

Tolerances.  m takes four fp32 roundings (the scaled gradient, a difference, a product, a sum) of values no larger than
|m| + |g|: 2^-22 of that sum.  v takes five of values no larger than the new v: 2^-21.  The weight takes the decay's (two,
2^-23 of itself), the last difference's (2^-24) and those of the update: m's error over the denominator, and six
roundings with v's error halved by the root, 2^-20 of the update.
"""

import math

import pytest
import torch

from mvp_engine import ops

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=3)


def f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def adamw64(p, g, m, v, scale):
    b1, b2 = f32(HYPER["beta1"]), f32(HYPER["beta2"])
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * scale
    size = m.abs() + g.abs()
    m = m + (1 - b1) * (g - m)
    v = v * b2 + (1 - b2) * g * g
    denom = (v / (1 - HYPER["beta2"] ** HYPER["step"])).sqrt() + f32(HYPER["eps"])
    rate = HYPER["lr"] / (1 - HYPER["beta1"] ** HYPER["step"])
    update = rate * m / denom
    new = p * (1 - HYPER["lr"] * HYPER["weight_decay"]) - update
    return new, m, v, 2.0**-22 * size, 2.0**-21 * v, \
        2.0**-22 * p.abs() + 2.0**-24 * new.abs() + 2.0**-20 * update.abs() + rate * 2.0**-22 * size / denom


@pytest.mark.parametrize("offsets", [(0, 0, 0, 0, 0), (1, 1, 1, 1, 1), (2, 2, 2, 2, 2), (3, 3, 3, 3, 3), (0, 0, 0, 0, 2),
                                     (4, 0, 3, 8, 4), (1155, 1155, 1155, 1155, 1155)])
@pytest.mark.parametrize("n", [1, 3, 125, 1027, 300001])
def test_adamw_step_on_slices_at_any_offset(n, offsets):
    g = torch.Generator(device="cuda").manual_seed(n * 31 + offsets[0])
    flat = [torch.full((n + 2000,), 7.0, device="cuda") for _ in range(4)]
    flat.append(torch.full((n + 2000,), 7.0, device="cuda", dtype=torch.bfloat16))
    views = [f[o:o + n] for f, o in zip(flat, offsets)]
    for t, size in zip(views, (0.02, 1e-3, 1e-3, 1e-6)):
        t.copy_(torch.randn(n, generator=g, device="cuda") * size)
    views[3].abs_()
    p, gr, m, v, shadow = views
    norm_sq = gr.square().sum()
    max_norm = 0.25 * math.sqrt(float(norm_sq))
    scale = 0.5 * f32(max_norm) / (math.sqrt(float(norm_sq)) * 0.5 + f32(1e-6))
    before = gr.clone()
    wp, wm, wv, tm, tv, tp = adamw64(p, gr, m, v, scale)
    ops.adamw_step_(p, gr, m, v, grad_scale=0.5, norm_sq=norm_sq, max_norm=max_norm, p_bf16=shadow, **HYPER)
    # the clip coefficient itself takes four roundings, 2^-22 of the gradient, twice that of its square
    assert bool(((m.double() - wm).abs() <= 2 * tm).all())
    assert bool(((v.double() - wv).abs() <= 2 * tv).all())
    assert bool(((p.double() - wp).abs() <= 2 * tp).all())
    assert torch.equal(shadow, p.to(torch.bfloat16)) and torch.equal(gr, before)
    for f, o in zip(flat, offsets):
        assert bool((f[:o] == 7.0).all()) and bool((f[o + n:] == 7.0).all())
