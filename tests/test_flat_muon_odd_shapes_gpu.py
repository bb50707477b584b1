"""FlatMuon on modules of odd widths on the GPU: matrices and what lies between them, against the formulas in 64 bits."""

import math

import pytest
import torch
import torch.nn as nn

from mvp_engine.ops import _ext
from mvp_engine.parallel.fsdp import NativeFSDP
from mvp_engine.parallel.optim import FlatMuon, is_hidden_matrix

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

NS_TOL = 3e-3  # documented for the iteration


def ns64(u):
    x = u / max(float(u.norm()), 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(5):
        s = x @ x.T
        x = 3.4445 * x + (-4.775 * s + 2.0315 * s @ s) @ x
    return x.T if tall else x


@pytest.mark.parametrize("param_dtype", [torch.bfloat16, torch.float32])
def test_step_of_odd_matrices_and_their_biases(param_dtype):
    torch.manual_seed(3)
    model = nn.Sequential(nn.Linear(33, 31), nn.GELU(), nn.Linear(31, 7), nn.Linear(7, 35, bias=False), nn.LayerNorm(35))
    fsdp = NativeFSDP(model, group=None, device=torch.device("cuda"), param_dtype=param_dtype)
    opt = FlatMuon(fsdp, lr=1e-2, momentum=0.9, weight_decay=0.1, betas=(0.9, 0.95))
    gen = torch.Generator(device="cuda").manual_seed(5)
    rest64 = {}
    for step in range(2):
        want = {}
        for u in fsdp.units:
            if not u.trainable:
                continue
            for e in u.entries:
                at = slice(e.offset, e.offset + e.numel)
                u.grad[at].copy_(torch.randn(e.numel, generator=gen, device="cuda") * 1e-2)
        norm = float(fsdp.clip_grad_norm_(0.05))
        for u in fsdp.units:
            if not u.trainable:
                continue
            for e in u.entries:
                at = slice(e.offset, e.offset + e.numel)
                g = u.grad[at].view(e.shape).double() * min(1.0, 0.05 / (norm + 1e-6))
                p = u.master.data[at].view(e.shape).double()
                name = e.fqns[0]
                if is_hidden_matrix(name, e.shape):
                    m = u.exp_avg[at].view(e.shape).double()
                    m = m + 0.1 * (g - m)
                    move = 1e-2 * 0.2 * math.sqrt(max(e.shape)) * ns64(g + 0.9 * (m - g))
                    want[name] = (u, at, p * (1 - 1e-3) - move, NS_TOL * float(move.norm()) + 2.0**-22 * float(p.norm()))
                else:
                    m, v = rest64.get(name, (torch.zeros_like(g), torch.zeros_like(g)))
                    m, v = m + 0.1 * (g - m), 0.95 * v + 0.05 * g * g
                    rest64[name] = (m, v)
                    move = 1e-2 / (1 - 0.9 ** (step + 1)) * m / ((v / (1 - 0.95 ** (step + 1))).sqrt() + 1e-8)
                    # moments within 2^-20 of themselves after two steps, sums of differently signed m within that of
                    # the gradients; an update is at most lr * sqrt(2 steps) large
                    want[name] = (u, at, p * (1 - 1e-3) - move, 2.0**-18 * 1e-2 * math.sqrt(p.numel()) + 2.0**-22 * float(p.norm()))
        opt.step()
        torch.cuda.synchronize()
        _ext.check_status()
        assert len(want) == 7
        for name, (u, at, p, bound) in want.items():
            got = u.master.data[at]
            assert float((got.double() - p.reshape(-1)).norm()) <= bound, name
            assert torch.equal(u.full[at], got.to(param_dtype)), name
