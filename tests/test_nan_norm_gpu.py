"""A gradient norm that is not a number, through AdamW and through both halves of FlatMuon, on the GPU."""

import pytest
import torch
import torch.nn as nn

from mvp_engine import ops
from mvp_engine.parallel import optim
from mvp_engine.parallel.fsdp import NativeFSDP

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]


@pytest.mark.parametrize("norm,scale", [(float("nan"), float("nan")), (float("inf"), 0.0), (4.0, 0.5), (0.25, 1.0)])
@pytest.mark.parametrize("offset", [0, 1])
def test_adamw_clips_as_clip_grad_norm_does(norm, scale, offset):
    p, g, m, v = (torch.full((70,), x, device="cuda")[offset:] for x in (1.0, 2.0, 0.0, 0.0))
    ops.adamw_step_(p, g, m, v, lr=0.1, beta1=0.5, beta2=0.5, eps=1e-8, weight_decay=0.0, step=1,
                    norm_sq=torch.tensor(norm * norm, device="cuda"), max_norm=2.0)
    torch.testing.assert_close(m, torch.full_like(m, 2.0 * scale * 0.5), equal_nan=True, rtol=1e-6, atol=0)
    assert bool(torch.isnan(p).all()) == (scale != scale)


@pytest.mark.parametrize("cls", ["FlatMuon", "FlatAdamW"])
def test_one_nan_reaches_matrices_and_the_rest_alike(cls):
    torch.manual_seed(1)
    model = nn.Sequential(nn.Linear(33, 31), nn.LayerNorm(31), nn.Linear(31, 7))
    fsdp = NativeFSDP(model, group=None, device=torch.device("cuda"), param_dtype=torch.bfloat16)
    opt = getattr(optim, cls)(fsdp, lr=1e-3)
    for u in fsdp.units:
        if u.trainable:
            u.grad.fill_(0.01)
            u.grad[0] = float("nan")  # one gradient value
    fsdp.clip_grad_norm_(1.0)
    opt.step()
    after = fsdp.checkpoint_state_dict(full=True)
    assert len(after) == 6
    for name, t in after.items():
        assert bool(torch.isnan(t).all()), name
