"""A gradient norm that is not a number, through AdamW and through both halves of FlatMuon, on CPU."""

import pytest
import torch
import torch.nn as nn

from mvp_engine import ops
from mvp_engine.parallel import optim
from mvp_engine.parallel.fsdp import NativeFSDP
from mvp_engine.testing import spawn_workers


@pytest.mark.parametrize("norm,scale", [(float("nan"), float("nan")), (float("inf"), 0.0), (4.0, 0.5), (0.25, 1.0)])
def test_adamw_clips_as_clip_grad_norm_does(norm, scale):
    """The coefficient of ``clip_grad_norm_`` for each norm, NaN and infinity included."""
    p, m, v = torch.ones(5), torch.zeros(5), torch.zeros(5)
    ops.adamw_step_(p, torch.full((5,), 2.0), m, v, lr=0.1, beta1=0.5, beta2=0.5, eps=1e-8, weight_decay=0.0, step=1,
                    norm_sq=torch.tensor(norm * norm), max_norm=2.0)
    torch.testing.assert_close(m, torch.full((5,), 2.0 * scale * 0.5), equal_nan=True, rtol=1e-6, atol=0)
    assert bool(torch.isnan(p).all()) == (scale != scale)


def _step(rank, world, port, cls):
    import torch.distributed as dist

    from mvp_engine.distributed.init import initialize_process_group

    if world > 1:
        initialize_process_group()
    torch.manual_seed(1)
    model = nn.Sequential(nn.Linear(33, 31), nn.LayerNorm(31), nn.Linear(31, 7))
    fsdp = NativeFSDP(model, group=dist.group.WORLD if world > 1 else None, device=torch.device("cpu"),
                      param_dtype=torch.float32)
    opt = getattr(optim, cls)(fsdp, lr=1e-3)
    for u in fsdp.units:
        if u.trainable:
            u.grad.fill_(0.01)
            u.grad[0] = float("nan")  # one gradient value
    fsdp.clip_grad_norm_(1.0)
    opt.step()
    return fsdp.checkpoint_state_dict(full=True)


@pytest.mark.parametrize("cls", ["FlatMuon", "FlatAdamW"])
def test_one_nan_reaches_matrices_and_the_rest_alike(cls):
    for after in (_step(0, 1, 0, cls), spawn_workers(_step, 2, cls)[1]):
        assert len(after) == 6
        for name, t in after.items():
            assert bool(torch.isnan(t).all()), name
