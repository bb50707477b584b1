"""FlatMuon's arguments: a name that it does not know is an error, not a setting that has no effect."""

import pytest
import torch
import torch.nn as nn

from mvp_engine.kit.optim import OptimKit
from mvp_engine.parallel.fsdp import NativeFSDP


@pytest.mark.parametrize("bad", [{"momentun": 0.9}, {"beta": (0.9, 0.99)}, {"adam_eps": 1e-6}, {"fused": True}])
def test_unknown_arguments_are_refused(bad):
    fsdp = NativeFSDP(nn.Linear(8, 8), group=None, device=torch.device("cpu"), param_dtype=torch.float32)
    with pytest.raises(TypeError, match=next(iter(bad))):
        OptimKit().build_optimizer(fsdp, "Muon", lr=1e-3, weight_decay=0.1, **bad)


def test_known_arguments_reach_the_step():
    fsdp = NativeFSDP(nn.Linear(8, 8), group=None, device=torch.device("cpu"), param_dtype=torch.float32)
    opt = OptimKit().build_optimizer(fsdp, "Muon", lr=1e-3, weight_decay=0.1, momentum=0.8, nesterov=False,
                                     ns_coefficients=(2.0, -1.5, 0.5), eps=1e-6, ns_steps=7, adjust_lr_fn="original",
                                     betas=(0.8, 0.9), adamw_eps=1e-7, adamw_lr_ratio=0.5, matrix_filter=lambda f, s: False)
    g = opt.param_groups[0]
    assert (g["momentum"], g["nesterov"], g["ns_eps"], g["eps"], g["betas"]) == (0.8, False, 1e-6, 1e-7, (0.8, 0.9))
    assert opt._ns == {"steps": 7, "coefficients": (2.0, -1.5, 0.5)} and opt._adjust == "original"
    assert opt._adamw_lr_ratio == 0.5 and not any(opt._matrices.values())
