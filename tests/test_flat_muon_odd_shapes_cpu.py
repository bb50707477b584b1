"""FlatMuon on modules of odd widths, on CPU: the ranges left to AdamW."""

import pytest
import torch
import torch.nn as nn

from mvp_engine.parallel.fsdp import _ALIGN, NativeFSDP
from mvp_engine.parallel.optim import FlatMuon


def odd_model():
    """Matrices whose sizes are no multiple of four, each followed by a bias."""
    torch.manual_seed(3)
    return nn.Sequential(nn.Linear(33, 31), nn.GELU(), nn.Linear(31, 7), nn.Linear(7, 35, bias=False), nn.LayerNorm(35))


@pytest.mark.parametrize("make", [odd_model, lambda: nn.Linear(33, 35), lambda: nn.Linear(1, 1),
                                  lambda: nn.Linear(64, 64, bias=False)])
def test_ranges_of_adamw_start_aligned_and_cover_the_rest(make):
    fsdp = NativeFSDP(make(), group=None, device=torch.device("cpu"), param_dtype=torch.float32)
    opt = FlatMuon(fsdp, lr=1e-3)
    for u in fsdp.units:
        if not u.trainable:
            continue
        covered = torch.zeros(u.padded, dtype=torch.int32)
        for a, b in opt._rest(u):
            assert a % _ALIGN == 0 and a < b <= u.padded
            covered[a:b] += 1
        for e in u.entries:
            want = 0 if any(e is m for m in opt._matrices[id(u)]) else 1
            assert bool((covered[e.offset:e.offset + e.numel] == want).all()), e.fqns
        assert int(covered.max()) <= 1
