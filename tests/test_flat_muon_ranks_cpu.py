"""FlatMuon on two ranks: the 8-bit decoder, bf16 weights, matrices of odd sizes that lie across the shards (gloo, CPU)."""

import pytest
import torch
import torch.nn as nn

from mvp_engine.models.qwen3 import build_qwen3
from mvp_engine.parallel.fsdp import NativeFSDP
from mvp_engine.parallel.optim import FlatMuon, is_hidden_matrix
from mvp_engine.testing import spawn_workers

TINY = dict(vocab_size=256, hidden_size=128, intermediate_size=256, num_attention_heads=2, num_key_value_heads=1)
LR, WD = 1e-3, 0.1


def _group(world):
    import torch.distributed as dist

    from mvp_engine.distributed.init import initialize_process_group

    if world == 1:
        return None
    initialize_process_group()
    return dist.group.WORLD


def _decoder(rank, world, port, precision):
    """One step; a rank's rows one at a time, so that 8-bit blocks hold the same tokens whatever the number of ranks."""
    group = _group(world)
    model = build_qwen3("mvp/qwen3-tiny", seed=3, **TINY)
    model.set_linear_precision(precision)
    fsdp = NativeFSDP(model, group=group, device=torch.device("cpu"), param_dtype=torch.float32)
    opt = FlatMuon(fsdp, lr=LR, weight_decay=WD)
    x = torch.randint(0, 256, (2, 48), generator=torch.Generator().manual_seed(5))
    for row in range(2):
        if world == 1 or row == rank:
            (fsdp(input_ids=x[row:row + 1], labels=x[row:row + 1])["loss"].sum() / 47).backward()
    if world == 1:
        fsdp.scale_gradients_(0.5)
    fsdp.clip_grad_norm_(1.0)
    opt.step()
    return {k: v.clone() for k, v in fsdp.checkpoint_state_dict(full=True).items()}


@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_every_matrix_of_a_layer_moves_the_same_on_two_ranks(precision):
    single = _decoder(0, 1, 0, precision)
    multi = spawn_workers(_decoder, 2, precision)
    start = build_qwen3("mvp/qwen3-tiny", seed=3, **TINY).state_dict()
    seen = 0
    for k, v in single.items():
        assert torch.equal(multi[0][k], multi[1][k])
        if not is_hidden_matrix(k, v.shape):
            continue
        moved = float((v - start[k] * (1 - LR * WD)).norm())
        # an orthogonalised update of a gradient of 94 tokens: at least 94 of 128 singular values, of 0.6 to 1.25 x lr x ratio
        assert moved >= 0.4 * LR * 0.2 * max(v.shape) ** 0.5 * min(v.shape) ** 0.5, k
        # the sum over the ranks and the norm are taken in another order: about 1e-6 of a gradient, at most 485 times in
        # five iterations, and fp32's rounding of the weight
        assert float((v - multi[0][k]).norm()) <= 1e-3 * moved + 2.0**-23 * float(v.norm()), k
        seen += 1
    assert seen == 14


def _odd(rank, world, port, dtype, steps):
    group = _group(world)
    torch.manual_seed(3)
    model = nn.Sequential(nn.Linear(33, 31), nn.GELU(), nn.Linear(31, 7), nn.Linear(7, 35, bias=False), nn.LayerNorm(35),
                          nn.Linear(35, 90))
    fsdp = NativeFSDP(model, group=group, device=torch.device("cpu"), param_dtype=dtype)
    opt = FlatMuon(fsdp, lr=LR, weight_decay=WD)
    straddle = [e.fqns[0] for u in fsdp.units for e in opt._matrices[id(u)]
                if e.offset < u.shard * (world - 1) < e.offset + e.numel] if world > 1 else []
    for step in range(steps):
        for r in range(2):
            g = torch.Generator().manual_seed(100 * step + r)
            for u in fsdp.units:
                for e in u.entries:
                    part = torch.randn(e.numel, generator=g) * 1e-2
                    if world == 1 or r == rank:
                        u.grad[e.offset:e.offset + e.numel].add_(part)
        if world == 1:
            fsdp.scale_gradients_(0.5)
        fsdp.clip_grad_norm_(0.05)
        opt.step()
        for u in fsdp.units:
            if u.trainable:
                own = u.own_compute_slice(rank)
                assert own.dtype == dtype and torch.equal(own, u.master.data.to(dtype))
    full = torch.cat([u.full for u in fsdp.units])  # what the next forward multiplies by
    return {k: v.clone() for k, v in fsdp.checkpoint_state_dict(full=True).items()}, full, straddle


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_that_the_next_step_uses_follow_the_masters(dtype):
    after, full, _ = _odd(0, 1, 0, dtype, 2)
    ranks = spawn_workers(_odd, 2, dtype, 2)
    assert ranks[0][2]  # a matrix lies across both shards
    assert torch.equal(ranks[0][1], ranks[1][1])
    for k, v in after.items():
        for got, _, _ in ranks:
            # per step at most 1e-3 of an update of lr x ratio x singular value, as above; AdamW's updates are at most lr each
            bound = 2e-3 * LR * 1.25 * (max(v.shape) * v.numel()) ** 0.5 + 2.0**-22 * float(v.norm())
            assert float((got[k] - v).norm()) <= bound, k
    for u_full in (full, ranks[0][1]):
        assert u_full.dtype == dtype and bool(torch.isfinite(u_full.float()).all())
