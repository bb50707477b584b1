"""Checkpoints of FlatMuon and FlatAdamW loaded into one another: whole files and DCP shards, one and two ranks (gloo)."""

import pytest
import torch

from mvp_engine.models.qwen3 import build_qwen3
from mvp_engine.parallel import optim
from mvp_engine.parallel.fsdp import NativeFSDP
from mvp_engine.testing import spawn_workers

TINY = dict(vocab_size=64, hidden_size=64, intermediate_size=128, num_hidden_layers=1, num_attention_heads=1,
            num_key_value_heads=1)


def build(cls, group=None, mesh=None):
    fsdp = NativeFSDP(build_qwen3("mvp/qwen3-tiny", seed=3, **TINY), group=group, device=torch.device("cpu"),
                      param_dtype=torch.float32, shard_mesh=mesh)
    return fsdp, getattr(optim, cls)(fsdp, lr=1e-3)


def steps(fsdp, opt, n):
    g = torch.Generator().manual_seed(1)
    for _ in range(n):
        x = torch.randint(0, 64, (1, 20), generator=g)
        (fsdp(input_ids=x, labels=x)["loss"].sum() / 19).backward()
        opt.step()


def _exchange(rank, world, port, wrote, reads, full):
    """What loading ``wrote``'s optimizer state into ``reads`` does."""
    import torch.distributed as dist

    from mvp_engine.distributed.init import initialize_process_group

    if world > 1:
        initialize_process_group()
    group = dist.group.WORLD if world > 1 else None
    mesh = dist.device_mesh.init_device_mesh("cpu", (world,)) if world > 1 else None
    a, oa = build(wrote, group, mesh)
    steps(a, oa, 2)
    msd, osd = a.checkpoint_state_dict(full=full), oa.checkpoint_state_dict(full=full)
    b, ob = build(reads, group, mesh)
    b.load_checkpoint_state_dict(msd, full=full)
    try:
        ob.load_checkpoint_state_dict(osd, full=full)
    except ValueError as e:
        assert not any(bool(u.exp_avg.any()) or bool(u.exp_avg_sq.any()) for u in ob.units)  # as a fresh optimizer's
        return str(e)
    if reads == "FlatMuon":
        for u in b.units:
            for e in ob._matrices[id(u)]:
                lo, hi = u.local_range(b.rank)
                assert not bool(u.exp_avg_sq[max(e.offset, lo) - lo:max(0, min(e.offset + e.numel, hi) - lo)].any())
    steps(b, ob, 1)
    return ""


@pytest.mark.parametrize("world", [1, 2])
@pytest.mark.parametrize("full", [True, False])
def test_adamw_refuses_a_muon_checkpoint_on_every_rank(world, full):
    got = ([_exchange(0, 1, 0, "FlatMuon", "FlatAdamW", full)] if world == 1 else
           spawn_workers(_exchange, world, "FlatMuon", "FlatAdamW", full))
    for message in got:
        assert "second moments" in message and "Muon" in message


@pytest.mark.parametrize("wrote,reads", [("FlatMuon", "FlatMuon"), ("FlatAdamW", "FlatAdamW"), ("FlatAdamW", "FlatMuon")])
@pytest.mark.parametrize("world", [1, 2])
def test_other_pairs_load(world, wrote, reads):
    got = ([_exchange(0, 1, 0, wrote, reads, True)] if world == 1 else spawn_workers(_exchange, world, wrote, reads, False))
    assert got == [""] * world


def test_muon_refuses_what_another_filter_orthogonalised():
    a, oa = build("FlatMuon")
    steps(a, oa, 2)
    osd = oa.checkpoint_state_dict(full=True)
    ob = optim.FlatMuon(build("FlatMuon")[0], lr=1e-3, matrix_filter=lambda fqn, shape: "mlp" in fqn)
    with pytest.raises(ValueError, match="matrix_filter"):
        ob.load_checkpoint_state_dict(osd, full=True)
    oc = optim.FlatMuon(build("FlatMuon")[0], lr=1e-3, matrix_filter=lambda fqn, shape: "norm" not in fqn)
    oc.load_checkpoint_state_dict(osd, full=True)  # more matrices than before need no second moments


def test_a_fresh_or_untouched_state_loads():
    """Zero moments on both sides, and first moments whose squares underflow."""
    a, oa = build("FlatAdamW")
    b, ob = build("FlatAdamW")
    ob.load_checkpoint_state_dict(oa.checkpoint_state_dict(full=True), full=True)
    for u in a.units:
        u.exp_avg.fill_(1e-30)
    ob.load_checkpoint_state_dict(oa.checkpoint_state_dict(full=True), full=True)
    assert float(b.units[0].exp_avg.max()) == torch.tensor(1e-30).item()


def _through_files(rank, world, port, folder, wrote, reads):
    import torch.distributed as dist

    from mvp_engine.distributed.init import initialize_process_group
    from mvp_engine.utils.checkpointing.parallel_sl_util import load_checkpoint, save_checkpoint

    initialize_process_group()
    mesh = dist.device_mesh.init_device_mesh("cpu", (world,), mesh_dim_names=("shard",))
    a, oa = build(wrote, dist.group.WORLD, mesh)
    steps(a, oa, 2)
    save_checkpoint(mesh, folder, a, oa, step=2)
    b, ob = build(reads, dist.group.WORLD, mesh)
    try:
        load_checkpoint(mesh, folder, b, ob)
    except ValueError as e:
        return str(e)
    steps(a, oa, 1)
    steps(b, ob, 1)
    return [(x, y) for x, y in zip(a.checkpoint_state_dict(full=True).values(), b.checkpoint_state_dict(full=True).values())]


@pytest.mark.parametrize("wrote,reads", [("FlatMuon", "FlatMuon"), ("FlatMuon", "FlatAdamW")])
def test_through_sharded_files(tmp_path, wrote, reads):
    for got in spawn_workers(_through_files, 2, str(tmp_path), wrote, reads):
        if reads == "FlatAdamW":
            assert "second moments" in got
        else:
            assert all(torch.equal(x, y) for x, y in got)
