"""The 8-bit decoder with resharded weights and recomputed layers on two ranks (gloo): the same weights as resident ones."""

import torch

from mvp_engine.models.qwen3 import build_qwen3
from mvp_engine.parallel.fsdp import NativeFSDP
from mvp_engine.parallel.optim import FlatMuon
from mvp_engine.testing import spawn_workers

TINY = dict(vocab_size=256, hidden_size=128, intermediate_size=256, num_hidden_layers=3, num_attention_heads=2,
            num_key_value_heads=1)


def _train(rank, world, port, reshard, ckpt):
    import torch.distributed as dist

    from mvp_engine.distributed.init import initialize_process_group

    initialize_process_group()
    model = build_qwen3("mvp/qwen3-tiny", seed=3, **TINY)
    model.set_linear_precision("fp8")
    if ckpt:
        model.gradient_checkpointing_enable()
    fsdp = NativeFSDP(model, group=dist.group.WORLD, device=torch.device("cpu"), param_dtype=torch.bfloat16,
                      reshard_after_forward=reshard)
    fsdp.train()
    opt = FlatMuon(fsdp, lr=1e-3)
    g = torch.Generator().manual_seed(5)
    for _ in range(2):
        x = torch.randint(0, 256, (2, 48), generator=g)[rank:rank + 1]
        (fsdp(input_ids=x, labels=x)["loss"].sum() / 47).backward()
        fsdp.clip_grad_norm_(1.0)
        opt.step()
        for u in fsdp.units:
            assert torch.equal(u.own_compute_slice(rank), u.master.data.to(torch.bfloat16))
    return {k: v.clone() for k, v in fsdp.checkpoint_state_dict(full=True).items()}


def test_resharded_and_recomputed_layers_give_the_same_weights():
    resident = spawn_workers(_train, 2, False, False)[0]
    for got in spawn_workers(_train, 2, True, True):
        for k, v in resident.items():
            assert torch.equal(got[k], v), k
