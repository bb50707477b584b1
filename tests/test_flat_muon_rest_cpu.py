"""What FlatMuon leaves to AdamW, with the gradient clip active: as FlatAdamW and as torch's own AdamW move it."""

import torch

from mvp_engine.models.qwen3 import build_qwen3
from mvp_engine.parallel.fsdp import NativeFSDP
from mvp_engine.parallel.optim import FlatAdamW, FlatMuon, is_hidden_matrix

TINY = dict(vocab_size=256, hidden_size=128, intermediate_size=256, num_attention_heads=2, num_key_value_heads=1)
HYPER = dict(lr=1e-3, weight_decay=0.1, betas=(0.9, 0.95))
STEPS, MAX_NORM = 3, 0.5


def gradients(step, named):
    g = torch.Generator().manual_seed(step)
    return {n: torch.randn(tuple(s), generator=g) * 1e-2 for n, s in named}


def run(cls):
    fsdp = NativeFSDP(build_qwen3("mvp/qwen3-tiny", seed=3, **TINY), group=None, device=torch.device("cpu"),
                      param_dtype=torch.float32)
    opt = cls(fsdp, **HYPER)
    entries = {e.fqns[0]: (u, e) for u in fsdp.units for e in u.entries}
    for step in range(STEPS):
        for n, grad in gradients(step, [(n, e.shape) for n, (_, e) in sorted(entries.items())]).items():
            u, e = entries[n]
            u.grad[e.offset:e.offset + e.numel].copy_(grad.view(-1))
        assert float(fsdp.clip_grad_norm_(MAX_NORM)) > 2 * MAX_NORM  # the clip does something
        opt.step()
    return fsdp.checkpoint_state_dict(full=True)


def test_rest_moves_as_adamw_moves_it_under_the_clip():
    muon, adamw = run(FlatMuon), run(FlatAdamW)
    plain = build_qwen3("mvp/qwen3-tiny", seed=3, **TINY)
    params = dict(plain.named_parameters())
    opt = torch.optim.AdamW(params.values(), eps=1e-8, **HYPER)
    for step in range(STEPS):
        for n, grad in gradients(step, [(n, params[n].shape) for n in sorted(params)]).items():
            params[n].grad = grad
        torch.nn.utils.clip_grad_norm_(params.values(), MAX_NORM)
        opt.step()
    rest = [n for n in params if not is_hidden_matrix(n, params[n].shape)]
    assert len(rest) == len(params) - 14
    for n in rest:
        assert torch.equal(muon[n], adamw[n]), n
        # the coefficient in another order, some 20 roundings of updates that are at most lr x 2 large, and the weight's own
        assert bool(((muon[n] - params[n].detach()).abs() <= STEPS * (20 * 2.0**-24 * 2e-3 + 2.0**-23 * muon[n].abs())).all()), n
    for n in set(params) - set(rest):
        assert not torch.equal(muon[n], adamw[n])
