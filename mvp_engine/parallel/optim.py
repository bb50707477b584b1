"""AdamW over the native data-parallel runtime's flat fp32 shards.

One fused kernel per unit does: gradient x (token-normalisation scale) x
(global-norm clip coefficient, computed on device from the all-reduced sum of
squares), decoupled weight decay, the Adam moments, and writes the bf16 copy
of the new weights straight into this rank's slice of the unit's compute
buffer, from where the next step's all-gather starts.  The update rule is
torch.optim.AdamW's single-tensor path, so results match the reference's
optimizer (reference: mvp_engine/kit/optim/__init__.py:11-35).

``param_groups`` behave like any torch optimizer's, so learning-rate
schedulers (e.g. transformers' cosine schedule) drive it unchanged.
"""

from __future__ import annotations

from typing import Any, Callable, Optional, Sequence

import torch
import torch.nn as nn

from .. import ops
from .fsdp import _ALIGN, NativeFSDP


class FlatAdamW(torch.optim.Optimizer):
    def __init__(self, fsdp: NativeFSDP, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, **unused: Any) -> None:
        self.fsdp = fsdp
        self.units = [u for u in fsdp.units if u.trainable]
        params = [u.master for u in self.units]
        if not params:
            raise ValueError("No trainable parameters found.")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self._step_count = 0
        self._mvp_native_step = True

    @torch.no_grad()
    def step(self, closure: Optional[Any] = None):
        loss = closure() if closure is not None else None
        f = self.fsdp
        f.finish_grad_sync()
        self._step_count += 1
        g = self.param_groups[0]
        b1, b2 = g["betas"]
        for u in self.units:
            own = u.own_compute_slice(f.rank)
            shadow = own if own.dtype == torch.bfloat16 else None
            ops.adamw_step_(u.master.data, u.grad_shard[: u.shard], u.exp_avg, u.exp_avg_sq, lr=float(g["lr"]), beta1=b1, beta2=b2,
                            eps=float(g["eps"]), weight_decay=float(g["weight_decay"]), step=self._step_count,
                            grad_scale=f._grad_scale, norm_sq=f._norm_sq,
                            max_norm=f._max_norm if f._max_norm is not None else 0.0, p_bf16=shadow)
            if shadow is None:
                own.copy_(u.master.to(own.dtype))
        f.after_optimizer_step()
        return loss

    def zero_grad(self, set_to_none: bool = True) -> None:
        """Gradient buffers are cleared by the runtime right after each update."""

    # ------------------------------------------------------- checkpoints
    def _group_meta(self, fqns: list[str]) -> dict[str, Any]:
        """The param-group entry torch.optim.AdamW of this torch version writes (same keys, so checkpoints
        load into either runtime), with this optimizer's hyper-parameters."""
        g = self.param_groups[0]
        meta = {k: v for k, v in torch.optim.AdamW([torch.zeros(1)]).param_groups[0].items() if k != "params"}
        meta.update(lr=g["lr"], betas=g["betas"], eps=g["eps"], weight_decay=g["weight_decay"], params=fqns)
        if "initial_lr" in g:  # present once a learning-rate scheduler drives the optimizer, as in torch
            meta["initial_lr"] = g["initial_lr"]
        return meta

    def checkpoint_state_dict(self, full: bool = False) -> dict[str, Any]:
        """``{"state": {fqn: {step, exp_avg, exp_avg_sq}}, "param_groups": [...]}`` keyed by HF names."""
        state: dict[str, Any] = {}
        names: list[str] = []
        step = torch.tensor(float(self._step_count))
        for fqns, avg, sq in self.fsdp.optimizer_state_views(full=full):
            for fqn in fqns[:1]:
                state[fqn] = {"step": step.clone(), "exp_avg": avg, "exp_avg_sq": sq}
                names.append(fqn)
        return {"state": state, "param_groups": [self._group_meta(names)]}

    def load_checkpoint_state_dict(self, sd: dict[str, Any], full: bool = False) -> None:
        state = sd.get("state", {})
        self.fsdp.load_optimizer_views(state)
        self._check_second_moments()
        steps = [v["step"] for v in state.values() if isinstance(v, dict) and "step" in v]
        if steps:
            self._step_count = int(float(steps[0]))
        groups = sd.get("param_groups") or []
        if groups:
            for k in ("lr", "betas", "eps", "weight_decay", "initial_lr"):
                if k in groups[0]:
                    self.param_groups[0][k] = groups[0][k]

    @torch.no_grad()
    def _check_second_moments(self) -> None:
        """Refuse first moments without second ones (a :class:`FlatMuon` checkpoint): AdamW would divide by their root.
        The moments are then those of a fresh optimizer.

        Every rank takes part and all refuse together.  First moments below 1e-15 prove nothing, their squares may have
        underflowed."""
        f = self.fsdp
        names = [(u, e) for u in self.units for e in u.entries if self._has_second_moment(u, e)]
        seen = torch.zeros(len(names), 2, device=f.device)
        for i, (u, e) in enumerate(names):
            lo, hi = u.local_range(f.rank)
            a, b = max(e.offset, lo) - lo, min(e.offset + e.numel, hi) - lo
            if a < b:
                seen[i, 0], seen[i, 1] = u.exp_avg[a:b].abs().max(), u.exp_avg_sq[a:b].max()
        for group, world in ((f.group, f.world), (f.tp_group, f.tp_world)):
            if world > 1:
                torch.distributed.all_reduce(seen, op=torch.distributed.ReduceOp.MAX, group=group)
        first, second = seen.cpu().unbind(1)
        bad = [e.fqns[0] for (_, e), x, y in zip(names, first.tolist(), second.tolist()) if x > 1e-15 and y == 0.0]
        if bad:
            for u in self.units:
                u.exp_avg.zero_()
                u.exp_avg_sq.zero_()
            raise ValueError(f"{type(self).__name__}: the checkpoint holds no second moments of {bad[0]} and {len(bad) - 1} more "
                             "parameters; Muon wrote it (resume with Muon and the same matrix_filter, or load the model alone)")

    def _has_second_moment(self, u: Any, e: Any) -> bool:
        """Whether AdamW updates this entry."""
        return True


def is_hidden_matrix(fqn: str, shape: Sequence[int]) -> bool:
    """The parameters :class:`FlatMuon` orthogonalises by default: matrices other than embeddings and output heads, which
    are told by their names (``embed``, ``head``, ``classifier``; a head under another name needs ``matrix_filter``)."""
    return len(shape) == 2 and not any(k in fqn for k in ("embed", "lm_head", "head.weight", "classifier"))


def _is_hidden_entry(e: Any) -> bool:
    """:func:`is_hidden_matrix` under every name of a parameter, none of whose owners is an embedding module."""
    return (all(is_hidden_matrix(f, tuple(e.shape)) for f in e.fqns) and
            not any(isinstance(mod, nn.Embedding) for mod, _ in e.owners))


class FlatMuon(FlatAdamW):
    """Muon over the native data-parallel runtime: hidden matrices take orthogonalised momentum updates
    (``ops.muon_step_``), everything else (embeddings, the head, norms, biases) the fused AdamW update.

    ``lr``, ``weight_decay``, ``momentum``, ``nesterov``, ``ns_coefficients``, ``eps``, ``ns_steps`` and
    ``adjust_lr_fn`` are those of ``torch.optim.Muon``, except that ``adjust_lr_fn`` defaults to
    ``"match_rms_adamw"``, since one learning rate drives both kinds; ``adamw_lr_ratio`` scales it for the AdamW part,
    whose other settings are ``betas`` and ``adamw_eps``.  ``matrix_filter(fqn, shape)`` decides which matrices are
    orthogonalised (default: :func:`is_hidden_matrix`, and no weight of an ``nn.Embedding``).

    On one rank the matrices of one shape go through the kernels together, momentum, products and the new bf16 weights
    in one chain.  Across ranks a matrix lies in several shards: each rank updates its momentum, the unit's
    updates are gathered, and a rank orthogonalises the matrices that its shard holds a part of.  The momentum lives in
    the first AdamW moment (``exp_avg`` in checkpoints); the second stays zero for matrices, also when an AdamW checkpoint
    is loaded, and :class:`FlatAdamW` refuses such a checkpoint.  Matrices split over a tensor-parallel group are not supported.
    """

    def __init__(self, fsdp: NativeFSDP, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95,
                 nesterov: bool = True, ns_coefficients: Sequence[float] = ops.NS_COEFFICIENTS, eps: float = ops.NS_EPS,
                 ns_steps: int = ops.NS_STEPS, adjust_lr_fn: Optional[str] = "match_rms_adamw",
                 betas: tuple[float, float] = (0.9, 0.95), adamw_eps: float = 1e-8, adamw_lr_ratio: float = 1.0,
                 matrix_filter: Optional[Callable[[str, Sequence[int]], bool]] = None) -> None:
        if fsdp.tp_world > 1:
            raise ValueError("FlatMuon: matrices split over a tensor-parallel group are not supported")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"FlatMuon: momentum must be in [0, 1), got {momentum}")
        ops.muon_lr_ratio(1, 1, adjust_lr_fn)  # refuses unknown names
        super().__init__(fsdp, lr=lr, betas=betas, eps=adamw_eps, weight_decay=weight_decay)
        self.param_groups[0].update(momentum=momentum, nesterov=nesterov, ns_eps=eps)
        self._ns = dict(steps=int(ns_steps), coefficients=tuple(float(c) for c in ns_coefficients))
        self._adjust = adjust_lr_fn
        self._adamw_lr_ratio = float(adamw_lr_ratio)
        keep = _is_hidden_entry if matrix_filter is None else lambda e: matrix_filter(e.fqns[0], tuple(e.shape))
        self._matrices = {id(u): [e for e in u.entries if len(e.shape) == 2 and e.numel and keep(e)] for u in self.units}

    def _rest(self, u: Any) -> list[tuple[int, int]]:
        """The ranges of a unit's flat buffer that AdamW updates: what lies between the matrices.  A matrix ends
        with the padding behind it (always zero), so a range starts where an entry does, aligned."""
        out, at = [], 0
        for e in sorted(self._matrices[id(u)], key=lambda e: e.offset):
            if e.offset > at:
                out.append((at, e.offset))
            at = e.offset + -(-e.numel // _ALIGN) * _ALIGN
        if at < u.padded:
            out.append((at, u.padded))
        return out

    @torch.no_grad()
    def step(self, closure: Optional[Any] = None):
        loss = closure() if closure is not None else None
        f = self.fsdp
        f.finish_grad_sync()
        self._step_count += 1
        g = self.param_groups[0]
        b1, b2 = g["betas"]
        lr, wd = float(g["lr"]), float(g["weight_decay"])
        clip = dict(grad_scale=f._grad_scale, norm_sq=f._norm_sq,
                    max_norm=f._max_norm if f._max_norm is not None else 0.0)
        stacks: dict[tuple[int, ...], list[tuple]] = {}
        for u in self.units:
            lo, hi = u.local_range(f.rank)
            own = u.own_compute_slice(f.rank)
            master, grad = u.master.data, u.grad_shard[: u.shard]
            shadow = own if own.dtype == torch.bfloat16 else None
            for a, b in self._rest(u):
                a, b = max(a, lo) - lo, min(b, hi) - lo
                if a < b:
                    ops.adamw_step_(master[a:b], grad[a:b], u.exp_avg[a:b], u.exp_avg_sq[a:b],
                                    lr=lr * self._adamw_lr_ratio, beta1=b1, beta2=b2, eps=float(g["eps"]),
                                    weight_decay=wd, step=self._step_count,
                                    p_bf16=shadow[a:b] if shadow is not None else None, **clip)
            if f.world == 1:
                for e in self._matrices[id(u)]:
                    at = slice(e.offset, e.offset + e.numel)
                    stacks.setdefault(tuple(e.shape), []).append(
                        tuple(t[at].view(e.shape) for t in (master, grad, u.exp_avg) + ((own,) if shadow is not None else ())))
            else:
                self._sharded_step(u, master, grad, lr, wd, clip)
        for same in stacks.values():
            cols = list(zip(*same))
            ops.muon_step_(cols[0], cols[1], cols[2], lr=lr, momentum=float(g["momentum"]), nesterov=bool(g["nesterov"]),
                           weight_decay=wd, eps=float(g["ns_eps"]), adjust_lr=self._adjust,
                           p_bf16=cols[3] if len(cols) > 3 else None, **self._ns, **clip)
        for u in self.units:
            own = u.own_compute_slice(f.rank)
            lo, _ = u.local_range(f.rank)
            if own.dtype != torch.bfloat16:
                own.copy_(u.master.to(own.dtype))
            elif f.world > 1:  # the matrices' part; AdamW has written its own
                for e in self._matrices[id(u)]:
                    a, b = max(e.offset - lo, 0), min(e.offset + e.numel - lo, u.shard)
                    if a < b:
                        own[a:b].copy_(u.master.data[a:b])
        f.after_optimizer_step()
        return loss

    def _sharded_step(self, u: Any, master: torch.Tensor, grad: torch.Tensor, lr: float, wd: float,
                      clip: dict[str, Any]) -> None:
        """Muon on a unit whose matrices lie across the shards of the data-parallel group."""
        if not self._matrices[id(u)]:
            return
        f, g = self.fsdp, self.param_groups[0]
        mu = float(g["momentum"])
        scale: Any = clip["grad_scale"]
        if clip["norm_sq"] is not None:  # on the device: no synchronisation
            scale = scale * (clip["max_norm"] / (clip["norm_sq"].sqrt() * scale + 1e-6)).clamp(max=1.0)
        lo, _ = u.local_range(f.rank)
        update = torch.zeros(u.shard, dtype=torch.float32, device=master.device)
        for e in self._matrices[id(u)]:
            a, b = max(e.offset - lo, 0), min(e.offset + e.numel - lo, u.shard)
            if a < b:
                ga, m = grad[a:b] * scale, u.exp_avg[a:b]
                m.lerp_(ga, 1 - mu)
                update[a:b] = ga.lerp(m, mu) if g["nesterov"] else m
        full = f._full_fp32(u, update)
        for e in self._matrices[id(u)]:
            a, b = max(e.offset - lo, 0), min(e.offset + e.numel - lo, u.shard)
            if a >= b:
                continue
            o = ops.orthogonalize(full[e.offset:e.offset + e.numel].view(e.shape), eps=float(g["ns_eps"]),
                                  out_dtype=torch.float32, **self._ns)
            part = o.view(-1)[lo + a - e.offset:lo + b - e.offset]
            master[a:b].mul_(1.0 - lr * wd).add_(part, alpha=-lr * ops.muon_lr_ratio(*e.shape, self._adjust))

    def load_checkpoint_state_dict(self, sd: dict[str, Any], full: bool = False) -> None:
        super().load_checkpoint_state_dict(sd, full)
        for u in self.units:  # an AdamW checkpoint's second moments of what Muon updates
            lo, hi = u.local_range(self.fsdp.rank)
            for e in self._matrices[id(u)]:
                a, b = max(e.offset, lo) - lo, min(e.offset + e.numel, hi) - lo
                if a < b:
                    u.exp_avg_sq[a:b].zero_()
        groups = sd.get("param_groups") or []
        if groups:
            for k in ("momentum", "nesterov", "ns_eps"):
                if k in groups[0]:
                    self.param_groups[0][k] = groups[0][k]

    def _has_second_moment(self, u: Any, e: Any) -> bool:
        return not any(e is m for m in self._matrices[id(u)])

    def _group_meta(self, fqns: list[str]) -> dict[str, Any]:
        g = self.param_groups[0]
        return {**super()._group_meta(fqns), "momentum": g["momentum"], "nesterov": g["nesterov"], "ns_eps": g["ns_eps"]}
