"""Orthogonalised matrix updates (Newton-Schulz) and the Muon optimizer step.

The arguments carry the names, the order and the defaults of ``torch.optim.Muon``.  On CUDA both operators run
the fp16 tensor-core kernels of ``csrc/muon_sm100.cu``; on CPU the same formulas run in 32 bits.
"""

from __future__ import annotations

import functools
import math
from typing import Optional, Sequence, Union

import torch

from . import _ext

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _check_iteration(steps: int, coefficients: Sequence[float], eps: float) -> tuple[int, tuple[float, ...], float]:
    """Refuse iterations whose singular values leave the range the kernels' fp16 products are scaled for."""
    return _checked(int(steps), tuple(float(c) for c in coefficients), float(eps))


@functools.lru_cache(maxsize=64)
def _checked(steps: int, coef: tuple[float, ...], eps: float) -> tuple[int, tuple[float, ...], float]:
    if not 1 <= steps <= 1000:
        raise ValueError(f"orthogonalize: steps must be in 1 .. 1000, got {steps}")
    if len(coef) != 3 or not all(math.isfinite(c) for c in coef):
        raise ValueError(f"orthogonalize: three finite coefficients are needed, got {coef!r}")
    if not 1e-100 <= eps <= 1e30:
        raise ValueError(f"orthogonalize: eps must be in 1e-100 .. 1e30, got {eps!r}")
    a, b, c = coef
    top = 1.0  # singular values lie in [0, top]; the Frobenius norm of the first X is at most 1
    for _ in range(min(steps, 64)):
        # extrema of a s + b s^3 + c s^5 on [0, top] and of b t + c t^2 on [0, top^2]
        points = [top]
        disc = 9 * b * b - 20 * a * c
        if c != 0 and disc >= 0:
            points += [math.sqrt(t) for r in (1, -1) if 0 < (t := (-3 * b + r * math.sqrt(disc)) / (10 * c)) < top * top]
        elif c == 0 and b != 0 and 0 < -a / (3 * b) < top * top:
            points.append(math.sqrt(-a / (3 * b)))
        inner = [top * top]
        if c != 0 and 0 < -b / (2 * c) < top * top:
            inner.append(-b / (2 * c))
        if max(abs(b * t + c * t * t) for t in inner) > 3.9:
            raise ValueError(f"orthogonalize: coefficients {coef} leave the range of the iteration")
        top = max(abs(a * s + b * s**3 + c * s**5) for s in points) * 1.001  # the kernels' rounding
        if top > 1.9:
            raise ValueError(f"orthogonalize: coefficients {coef} let singular values grow to {top:.3g}; "
                             "at most 1.9 is supported")
        top = max(top, 1e-6)
    return steps, coef, eps


def _newton_schulz(u: torch.Tensor, steps: int, coefficients: Sequence[float], eps: float) -> torch.Tensor:
    a, b, c = coefficients
    norm = u.double().square().sum(dim=(-2, -1), keepdim=True).sqrt()
    x = (u.double() / norm.clamp(min=eps)).float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if tall else x


def orthogonalize(x: torch.Tensor, *, steps: int = NS_STEPS, coefficients: Sequence[float] = NS_COEFFICIENTS,
                  eps: float = NS_EPS, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Bring the singular values of each matrix of ``x [..., m, n]`` near 1 (``U V^T`` of its SVD, roughly).

    ``X = x / max(|x|_F, eps)``, then ``steps`` times ``X <- a X + (b A + c A A) X`` with ``A = X X^T`` over the
    shorter side.  ``x`` is fp32, bf16 or fp16; the result has ``out_dtype`` (one of the three).  On CUDA it is within
    0.3 % (Frobenius) of 64-bit arithmetic plus its own rounding in up to five steps (an fp32 result of sides up to 256, the
    shorter up to 64: 0.03 %), and ``sqrt(steps / 5)`` times that in more, where ``|x|_F`` is at least ``1e-4 eps``.  Smaller
    matrices, whose first X is that far below 1, keep fewer bits of fp16: what they lose is below 3e-5 (Frobenius, five steps
    of the default coefficients).  A matrix with a value that is not finite comes back as NaN, a zero matrix as zeros.  No
    gradient is defined.
    """
    if x.dim() < 2:
        raise ValueError(f"orthogonalize: matrices are needed, got shape {tuple(x.shape)}")
    if x.dtype not in _FLOATS or out_dtype not in _FLOATS:
        raise TypeError(f"orthogonalize: fp32, bf16 or fp16 values, got {x.dtype} -> {out_dtype}")
    steps, coef, eps = _check_iteration(steps, coefficients, eps)
    x = x.detach()
    from . import _native

    if not _native(x):
        return _newton_schulz(x, steps, coef, eps).to(out_dtype).contiguous()
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    if x.numel():
        m, n = x.shape[-2:]
        _ext.ext().orthogonalize(x.reshape(-1, m, n).contiguous(), out.view(-1, m, n), steps, coef, eps,
                                 _ext.status_buffer(x.device).data_ptr())
    return out


Matrices = Union[torch.Tensor, Sequence[torch.Tensor]]


def _as_list(name: str, t: Matrices, count: Optional[int] = None) -> list[torch.Tensor]:
    ts = [t] if isinstance(t, torch.Tensor) else list(t)
    if not all(isinstance(v, torch.Tensor) and v.dim() == 2 for v in ts):
        raise ValueError(f"muon_step_: {name} must be matrices")
    if count is not None and len(ts) != count:
        raise ValueError(f"muon_step_: {len(ts)} tensors in {name} for {count} weights")
    return ts


def muon_lr_ratio(rows: int, cols: int, adjust_lr: Optional[str] = None) -> float:
    """The factor on the learning rate of a ``[rows, cols]`` matrix: ``"original"`` (or None)
    ``sqrt(max(1, rows / cols))``, ``"match_rms_adamw"`` ``0.2 sqrt(max(rows, cols))``."""
    if adjust_lr is None or adjust_lr == "original":
        return math.sqrt(max(1.0, rows / cols))
    if adjust_lr == "match_rms_adamw":
        return 0.2 * math.sqrt(max(rows, cols))
    raise ValueError(f"muon: adjust_lr must be 'original' or 'match_rms_adamw', got {adjust_lr!r}")


def muon_step_(
    p: Matrices,
    g: Matrices,
    m: Matrices,
    *,
    lr: float,
    momentum: float = 0.95,
    nesterov: bool = True,
    weight_decay: float = 0.1,
    steps: int = NS_STEPS,
    coefficients: Sequence[float] = NS_COEFFICIENTS,
    eps: float = NS_EPS,
    adjust_lr: Optional[str] = None,
    grad_scale: float = 1.0,
    norm_sq: Optional[torch.Tensor] = None,
    max_norm: float = 0.0,
    p_bf16: Optional[Matrices] = None,
) -> None:
    """One Muon step on a matrix, or on a list of matrices of one shape (one launch per product for all).

    ``m <- m + (1 - momentum) (g - m)``, ``u = g + momentum (m - g)`` (or ``m`` without ``nesterov``),
    ``p <- p (1 - lr weight_decay) - lr ratio orthogonalize(u)`` with the ratio of :func:`muon_lr_ratio`.
    ``p``, ``g`` and ``m`` are contiguous fp32; ``p_bf16`` (optional) receives the new weights in bf16.  The gradient is
    scaled by ``grad_scale`` and, when ``norm_sq`` is given, by the clip coefficient, as in :func:`adamw_step_`.
    Matrices must not overlap one another.
    """
    ps = _as_list("p", p)
    if not ps:
        return
    gs, ms = _as_list("g", g, len(ps)), _as_list("m", m, len(ps))
    shadows = [] if p_bf16 is None else _as_list("p_bf16", p_bf16, len(ps))
    shape, dev = ps[0].shape, ps[0].device
    for name, ts, dt in (("p", ps, torch.float32), ("g", gs, torch.float32), ("m", ms, torch.float32),
                         ("p_bf16", shadows, torch.bfloat16)):
        for t in ts:
            if t.shape != shape or t.dtype != dt or t.device != dev or not t.is_contiguous():
                raise ValueError(f"muon_step_: {name} must be contiguous {dt} matrices of shape {tuple(shape)} on {dev}, "
                                 f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    steps, coef, eps = _check_iteration(steps, coefficients, eps)
    if ps[0].numel() == 0:
        return
    ptrs = [t.data_ptr() for t in ps + ms + shadows]
    if len(set(ptrs)) != len(ptrs) or not set(ptrs).isdisjoint(t.data_ptr() for t in gs):
        raise ValueError("muon_step_: a weight, momentum or bf16 copy is given twice, or as a gradient")
    rate = float(lr) * muon_lr_ratio(shape[0], shape[1], adjust_lr)
    decay = 1.0 - float(lr) * float(weight_decay)
    from . import _native

    with torch.no_grad():
        if _native(ps[0]):
            _ext.ext().muon_step_([t.detach() for t in ps], [t.detach() for t in gs], ms, shadows, rate, decay,
                                  float(momentum), bool(nesterov), steps, coef, eps, float(grad_scale), norm_sq,
                                  float(max_norm), _ext.status_buffer(dev).data_ptr())
            return
        scale = float(grad_scale)
        if norm_sq is not None:
            clip = float(max_norm) / (float(norm_sq.sqrt()) * scale + 1e-6)
            scale *= 1.0 if clip > 1.0 else clip  # a norm that is not a number reaches the weights
        for i, w in enumerate(ps):
            gi = gs[i] * scale
            ms[i].lerp_(gi, 1 - momentum)
            u = gi.lerp(ms[i], momentum) if nesterov else ms[i]
            w.mul_(decay).add_(_newton_schulz(u, steps, coef, eps), alpha=-rate)
            if shadows:
                shadows[i].copy_(w)
