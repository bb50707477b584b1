"""8-bit floating point matrices with a scale for each block of 128, their product, and the linear layer on it.

A block is 128 consecutive values of a row (``block="row"``: activations, gradients) or a 128 x 128 tile
(``block="tile"``: weights, whose rows and columns then share codes).  Its scale is the smallest power of two that
keeps the block within the 8-bit type's range; codes are rounded to nearest, ties to even.  On CUDA the kernels of
``csrc/fp8_sm100.cu`` run (block-scaled tcgen05 products, fp32 accumulation); on CPU the same values are computed with
plain torch operations.
"""

from __future__ import annotations

import os
from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _ext

BLOCK = 128
# largest value of each type, as a power of two times 1.75
_MAX_EXPONENT = {torch.float8_e4m3fn: 8, torch.float8_e5m2: 15}


def _native(t: torch.Tensor) -> bool:
    # as ops._native, without asking for the device that a CUDA tensor proves
    return t.is_cuda and (os.environ.get("MVP_ALLOW_EAGER", "0") != "1" or _ext.available())


class Fp8Matrix:
    """A ``[rows, cols]`` matrix in 8-bit codes with one scale per block of 128 columns of a row.

    ``data`` holds the codes, ``[rows, blocks * 128]`` (zero beyond ``cols``), in ``float8_e4m3fn`` or ``float8_e5m2``.
    ``scale`` holds the scales' exponents plus 127 as bytes, ``[rows / 128, blocks / 4, 32, 4, 4]`` (both rounded up, zero
    padded): row ``r`` and block ``k`` are at ``[r // 128, k // 4, r % 32, r // 32 % 4, k % 4]``.
    """

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, cols: int) -> None:
        self.data = data
        self.scale = scale
        self.cols = int(cols)

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    @property
    def shape(self) -> tuple[int, int]:
        return (self.rows, self.cols)

    @property
    def dtype(self) -> torch.dtype:
        return self.data.dtype

    @property
    def device(self) -> torch.device:
        return self.data.device

    def exponents(self) -> torch.Tensor:
        """The scales' exponents, int32 ``[rows, blocks]``: a value is its code times ``2 ** exponent``."""
        s = self.scale.permute(0, 3, 2, 1, 4).reshape(self.scale.shape[0] * BLOCK, -1)
        return s[: self.rows, : self.data.shape[1] // BLOCK].to(torch.int32) - 127

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the codes stand for, ``[rows, cols]``."""
        # codes are whole multiples of 2^-16, scales powers of two down to 2^-127: 64 bits hold every product
        v = self.data.to(torch.float64).view(self.rows, -1, BLOCK) * _exp2(self.exponents())[..., None]
        return v.view(self.rows, -1)[:, : self.cols].to(dtype)

    def __repr__(self) -> str:
        return f"Fp8Matrix({self.rows} x {self.cols}, {self.dtype}, {self.device})"


def _exp2(e: torch.Tensor) -> torch.Tensor:
    """``2 ** e`` in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _up(n: int, m: int) -> int:
    return -(-n // m) * m


def _pack_scale(byte: torch.Tensor) -> torch.Tensor:
    rows, blocks = byte.shape
    p = byte.new_zeros(_up(rows, BLOCK), _up(blocks, 4))
    p[:rows, :blocks] = byte
    return p.view(-1, 4, 32, p.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


def _quantize_plain(x: torch.Tensor, tile: bool, dtype: torch.dtype) -> Fp8Matrix:
    rows, cols = x.shape
    pr, pc = _up(rows, BLOCK) if tile else rows, _up(cols, BLOCK)
    v = torch.zeros(pr, pc, dtype=torch.float32, device=x.device)
    v[:rows, :cols] = x
    b = v.view(pr // BLOCK, BLOCK, pc // BLOCK, BLOCK) if tile else v.view(pr, 1, pc // BLOCK, BLOCK)
    amax = b.abs().amax(dim=(1, 3), keepdim=True)
    bad = ~torch.isfinite(amax)
    f, k = torch.frexp(torch.where(bad, torch.ones_like(amax), amax))  # f in [0.5, 1); the range is 0.875 * 2^(p + 1)
    e = k - (_MAX_EXPONENT[dtype] + 1) + (f > 0.875).to(k.dtype)
    e = torch.where(amax == 0, torch.full_like(e, -127), e.clamp(min=-127))
    e = torch.where(bad, torch.zeros_like(e), e)
    q = torch.where(bad, torch.full_like(b, float("nan")), (b.double() * _exp2(-e)).float())
    q = q.reshape(pr, pc)[:rows]
    if cols < pc:
        q[:, cols:] = 0
    byte = (e + 127).to(torch.uint8).expand(-1, BLOCK if tile else 1, -1, 1).reshape(pr, -1)[:rows]
    return Fp8Matrix(q.to(dtype), _pack_scale(byte), cols)


def quantize_fp8(x: torch.Tensor, block: str = "row", *, rows: bool = True, columns: bool = False,
                 dtype: torch.dtype = torch.float8_e4m3fn) -> tuple[Optional[Fp8Matrix], Optional[Fp8Matrix]]:
    """``(matrix, transposed)`` of ``x [R, C]`` (bf16 or fp32) in 8-bit blocks, in one pass over ``x``.

    ``rows`` asks for ``x`` itself (blocks of 128 along its rows), ``columns`` for its transpose ``[C, R]`` (blocks of
    128 along its columns); what is not asked for is ``None``.  With ``block="tile"`` both share the scales of
    128 x 128 tiles.  Zero blocks have the exponent -127; a block with a value that is not finite has NaN codes
    (within the matrix) and the exponent 0.
    """
    if block not in ("row", "tile"):
        raise ValueError(f"quantize_fp8: block must be 'row' or 'tile', got {block!r}")
    if dtype not in _MAX_EXPONENT:
        raise TypeError(f"quantize_fp8: float8_e4m3fn or float8_e5m2, got {dtype}")
    if x.dim() != 2 or x.numel() == 0:
        raise ValueError(f"quantize_fp8: a matrix with at least one value is needed, got shape {tuple(x.shape)}")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"quantize_fp8: bf16 or fp32 values, got {x.dtype}")
    if not (rows or columns):
        raise ValueError("quantize_fp8: neither rows nor columns asked for")
    if not _native(x):
        x = x.detach()
        return (_quantize_plain(x, block == "tile", dtype) if rows else None,
                _quantize_plain(x.t(), block == "tile", dtype) if columns else None)
    if x.stride(1) != 1 and x.shape[1] > 1:
        x = x.contiguous()
    q, s, t, st = _ext.ext().quantize_fp8(x, block == "tile", bool(rows), bool(columns), dtype == torch.float8_e5m2)
    return (Fp8Matrix(q, s, x.shape[1]) if rows else None, Fp8Matrix(t, st, x.shape[0]) if columns else None)


def gemm_fp8(a: Fp8Matrix, b: Fp8Matrix, *, out: Optional[torch.Tensor] = None, accumulate: bool = False,
             out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``C (+)= A B^T`` of ``a [M, K]`` and ``b [N, K]`` with fp32 accumulation; ``C`` is bf16 or fp32 (:func:`gemm`)."""
    if not isinstance(a, Fp8Matrix) or not isinstance(b, Fp8Matrix):
        raise TypeError("gemm_fp8: Fp8Matrix operands are needed")
    if a.cols != b.cols:
        raise ValueError(f"gemm_fp8: reduction sizes differ, {a.cols} and {b.cols}")
    if a.device != b.device:
        raise ValueError(f"gemm_fp8: operands on {a.device} and {b.device}")
    if out is None:
        if accumulate:
            raise ValueError("gemm_fp8: accumulate needs out")
        if out_dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"gemm_fp8: bf16 or fp32 output, got {out_dtype}")
        out = torch.empty(a.rows, b.rows, dtype=out_dtype, device=a.device)
    elif (out.shape != (a.rows, b.rows) or out.device != a.device or
          out.dtype not in (torch.bfloat16, torch.float32) or (accumulate and out.dtype != torch.float32)):
        raise ValueError(f"gemm_fp8: out must be a {a.rows} x {b.rows} bf16 or fp32 matrix on {a.device} (fp32 to "
                         f"accumulate), got {out.dtype} {tuple(out.shape)} on {out.device}")
    if not _native(a.data):
        res = a.dequantize() @ b.dequantize().t()
        out.add_(res) if accumulate else out.copy_(res)
        return out
    _ext.ext().gemm_fp8(a.data, a.scale, b.data, b.scale, a.cols, out, accumulate,
                        _ext.status_buffer(a.device).data_ptr())
    return out


def _forward(x2, w, w8, need_xt, need_wt):
    """``(y, [x^T codes, scales, w^T codes, scales])``; what is not needed is ``None``."""
    if _native(x2):
        y, *kept = _ext.ext().linear_fp8_fwd(x2, w, w8[0].data if w8 else None, w8[0].scale if w8 else None,
                                             need_xt, need_wt, _ext.status_buffer(x2.device).data_ptr())
        if need_wt and w8:
            kept[2:] = [w8[1].data, w8[1].scale]
        return y, kept
    x8, xt8 = quantize_fp8(x2, "row", rows=True, columns=need_xt)
    q, t = w8 if w8 else quantize_fp8(w, "tile", rows=True, columns=need_wt)
    y = gemm_fp8(x8, q, out_dtype=torch.float32).to(x2.dtype)
    return y, [v for m, need in ((xt8, need_xt), (t, need_wt)) for v in ((m.data, m.scale) if need else (None, None))]


class _LinearFp8(torch.autograd.Function):
    """Forward ``Q(x) Q(w)^T``; backward ``dx = Q(dy) Q(w)`` and ``dw = Q(dy^T) Q(x^T)^T``, each operand in blocks along
    its own reduction.  What is kept for the backward is 8 bits wide: x's columns and w's."""

    @staticmethod
    def forward(ctx, x2, w, w8, need_dx, need_dw, grad_dtype, acc):
        y, kept = _forward(x2, w, w8, need_dw, need_dx)
        ctx.save_for_backward(*kept)
        ctx.meta = (need_dx, need_dw, grad_dtype, acc, x2.shape, w.shape, w.dtype, x2.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_dx, need_dw, grad_dtype, acc, x_shape, w_shape, w_dtype, x_dtype = ctx.meta
        xt, sxt, wt, swt = ctx.saved_tensors
        if dy.stride(1) != 1 and dy.shape[1] > 1:
            dy = dy.contiguous()
        if _native(dy):
            dx, dw = _ext.ext().linear_fp8_bwd(dy, xt if need_dw else None, sxt if need_dw else None,
                                               wt if need_dx else None, swt if need_dx else None,
                                               grad_dtype == torch.float8_e5m2, acc,
                                               _ext.status_buffer(dy.device).data_ptr())
            return dx, dw, None, None, None, None, None
        dx = dw = None
        dy8, dyt8 = quantize_fp8(dy.float(), "row", rows=need_dx, columns=need_dw, dtype=grad_dtype)
        if need_dw:
            xt8 = Fp8Matrix(xt, sxt, x_shape[0])
            if acc is not None:
                gemm_fp8(dyt8, xt8, out=acc, accumulate=True)
            else:
                dw = gemm_fp8(dyt8, xt8, out_dtype=torch.float32).to(w_dtype)
        if need_dx:
            dx = gemm_fp8(dy8, Fp8Matrix(wt, swt, w_shape[0]), out_dtype=torch.float32).to(x_dtype)
        return dx, dw, None, None, None, None, None


def linear_fp8(x: torch.Tensor, w: torch.Tensor, w8: Optional[tuple[Fp8Matrix, Fp8Matrix]] = None, *,
               grad_dtype: torch.dtype = torch.float8_e4m3fn) -> torch.Tensor:
    """``x @ w.T`` (no bias) with both operands, and in the backward the gradient, in 8-bit blocks of 128.

    ``x [..., K]`` is quantised in row blocks and ``w [N, K]`` in 128 x 128 tiles; the backward quantises ``dy`` in row
    blocks for ``dx`` and in column blocks, with x's, for ``dw`` (``grad_dtype``: the gradient's 8-bit type).  The
    weight gradient goes into ``w._mvp_grad_acc`` when present, as in :func:`linear`.  ``w8`` is ``quantize_fp8(w, "tile",
    rows=True, columns=True)`` of the present weights, for a caller that keeps it between calls; without it the
    call quantises ``w`` itself.  Not differentiable twice.  A backward pass may be captured into a CUDA graph; as with every
    torch operator, no eager autograd graph of the same leaf tensors may be alive meanwhile.
    """
    from . import grad_acc, linear

    if w.dim() != 2 or x.dim() < 1 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"linear_fp8: x [..., K] and w [N, K] are needed, got {tuple(x.shape)} and {tuple(w.shape)}")
    if x.device != w.device:
        raise ValueError(f"linear_fp8: x on {x.device}, w on {w.device}")
    if grad_dtype not in _MAX_EXPONENT:
        raise TypeError(f"linear_fp8: grad_dtype must be float8_e4m3fn or float8_e5m2, got {grad_dtype}")
    if x.is_cuda and _native(x):
        if x.dtype != torch.bfloat16:
            x = x.to(torch.bfloat16)
        if w.dtype != torch.bfloat16:
            raise TypeError("linear_fp8: the CUDA path expects bf16 weights (cast by the data-parallel wrapper)")
    if w8 is not None:
        q, t = w8
        if q is None or t is None or q.shape != tuple(w.shape) or t.shape != (w.shape[1], w.shape[0]) or \
                q.device != x.device or t.device != x.device:
            raise ValueError("linear_fp8: w8 must be quantize_fp8(w, 'tile', rows=True, columns=True)")
    if x.numel() == 0 or w.numel() == 0:
        return linear(x, w) if not x.is_cuda else F.linear(x, w)
    grad = torch.is_grad_enabled()
    acc = grad_acc(w)
    if acc is not None and (acc.dtype != torch.float32 or acc.shape != w.shape or acc.stride(-1) != 1):
        raise ValueError("linear_fp8: the gradient accumulator must be fp32 of the weight's shape")
    need_dx = grad and x.requires_grad
    need_dw = grad and (w.requires_grad or (acc is not None and need_dx))
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.stride(1) != 1 and x2.shape[1] > 1:
        x2 = x2.contiguous()
    if w.is_cuda and w.stride(1) != 1 and w.shape[1] > 1:
        w = w.contiguous()
    if need_dx or need_dw:
        y = _LinearFp8.apply(x2, w, w8, need_dx, need_dw, grad_dtype, acc if need_dw else None)
    else:
        with torch.no_grad():
            y = _forward(x2, w, w8, False, False)[0]
    return y if x.dim() == 2 else y.view(*x.shape[:-1], w.shape[0])
