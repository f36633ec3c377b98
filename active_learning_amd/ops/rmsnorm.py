"""Root-mean-square norm, with a residual's addition and an e4m3 output.

    s = x + residual (rounded to their type)      rstd = 1 / sqrt(mean(s^2) + eps)
    y = s * rstd * weight

The norm is that of the rounded sum, which is also what comes back for the next
residual and what the backward pass reads. Squares are summed in 64 bits; the other
arithmetic is in 32 (64 in front of an e4m3 output) and rounded to the type once. GPU tensors run rmsnorm.hip;
CPU tensors run the torch math below, which defines the semantics that the kernels
are tested against.

Stands beside batch_norm_act (ops/functional.py): a norm for embeddings and
heads, whose rows are independent of the batch.
"""

import torch
import torch.nn as nn
from torch.autograd import Function

from .extension import require_extension
from .fp8 import Fp8Blocks, check_scale_kind, no_tangent, once, quantize_fp8

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check(x, weight, residual, eps):
    if x.dtype not in _TYPES:
        raise TypeError(f"rms_norm takes bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("rms_norm needs a last axis of at least one value")
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"weight has shape {tuple(weight.shape)}, not {tuple(x.shape[-1:])}")
    if weight.dtype not in (torch.float32, x.dtype):
        raise TypeError(f"weight must be float32 or {x.dtype}, got {weight.dtype}")
    if weight.device != x.device:
        raise ValueError(f"weight is on {weight.device}, the input on {x.device}")
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError("residual must have the input's shape and type: "
                             f"{tuple(residual.shape)} {residual.dtype}, not "
                             f"{tuple(x.shape)} {x.dtype}")
        if residual.device != x.device:
            raise ValueError(f"residual is on {residual.device}, the input on {x.device}")
    if not torch.tensor(eps, dtype=torch.float32) > 0:
        raise ValueError(f"eps must be positive, got {eps}")


def _forward_cpu(x, weight, residual, eps, wide=torch.float32):
    total = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    mean = total.double().square().mean(-1, keepdim=True)  # squares may leave the range of 32 bits
    rstd = (1.0 / torch.sqrt(mean + eps)).to(wide)
    return total.to(wide) * rstd * weight.to(wide), total, rstd


class _RMSNormCPU(Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        y, total, rstd = _forward_cpu(x, weight, residual, eps)
        ctx.save_for_backward(total, weight, rstd)
        y = y.to(x.dtype)
        return y if residual is None else (y, total)

    @staticmethod
    def backward(ctx, dy, dsum=None):
        need_x, need_w, need_r, _ = ctx.needs_input_grad
        if dy is None:  # only the sum was used
            dx, dw = dsum, torch.zeros_like(ctx.saved_tensors[1])
        else:
            with torch.no_grad():
                dx, dw = _RMSNormCPU.gradients(ctx, dy, dsum)
            outer = dy.requires_grad or (dsum is not None and dsum.requires_grad)
            dx = once(dx, outer or need_x or need_r or need_w, "rms_norm")
            dw = once(dw, outer or need_x or need_r, "rms_norm")
        return dx if need_x else None, dw if need_w else None, dx if need_r else None, None

    @staticmethod
    def gradients(ctx, dy, dsum):
        total, weight, rstd = ctx.saved_tensors
        u = total.float() * rstd
        g = dy.float() * weight.float()
        dx = (g - u * (g * u).mean(-1, keepdim=True)) * rstd
        if dsum is not None:
            dx = dx + dsum.float()
        dx = dx.to(total.dtype)
        dw = (dy.float() * u).reshape(-1, u.shape[-1]).sum(0).to(weight.dtype)
        return dx, dw


def rms_norm(x, weight, residual=None, eps=1e-6):
    """The norm of ``x`` over its last axis, or of ``x + residual``.

    ``x``: (..., dim) in bfloat16, float16 or float32; ``residual``: the same
    shape and type; ``weight``: (dim,) in float32 or x's type. Returns y, or
    (y, sum) where a residual is given. Differentiable in all three, once, and not in
    forward mode.
    """
    if x.is_cuda:  # checked, and differentiated, by the extension
        out = require_extension().rms_norm(x, weight, residual, eps)
        return out[0] if residual is None else tuple(out)
    _check(x, weight, residual, eps)
    return _RMSNormCPU.apply(x, weight, residual, eps)


def rms_norm_fp8(x, weight, residual=None, eps=1e-6, scale="e8m0"):
    """``rms_norm`` straight into e4m3 with a scale for each 128 values of a row.

    Returns Fp8Blocks of (rows, dim), the leading axes flattened, or (blocks,
    sum) where a residual is given. Codes and scales are those of the norm in 64 bits,
    without a rounding to x's type between. For inference: it has no gradient, and inputs
    that ask for one are refused.
    """
    kind = check_scale_kind(scale)
    if x.is_cuda:
        codes, scales, total = require_extension().rms_norm_quant(x, weight, residual, eps, kind)
        blocks = Fp8Blocks._of(codes, scales, (codes.shape[0], x.shape[-1]), False)
        return blocks if residual is None else (blocks, total)
    _check(x, weight, residual, eps)
    no_tangent("rms_norm_fp8", x, weight, residual)
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_fp8 has no gradient: use rms_norm and fp8_linear to "
                           "train, or torch.no_grad()")
    y, total, _ = _forward_cpu(x, weight, residual, eps, torch.float64)
    blocks = quantize_fp8(y.float().reshape(-1, y.shape[-1]), scale=scale)
    return blocks if residual is None else (blocks, total)


class RMSNorm(nn.Module):
    """Module form of ``rms_norm``; ``quantize`` gives the e4m3 form."""

    def __init__(self, dim, eps=1e-6):
        super().__init__()
        self.dim = dim
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, residual, self.eps)

    def quantize(self, x, residual=None, scale="e8m0"):
        with torch.no_grad():
            return rms_norm_fp8(x, self.weight, residual, self.eps, scale)

    def extra_repr(self):
        return f"{self.dim}, eps={self.eps}"
