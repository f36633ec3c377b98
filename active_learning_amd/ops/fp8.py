"""Matrices in e4m3 with a scale for each block of 128, and products of them.

A block is 128 neighbouring values of a row (activations, gradients) or a
128x128 tile (weights). Its scale is a power of two held in one e8m0 byte, which
the matrix cores apply by themselves, or a float32. With a = max|v| of the
block, at least 2^-110:

    e8m0:  scale = the smallest 2^e with a <= 448 * 2^e,   code = e4m3(v / scale)
    fp32:  scale = a / 448,                                code = e4m3(v * (448 / a))

An infinity or a NaN makes its block's scale and codes NaN, and with them every
product that the block enters.

    C[m, n] = sum over blocks of scale_a * scale_b * (sum in the block of a * b) + bias[n]

GPU tensors run fp8.hip; CPU tensors run the torch math below, which defines the
semantics that the kernels are tested against. Stands beside the float32 head of
ops/linear.py, for heads and pools large enough that its rate counts.
"""

import torch
from torch.autograd import Function, forward_ad

from .extension import require_extension
from .linear import NativeLinear

BLOCK = 128
FP8_MAX = 448.0
_AMAX_FLOOR = 2.0 ** -110
_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_KINDS = {"e8m0": 0, "fp32": 1}
_SCALE_TYPES = {torch.float8_e8m0fnu: "e8m0", torch.float32: "fp32"}


def check_scale_kind(scale):
    if scale not in _KINDS:
        raise ValueError(f"scale must be one of {sorted(_KINDS)}, got {scale!r}")
    return _KINDS[scale]


def _blocks(n):
    return -(-n // BLOCK)


class Fp8Blocks:
    """A matrix of e4m3 values with block scales.

    ``values`` (rows, cols) are the codes, ``scale`` the factors: (rows, blocks)
    of 1x128 blocks, or with ``tile`` (row blocks, blocks) of 128x128 tiles.
    Kernels read whole blocks and four scales at a time, so the storage is padded
    (zero behind the last column). The constructor copies into that layout what
    does not have it already: build it once and keep it, as a program keeps its
    weights. quantize_fp8 and rms_norm_fp8 write it themselves. Values times scales
    have to lie in float32's range.
    """

    __slots__ = ("_codes", "_scales", "shape", "tile")

    def __init__(self, values, scale, tile=False):
        if values.dtype != torch.float8_e4m3fn or values.dim() != 2:
            raise TypeError("values must be a float8_e4m3fn matrix, got "
                            f"{values.dtype} with {values.dim()} axes")
        if scale.dtype not in _SCALE_TYPES:
            raise TypeError(f"scale must be float8_e8m0fnu or float32, got {scale.dtype}")
        rows, cols = values.shape
        if cols == 0:
            raise ValueError("values must have at least one column")
        want = (_blocks(rows) if tile else rows, _blocks(cols))
        if tuple(scale.shape) != want:
            raise ValueError(f"scale must have shape {want} for values of shape "
                             f"{(rows, cols)}, got {tuple(scale.shape)}")
        if scale.device != values.device:
            raise ValueError(f"scale is on {scale.device}, the values on {values.device}")
        values, scale = values.detach(), scale.detach()
        if (cols % BLOCK or not values.is_contiguous()
                or (values.is_cuda and values.data_ptr() % 16)):
            codes = torch.zeros(rows, _blocks(cols) * BLOCK, dtype=torch.uint8,
                                device=values.device)
            codes[:, :cols] = values.view(torch.uint8)
            values = codes.view(torch.float8_e4m3fn)
        size = scale.element_size()
        if (want[1] % 4 or not scale.is_contiguous()
                or (scale.is_cuda and scale.data_ptr() % (4 * size))):
            fours = torch.zeros(want[0], -(-want[1] // 4) * 4 * size, dtype=torch.uint8,
                                device=scale.device)
            fours[:, :want[1] * size] = scale.contiguous().view(torch.uint8)
            scale = fours.view(scale.dtype)
        self._codes, self._scales = values, scale
        self.shape, self.tile = torch.Size((rows, cols)), bool(tile)

    @classmethod
    def _of(cls, codes, scales, shape, tile):
        """From storage that is already laid out, as the kernels write it."""
        self = cls.__new__(cls)
        self._codes, self._scales = codes, scales
        self.shape, self.tile = torch.Size(shape), tile
        return self

    @property
    def values(self):
        cols = self.shape[1]
        return self._codes if self._codes.shape[1] == cols else self._codes[:, :cols]

    @property
    def scale(self):
        blocks = _blocks(self.shape[1])
        return self._scales if self._scales.shape[1] == blocks else self._scales[:, :blocks]

    @property
    def device(self):
        return self._codes.device

    @property
    def scale_kind(self):
        return _SCALE_TYPES[self._scales.dtype]

    def to(self, device):
        return Fp8Blocks._of(self._codes.to(device), self._scales.to(device),
                             self.shape, self.tile)

    def dequantize(self, dtype=torch.float32):
        """The matrix that the codes and scales stand for."""
        rows, cols = self.shape
        scale = self.scale.float().repeat_interleave(BLOCK, 1)[:, :cols]
        if self.tile:
            scale = scale.repeat_interleave(BLOCK, 0)[:rows]
        return (self.values.float() * scale).to(dtype)

    def __repr__(self):
        return (f"Fp8Blocks({self.shape[0]}x{self.shape[1]}, "
                f"{'128x128' if self.tile else '1x128'} {self.scale_kind} scales, "
                f"{self.device})")


def _quantize_cpu(x, kind, tile):
    rows, cols = x.shape
    up, across = (_blocks(rows) * BLOCK if tile else rows), _blocks(cols) * BLOCK
    wide = torch.zeros(up, across, dtype=torch.float32)
    wide[:rows, :cols] = x
    tall = BLOCK if tile else 1
    grid = wide.view(up // tall, tall, across // BLOCK, BLOCK)
    amax = grid.abs().amax((1, 3))  # NaN stays
    bad = ~torch.isfinite(amax)
    amax = torch.where(bad, amax.new_ones(()), amax).clamp_min(_AMAX_FLOOR)
    if kind == 0:
        code = ((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8
        inverse = ((254 - code) << 23).view(torch.float32)
        scale = torch.where(bad, 255, code).to(torch.uint8).view(torch.float8_e8m0fnu)
    else:
        # a tensor over a tensor: a number over one is rounded twice
        inverse = torch.full_like(amax, FP8_MAX) / amax
        scale = torch.where(bad, amax.new_tensor(float("nan")), amax / FP8_MAX)
    inverse = torch.where(bad, amax.new_tensor(float("nan")), inverse)
    scaled = (grid * inverse[:, None, :, None]).reshape(up, across)[:rows, :cols]
    values = scaled.clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    if cols == 0:  # the transpose of no rows
        return Fp8Blocks._of(values, scale, x.shape, tile)
    return Fp8Blocks(values, scale, tile)


def no_tangent(name, *tensors):
    """Refuses dual tensors, whose output without a tangent would read as a derivative
    of zero."""
    if torch._C._is_fwd_grad_enabled() and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def _matrix(x, name):
    if x.dtype not in _TYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"{name} must be a matrix with at least one column, got shape "
                         f"{tuple(x.shape)}")
    return x.detach()


def _dense_rows(x):
    return x if x.shape[1] == 1 or x.stride(1) == 1 else x.contiguous()


def _pair(x, kind, tile, plain, transposed, sums=None):
    """(blocks, blocks of the transpose, column sums) of ``x``, each None where it
    is not asked for."""
    x = x.float()
    return (_quantize_cpu(x, kind, tile) if plain else None,
            _quantize_cpu(x.t(), kind, tile) if transposed else None,
            x.sum(0, dtype=torch.float64).float().to(sums) if sums is not None else None)


def quantize_fp8(x, tile=False, scale="e8m0"):
    """e4m3 blocks of a matrix: 1x128 along its rows, or 128x128 with ``tile``.

    ``x``: (rows, cols) in bfloat16, float16 or float32, of any strides; a
    transposed matrix is read along its memory. Not differentiable.
    """
    kind = check_scale_kind(scale)
    x = _matrix(x, "x")
    if not x.is_cuda:
        return _quantize_cpu(x.float(), kind, tile)
    ext = require_extension()
    if x.stride(1) != 1 and x.stride(0) == 1 and x.shape[0] > 0:
        # the transpose of a matrix with dense rows
        _, _, codes, scales, _ = ext.fp8_quant_tile(x.t(), kind, tile, False, True, None)
    elif tile:
        codes, scales, _, _, _ = ext.fp8_quant_tile(_dense_rows(x), kind, True, True, False, None)
    else:
        codes, scales = ext.fp8_quant_rows(x, kind)
    return Fp8Blocks._of(codes, scales, x.shape, tile)


def _check_product(a_kind, a_cols, a_device, b, bias):
    if a_cols != b.shape[1]:
        raise ValueError(f"the operands' rows are {a_cols} and {b.shape[1]} values long")
    if a_kind != b.scale_kind:
        raise ValueError(f"the operands' scales are {a_kind} and {b.scale_kind}")
    if a_device != b.device:
        raise ValueError(f"the operands are on {a_device} and {b.device}")
    if bias is not None:
        if bias.shape != (b.shape[0],):
            raise ValueError(f"bias has shape {tuple(bias.shape)}, not ({b.shape[0]},)")
        if bias.dtype not in _TYPES:
            raise TypeError(f"bias must be bfloat16, float16 or float32, got {bias.dtype}")
        if bias.device != b.device:
            raise ValueError(f"bias is on {bias.device}, the operands on {b.device}")


def _product(a, b, bias, out_dtype):
    if a.device.type != "cpu":
        return require_extension().fp8_gemm(
            a._codes, a._scales, b._codes, b._scales, b.tile, a.shape[0], b.shape[0],
            a.shape[1], bias, out_dtype)
    y = a.dequantize() @ b.dequantize().t()
    return (y if bias is None else y + bias.float()).to(out_dtype)


def fp8_matmul(a, b, bias=None, out_dtype=torch.bfloat16):
    """``a @ b.T + bias`` of two Fp8Blocks, (m, k) with 1x128 blocks and (n, k)
    with 1x128 blocks or 128x128 tiles, both with one kind of scale.

    Sums are held in 32 bits. Products for a bfloat16 or float16 result are added
    by the 8-bit matrix instruction, which is a few 1e-5 off; for a float32 result
    they are computed by bf16 instructions, exactly (with e8m0 scales of values
    under 2^-126 what bf16 holds), at half the rate. Not differentiable.
    """
    if not isinstance(a, Fp8Blocks) or not isinstance(b, Fp8Blocks):
        raise TypeError("fp8_matmul takes two Fp8Blocks")
    if a.tile:
        raise ValueError("the left operand's blocks must be 1x128")
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    _check_product(a.scale_kind, a.shape[1], a.device, b, bias)
    return _product(a, b, bias if bias is None else bias.detach().contiguous(), out_dtype)


class _Once(Function):
    @staticmethod
    def forward(ctx, grad, name):
        ctx.name = name
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.name} is differentiable once: its backward pass has no gradient")


def once(grad, asked, name):
    """A gradient that has none of its own though what it depends on asks for one
    (``asked``): where it is to be differentiable, differentiating it raises."""
    if grad is None or not asked or not torch.is_grad_enabled():
        return grad
    return _Once.apply(grad.detach().requires_grad_(), name)


class _Fp8LinearCPU(Function):
    """y = Q(x) Q(w)^T + b,  dx = Q(dy) Q(w),  dw = Q(dy^T) Q(x^T)^T: each
    operand in blocks along its product's contraction. The weight's tiles are the
    same for both of its products."""

    @staticmethod
    def forward(ctx, x, weight, bias, kind):
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        xq, xt, _ = _pair(x, kind, False, True, need_w)
        wq, wt, _ = _pair(weight, kind, True, True, need_x)
        ctx.kind, ctx.types = kind, (x.dtype, weight.dtype, None if bias is None else bias.dtype)
        ctx.shapes = [None if q is None else q.shape for q in (xt, wt)]
        ctx.save_for_backward(*(t for q in (xt, wt) for t in (
            (None, None) if q is None else (q._codes, q._scales))))
        return _product(xq, wq, bias, x.dtype)

    @staticmethod
    def backward(ctx, dy):
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        with torch.no_grad():
            dx, dw, db = _Fp8LinearCPU.gradients(ctx, dy)
        outer = dy.requires_grad
        return (once(dx, outer or need_w, "fp8_linear"), once(dw, outer or need_x, "fp8_linear"),
                once(db, outer, "fp8_linear"), None)

    @staticmethod
    def gradients(ctx, dy):
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        xc, xs, wc, ws = ctx.saved_tensors
        dq, dt, db = _pair(dy, ctx.kind, False, need_x, need_w,
                           ctx.types[2] if need_b else None)
        dx = dw = None
        if need_x:
            dx = _product(dq, Fp8Blocks._of(wc, ws, ctx.shapes[1], True), None, ctx.types[0])
        if need_w:
            dw = _product(dt, Fp8Blocks._of(xc, xs, ctx.shapes[0], False), None, ctx.types[1])
        return dx, dw, db if need_b else None


def fp8_linear(x, weight, bias=None, scale="e8m0"):
    """``x @ weight.T + bias`` with both operands in e4m3 blocks.

    ``x``: (..., in) in bfloat16, float16 or float32; the result has its type.
    ``weight``: Fp8Blocks (out, in), to serve with a weight that is kept
    quantised (``scale`` is then the weight's own), or a tensor (out, in), which
    is quantised by 128x128 tiles in every call and is differentiable once, as are
    x and bias: both of the gradients' products are e4m3 products too.

    Products for a bfloat16 or float16 result (y and dx in x's type, dw in the
    weight's) are added by the 8-bit matrix instruction, which is a few 1e-5 off;
    float32 ones by bf16 instructions, exactly, as in fp8_matmul. The bias' gradient
    is summed in 64 bits. Forward-mode differentiation is refused.
    """
    kept = isinstance(weight, Fp8Blocks)
    if x.is_cuda:  # checked, and differentiated, by the extension
        if kept:
            return require_extension().fp8_linear_kept(
                x, weight._codes, weight._scales, weight.tile, *weight.shape, bias)
        return require_extension().fp8_linear(x, weight, bias, check_scale_kind(scale))
    kind = check_scale_kind(weight.scale_kind if kept else scale)
    if x.dtype not in _TYPES:
        raise TypeError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("x needs a last axis of at least one value")
    flat = x.reshape(-1, x.shape[-1])
    if bias is not None:
        bias = bias.contiguous()
    if kept:
        _check_product(weight.scale_kind, flat.shape[1], x.device, weight, bias)
        no_tangent("fp8_linear", x, bias)
        if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
            raise RuntimeError("a weight kept in Fp8Blocks has no gradient: pass the weight "
                               "itself to train, or use torch.no_grad()")
        y = _product(quantize_fp8(flat, scale=weight.scale_kind), weight, bias, x.dtype)
    else:
        if weight.dim() != 2 or weight.dtype not in _TYPES:
            raise TypeError("weight must be Fp8Blocks or a bfloat16, float16 or float32 matrix")
        if weight.shape[1] != flat.shape[1]:
            raise ValueError(f"the operands' rows are {flat.shape[1]} and {weight.shape[1]} "
                             "values long")
        if weight.device != x.device:
            raise ValueError(f"the operands are on {x.device} and {weight.device}")
        if bias is not None and (bias.shape != weight.shape[:1] or bias.dtype not in _TYPES
                                 or bias.device != x.device):
            raise ValueError(f"bias must be a vector of {weight.shape[0]} values on {x.device}")
        y = _Fp8LinearCPU.apply(flat, weight, bias, kind)
    return y.view(*x.shape[:-1], y.shape[1])


class Fp8Linear(NativeLinear):
    """NativeLinear whose products run in e4m3 blocks; the same parameters and
    state_dict keys. ``quantized`` gives the weight to keep for serving."""

    def forward(self, x):
        return fp8_linear(x, self.weight, self.bias)

    def quantized(self, scale="e8m0"):
        return quantize_fp8(self.weight, tile=True, scale=scale)
