"""The operators around a classifier head held in 8 bits, as they are timed and checked.

Five ways into three operators:

  norm_fp8      root-mean-square norm of embeddings, with a residual's addition, straight into e4m3 and its block scales
  norm_train    the same norm in a training step: outputs and the gradients of input, residual and weight
  linear        the head on embeddings: quantise them by row and block of 128, multiply with a weight kept in e4m3
  matmul        the product of two matrices that are both kept in e4m3 with block scales
  linear_train  the head in a training step: all three products in e4m3, gradients of input, weight and bias
  sgd_clip      an SGD step whose gradients are clipped by their norm over all tensors

Where ``own`` is false everything is computed in 32 bits (sums of many squares in 64) from the formulas.
"""

import math

import torch

own = False

EPS = 1e-6
BLOCK = 128
FP8_MAX = 448.0
AMAX_FLOOR = 2.0 ** -110
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
#: ResNet stage plans: (blocks, width, expansion), and the classes of the head.
NETS = {"resnet18": ((2, 2, 2, 2), 1, 10), "resnet50": ((3, 4, 6, 3), 4, 1000)}


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #

def listed():
    return [
        # one embedding of a ResNet-50 on its way into the head: latency is all there is
        {"name": "norm-fp8-one", "op": "norm_fp8", "rows": 1, "dim": 2048, "dtype": "bf16", "residual": True, "scale": "e8m0"},
        # a whole unlabelled pool of embeddings, normalised before the head scores it
        {"name": "norm-fp8-pool", "op": "norm_fp8", "rows": 130000, "dim": 2048, "dtype": "bf16", "residual": True, "scale": "e8m0"},
        # a training batch of embeddings in 32 bits, as the encoder hands them to the head
        {"name": "norm-train-batch", "op": "norm_train", "rows": 256, "dim": 2048, "dtype": "fp32", "residual": False},
        # many positions of a wide model, with an odd count of rows and the residual stream's gradient
        {"name": "norm-train-wide", "op": "norm_train", "rows": 16383, "dim": 4096, "dtype": "bf16", "residual": True},
        # one embedding through the 1000-class head
        {"name": "linear-one", "op": "linear", "rows": 1, "out": 1000, "inner": 2048, "dtype": "bf16", "bias": True, "scale": "e8m0"},
        # sixteen single tokens against a large weight: the weight's bytes are what it costs
        {"name": "linear-sixteen", "op": "linear", "rows": 16, "out": 8192, "inner": 8192, "dtype": "bf16", "bias": False, "scale": "e8m0"},
        # a chunk of the pool through the 1000-class head: rows by the ten thousand, an output that no tile divides
        {"name": "linear-pool", "op": "linear", "rows": 65536, "out": 1000, "inner": 2048, "dtype": "bf16", "bias": True, "scale": "e8m0"},
        # a large square product: the matrix cores' own rate
        {"name": "matmul-square", "op": "matmul", "rows": 8192, "out": 8192, "inner": 8192, "scale": "e8m0"},
        # weights that come with 32-bit scales, every side odd or ragged
        {"name": "matmul-ragged", "op": "matmul", "rows": 4099, "out": 5003, "inner": 4100, "scale": "fp32"},
        # a training step of a wide layer: forward, both gradients' products and the bias
        {"name": "linear-train", "op": "linear_train", "rows": 8192, "out": 4096, "inner": 2048, "dtype": "bf16", "bias": True},
        # a clipped step of the 10-class network, mostly launches
        {"name": "clip-resnet18", "op": "sgd_clip", "net": "resnet18", "tensors": 0, "total": 0},
        # a clipped step over many tensors of uneven, odd sizes: as much memory as a large model's shard
        {"name": "clip-many", "op": "sgd_clip", "net": "", "tensors": 301, "total": 400000000},
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["norm_fp8", "norm_train", "linear", "matmul", "linear_train", "sgd_clip"])
    if op in ("norm_fp8", "norm_train"):
        dim = size(33, 8192)
        case = {"op": op, "rows": size(1, min(130000, 130000 * 2048 // dim if op == "norm_fp8" else 16383 * 4096 // dim)), "dim": dim,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "residual": rng.random() < 0.5}
        if op == "norm_fp8":
            case["scale"] = rng.choice(["e8m0", "fp32"])
        return case
    if op == "sgd_clip":
        tensors = size(1, 301)
        return {"op": op, "net": "", "tensors": tensors, "total": size(1000 * tensors, 200000000)}
    out, inner = size(10, 8192), size(64, 8192)
    case = {"op": op, "rows": size(1, 65536 if op == "linear" else 8192), "out": out, "inner": inner}
    if op == "linear_train":
        case["rows"] = size(8, 8192)
    if op == "matmul":
        case["scale"] = rng.choice(["e8m0", "fp32"])
        return case
    case.update(dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), bias=rng.random() < 0.5)
    if op == "linear":
        case["rows"] = min(case["rows"], 2 ** 28 // max(out, inner))
        case["scale"] = rng.choice(["e8m0", "fp32"])
    return case


def work(case):
    op, size = case["op"], {"bf16": 2, "fp16": 2, "fp32": 4}.get(case.get("dtype"), 4)
    if op in ("norm_fp8", "norm_train"):
        n, streams = case["rows"] * case["dim"], 2 if case["residual"] else 1
        if op == "norm_fp8":  # input (and residual) in, e4m3 (and the sum) out
            scales = case["rows"] * -(-case["dim"] // BLOCK) * (1 if case["scale"] == "e8m0" else 4)
            return {"bytes": n * (size * (2 * streams - 1) + 1) + scales + 4 * case["dim"], "flops": 6 * n}
        # x (and residual) in, y (and the sum) out, their gradients in, the input's gradient out; weight in and its gradient out
        return {"bytes": n * size * (3 * streams + 1) + 8 * case["dim"], "flops": 14 * n}
    if op == "sgd_clip":
        return {"bytes": 20 * sum(_tensor_sizes(case, 0)), "flops": 7 * sum(_tensor_sizes(case, 0))}
    m, n, k = case["rows"], case["out"], case["inner"]
    if op == "linear_train":  # x, w, dy in; y, dx, dw out
        return {"bytes": size * (2 * m * k + 2 * m * n) + 8 * n * k, "flops": 6 * m * n * k}
    kb = -(-k // BLOCK)
    scale = 1 if case["scale"] == "e8m0" else 4
    if op == "linear":
        return {"bytes": size * (m * k + m * n) + n * k + scale * kb * -(-n // BLOCK), "flops": 2 * m * n * k}
    return {"bytes": m * k + n * k + 2 * m * n + scale * kb * (m + -(-n // BLOCK)), "flops": 2 * m * n * k}


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #

def _tensor_sizes(case, seed):
    """How many values each parameter has: a network's own list, or a random split of the total into uneven parts."""
    if not case["net"]:
        g = torch.Generator().manual_seed(seed)
        share = torch.rand(case["tensors"], generator=g, dtype=torch.float64).pow(4) + 1e-4
        sizes = (share / share.sum() * (case["total"] - case["tensors"])).long() + 1
        sizes[0] += case["total"] - int(sizes.sum())
        return sizes.tolist()
    blocks, expansion, classes = NETS[case["net"]]
    sizes, width_in = [64 * 3 * (9 if classes == 10 else 49), 64, 64], 64
    for stage, count in enumerate(blocks):
        width = 64 << stage
        for i in range(count):
            wide = width * expansion
            convs = [9 * width_in * width, 9 * width * width] if expansion == 1 else [width_in * width, 9 * width * width, width * wide]
            outs = [width, width] if expansion == 1 else [width, width, wide]
            if i == 0 and (stage > 0 or expansion > 1):
                convs, outs = convs + [width_in * wide], outs + [wide]
            sizes += [v for c, o in zip(convs, outs) for v in (c, o, o)]
            width_in = wide
    return sizes + [classes * width_in, classes]


def _embeddings(rows, dim, gen):
    """Activations with a few channels far above the others, as trained networks have them."""
    x = torch.randn(rows, dim, device="cuda", generator=gen)
    loud = torch.rand(dim, device="cuda", generator=gen) < 0.01
    return x.mul_(torch.where(loud, 20.0, 1.0))


def prepare(case, seed):
    op, gen = case["op"], torch.Generator("cuda").manual_seed(seed)
    s = {"op": op, "scale": case.get("scale", "e8m0")}
    if op == "sgd_clip":
        sizes = _tensor_sizes(case, seed)
        total = sum(sizes)
        s["param"] = torch.randn(total, device="cuda", generator=gen).mul_(0.05)
        s["momentum"] = torch.randn(total, device="cuda", generator=gen).mul_(1e-3)
        s["grad"] = torch.randn(total, device="cuda", generator=gen).mul_(1e-2)
        s["args"] = dict(lr=0.1, momentum=0.9, weight_decay=1e-4, max_grad_norm=1.0)
        if own:
            from active_learning_amd.ops.optim import FusedSGD
            params = [torch.nn.Parameter(v) for v in s["param"].split(sizes)]
            s["optimizer"] = FusedSGD(params, **s["args"])
            for p, g, b in zip(params, s["grad"].split(sizes), s["momentum"].split(sizes)):
                p.grad = g
                s["optimizer"].state[p]["momentum_buffer"] = b
        return s
    dtype = DTYPES[case.get("dtype", "bf16")]
    if op in ("norm_fp8", "norm_train"):
        rows, dim = case["rows"], case["dim"]
        s["x"] = _embeddings(rows, dim, gen).to(dtype)
        s["weight"] = torch.rand(dim, device="cuda", generator=gen).add_(0.5)
        s["residual"] = _embeddings(rows, dim, gen).to(dtype) if case["residual"] else None
        if op == "norm_train":
            s["dy"] = torch.randn(rows, dim, device="cuda", generator=gen).to(dtype)
            s["dsum"] = torch.randn(rows, dim, device="cuda", generator=gen).to(dtype) if case["residual"] else None
            s["leaves"] = [t.requires_grad_() for t in (s["x"], s["weight"], s["residual"]) if t is not None]
        return s
    m, n, k = case["rows"], case["out"], case["inner"]
    x = _embeddings(m, k, gen)
    w = torch.randn(n, k, device="cuda", generator=gen).div_(math.sqrt(k))
    s["bias"] = torch.randn(n, device="cuda", generator=gen).mul_(0.1) if case.get("bias") else None
    if op == "linear_train":
        s["x"], s["weight"] = x.to(dtype).requires_grad_(), w.requires_grad_()
        s["dy"] = torch.randn(m, n, device="cuda", generator=gen).mul_(1e-3).to(dtype)
        if s["bias"] is not None:
            s["bias"].requires_grad_()
        s["leaves"] = [t for t in (s["x"], s["weight"], s["bias"]) if t is not None]
        return s
    s["weight"] = _quantise(w, s["scale"], tile=True)
    s["x"] = x.to(dtype) if op == "linear" else _quantise(x, s["scale"])
    if own:
        from active_learning_amd.ops.fp8 import Fp8Blocks
        s["weight"] = Fp8Blocks(*s["weight"], tile=True)
        if op == "matmul":
            s["x"] = Fp8Blocks(*s["x"])
    return s


# --------------------------------------------------------------------------- #
# plain forms
# --------------------------------------------------------------------------- #

def _spread(scale, rows, cols, tile):
    """One factor for each value: the block scales repeated over their blocks."""
    scale = scale.float().repeat_interleave(BLOCK, 1)[:, :cols]
    return scale.repeat_interleave(BLOCK, 0)[:rows] if tile else scale


def _quantise(x, kind, tile=False):
    """e4m3 values of ``x`` (32 bits) and the scales of its blocks: 1 x 128, or 128 x 128."""
    rows, cols = x.shape
    up, across = -(-rows // BLOCK) * BLOCK if tile else rows, -(-cols // BLOCK) * BLOCK
    wide = x.new_zeros(up, across)
    wide[:rows, :cols] = x
    if tile:
        amax = wide.abs().view(up // BLOCK, BLOCK, across // BLOCK, BLOCK).amax((1, 3))
    else:
        amax = wide.abs().view(rows, across // BLOCK, BLOCK).amax(2)
    amax = amax.clamp_min(AMAX_FLOOR)
    if kind == "e8m0":  # the smallest power of two that brings the block's largest magnitude to 448 or less
        code = ((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8
        scale, inverse = code.to(torch.uint8).view(torch.float8_e8m0fnu), ((254 - code) << 23).view(torch.float32)
    else:
        scale, inverse = amax / FP8_MAX, torch.full_like(amax, FP8_MAX) / amax  # a number over a tensor would round twice
    return (x * _spread(inverse, rows, cols, tile)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scale


def _value(q, scale, tile=False):
    return q.float() * _spread(scale, q.shape[0], q.shape[1], tile)


def _rounded(x, kind, tile=False):
    return _value(*_quantise(x, kind, tile), tile)


def _plain(s):
    op = s["op"]
    if op == "sgd_clip":
        a, g = s["args"], s["grad"]
        norm = g.square().sum(dtype=torch.float64).sqrt().float()
        factor = (a["max_grad_norm"] / (norm + 1e-6)).clamp(max=1.0)
        s["momentum"].mul_(a["momentum"]).add_(g * factor).add_(s["param"], alpha=a["weight_decay"])
        s["param"].sub_(s["momentum"], alpha=a["lr"])
        return s["param"], s["momentum"], norm
    x = s["x"]
    if op in ("norm_fp8", "norm_train"):
        total = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
        v = total.float()
        rstd = (v.square().mean(1, keepdim=True) + EPS).rsqrt()
        unit = v * rstd
        y = unit * s["weight"]
        if op == "norm_fp8":
            return (*_quantise(y, s["scale"]), None if s["residual"] is None else total)
        dy = s["dy"].float()
        wdy = dy * s["weight"]
        dx = (wdy - unit * (wdy * unit).mean(1, keepdim=True)) * rstd
        dw = (dy * unit).sum(0)
        if s["residual"] is None:
            return y.to(x.dtype), dx.to(x.dtype), dw
        dx = (dx + s["dsum"].float()).to(x.dtype)
        return y.to(x.dtype), total, dx, dw, dx
    if op == "matmul":
        return (_value(*x) @ _value(*s["weight"], tile=True).t()).bfloat16()
    if op == "linear":
        y = _rounded(x.float(), s["scale"]) @ _value(*s["weight"], tile=True).t()
        return (y if s["bias"] is None else y + s["bias"]).to(x.dtype)
    wide, w, dy = x.float(), _rounded(s["weight"], s["scale"], tile=True), s["dy"].float()
    y = _rounded(wide, s["scale"]) @ w.t()
    dx = _rounded(dy, s["scale"]) @ w
    dw = _rounded(dy.t().contiguous(), s["scale"]) @ _rounded(wide.t().contiguous(), s["scale"]).t()
    if s["bias"] is None:
        return y.to(x.dtype), dx.to(x.dtype), dw
    return (y + s["bias"]).to(x.dtype), dx.to(x.dtype), dw, dy.sum(0, dtype=torch.float64).float()


def run(state):
    if not own:
        with torch.no_grad():
            return _plain(state)
    op = state["op"]
    if op == "sgd_clip":
        state["optimizer"].step()
        return state["param"], state["momentum"], state["optimizer"].last_grad_norm
    if op == "norm_fp8":
        from active_learning_amd.ops.rmsnorm import rms_norm_fp8
        out = rms_norm_fp8(state["x"], state["weight"], residual=state["residual"], eps=EPS, scale=state["scale"])
        out, total = (out, None) if state["residual"] is None else out
        return out.values, out.scale, total
    if op == "norm_train":
        from active_learning_amd.ops.rmsnorm import rms_norm
        if state["residual"] is None:
            y = rms_norm(state["x"], state["weight"], eps=EPS)
            return (y.detach(), *torch.autograd.grad(y, state["leaves"], state["dy"]))
        y, total = rms_norm(state["x"], state["weight"], residual=state["residual"], eps=EPS)
        return (y.detach(), total.detach(), *torch.autograd.grad((y, total), state["leaves"], (state["dy"], state["dsum"])))
    if op == "matmul":
        from active_learning_amd.ops.fp8 import fp8_matmul
        return fp8_matmul(state["x"], state["weight"], out_dtype=torch.bfloat16)
    from active_learning_amd.ops.fp8 import fp8_linear
    y = fp8_linear(state["x"], state["weight"], state["bias"])
    if op == "linear":
        return y
    return (y.detach(), *torch.autograd.grad(y, state["leaves"], state["dy"]))


# --------------------------------------------------------------------------- #
# the definitions in 64 bits
# --------------------------------------------------------------------------- #

def _exact_blocks(x, kind, high, tile=False):
    """(values, scales, their product) of a 64-bit matrix. ``high``: blocks over rows as well."""
    rows, cols = x.shape
    tall = BLOCK if high else 1
    pad = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % tall))
    grid = pad.view(pad.shape[0] // tall, tall, pad.shape[1] // BLOCK, BLOCK)
    top = torch.maximum(grid.amax((1, 3)), -grid.amin((1, 3))).clamp_min(AMAX_FLOOR)
    if kind == "e8m0":
        scale = torch.exp2(torch.ceil(torch.log2(top / FP8_MAX)))
        factor = 1 / scale
    else:  # both are 32-bit numbers by definition
        scale, factor = (top / FP8_MAX).float().double(), (torch.full_like(top, FP8_MAX) / top).float().double()
    by = scale[:, None, :, None]
    codes = (grid * factor[:, None, :, None]).clamp(-FP8_MAX, FP8_MAX).float().to(torch.float8_e4m3fn)
    back = lambda t: t.reshape(pad.shape)[:rows, :cols]  # noqa: E731
    return back(codes), scale, back(codes.double() * by)


def _decoded(q, scale, high):
    """The 64-bit matrix that stored e4m3 values and scales stand for."""
    rows = torch.arange(q.shape[0], device=q.device) // (BLOCK if high else 1)
    cols = torch.arange(q.shape[1], device=q.device) // BLOCK
    return q.double() * scale.double()[rows][:, cols]


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    with torch.no_grad():
        if op == "sgd_clip":
            p, b, g, a = s["param"].double(), s["momentum"].double(), s["grad"].double(), s["args"]
            norm = torch.linalg.vector_norm(g)
            b = a["momentum"] * b + g * min(1.0, a["max_grad_norm"] / (float(norm) + 1e-6)) + a["weight_decay"] * p
            return p - a["lr"] * b, b, norm
        if op in ("norm_fp8", "norm_train"):
            kept = s["x"].detach()
            if s["residual"] is not None:  # the stored sum is rounded to the stream's type, and the norm is that of the stored sum
                kept = (kept.double() + s["residual"].detach().double()).to(kept.dtype)
            v, w = kept.double(), s["weight"].detach().double()
            root = torch.sqrt((v * v).sum(1, keepdim=True) / v.shape[1] + EPS)
            if op == "norm_fp8":
                codes, scale, _ = _exact_blocks(v / root * w, case["scale"], False)
                return codes, scale, None if s["residual"] is None else kept.double()
            dy = s["dy"].double()
            dv = dy * w / root - v * (dy * w * v).sum(1, keepdim=True) / (v.shape[1] * root ** 3)
            dw = (dy * v / root).sum(0)
            y = v / root * w
            if s["residual"] is None:
                return y, dv, dw
            dv = dv + s["dsum"].double()
            return y, v, dv, dw, dv
        if op == "matmul":
            return _decoded(*s["x"], False) @ _decoded(*s["weight"], True).t()
        x = s["x"].detach().double()
        bias = 0.0 if s["bias"] is None else s["bias"].detach().double()
        if op == "linear":
            return _exact_blocks(x, case["scale"], False)[2] @ _decoded(*s["weight"], True).t() + bias
        w, dy = _exact_blocks(s["weight"].detach().double(), "e8m0", True)[2], s["dy"].double()
        y = _exact_blocks(x, "e8m0", False)[2] @ w.t() + bias
        dx = _exact_blocks(dy, "e8m0", False)[2] @ w
        dw = _exact_blocks(dy.t().contiguous(), "e8m0", False)[2] @ _exact_blocks(x.t().contiguous(), "e8m0", False)[2].t()
        return (y, dx, dw) if s["bias"] is None else (y, dx, dw, dy.sum(0))
