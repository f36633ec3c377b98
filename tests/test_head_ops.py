"""The norm, the e4m3 products and clipping on the CPU: the semantics that the
kernels are tested against, checked against 64-bit formulas, differences and
hand-made values; and what each entry point refuses."""

import math

import pytest
import torch

from active_learning_amd.ops.fp8 import (Fp8Blocks, Fp8Linear, fp8_linear, fp8_matmul,
                                         quantize_fp8)
from active_learning_amd.ops.grad_clip import clip_grad_norm_, grad_norm
from active_learning_amd.ops.optim import FusedAdam, FusedSGD, build_optimizer
from active_learning_amd.ops.rmsnorm import RMSNorm, rms_norm, rms_norm_fp8

U32 = 2.0 ** -24  # a rounding to 32 bits


# --------------------------------------------------------------------------- #
# norm
# --------------------------------------------------------------------------- #

@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_gradients_against_differences(residual):
    """Central differences of step h in 32 bits: truncation h^2 / 6 times a third
    derivative of order one, rounding 2^-24 * |loss| / h; h = 2^-7 puts both under
    1e-4 of sums of 12 terms of order one."""
    x, r, w = torch.randn(3, 4), torch.randn(3, 4), torch.rand(4) + 0.5
    dy, ds = torch.randn(3, 4), torch.randn(3, 4)
    leaves = [x, w] + ([r] if residual else [])

    def loss():
        if not residual:
            return (rms_norm(x, w).double() * dy).sum()
        y, s = rms_norm(x, w, residual=r)
        return (y.double() * dy).sum() + (s.double() * ds).sum()

    for t in leaves:
        t.requires_grad_()
    grads = torch.autograd.grad(loss(), leaves)
    h = 2.0 ** -7
    with torch.no_grad():
        for t, g in zip(leaves, grads):
            flat, gf = t.view(-1), g.reshape(-1)
            for i in range(flat.numel()):
                keep = flat[i].item()
                flat[i] = keep + h
                up = loss()
                flat[i] = keep - h
                down = loss()
                flat[i] = keep
                assert abs((up - down) / (2 * h) - gf[i]) < 2e-3 * (1 + abs(gf[i]))


def test_rms_norm_only_the_sum_is_used():
    x, r, w = (torch.randn(2, 8, requires_grad=True), torch.randn(2, 8, requires_grad=True),
               torch.ones(8, requires_grad=True))
    _, s = rms_norm(x, w, residual=r)
    dx, dr, dw = torch.autograd.grad(s.sum(), (x, r, w))
    assert torch.equal(dx, torch.ones(2, 8)) and torch.equal(dr, dx)
    assert torch.equal(dw, torch.zeros(8))


def test_rms_norm_module_and_quantize():
    m = RMSNorm(130)
    x = torch.randn(2, 3, 130)
    y = m(x)
    assert y.shape == x.shape
    q = m.quantize(x)
    assert tuple(q.shape) == (6, 130)
    assert torch.equal(q.values.float(), quantize_fp8(y.detach().view(6, 130)).values.float())


@pytest.mark.parametrize("bad", [
    lambda: rms_norm(torch.ones(2, 4, dtype=torch.float64), torch.ones(4)),
    lambda: rms_norm(torch.ones(2, 4), torch.ones(5)),
    lambda: rms_norm(torch.ones(2, 4), torch.ones(4, dtype=torch.float16)),
    lambda: rms_norm(torch.ones(2, 4), torch.ones(4), residual=torch.ones(1, 4)),
    lambda: rms_norm(torch.ones(2, 4), torch.ones(4), residual=torch.ones(2, 4).bfloat16()),
    lambda: rms_norm(torch.ones(2, 0), torch.ones(0)),
    lambda: rms_norm(torch.ones(2, 4), torch.ones(4), eps=0.0),
    lambda: rms_norm_fp8(torch.ones(2, 4), torch.ones(4), scale="bf16"),
    lambda: rms_norm_fp8(torch.ones(2, 4, requires_grad=True), torch.ones(4)),
])
def test_rms_norm_refusals(bad):
    with pytest.raises((TypeError, ValueError, RuntimeError)):
        bad()


# --------------------------------------------------------------------------- #
# blocks
# --------------------------------------------------------------------------- #

def test_e8m0_scale_is_the_smallest_power_of_two():
    for top in (448.0, 448.0 * (1 + 2 ** -20), 1.0, 1.75, 1.7500001, 3e38, 2.0 ** -110, 1e-30):
        x = torch.zeros(1, 128)
        x[0, 5] = top
        q = quantize_fp8(x)
        s = q.scale.double().item()
        v = x[0, 5].double().item()
        assert v <= 448 * s and v > 448 * s / 2
        assert math.log2(s) == int(math.log2(s))
        assert abs(q.dequantize()[0, 5].double().item() - v) <= 2 ** -4 * v


def test_block_of_zeros_and_below_the_floor():
    x = torch.zeros(2, 200)
    x[1] = 2.0 ** -140
    for kind in ("e8m0", "fp32"):
        q = quantize_fp8(x, scale=kind)
        assert torch.equal(q.dequantize(), torch.zeros(2, 200))
        assert (q.scale.float() > 0).all()


@pytest.mark.parametrize("kind", ["e8m0", "fp32"])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_not_finite_spreads_over_its_block_only(kind, bad):
    x = torch.randn(3, 300)
    x[1, 130] = bad
    q = quantize_fp8(x, scale=kind)
    nan = torch.isnan(q.dequantize())
    assert nan[1, 128:256].all() and nan.sum() == 128
    y = fp8_matmul(q, quantize_fp8(torch.randn(4, 300), tile=True, scale=kind),
                   out_dtype=torch.float32)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[[0, 2]]).all()


@pytest.mark.parametrize("kind", ["e8m0", "fp32"])
@pytest.mark.parametrize("tile", [False, True])
def test_quantize_error(kind, tile):
    x = torch.randn(130, 261) * torch.logspace(-3, 3, 261)
    q = quantize_fp8(x, tile=tile, scale=kind)
    assert tuple(q.scale.shape) == ((2 if tile else 130), 3)
    factor = q.scale.float().repeat_interleave(128, 1)[:, :261]
    if tile:
        factor = factor.repeat_interleave(128, 0)[:130]
    # half a step of a normal code is 2^-4 of it, of a subnormal one 2^-10;
    # two 32-bit roundings in the factor and its inverse
    assert ((q.dequantize() - x).abs() <= (2 ** -4 + 4 * U32) * x.abs() + 2 ** -10 * factor).all()


def test_blocks_from_parts_copy_what_is_not_laid_out():
    big = torch.randn(6, 400)
    q = quantize_fp8(big[:, :300].contiguous())
    wide = torch.full((6, 400), float("nan")).to(torch.float8_e4m3fn)
    wide[:, :300] = q.values
    again = Fp8Blocks(wide[:, :300], q.scale)
    assert torch.equal(again.dequantize(), q.dequantize())
    assert torch.equal(again._codes[:, 300:].float(), torch.zeros(6, 84))
    w = torch.randn(5, 300)
    wq = quantize_fp8(w, tile=True)
    assert torch.equal(fp8_matmul(again, wq), fp8_matmul(q, wq))


def _parts(rows=4, cols=256, tile=False):
    q = quantize_fp8(torch.randn(rows, cols), tile=tile)
    return q.values, q.scale


@pytest.mark.parametrize("bad", [
    lambda: Fp8Blocks(torch.ones(4, 256), _parts()[1]),
    lambda: Fp8Blocks(_parts()[0], _parts()[1].float().double()),
    lambda: Fp8Blocks(_parts()[0], _parts()[1][:, :1]),
    lambda: Fp8Blocks(_parts()[0], _parts()[1], tile=True),
    lambda: Fp8Blocks(_parts()[0][:, :0], _parts()[1][:, :0]),
    lambda: quantize_fp8(torch.ones(4, 4, dtype=torch.float64)),
    lambda: quantize_fp8(torch.ones(4)),
    lambda: quantize_fp8(torch.ones(4, 0)),
    lambda: quantize_fp8(torch.ones(4, 4), scale="e5m2"),
    lambda: fp8_matmul(torch.ones(4, 4), quantize_fp8(torch.ones(4, 4))),
    lambda: fp8_matmul(quantize_fp8(torch.ones(4, 4), tile=True), quantize_fp8(torch.ones(4, 4))),
    lambda: fp8_matmul(quantize_fp8(torch.ones(4, 4)), quantize_fp8(torch.ones(4, 5))),
    lambda: fp8_matmul(quantize_fp8(torch.ones(4, 4)), quantize_fp8(torch.ones(4, 4), scale="fp32")),
    lambda: fp8_matmul(quantize_fp8(torch.ones(4, 4)), quantize_fp8(torch.ones(4, 4)),
                       bias=torch.ones(3)),
    lambda: fp8_matmul(quantize_fp8(torch.ones(4, 4)), quantize_fp8(torch.ones(4, 4)),
                       out_dtype=torch.float64),
    lambda: fp8_linear(torch.ones(2, 4, requires_grad=True), quantize_fp8(torch.ones(3, 4), tile=True)),
    lambda: fp8_linear(torch.ones(2, 5), torch.ones(3, 4)),
    lambda: fp8_linear(torch.ones(2, 4), torch.ones(3, 4), torch.ones(4)),
    lambda: fp8_linear(torch.ones(2, 4).double(), torch.ones(3, 4)),
])
def test_fp8_refusals(bad):
    with pytest.raises((TypeError, ValueError, RuntimeError)):
        bad()


# --------------------------------------------------------------------------- #
# the head in training
# --------------------------------------------------------------------------- #

def test_fp8_linear_gradients_are_the_formulas():
    x = torch.randn(2, 65, 200, requires_grad=True)
    layer = Fp8Linear(200, 130)
    y = layer(x)
    dy = torch.randn_like(y)
    dx, dw, db = torch.autograd.grad(y, (x, layer.weight, layer.bias), dy)
    flat, g = x.detach().view(130, 200), dy.view(130, 130)
    w = quantize_fp8(layer.weight, tile=True).dequantize().double()
    want_y = quantize_fp8(flat).dequantize().double() @ w.t() + layer.bias.double()
    want_dx = quantize_fp8(g).dequantize().double() @ w
    want_dw = (quantize_fp8(g.t()).dequantize().double()
               @ quantize_fp8(flat.t()).dequantize().double().t())
    # 32-bit sums of at most 200 products: 201 roundings of the sum of magnitudes
    for got, want, scale in ((y.view(130, 130), want_y, 20.0), (dx.view(130, 200), want_dx, 20.0),
                             (dw, want_dw, 200.0), (db, g.double().sum(0), 200.0)):
        assert (got.double() - want).abs().max() <= 201 * U32 * scale * 10


def test_fp8_linear_gradients_against_differences():
    """The loss is linear in each input but for the rounding to e4m3, so a whole
    step's difference is the gradient's product with it, to the roundings: each
    value is off by at most 2^-4 of itself, independently of the others, so the
    sum of n products by about sqrt(2 n) 2^-4 / sqrt(3) of a product; five times
    that is allowed."""
    x, w = torch.randn(64, 256), torch.randn(96, 256) / 16
    dy = torch.randn(64, 96)
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(fp8_linear(x, w), (x, w), dy)
    with torch.no_grad():
        for t, g, other in ((x, dx, w), (w, dw, x)):
            d = torch.randn_like(t)
            args = lambda v: (v, w) if t is x else (x, v)  # noqa: E731
            change = ((fp8_linear(*args(t + d)) - fp8_linear(*args(t - d))) * dy).sum() / 2
            n = 64 * 96 * 256
            size = 5 * math.sqrt(4 * n) * 2 ** -4 / math.sqrt(3) * (1 if t is w else 1 / 16)
            assert abs(change - (g * d).sum()) < size


def test_weight_kept_in_blocks_gives_the_same_head():
    x, layer = torch.randn(7, 200), Fp8Linear(200, 30)
    with torch.no_grad():
        assert torch.equal(fp8_linear(x, layer.quantized(), layer.bias), layer(x))
    assert list(layer.state_dict()) == list(torch.nn.Linear(200, 30).state_dict())


# --------------------------------------------------------------------------- #
# clipping
# --------------------------------------------------------------------------- #

def _params(sizes, scale=1.0):
    ps = [torch.nn.Parameter(torch.randn(s)) for s in sizes]
    for p in ps:
        p.grad = torch.randn_like(p) * scale
    return ps


def test_clip_grad_norm_matches_formula():
    ps = _params([(3, 4), (5,), (1,)])
    want = math.sqrt(sum(p.grad.double().square().sum().item() for p in ps))
    before = [p.grad.clone() for p in ps]
    norm = clip_grad_norm_(ps, 0.5)
    assert abs(norm.item() - want) <= 2 * U32 * want
    for p, b in zip(ps, before):
        assert torch.allclose(p.grad, b * (0.5 / (want + 1e-6)), rtol=8 * U32, atol=0)
    kept = [p.grad.clone() for p in ps]
    clip_grad_norm_(ps, 10.0)
    assert all(torch.equal(p.grad, k) for p, k in zip(ps, kept))


def test_norm_range_repeats_and_nothing():
    big, small = torch.full((4,), 1e30), torch.full((4,), 1e-30)
    assert abs(grad_norm([big]).item() / 2e30 - 1) < 4 * U32
    assert abs(grad_norm([small]).item() / 2e-30 - 1) < 4 * U32
    assert grad_norm([big, big, None]).item() == grad_norm(big).item()
    assert grad_norm([]).item() == 0
    p = torch.nn.Parameter(torch.ones(3))
    assert clip_grad_norm_([p], 1.0).item() == 0
    p.grad = torch.full((3,), 2.0)
    clip_grad_norm_([p, p], 1.0)
    assert abs(p.grad.norm().item() - 1) < 1e-5


@pytest.mark.parametrize("bad", [
    lambda: clip_grad_norm_(_params([(3,)]), -1.0),
    lambda: clip_grad_norm_(_params([(3,)]), float("nan")),
    lambda: grad_norm([torch.ones(3, dtype=torch.int32)]),
    lambda: FusedSGD(_params([(3,)]), lr=0.1, max_grad_norm=-1),
    lambda: FusedAdam(_params([(3,)]), max_grad_norm=float("nan")),
])
def test_clip_refusals(bad):
    with pytest.raises((TypeError, ValueError)):
        bad()


@pytest.mark.parametrize("name,args", [("SGD", {"lr": 0.1, "momentum": 0.9, "weight_decay": 1e-2}),
                                       ("Adam", {"lr": 0.1, "weight_decay": 1e-2})])
def test_optimizer_clips_inside_its_step(name, args):
    """The clipped step equals clipping first and stepping then, and leaves the
    gradients as they are; a bound that is not reached changes no bit."""
    sizes = [(3, 4), (5,), (130,)]
    torch.manual_seed(1)
    a = _params(sizes)
    torch.manual_seed(1)
    b = _params(sizes)
    grads = [p.grad.clone() for p in a]
    oa, ob = build_optimizer(name, a, max_grad_norm=0.5, **args), build_optimizer(name, b, **args)
    for _ in range(3):
        oa.step()
        for p, g in zip(b, grads):
            p.grad = g.clone()
        norm = clip_grad_norm_(b, 0.5)
        ob.step()
        assert torch.equal(oa.last_grad_norm, norm)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(p.grad, g) for p, g in zip(a, grads))
    oa.max_grad_norm = 1e9
    for p, g in zip(b, grads):
        p.grad = g.clone()
    oa.step()
    ob.step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert "max_grad_norm" not in oa.param_groups[0]


def test_head_step_from_norm_to_clipped_update():
    """Norm, e4m3 head, loss and clipped step together, run twice from one seed."""
    from active_learning_amd.ops.loss import cross_entropy

    def train():
        torch.manual_seed(3)
        norm, head = RMSNorm(64), Fp8Linear(64, 10)
        params = [*norm.parameters(), *head.parameters()]
        opt = FusedSGD(params, lr=0.1, momentum=0.9, max_grad_norm=0.1)
        x, y = torch.randn(32, 64), torch.randint(0, 10, (32,))
        for _ in range(3):
            opt.zero_grad()
            cross_entropy(head(norm(x)), y).backward()
            opt.step()
        return [p.detach() for p in params], opt.last_grad_norm

    (a, na), (b, nb) = train(), train()
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(na, nb)
    assert all(torch.isfinite(p).all() for p in a) and na > 0


def test_outputs_may_be_changed_in_place():
    x = torch.randn(2, 3, 64, requires_grad=True)
    w = torch.nn.Parameter(torch.randn(64))
    y = rms_norm(x, w)
    y.mul_(2)
    y.sum().backward()
    want = torch.autograd.grad((rms_norm(x, w) * 2).sum(), (x, w))
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
    y, total = rms_norm(x, w, residual=x.detach())
    total.add_(1)  # the backward pass needs it
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("eps", [0.0, -1.0, 1e-46, float("nan")])
def test_eps_that_32_bits_do_not_hold(eps):
    with pytest.raises(ValueError, match="eps must be positive"):
        rms_norm(torch.zeros(1, 8), torch.ones(8), eps=eps)


def test_clip_refuses_shared_memory_and_leaves_all_without_a_bound():
    both = torch.randn(6)
    p, q = torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4))
    p.grad, q.grad = both[:4], both[2:]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_([p, q], 0.1)
    p.grad, q.grad = torch.full((4,), float("inf")), torch.ones(4)
    assert clip_grad_norm_([p, q], float("inf")) == float("inf")
    assert torch.equal(q.grad, torch.ones(4))


def test_no_rows_and_no_outputs():
    x, w = torch.zeros(3, 0, 256, requires_grad=True), torch.ones(256, requires_grad=True)
    weight = torch.randn(40, 256, requires_grad=True)
    y, total = rms_norm(x, w, residual=x.detach())
    z = fp8_linear(y, weight)
    assert z.shape == (3, 0, 40) and total.shape == x.shape
    grads = torch.autograd.grad(z.sum(), (x, w, weight))
    assert all((g == 0).all() for g in grads)
    x = torch.randn(5, 256, requires_grad=True)
    z = fp8_linear(x, weight[:0])
    (dx,) = torch.autograd.grad(z.sum(), x)
    assert z.shape == (5, 0) and (dx == 0).all()
