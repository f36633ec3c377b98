"""The norm, the e4m3 products and the clipped steps on the CPU: calls that used to be
answered wrongly or forgotten, each with what it has to give."""

import pytest
import torch

from active_learning_amd.ops.fp8 import fp8_linear, quantize_fp8
from active_learning_amd.ops.grad_clip import clip_grad_norm_
from active_learning_amd.ops.optim import FusedSGD, build_optimizer
from active_learning_amd.ops.rmsnorm import rms_norm, rms_norm_fp8


def _params(sizes):
    ps = [torch.nn.Parameter(torch.randn(s)) for s in sizes]
    for p in ps:
        p.grad = torch.randn_like(p)
    return ps


@pytest.fixture
def capturing(monkeypatch):
    """A switch that makes the optimizer see a stream that is being captured."""
    from active_learning_amd.ops import optim
    state = {"on": False}
    monkeypatch.setattr(optim, "_stream_capturing", lambda: state["on"])
    return lambda on: state.update(on=on)


@pytest.mark.parametrize("bound", [None, 0.5])
def test_momentum_cannot_come_after_the_capture(capturing, bound):
    """A step that is captured without momentum has no buffers for it."""
    opt = FusedSGD(_params([(3, 4)]), lr=0.1, max_grad_norm=bound)
    opt.enable_device_hyper("cpu")
    opt.step()
    capturing(True)
    opt.step()
    capturing(False)
    opt.param_groups[0]["lr"] = 0.05
    opt.sync_hyper()
    opt.param_groups[0]["momentum"] = 0.9
    with pytest.raises(ValueError, match="captured without momentum"):
        opt.sync_hyper()
    assert opt._hyper_dev[1] == 0
    # with buffers at the capture it may come and go
    opt = FusedSGD(_params([(3, 4)]), lr=0.1, momentum=0.9, max_grad_norm=bound)
    opt.enable_device_hyper("cpu")
    opt.step()
    opt.param_groups[0]["momentum"] = 0.0
    opt.sync_hyper()
    capturing(True)
    opt.step()
    capturing(False)
    opt.param_groups[0]["momentum"] = 0.9
    opt.sync_hyper()
    assert abs(opt._hyper_dev[1] - 0.9) < 1e-6


@pytest.fixture
def norm_calls(monkeypatch):
    """What each step hands to the norm: the bound on the host, on the device, and where to."""
    from active_learning_amd.ops import optim
    calls, real = [], optim._params_norm_factor

    def spy(params, max_norm, max_dev=None, to=None):
        calls.append((max_norm, max_dev, to))
        return real(params, max_norm)

    monkeypatch.setattr(optim, "_params_norm_factor", spy)
    return calls


def test_bound_set_at_the_capture_is_followed(capturing, norm_calls):
    """A bound that is set or changed on exactly the step that is captured is read from
    the device, so that later changes reach the captured step."""
    opt = FusedSGD(_params([(3, 4)]), lr=0.1)
    opt.enable_device_hyper("cpu")
    opt.step()
    assert not norm_calls
    opt.max_grad_norm = 0.5
    with opt.capture_of(test_bound_set_at_the_capture_is_followed):
        capturing(True)
        with pytest.raises(RuntimeError, match="sync_hyper"):  # refused, not forgotten
            opt.step()
        capturing(False)
        opt.sync_hyper()
        capturing(True)
        opt.step()
        capturing(False)
    _, on_device, to = norm_calls[-1]
    assert on_device is not None and to is not None and on_device.item() == 0.5
    opt.max_grad_norm = 0.25
    opt.sync_hyper()
    assert on_device.item() == 0.25
    opt.max_grad_norm = None
    opt.sync_hyper()
    assert on_device.item() == float("inf")
    # an eager step between, and another user of the same optimizer, leave it in place
    opt.max_grad_norm = 0.125
    opt.step()
    opt.enable_device_hyper("cpu")
    assert norm_calls[-1][1] is on_device and on_device.item() == 0.125 and opt._clip_dev is on_device


def test_refusals_last_as_long_as_the_captured_step(capturing):
    class Owner:
        pass

    opt = FusedSGD(_params([(3, 4)]), lr=0.1)
    opt.enable_device_hyper("cpu")

    def capture(owner, fails=False):
        with opt.capture_of(owner):
            capturing(True)
            opt.step()
            capturing(False)
            if fails:
                raise OSError("capture")

    def set_all():
        opt.max_grad_norm, opt.param_groups[0]["momentum"] = 0.5, 0.9
        try:
            opt.sync_hyper()
        finally:
            opt.max_grad_norm, opt.param_groups[0]["momentum"] = None, 0.0

    failed, kept = Owner(), Owner()
    with pytest.raises(OSError):
        capture(failed, fails=True)
    set_all()
    capture(kept)
    with pytest.raises(ValueError, match="captured without"):
        set_all()
    del kept
    set_all()


def test_hyperparameters_on_their_way_keep_their_values():
    """A copy to the device runs behind the steps that are queued: the next change does
    not write into the host memory that it reads."""
    opt = FusedSGD(_params([(3, 4)]), lr=0.1, momentum=0.9)
    opt.enable_device_hyper("cpu")
    sent = []

    class Device:
        is_cuda = False

        def copy_(self, host, non_blocking=False):
            sent.append(host)

    opt._hyper_dev = Device()
    for lr in (0.5, 0.25):
        opt.param_groups[0]["lr"] = lr
        opt.sync_hyper()
        opt.sync_hyper()
    assert [t[0].item() for t in sent] == [0.5, 0.25]


@pytest.mark.parametrize("name", ["SGD", "Adam"])
@pytest.mark.parametrize("bound", [-1.0, float("nan")])
def test_a_bound_that_is_set_later_is_checked(name, bound):
    """A negative one would turn the gradients round."""
    opt = build_optimizer(name, _params([(3, 4)]), lr=0.1, max_grad_norm=1.0)
    with pytest.raises(ValueError, match="max_grad_norm"):
        opt.max_grad_norm = bound
    assert opt.max_grad_norm == 1.0
    opt.max_grad_norm = None
    opt.step()
    assert opt.last_grad_norm is None


def _with_tangents(device):
    """Calls with one dual tensor each, by name."""
    from torch.autograd import forward_ad
    x, w = torch.randn(20, 8, device=device), torch.randn(8, device=device)
    weight, bias = torch.randn(3, 8, device=device), torch.randn(3, device=device)
    kept = quantize_fp8(weight, tile=True)

    def dual(t):
        return forward_ad.make_dual(t, torch.ones_like(t))

    return {
        "norm": lambda: rms_norm(dual(x), w), "norm's weight": lambda: rms_norm(x, dual(w)),
        "residual": lambda: rms_norm(x, w, residual=dual(x)), "codes": lambda: rms_norm_fp8(dual(x), w),
        "codes' residual": lambda: rms_norm_fp8(x, w, residual=dual(x)),
        "linear": lambda: fp8_linear(dual(x), weight), "weight": lambda: fp8_linear(x, dual(weight)),
        "bias": lambda: fp8_linear(x, weight, dual(bias)), "kept": lambda: fp8_linear(dual(x), kept),
        "kept, one row": lambda: fp8_linear(dual(x[:1]), kept),
        "kept weight's bias": lambda: fp8_linear(x, kept, dual(bias)),
    }


@pytest.mark.parametrize("name", list(_with_tangents("cpu")))
def test_forward_mode_is_refused(name):
    """An output without a tangent would read as a derivative of zero."""
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        call = _with_tangents("cpu")[name]
        with pytest.raises(NotImplementedError):
            call()
        with torch.no_grad(), pytest.raises(NotImplementedError):  # it has no say in this mode
            call()


@pytest.mark.parametrize("device", ["cpu"])
def test_second_gradients_are_refused_not_zero(device):
    """A penalty on a gradient would have no effect; what does not depend on anything that
    asks for a gradient may be used as the constant that it is."""
    x, r, w = (torch.randn(*s, device=device).requires_grad_() for s in ((20, 8), (20, 8), (8,)))
    weight = torch.randn(3, 8, device=device).requires_grad_()
    bias = torch.randn(3, device=device).requires_grad_()
    cases = [
        (lambda: rms_norm(x, w), (x, w)), (lambda: rms_norm(x, w), (x,)), (lambda: rms_norm(x, w.detach()), (x,)),
        (lambda: rms_norm(x, w), (w,)), (lambda: rms_norm(x.detach(), w, residual=r)[0], (r, w)),
        (lambda: sum(rms_norm(x, w, residual=r)), (x, r, w)),
        (lambda: fp8_linear(x, weight, bias), (x,)), (lambda: fp8_linear(x, weight, bias), (weight,)),
    ]
    for f, leaves in cases:
        want = torch.autograd.grad(f().sum(), leaves)
        grads = torch.autograd.grad(f().sum(), leaves, create_graph=True)
        for g, v in zip(grads, want):
            assert torch.equal(g, v)
            with pytest.raises(RuntimeError, match="differentiable once"):
                g.square().sum().backward(retain_graph=True)
    constants = [
        (lambda: rms_norm(x.detach(), w), w), (lambda: fp8_linear(x, weight.detach()), x),
        (lambda: fp8_linear(x.detach(), weight), weight), (lambda: fp8_linear(x, weight, bias), bias),
        (lambda: rms_norm(x, w, residual=r)[1], x),
    ]
    for f, leaf in constants:
        (g,) = torch.autograd.grad(f().sum(), leaf, create_graph=True)
        assert not g.requires_grad
    # the sum's gradient goes through as it is
    dsum = torch.randn(20, 8, device=device).requires_grad_()
    (g,) = torch.autograd.grad(rms_norm(x, w, residual=r)[1], r, dsum, create_graph=True)
    (back,) = torch.autograd.grad(g.square().sum(), dsum)
    assert torch.equal(back, 2 * dsum)


@pytest.mark.parametrize("size", [1e-30, 1e19, 3e19, 1e20, 1e30, 1e37])
@pytest.mark.parametrize("dim", [8, 300, 2048, 5000, 40000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_of_large_and_small_values(dim, size, dtype):
    """Squares that leave the range of 32 bits: the norm is that of any other row, forward,
    backward and in front of codes."""
    x = (torch.randn(3, dim, device="cpu") * size).to(dtype).requires_grad_()
    w = (torch.rand(dim, device="cpu") + 0.5).requires_grad_()
    dy = torch.randn(3, dim, device="cpu").to(dtype)
    eps = 1e-6 if size > 1 else 1e-38  # the smallest normal one and a root that counts in 64 bits
    y = rms_norm(x, w, eps=eps)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    s = x.detach().double()
    root = (s.square().mean(-1, keepdim=True) + torch.tensor(eps).double().item()).sqrt()
    u, g = s / root, dy.double() * w.detach().double()
    half = torch.finfo(dtype).eps / 2
    # 1 / root, two products and a rounding; the dot product's 32-bit sum of dim / 1024 + 24 terms
    # behind each other at most, which the gradients are off by as well (CPU: pairwise sums, fewer)
    many = (dim / 1024 + 24) * 2.0 ** -24
    want = u * w.detach().double()
    assert ((y.double() - want).abs() <= (half + 4 * 2.0 ** -24) * want.abs() + 2.0 ** -133).all()
    dot = (g * u).mean(-1, keepdim=True)
    want = (g - u * dot) / root
    scale = (g.abs() + u.abs() * (g * u).abs().mean(-1, keepdim=True)) / root
    least = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -148
    assert ((dx.double() - want).abs() <= half * want.abs() + 4 * many * scale + least).all()
    want = (dy.double() * u).sum(0)
    assert ((dw.double() - want).abs() <= 6 * 2.0 ** -24 * (dy.double() * u).abs().sum(0)).all()
    with torch.no_grad():
        q = rms_norm_fp8(x, w, eps=eps)
    spread = q.scale.double().repeat_interleave(128, 1)[:, :dim]
    want = u * w.detach().double()
    assert ((q.values.double() * spread - want).abs() <= (2.0 ** -4 + 2.0 ** -20) * want.abs() + 2.0 ** -10 * spread).all()


@pytest.mark.parametrize("rows,cols", [(300, 20), (8000, 300)])
def test_bias_gradient_is_rounded_once(rows, cols):
    """Its sum is held in 64 bits: off by the one rounding to its type."""
    x, w = torch.randn(rows, 64, device="cpu"), torch.randn(cols, 64, device="cpu")
    for dtype in (torch.float32, torch.bfloat16):
        bias = torch.zeros(cols, device="cpu", dtype=dtype).requires_grad_()
        for kind in ("e8m0", "fp32"):
            y = fp8_linear(x, w, bias, scale=kind)
            dy = torch.randn_like(y)
            (db,) = torch.autograd.grad(y, bias, dy)
            want, size = dy.double().sum(0), dy.double().abs().sum(0)
            # a 16-bit one through 32 bits
            half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8 + 2.0 ** -23
            assert ((db.double() - want).abs() <= half * want.abs() + rows * 2.0 ** -52 * size).all()


def test_only_steps_that_a_replay_can_follow_are_captured():
    from active_learning_amd.ops.graph import GraphedTrainStep
    net = torch.nn.Linear(4, 3)
    for opt in (build_optimizer("Adam", net.parameters(), max_grad_norm=0.5),
                FusedSGD([{"params": [net.weight]}, {"params": [net.bias]}], lr=0.1)):
        assert GraphedTrainStep(net, opt, torch.nn.CrossEntropyLoss(), torch.device("cuda"))._failed


def test_clip_scales_shared_memory_once_or_refuses():
    base = torch.arange(1.0, 13.0, device="cpu")

    def clip(*grads):
        ps = [torch.nn.Parameter(torch.zeros(g.shape, device="cpu")) for g in grads]
        for p, g in zip(ps, grads):
            p.grad = g
        return clip_grad_norm_(ps, 1.0)

    keep, square = base.clone(), base.view(3, 4)
    for shared in ((square, square.t()), (torch.ones(1, device="cpu").expand(5),),
                   (base, torch.ones(2, 1, device="cpu").expand(2, 4)), (base[:8], base[4:])):
        before = [g.clone() for g in shared]
        with pytest.raises(RuntimeError, match="share memory"):
            clip(*shared)
        assert all(torch.equal(g, b) for g, b in zip(shared, before))
    # every second value is there twice: it counts twice in the norm, and is scaled once
    norm = (keep.double().square().sum() + keep[::2].double().square().sum()).sqrt().item()
    assert abs(clip(base, base[::2]).item() - norm) <= 2 * 2.0 ** -24 * norm
    assert ((base.double() - keep.double() / (norm + 1e-6)).abs() <= 4 * 2.0 ** -24 * base.double()).all()
    empty = torch.empty(3, 0, device="cpu")
    assert clip(empty, empty.t()).item() == 0.0


@pytest.mark.parametrize("bad", [torch.zeros(11), torch.zeros(12, dtype=torch.float64), torch.zeros(3, 4).t(), torch.zeros(12).expand(2, 12)[:, ::2]])
def test_momentum_that_does_not_fit_is_refused(bad):
    """The table of the multi-tensor step takes addresses only of what fits its parameter."""
    from active_learning_amd.ops.extension import load_extension
    ext, p = load_extension(), torch.nn.Parameter(torch.zeros(3, 4))
    p.grad = torch.zeros(3, 4)
    assert len(ext.sgd_addresses([p], [torch.zeros(12)], [None])) == 40
    with pytest.raises(ValueError, match="momentum_buffer"):
        ext.sgd_addresses([p], [bad], [None])
    with pytest.raises(ValueError, match="bf16"):
        ext.sgd_addresses([p], [None], [bad])


def test_default_type_of_64_bits():
    """What torch makes by default has no say in types that are fixed."""
    x, w = torch.randn(20, 300, device="cpu"), torch.randn(40, 300, device="cpu")
    norm_weight = torch.rand(300, device="cpu")
    x[3, 7] = float("nan")

    def run():
        out = []
        for kind in ("e8m0", "fp32"):
            q = rms_norm_fp8(x, norm_weight, scale=kind)
            out += [q.values.float(), q.scale.float(), fp8_linear(x, quantize_fp8(w, tile=True, scale=kind))]
        p = torch.nn.Parameter(x[:2].clone())
        p.grad = x[4:6].clone()
        opt = FusedSGD([p], lr=0.5, momentum=0.9, max_grad_norm=0.5)
        opt.enable_device_hyper("cpu")
        opt.step()
        return [*out, rms_norm(x, norm_weight), p.detach(), opt.last_grad_norm, clip_grad_norm_([], 1.0)]

    want = run()
    torch.set_default_dtype(torch.float64)
    try:
        got = run()
    finally:
        torch.set_default_dtype(torch.float32)
    for g, v in zip(got, want):
        assert g.dtype == v.dtype == torch.float32 and torch.equal(g.nan_to_num(9), v.nan_to_num(9))
