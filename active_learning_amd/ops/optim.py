"""Fused optimizers.

Reference reaches SGD+momentum+weight-decay through torch.optim (built from
config strings by eval at strategy.py:345-350; hyperparameters in
arg_pools/default.py:39-40). Here: an SGD with a single fused HIP update
kernel per tensor on GPU (update + momentum + weight decay in one pass over
fp32 master params), torch math on CPU. Adam (VAAL's VAE/discriminator,
vaal_sampler.py:139-140) likewise.

Constructor signatures match torch.optim so arg-pool optimizer_args apply
unchanged; the trainer maps names through OPTIMIZERS.
"""

import contextlib
import struct
import weakref

import torch

from .extension import extension_available, load_extension
from .functional import bump_tick
from .grad_clip import _params_norm_factor


def _invalidate(p):
    """Native updates mutate storage without bumping torch's version counter;
    drop the per-version bf16 weight cache (ops/functional.cast_cached)."""
    if getattr(p, "_al_cast", None) is not None:
        p._al_cast = None


def _check_max_norm(max_grad_norm):
    if max_grad_norm is not None and not float(max_grad_norm) >= 0:
        raise ValueError(f"max_grad_norm must not be negative, got {max_grad_norm}")
    return max_grad_norm


def _stream_capturing():
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


class _Clips:
    """The bound of an optimizer that clips, checked whenever it is set."""

    @property
    def max_grad_norm(self):
        return self._max_grad_norm

    @max_grad_norm.setter
    def max_grad_norm(self, bound):
        self._max_grad_norm = _check_max_norm(bound)


def _all_params(optimizer):
    return [p for group in optimizer.param_groups for p in group["params"]]


class FusedSGD(_Clips, torch.optim.Optimizer):
    """SGD with momentum and weight decay.

    ``max_grad_norm``: the step uses gradients scaled so that their norm over all
    parameters is at most this (ops/grad_clip.py). The scaling happens as the
    update reads them: ``p.grad`` keeps its values, and the norm they had is
    ``last_grad_norm``, a 0-d tensor on the device that later steps leave alone.
    """

    _CHUNK = 32768  # elements per workgroup in the multi-tensor kernel

    def __init__(self, params, lr, momentum=0.0, weight_decay=0.0, dampening=0.0,
                 nesterov=False, max_grad_norm=None):
        if nesterov:
            raise ValueError("nesterov not supported")
        if dampening != 0:
            raise ValueError("dampening not supported")
        defaults = dict(lr=lr, momentum=momentum, weight_decay=weight_decay,
                        dampening=dampening)
        super().__init__(params, defaults)
        self._mt_cache = {}  # group idx -> (fingerprint, device table, nchunks)
        self._wt_cache = {}  # group idx -> (fingerprint, tile table, nrows)
        self._mt_keepalive = []  # device tables that a captured step reads, and outgrown ones
        self._hyper_dev = None   # device (lr, momentum, wd); graph-capture mode
        self._hyper_host = None
        self._persistent = False  # grads kept in stable storage, zeroed in-kernel
        self.max_grad_norm = max_grad_norm
        self._last_norm = None
        self._clip_dev = None    # device max_grad_norm; graph-capture mode
        self._clip_to = None     # where captured and eager steps alike leave norm and factor
        self._clip_host = None
        # who holds a captured step -> what that step cannot follow: "max_grad_norm"
        # where it was captured without, "momentum" where a buffer was missing
        self._left_out = weakref.WeakKeyDictionary()
        self._capture_owner = None

    def enable_persistent_grads(self):
        """Persistent-grad mode for hipGraph capture: the caller must NOT call
        zero_grad — gradient tensors keep their storage across steps (backward
        accumulates in place) and the fused update zeroes them after
        consumption. This keeps the captured step allocation-free."""
        self._persistent = True

    def enable_device_hyper(self, device):
        """Switch the fused update to read (lr, momentum, wd) and the clipping bound
        from device memory so a hipGraph-captured step tracks their changes without
        re-capture; call sync_hyper() OUTSIDE capture right before it and whenever
        one of them changed. What a captured step has no part for (momentum, where
        a buffer was missing; a clipping bound, where there was none) cannot come
        later: sync_hyper refuses it as long as the step is there."""
        assert len(self.param_groups) == 1, "device-hyper mode: single group"
        device = torch.empty(0, device=device).device
        if self._hyper_dev is None or self._hyper_dev.device != device:
            # otherwise a step that was captured before goes on to follow
            self._hyper_host = None
            self._hyper_dev = torch.zeros(3, dtype=torch.float32, device=device)
            self._clip_dev = torch.full((1,), float("inf"), dtype=torch.float32, device=device)
            self._clip_to = torch.zeros(2, dtype=torch.float32, device=device)
            self._clip_host = None
        self.sync_hyper()

    @property
    def last_grad_norm(self):
        # with device hyperparameters all steps leave theirs in one place
        if self._last_norm is None or self._clip_to is None:
            return self._last_norm
        return self._last_norm.clone()

    @contextlib.contextmanager
    def capture_of(self, owner):
        """Around a capture of step(): ``owner`` is what holds the captured step. A
        capture outside of this counts as the optimizer's own, for good."""
        self._capture_owner = owner
        try:
            yield
        except BaseException:
            self._left_out.pop(owner, None)
            raise
        finally:
            self._capture_owner = None

    def _leave_out(self, what):
        owner = self if self._capture_owner is None else self._capture_owner
        self._left_out.setdefault(owner, set()).add(what)

    def _capturing(self):
        return self._hyper_dev is not None and _stream_capturing()

    def sync_hyper(self):
        g = self.param_groups[0]
        vals = (float(g["lr"]), float(g["momentum"]), float(g["weight_decay"]))
        left_out = set().union(*self._left_out.values())
        if "momentum" in left_out and vals[1] != 0:
            raise ValueError("the step was captured without momentum: set it before the capture")
        if "max_grad_norm" in left_out and self.max_grad_norm is not None:
            raise ValueError("the step was captured without max_grad_norm: set it before the "
                             "capture")
        if self._hyper_host != vals:
            # host memory of its own: the copy before may still be on its way, behind
            # steps that are queued and read the values that it brings
            host = torch.tensor(vals, dtype=torch.float32)
            if self._hyper_dev.is_cuda:
                host = host.pin_memory()
            self._hyper_dev.copy_(host, non_blocking=True)
            self._hyper_host = vals
        self._sync_bound()

    def _sync_bound(self):
        bound = self.max_grad_norm
        if self._clip_host != bound:
            # a captured step goes on to look at the bound: none is an infinite one
            self._clip_dev.fill_(float("inf") if bound is None else float(bound))
            self._clip_host = bound

    def _clip(self):
        """(norm, factor) of this step's gradients on their device; None without
        max_grad_norm or gradients."""
        capturing = self._capturing()
        if self.max_grad_norm is None:
            if capturing:
                self._leave_out("max_grad_norm")
            return None
        if self._clip_dev is not None:
            if not capturing:
                self._sync_bound()
            elif self._clip_host != self.max_grad_norm:
                raise RuntimeError("max_grad_norm changed: call sync_hyper() before the capture")
        both = _params_norm_factor(_all_params(self), float(self.max_grad_norm),
                                   self._clip_dev, self._clip_to)
        if both is not None:
            self._last_norm = both[0]
        return both

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        ext = load_extension() if extension_available() else None
        clip = self._clip()
        capturing = self._capturing()
        for gi, group in enumerate(self.param_groups):
            lr = group["lr"]
            momentum = group["momentum"]
            wd = group["weight_decay"]
            fused = []
            params = [p for p in group["params"] if p.grad is not None and p.numel()]
            if capturing and momentum == 0 and any(
                    "momentum_buffer" not in self.state.get(p, ()) for p in params):
                self._leave_out("momentum")
            if ext is not None and params and ext.sgd_fusable(params):
                fused, params = params, []  # all of them: no look at each in Python
            for p in params:
                if (ext is not None and p.is_cuda
                        and p.dtype == torch.float32 and p.is_contiguous()
                        and p.grad.dtype == torch.float32
                        and p.grad.is_contiguous()):
                    fused.append(p)
                    continue
                g = p.grad
                state = self.state[p]
                if momentum != 0 and "momentum_buffer" not in state:
                    state["momentum_buffer"] = self._new_buffer(p)
                buf = state.get("momentum_buffer")
                if p.is_cuda and ext is not None and p.is_contiguous():
                    cache = getattr(p, "_al_cast", None)
                    shadow = (cache[1] if cache is not None
                              and cache[1].numel() == p.numel()
                              and cache[1].dtype == torch.bfloat16
                              else p.new_empty(0, dtype=torch.bfloat16))
                    self._sgd_step(ext, p, g.to(torch.float32), buf, lr, momentum, wd,
                                   shadow, clip)
                    if shadow.numel():
                        # the kernel refreshed the bf16 copy in-pass; derived
                        # caches (bwd-data permute) must be recomputed
                        if getattr(cache[1], "_al_wt", None) is not None:
                            cache[1]._al_wt = None
                        p._al_cast = (p._version, cache[1])
                    else:
                        _invalidate(p)
                    bump_tick(p)  # in-kernel update: no _version bump
                else:  # on the CPU, or of other strides than the kernels take
                    if p.is_cuda and capturing:
                        raise RuntimeError("a step that follows hyperparameters on the device "
                                           "needs contiguous parameters")
                    gf = g.float()
                    if clip is not None:
                        gf = gf * clip[1]
                    if wd != 0:
                        gf = gf.add(p, alpha=wd)
                    if momentum != 0:
                        buf.mul_(momentum).add_(gf)
                        gf = buf
                    p.add_(gf, alpha=-lr)
                if self._persistent:
                    g.zero_()
            if fused:
                self._multi_tensor_step(ext, gi, fused, lr, momentum, wd, clip)
        return loss

    @staticmethod
    def _new_buffer(p):
        if p.is_cuda and _stream_capturing():
            # each replay would fill it with zeros again
            raise RuntimeError("a step without its momentum buffers cannot be captured: take one "
                               "before")
        return torch.zeros_like(p, dtype=torch.float32)

    def _sgd_step(self, ext, p, g, buf, lr, momentum, wd, shadow, clip):
        if buf is None:
            buf = p.new_empty(0)
        if clip is None:
            ext.sgd_step(p, g, buf, lr, momentum, wd, shadow)
        else:
            ext.sgd_step_clip(p, g.contiguous(), buf, lr, momentum, wd, self._hyper_dev,
                              shadow, clip)

    def _multi_tensor_step(self, ext, gi, params, lr, momentum, wd, clip):
        """ONE kernel launch for the whole parameter set (the per-tensor path
        cost 161 launches/step on ResNet-50). Packs a chunk table of
        (p, grad, momentum-buf, bf16-shadow, offset, count) int64 rows; the
        device copy is cached and only refreshed when any pointer moves, so
        steady-state steps (and hipGraph captures) launch with no H2D
        traffic."""
        state = self.state
        if momentum != 0:
            for p in params:
                if "momentum_buffer" not in state[p]:
                    state[p]["momentum_buffer"] = self._new_buffer(p)
        bufs = [state[p].get("momentum_buffer") for p in params]
        shadows = []
        for p in params:
            cache = getattr(p, "_al_cast", None)
            shadows.append(cache[1] if cache is not None
                           and cache[1].numel() == p.numel()
                           and cache[1].dtype == torch.bfloat16 else None)
        # five words a parameter: its address, its gradient's, momentum's and
        # shadow's (0: none), and its length
        fp = ext.sgd_addresses(params, bufs, shadows)
        entry = self._mt_cache.get(gi)
        capturing = _stream_capturing()
        if entry is None or entry[0] != fp:
            if capturing:
                # a table rebuild needs host allocations, which invalidate
                # hipGraph capture — fall back to per-tensor launches for
                # this (captured) step. With persistent grads the
                # fingerprint is stable and this path never triggers.
                self._per_tensor_fallback(ext, params, lr, momentum, wd, clip)
                return
            rows = []
            for pp, gp, bp, sp, n in struct.iter_unpack("5q", fp):
                off = 0
                while off < n:
                    rows.append((pp, gp, bp, sp, off, min(self._CHUNK, n - off)))
                    off += self._CHUNK
            entry = self._new_table(self._mt_cache, gi, fp, rows, params[0].device)
        if capturing:
            self._keep(entry[1])
        if clip is not None:
            ext.sgd_step_multi_clip(entry[1], entry[2], lr, momentum, wd,
                                    self._hyper_dev, clip, self._persistent)
        elif self._hyper_dev is not None:
            ext.sgd_step_multi_dev(entry[1], entry[2], self._hyper_dev,
                                   self._persistent)
        else:
            ext.sgd_step_multi(entry[1], entry[2], lr, momentum, wd,
                               self._persistent)
        wt_fp, wt_entries = [], []
        for p, shadow in zip(params, shadows):
            if shadow is not None:
                wt = getattr(shadow, "_al_wt", None)
                if wt is not None:
                    if (shadow.dim() == 4 and shadow.shape[0] % 64 == 0
                            and shadow.shape[3] % 64 == 0):
                        # refreshed by ONE batched transpose kernel below
                        # instead of a per-conv ATen permute+clone
                        wt_fp.append((shadow.data_ptr(), wt.data_ptr())
                                     + tuple(shadow.shape))
                        wt_entries.append(shadow)
                    else:
                        shadow._al_wt = None
                p._al_cast = (p._version, shadow)
            else:
                _invalidate(p)
            bump_tick(p)
        if wt_fp:
            self._launch_wt_refresh(ext, gi, tuple(wt_fp), wt_entries)

    def _keep(self, table):
        if not any(table is t for t in self._mt_keepalive):
            self._mt_keepalive.append(table)

    def _new_table(self, cache, gi, fp, rows, device):
        """Copies a table to the device, over the one that it replaces: a step whose
        addresses changed (new gradients) takes no more memory than the one before.
        Where a captured step reads that one, or it is too short, the new one gets
        memory of its own, and an outgrown one stays, since a step on another stream
        may still read it; sizes double, so that these are few."""
        host = torch.tensor(rows, dtype=torch.int64).pin_memory()
        dev = cache[gi][1] if gi in cache else None
        if dev is None or len(dev) < len(rows) or any(dev is t for t in self._mt_keepalive):
            size = len(rows)
            if dev is not None and len(dev) < size:
                self._keep(dev)
                size = max(size, 2 * len(dev))
            dev = torch.empty(size, host.shape[1], dtype=torch.int64, device=device)
        dev[:len(rows)].copy_(host, non_blocking=True)
        cache[gi] = entry = (fp, dev, len(rows))
        return entry

    def _launch_wt_refresh(self, ext, gi, fp, shadows):
        """Refresh every cached (C,R,S,K) bwd-data weight permutation in one
        launch (64x64 tiles; only full tiles are enqueued — the host gates on
        K, C % 64). Table cached by pointer fingerprint like the sgd chunk
        table, so steady-state (and captured) steps launch with no H2D."""
        entry = self._wt_cache.get(gi)
        capturing = _stream_capturing()
        if entry is None or entry[0] != fp:
            if capturing:
                for shadow in shadows:
                    shadow._al_wt = None  # lazy ATen rebuild for this step
                return
            rows = []
            for (sp, dp, K, R, S, C) in fp:
                RS = R * S
                for rs in range(RS):
                    for k0 in range(0, K, 64):
                        for c0 in range(0, C, 64):
                            rows.append((sp, dp,
                                         k0 | (c0 << 16) | (rs << 32),
                                         K | (C << 16) | (RS << 32)))
            entry = self._new_table(self._wt_cache, gi, fp, rows, shadows[0].device)
        if capturing:
            self._keep(entry[1])
        ext.wt_refresh_multi(entry[1], entry[2])

    def _per_tensor_fallback(self, ext, params, lr, momentum, wd, clip):
        for p in params:
            buf = self.state[p].get("momentum_buffer")
            cache = getattr(p, "_al_cast", None)
            shadow = (cache[1] if cache is not None
                      and cache[1].numel() == p.numel()
                      and cache[1].dtype == torch.bfloat16
                      else p.new_empty(0, dtype=torch.bfloat16))
            self._sgd_step(ext, p, p.grad, buf, lr, momentum, wd, shadow, clip)
            if self._persistent:
                p.grad.zero_()
            if shadow.numel():
                if getattr(shadow, "_al_wt", None) is not None:
                    shadow._al_wt = None
                p._al_cast = (p._version, shadow)
            else:
                _invalidate(p)
            bump_tick(p)


class FusedAdam(_Clips, torch.optim.Optimizer):
    """Adam; ``max_grad_norm`` and ``last_grad_norm`` as in FusedSGD."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0,
                 max_grad_norm=None):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        super().__init__(params, defaults)
        self.max_grad_norm = max_grad_norm
        self.last_grad_norm = None

    def _clip(self):
        if self.max_grad_norm is None:
            return None
        both = _params_norm_factor(_all_params(self), float(self.max_grad_norm))
        if both is not None:
            self.last_grad_norm = both[0]
        return both

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        ext = load_extension() if extension_available() else None
        clip = self._clip()
        for group in self.param_groups:
            lr = group["lr"]
            beta1, beta2 = group["betas"]
            eps = group["eps"]
            wd = group["weight_decay"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state["step"] = 0
                    state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
                    state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
                state["step"] += 1
                t = state["step"]
                bc1 = 1 - beta1 ** t
                bc2 = 1 - beta2 ** t
                if p.is_cuda and ext is not None and p.is_contiguous():
                    if clip is not None:
                        ext.adam_step_clip(p, p.grad.to(torch.float32).contiguous(),
                                           state["exp_avg"], state["exp_avg_sq"], lr, beta1,
                                           beta2, eps, wd, bc1, bc2, clip)
                    else:
                        ext.adam_step(p, p.grad.to(torch.float32), state["exp_avg"],
                                      state["exp_avg_sq"], lr, beta1, beta2, eps, wd,
                                      bc1, bc2)
                    _invalidate(p)
                    bump_tick(p)  # in-kernel update: no _version bump
                else:
                    gf = p.grad.float()
                    if clip is not None:
                        gf = gf * clip[1]
                    if wd != 0:
                        gf = gf.add(p, alpha=wd)
                    state["exp_avg"].mul_(beta1).add_(gf, alpha=1 - beta1)
                    state["exp_avg_sq"].mul_(beta2).addcmul_(gf, gf, value=1 - beta2)
                    denom = (state["exp_avg_sq"] / bc2).sqrt_().add_(eps)
                    p.addcdiv_(state["exp_avg"] / bc1, denom, value=-lr)
        return loss


OPTIMIZERS = {
    "SGD": FusedSGD,
    "Adam": FusedAdam,
}


def build_optimizer(name: str, params, **kwargs):
    """Explicit registry replacing the reference's eval-based dispatch
    (strategy.py:345-346)."""
    if name not in OPTIMIZERS:
        raise ValueError(f"Unknown optimizer {name!r}")
    return OPTIMIZERS[name](params, **kwargs)


SCHEDULERS = {
    "CosineAnnealingLR": torch.optim.lr_scheduler.CosineAnnealingLR,
    "StepLR": torch.optim.lr_scheduler.StepLR,
    "MultiStepLR": torch.optim.lr_scheduler.MultiStepLR,
}


def build_scheduler(name: str, optimizer, **kwargs):
    """Explicit registry replacing eval-based dispatch (strategy.py:348-350).
    LR schedules are host-side scalar math."""
    if name not in SCHEDULERS:
        raise ValueError(f"Unknown lr scheduler {name!r}")
    return SCHEDULERS[name](optimizer, **kwargs)
