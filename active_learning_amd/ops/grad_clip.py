"""The norm of all gradients together, and clipping by it.

    norm = sqrt(sum over all tensors of g^2),   factor = min(1, max_norm / (norm + 1e-6))

Gradients are bfloat16, float16 or float32; others are refused. Squares are summed
in 64 bits in a fixed order: the norm is exact to its 32-bit rounding, has the
range of a float, and does not change from run to run. GPU tensors run optim.hip;
nothing here waits for the device. The optimizers of ops/optim.py clip inside
their step (``max_grad_norm``), without the pass over the gradients that
clip_grad_norm_ writes.
"""

import torch

from .extension import require_extension

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _distinct(tensors):
    """The tensors without None and without repeats: a parameter that is listed
    twice has one gradient."""
    seen, kept = set(), []
    for t in tensors:
        if t is not None and id(t) not in seen:
            seen.add(id(t))
            kept.append(t.detach())
    for t in kept:
        if t.dtype not in _TYPES:
            raise TypeError(f"gradients must be bfloat16, float16 or float32, got {t.dtype}")
        if t.device != kept[0].device:
            raise ValueError(f"gradients are on {kept[0].device} and {t.device}")
    return kept


def _dense(t):
    """Whether the values fill their memory, in any order."""
    size = 1
    for stride, n in sorted((t.stride(i), t.shape[i]) for i in range(t.dim()) if t.shape[i] != 1):
        if stride != size:
            return False
        size *= n
    return True


def _scale(grads, factor):
    """Scales gradients on the CPU in place."""
    spans, copies = [], []
    for g in grads:
        if not g.numel():
            continue
        if any(n > 1 and s == 0 for n, s in zip(g.shape, g.stride())):
            raise RuntimeError("a gradient whose values share memory cannot be scaled in place")
        if _dense(g):
            spans.append((g.data_ptr(), g.data_ptr() + g.numel() * g.element_size()))
        else:  # may be part of another one
            copies.append((g, g * factor))
    spans.sort()
    if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
        raise RuntimeError("gradients that share memory cannot be scaled in place")
    apart = {id(g) for g, _ in copies}
    for g in grads:
        if id(g) not in apart:
            g.mul_(factor)
    for g, scaled in copies:
        g.copy_(scaled)


def _norm_factor(grads, max_norm):
    """Norm and factor of gradients on the CPU."""
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    factor = (torch.ones_like(norm) if max_norm == float("inf")
              else (max_norm / (norm + 1e-6)).clamp(max=1.0))
    return torch.stack([norm, factor]).float()


def _params_norm_factor(params, max_norm, max_dev=None, to=None):
    """Two floats on the device of the parameters' gradients (GPU: in ``to`` where it
    is given), or None where there are no gradients."""
    on_gpu = next((p.is_cuda for p in params if p.grad is not None), None)
    if on_gpu:
        return require_extension().params_norm_factor(params, max_norm, max_dev, to)
    if on_gpu is None:
        return None
    return _norm_factor(_distinct(p.grad for p in params), max_norm)


def grad_norm(tensors):
    """The 2-norm of all ``tensors`` together, a 0-d float32 tensor on their
    device. None is skipped; a tensor that is listed twice counts once."""
    if isinstance(tensors, torch.Tensor):
        tensors = [tensors]
    tensors = [t for t in tensors if t is not None]
    if not tensors:
        return torch.zeros((), dtype=torch.float32)
    if tensors[0].is_cuda:
        return require_extension().grad_norm_factor(tensors, float("inf"), None)[0]
    return _norm_factor(_distinct(tensors), float("inf"))[0]


def clip_grad_norm_(parameters, max_norm):
    """Scales the parameters' gradients in place so that their norm is at most
    ``max_norm``, and returns the norm they had.

    A NaN makes all gradients NaN; an infinity makes the factor zero, so that it
    becomes NaN itself and everything else zero; an infinite ``max_norm`` leaves
    everything as it is. Gradients that share memory, and a gradient whose own values
    do (an expanded one), are refused; one that is a sparse part of another's memory
    is scaled once.
    """
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    both = _params_norm_factor(parameters, max_norm)
    if both is None:
        return torch.zeros((), dtype=torch.float32)
    with torch.no_grad():
        if both.is_cuda:
            require_extension().scale_grads(parameters, both)
        else:
            _scale(_distinct(p.grad for p in parameters), both[1])
    return both[0]
