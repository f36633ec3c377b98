"""The norm of all gradients together, and clipping by it.

    norm = sqrt(sum over all tensors of g^2),   factor = min(1, max_norm / (norm + 1e-6))

Squares are summed in 64 bits in a fixed order: the norm is exact to its 32-bit
rounding, has the range of a float, and does not change from run to run. GPU
tensors run optim.hip; nothing here waits for the device. The optimizers of
ops/optim.py clip inside their step (``max_grad_norm``), without the pass over
the gradients that clip_grad_norm_ writes.
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


def _norm_factor(grads, max_norm, max_dev=None):
    """Two floats on the gradients' device: norm, factor."""
    if grads[0].is_cuda:
        return require_extension().grad_norm_factor(grads, max_norm, max_dev)
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    return torch.stack([norm, factor]).float()


def grad_norm(tensors):
    """The 2-norm of all ``tensors`` together, a 0-d float32 tensor on their
    device. None is skipped; a tensor that is listed twice counts once."""
    if isinstance(tensors, torch.Tensor):
        tensors = [tensors]
    grads = _distinct(tensors)
    if not grads:
        return torch.zeros(())
    return _norm_factor(grads, float("inf"))[0]


def clip_grad_norm_(parameters, max_norm):
    """Scales the parameters' gradients in place so that their norm is at most
    ``max_norm``, and returns the norm they had.

    A gradient with a NaN makes all of them NaN; an infinity makes its own tensor
    NaN where it stands and the others zero. Gradients that share memory are refused.
    """
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    seen = {id(p): p for p in parameters}
    grads = _distinct(p.grad for p in seen.values())
    if not grads:
        return torch.zeros(())
    both = _norm_factor(grads, max_norm)
    with torch.no_grad():
        if grads[0].is_cuda:
            require_extension().scale_by_factor(grads, both)
            torch.autograd.graph.increment_version(grads)
        else:
            for g in grads:
                g.mul_(both[1])
    return both[0]
