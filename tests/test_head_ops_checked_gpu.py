"""The norm, the e4m3 products and the clipped steps on the GPU: calls that used to be
answered wrongly or that no other test reaches. Tolerances count roundings as in
test_head_ops_gpu.py."""

import pytest
import torch

from active_learning_amd.ops.extension import require_extension

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def randn(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("clip", [False, True])
def test_momentum_without_buffers_is_none(clip):
    """Device hyperparameters that ask for momentum where a step has no buffers."""
    ext = require_extension()
    p, g = randn(1000, seed=1), randn(1000, seed=2)
    want = p.double() - 0.1 * (g.double() + 0.01 * p.double())
    hyper = torch.tensor([0.1, 0.9, 0.01], device="cuda")
    table = torch.tensor([[p.data_ptr(), g.data_ptr(), 0, 0, 0, 1000]], device="cuda")
    one = torch.ones(2, device="cuda")  # norm and factor
    done = [p]
    if clip:
        done.append(p.clone())
        ext.sgd_step_clip(done[1], g, p.new_empty(0), 0.1, 0.0, 0.01, hyper,
                          p.new_empty(0, dtype=torch.bfloat16), one)
        ext.sgd_step_multi_clip(table, 1, 0.1, 0.0, 0.01, hyper, one, False)
    else:
        ext.sgd_step_multi_dev(table, 1, hyper, False)
    for got in done:  # 0.1 and 0.01 as 32-bit numbers, two products, two sums
        assert ((got.double() - want).abs() <= 6 * U32 * (want.abs() + g.double().abs())).all()
