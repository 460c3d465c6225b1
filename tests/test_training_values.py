"""Values of a trainer's operators (p2pdl_amd/training.py) at the ends of their types' ranges, and what a
call may not depend on: where its operands lie, which host path made it.

Bounds as in test_training_ops.py, whose forms in 64 bits these tests share; `strict` compares infinities
and NaN too.
"""
import pytest
import torch

import test_training_ops as ops
from p2pdl_amd import training as T
from test_training_ops import DTYPES, U, gpu, randn, rounded, same_bits


def strict(got, want, bound, what):
    """|got - want| <= bound wherever want is finite, the same infinity or a NaN elsewhere."""
    got, want, bound = got.detach().double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (what, "NaN")
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]), (what, "infinities")
    fine = torch.isfinite(want)
    assert torch.isfinite(bound.expand_as(want)[fine]).all(), (what, "no bound")
    bad = fine & ~((got - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs()[bad].max()))


# ------------------------------------------------------------------ layer norm
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [1, 3, 8, 10, 24, 100])
def test_layer_norm_backward_of_large_constant_rows(cuda, dtype, cols):
    """A constant row of 2^120: rstd is 1 / sqrt(eps), so (0 - mean) * rstd leaves float32's range in the lanes past
    the row, which add nothing.  Its sums are exact, x - mean is 0: dx = rstd * (g - mean(g)) and dw = 0."""
    x = torch.full((5, cols), 2.0 ** 120, dtype=dtype, device="cuda")
    x[1::2] = 0.5
    dy, w = randn((5, cols), dtype, 70), randn((cols,), dtype, 71)
    y, mean, rstd = T.layer_norm_forward(x, w)
    assert torch.equal(mean, x[:, 0].float()) and not y.any()
    dx, dw, db = T.layer_norm_backward(dy, x, mean, rstd, w)
    g, r = dy.double().cpu() * w.double().cpu(), rstd.double().cpu()[:, None]
    want = r * (g - g.mean(1, keepdim=True))
    bound = r * 16 * U * (g.abs() + g.abs().mean(1, keepdim=True))
    strict(dx, want, rounded(want, bound, dtype), "dx")
    strict(dw, torch.zeros(cols), torch.zeros(cols), "dw")
    total = dy.double().cpu().sum(0)
    strict(db, total, rounded(total, 16 * U * dy.double().cpu().abs().sum(0), dtype), "db")
