"""Softmax cross entropy, gradient norm and clipping on the GPU: what test_operators_gpu.py leaves out, with its problems and its bounds (u = half a
step of the type, v = 2^-24)."""
import math

import pytest
import torch

import nmfx
from test_operators_gpu import DEV, HALF_STEP, TYPES, V, check, near, oracle, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p,n,k", [(300, 40, 64), (900, 300, 129), (5000, 1000, 100), (20000, 130, 300)])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("order", ["r", "c"])
def test_an_ignored_column_has_a_zero_gradient_whatever_the_factor(dtype, p, n, k, reduction, order):
    """A loss scale that has overflowed: infinite or NaN gradients, but not in the columns that are left out (dH of either order, summed from
    parts and directly)."""
    W, H, y = problem(p, n, k, dtype, seed=1)
    y[::3] = -100
    for gout in (math.inf, -math.inf, math.nan):
        dH = torch.full((k, n), 3.0, dtype=H.dtype, device=DEV) if order == "r" else torch.full((n, k), 3.0, dtype=H.dtype, device=DEV).t()
        dW = nmfx.softmax_xent_grad(W, H, y, reduction=reduction, gout=torch.tensor(gout, device=DEV), dH=dH)[2]
        assert (dH[:, ::3] == 0).all() and not dH[:, 1::3].isfinite().any() and not dW.isfinite().any()
    y[:] = -100
    _, _, dW, dH = nmfx.softmax_xent_grad(W, H, y, reduction=reduction, gout=torch.tensor(math.inf, device=DEV))
    assert (dW == 0).all() and (dH == 0).all()
