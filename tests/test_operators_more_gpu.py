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


@pytest.mark.parametrize("p,n,k", [(1024, 300, 300), (5000, 1000, 100)])
@pytest.mark.parametrize("gout", [1e-12, 1e-30, 1e20])
def test_small_and_large_factors_of_badly_predicted_columns(p, n, k, gout):
    """Sizes that form the logits once.  Columns with losses of 60, H of 10^-3 and factors far from 1 among well predicted ones: rows of dW that
    hold little else must keep their bits.  (10^-30: dW's entries are of 10^-33, far above the smallest step of 2^-149.)"""
    W, H, y = problem(p, n, k, "f32", seed=k)
    z = W.double() @ H.double()
    scale = 60.0 / (z.max(0).values - z.min(0).values).mean()
    W, H = (W.double() * scale * 1e3).float(), (H.double() * 1e-3).float()
    z = W.double() @ H.double()
    y = z.argmax(0)
    bad = torch.tensor([2, 3, n // 2, n - 1], device=DEV)
    y[bad] = z.argmin(0)[bad]
    g = torch.ones(n, device=DEV) * min(1.0, gout * 1e3)
    g[bad] = gout
    check(W, H, y, "f32", reduction="none", gout=g)
