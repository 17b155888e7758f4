"""Softmax cross entropy, gradient norm and clipping on the GPU: what test_operators_gpu.py leaves out, with its problems and its bounds (u = half a
step of the type, v = 2^-24)."""
import math

import pytest
import torch

import nmfx
from test_operators_gpu import ALL, DEV, TYPES, V, check, near, oracle, problem, total

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


def outlier(W, H, y, column):
    """H and y with a loss in one column that no exponential holds."""
    H, y = H.clone(), y.clone()
    H[:, column] *= 300
    y[column] = (W.double() @ H[:, column].double()).argmin()
    return H, y


@pytest.mark.parametrize("p,n,k", [(5000, 1000, 100), (4097, 1100, 520)])
@pytest.mark.parametrize("eps", [0.0, 0.1])
def test_an_outlier_leaves_the_other_columns_as_they_were(p, n, k, eps):
    W, H, y = problem(p, n, k, "f32", seed=k, ignored=0.2)
    y[77] = 5
    kw = dict(reduction="none", label_smoothing=eps)
    clean = nmfx.softmax_xent_grad(W, H, y, **kw)
    H2, y2 = outlier(W, H, y, 77)
    assert float(oracle(W, H2, y2, eps, "none")["loss"][77]) > 100 * (1 - eps)
    got = nmfx.softmax_xent_grad(W, H2, y2, **kw)
    others = torch.arange(n, device=DEV) != 77
    for a, b in zip((got[0], got[1], got[3]), (clean[0], clean[1], clean[3])):
        assert torch.equal(a[..., others], b[..., others])
    check(W, H2, y2, "f32", eps=eps, reduction="none")


def test_an_outlier_does_not_hold_up_the_call():
    """One column whose logits are formed again, among 2048: a few more microseconds, not another kernel's length for every tile of classes."""
    W, H, y = problem(16384, 2048, 512, "f32")
    times = {}
    for name, (h, labels) in {"none": (H, y), "one": outlier(W, H, y, 700)}.items():
        nmfx.softmax_xent_grad(W, h, labels)
        best = math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            nmfx.softmax_xent_grad(W, h, labels)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        times[name] = best
    assert times["one"] < 2 * times["none"], times


@pytest.mark.parametrize("dtype,k", [(d, k) for d in ("bf16", "f16") for k in (264, 512, 1000, 2048)] + [("f32", k) for k in (132, 500, 1024)])
@pytest.mark.parametrize("n", [1, 7, 16])
@pytest.mark.parametrize("p", [1031, 70001])
def test_scoring_of_many_components(dtype, k, n, p):
    """Up to 16 columns against rows of W that a wave reads in several parts (up to all of H's 64 KB), in one and in several groups of rows."""
    W, H, y = problem(p, n, k, dtype, seed=k + n)
    if n > 1:
        y[n // 2] = -100
    for eps in (0.0, 0.1):
        want = oracle(W, H, y, eps, "none", dtype=dtype)
        loss, lse = nmfx.softmax_xent(W, H, y, label_smoothing=eps, reduction="none")
        near("loss", loss, want["loss"], want["eloss"])
        near("lse", lse, want["lse"], want["else_"])
    want = oracle(W, H, y, 0.1, "mean", dtype=dtype)
    near("mean", nmfx.softmax_xent(W, H, y, label_smoothing=0.1)[0], want["loss"], want["eloss"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("p,n,k", [(300, 40, 64), (1024, 300, 300), (5000, 1000, 100), (2000, 7, 64)])
@pytest.mark.parametrize("size", [1e6, 1e8, 1e9, 1e12])
def test_logits_so_large_that_their_rounding_is(dtype, p, n, k, size):
    """Float32 sums whose own rounding is beyond any exponential: exp(z - lse) still is between 0 and 1 (as the bounds take for granted), and
    everything finite."""
    W, H, y = problem(p, n, k, dtype, seed=3)
    W, H = (W.double() * math.sqrt(size)).to(W.dtype), (H.double() * math.sqrt(size)).to(H.dtype)
    for eps in (0.0, 0.1):
        check(W, H, y, dtype, eps=eps, reduction="none")


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("size", [300, 50001])
def test_clip_by_a_coefficient_that_is_no_normal_float32(dtype, size):
    """Gradients near the largest numbers of their type and norms to clip to that are small beside them: the coefficient is near and below 2^-126,
    the results are not."""
    big = {torch.float32: 3e38, torch.bfloat16: 3e38, torch.float16: 65504.0, torch.float64: 1e100}[dtype]
    for max_norm in (1e10, 1e6, 1e4, 100.0, 10.0, 1.0, 1e-3, 1e-20, 1e-30):
        for out in (False, True):
            ts = [torch.full((size,), big, device=DEV, dtype=torch.float64).to(dtype), torch.linspace(-big, big, 77, device=DEV, dtype=torch.float64).to(dtype)]
            ts[0][::3] = 0
            before, norm = [t.clone() for t in ts], total(ts)
            res = [torch.full_like(t, 7) for t in ts] if out else ts
            nmfx.clip_grad_norm(ts, max_norm, out=res if out else None)
            u = {torch.float32: V, torch.float64: 2.0 ** -50, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
            tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150, torch.float64: 0.0}[dtype]   # half the smallest step
            for b, t in zip(before, res):
                want = b.double() * min(1.0, max_norm / (norm + 1e-6))
                assert ((t.double() - want).abs() <= (u + (3 * V if dtype != torch.float64 else 0.0)) * want.abs() + tiny).all()


@pytest.mark.parametrize("n", [3, 100])
def test_a_backward_pass_through_softmax_xent_is_refused(n):
    """Its results have no graph: added to another loss, their part of the gradient must not be left out without a word."""
    W, H, y = problem(200, n, 40, "f32")
    want = nmfx.softmax_xent(W, H, y)
    hidden = H.t().detach().clone().requires_grad_()
    for a, b in ((W.clone().requires_grad_(), H), (W, hidden.t()), (torch.nn.Parameter(W), hidden.t())):
        leaf = a if a.requires_grad else hidden
        for part in (0, 1):
            got = nmfx.softmax_xent(a, b, y)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            with pytest.raises(nmfx.ArgumentError, match="softmax_xent_grad"):
                (got[part].sum() + leaf.sum()).backward()
            with pytest.raises(nmfx.ArgumentError, match="softmax_xent_grad"):
                torch.autograd.grad(got[part].sum(), leaf)
        with torch.no_grad():
            assert not nmfx.softmax_xent(a, b, y)[0].requires_grad
        leaf.grad = None
        loss, lse = (t.detach() for t in nmfx.softmax_xent(a, b, y))
        (loss + lse.sum() + leaf.sum()).backward()                    # a constant, and said to be one
        assert (leaf.grad == 1).all()
        for call in (lambda w, h: nmfx.softmax_xent_grad(w, h, y), lambda w, h: nmfx.softmax_xent_backward(w, h, y, lse)):
            for g, x in zip(call(a, b), call(W, H)):
                assert not g.requires_grad and torch.equal(g, x)
    with pytest.raises(nmfx.DimensionMismatch):
        nmfx.softmax_xent(torch.nn.Parameter(W), H[:, :2], y)


def test_what_is_written_in_place_shows_to_autograd():
    """A graph that has saved a tensor which is then written over must not go on with the new values."""
    W, H, y = problem(60, 20, 16, "f32")

    def saved(t):
        x = torch.ones_like(t).requires_grad_()
        return (x * t).sum()

    t, u = torch.randn(40, 30, device=DEV), torch.randn(300, device=DEV)
    out = [torch.empty_like(t), torch.empty_like(u)]
    dW, dH = torch.empty_like(W), torch.empty_like(H)
    with torch.inference_mode():
        apart = torch.randn(10, device=DEV)
    for targets, call in (([t, u], lambda: nmfx.clip_grad_norm([t, u, apart], 1.0)), (out, lambda: nmfx.clip_grad_norm([t, u], 1.0, out=out)),
                          ([t[:, :7]], lambda: nmfx.clip_grad_norm([t[:, :7]], 1.0)), ([dW, dH], lambda: nmfx.softmax_xent_grad(W, H, y, dW=dW, dH=dH)),
                          ([dH], lambda: nmfx.softmax_xent_backward(W, H, y, torch.zeros(20, device=DEV), dH=dH))):
        graphs = [saved(x) for x in targets]
        call()
        for g in graphs:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                g.backward()
    read = [saved(t), saved(u)]
    nmfx.grad_norm([t, u])                                            # reads only
    nmfx.clip_grad_norm([t, u], 1.0, out=out)
    for g in read:
        g.backward()
    graph = saved(t)
    with pytest.raises(nmfx.ArgumentError):
        nmfx.clip_grad_norm([t], -1.0)                                # refused: nothing is written
    graph.backward()
