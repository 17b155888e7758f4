"""Softmax cross entropy of W*H with its gradients, the gradient norm and clipping, on the GPU against the formulas in Float64.

Tolerances are bounds on the rounding, element by element, computed from the inputs (u = half a step of the type, v = 2^-24):
  logits      e_z    = (k + 2) v (|W| |H|)                                  a Float32 sum of k products
  exp(z - m)  d      = 4 v max|z| + 4 v                                     the difference's rounding and exp2's two units
  lse         e_lse  = max e_z + d + (512 + p / 128) v + 2 v |lse|          the tree of sums, the logarithm
  dz          e_dz   = |g| (P (e_z + e_lse + d) + 4 v) + u |dz|             (Float16: + 2^-39 max|g|, its smallest step after the scaling)
  dW          e_dz |H'| + (n + 8) v |dz| |H'| + u |dW| + tiny               (tiny: half the smallest Float16 step, where gradients are Float16)
  dH          |W'| e_dz + (p + 8) v |W'| |dz| + u |dH| + tiny
"""
import math

import numpy as np
import pytest
import torch

import nmfx

pytestmark = pytest.mark.gpu
V = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
DEV = "cuda"


def lay(t, how):
    """The same matrix stored otherwise: 'r' rows contiguous, 'c' columns contiguous; '+' padded, with NaN between; 'o' off by one element."""
    r, c = t.shape
    a = t if how[0] == "r" else t.t()
    pad, off = (13 if "+" in how else 0), (1 if "o" in how else 0)
    buf = torch.full((a.shape[0] * (a.shape[1] + pad) + off,), float("nan"), dtype=t.dtype, device=t.device)
    v = buf[off:].view(a.shape[0], a.shape[1] + pad)[:, :a.shape[1]]
    v.copy_(a)
    return v if how[0] == "r" else v.t()


def problem(p, n, k, dtype, seed=0, ignored=0.0, spread=2.0, wl="r", hl="c"):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000 + seed)
    W = (torch.randn(p, k, generator=g, device=DEV) * (spread / math.sqrt(k))).to(TYPES[dtype])
    H = torch.randn(k, n, generator=g, device=DEV).to(TYPES[dtype])
    y = torch.randint(0, p, (n,), generator=g, device=DEV)
    if ignored:
        y[torch.rand(n, generator=g, device=DEV) < ignored] = -100
    return lay(W, wl), lay(H, hl), y


def oracle(W, H, y, eps=0.0, reduction="mean", gout=None, ignore=-100, dtype="f32"):
    """Values and bounds in Float64."""
    W, H = W.double(), H.double()
    p, k = W.shape
    n = H.shape[1]
    on = y != ignore
    H = torch.where(on[None, :], H, 0.0)
    z = W @ H
    ez = (k + 2) * V * (W.abs() @ H.abs())
    zmax = z.abs().max(0).values if n else z.new_zeros(0)
    lse = torch.logsumexp(z, 0)
    d = 4 * V * zmax + 4 * V
    elz = ez.max(0).values if n else ez.new_zeros(0)
    elog = elz + d + (512 + p / 128) * V + 2 * V * lse.abs()
    yy = torch.where(on, y, 0)
    T = torch.full_like(z, eps / p)
    T[yy, torch.arange(n, device=DEV)] += 1 - eps
    loss = torch.where(on, lse - (T * z).sum(0), 0.0)
    eloss = torch.where(on, elog + elz + (8 + p / 128) * V * (zmax + lse.abs()), 0.0)
    g = torch.ones(n, dtype=torch.float64, device=DEV) if gout is None else gout.double().expand(n).clone()
    cnt = max(1, int(on.sum()))
    if reduction == "mean":
        g /= cnt
    g = torch.where(on, g, 0.0)
    P = torch.exp(z - lse)
    dz = g * (P - T)
    u = HALF_STEP[dtype]
    edz = g.abs() * (P * (ez + elog + d) + 4 * V) + u * dz.abs()
    tiny = 0.0
    if dtype == "f16":
        edz = edz + (g.abs().max() * 2.0 ** -39 if n else 0.0)
        tiny = 2.0 ** -25
    dW, dH = dz @ H.t(), W.t() @ dz
    edW = edz @ H.t().abs() + (n + 8) * V * (dz.abs() @ H.t().abs()) + u * dW.abs() + tiny
    edH = W.t().abs() @ edz + (p + 8) * V * (W.t().abs() @ dz.abs()) + u * dH.abs() + tiny
    edH = torch.where(on[None, :], edH, 0.0)
    if reduction == "none":
        total, etotal = loss, eloss
    else:
        total, etotal = loss.sum(), eloss.sum() + V * loss.abs().sum()
        if reduction == "mean":
            total, etotal = total / cnt, etotal / cnt
    return dict(loss=total, lse=torch.where(on, lse, 0.0), dW=dW, dH=dH, eloss=etotal, else_=torch.where(on, elog, 0.0), edW=edW, edH=edH)


def near(name, got, want, bound):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), name
    over = off - bound
    assert (over <= 0).all(), f"{name}: off by {float(off.flatten()[over.argmax()]):.3e} where {float(bound.expand_as(off).flatten()[over.argmax()]):.3e} is allowed"


def check(W, H, y, dtype, eps=0.0, reduction="mean", gout=None, ignore=-100):
    kw = dict(ignore_index=ignore, label_smoothing=eps, reduction=reduction)
    want = oracle(W, H, y, eps, reduction, gout, ignore, dtype)
    loss, lse = nmfx.softmax_xent(W, H, y, **kw)
    near("loss", loss, want["loss"], want["eloss"])
    near("lse", lse, want["lse"], want["else_"])
    loss2, lse2, dW, dH = nmfx.softmax_xent_grad(W, H, y, gout=gout, **kw)
    near("loss (with gradients)", loss2, want["loss"], want["eloss"])
    near("lse (with gradients)", lse2, want["lse"], want["else_"])
    assert dW.dtype == W.dtype and dH.dtype == H.dtype and dW.shape == W.shape and dH.shape == H.shape
    near("dW", dW, want["dW"], want["edW"])
    near("dH", dH, want["dH"], want["edH"])
    bW, bH = nmfx.softmax_xent_backward(W, H, y, lse, gout=gout, **kw)
    near("dW (from lse)", bW, want["dW"], want["edW"])
    near("dH (from lse)", bH, want["dH"], want["edH"])
    return loss2, lse2, dW, dH


SIZES = [(1, 1, 1), (2, 3, 5), (5, 2, 1), (31, 1, 64), (64, 64, 64), (127, 33, 40), (129, 128, 8), (257, 130, 65), (300, 7, 129), (1000, 17, 200), (513, 1025, 24), (4099, 259, 72)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p,n,k", SIZES)
def test_xent_sizes(dtype, p, n, k):
    check(*problem(p, n, k, dtype, seed=p + n), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 9, 15, 16, 20, 31, 32, 48, 63, 65])
def test_xent_few_columns(dtype, n):
    check(*problem(777, n, 96, dtype, seed=n), dtype, reduction="none")
    check(*problem(1030, n, 1000, dtype, seed=n, wl="c"), dtype, reduction="none")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p,n,k", [(5000, 3000, 96), (2048, 8192, 64), (20000, 700, 520)])
def test_xent_many_tiles(dtype, p, n, k):
    check(*problem(p, n, k, dtype, seed=3), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("wl,hl", [("r", "r"), ("c", "c"), ("c", "r"), ("r+", "c+"), ("c+", "r+"), ("ro", "co"), ("co", "ro"), ("r+o", "c"), ("c+o", "r+o")])
def test_xent_layouts(dtype, n, wl, hl):
    for p, k in ((264, 72), (263, 71)):
        W, H, y = problem(p, n, k, dtype, seed=5, ignored=0.2, wl=wl, hl=hl)
        _, _, dW, dH = check(W, H, y, dtype, eps=0.05)
        if p > 1 and k > 1:
            assert (dW.stride(0) == 1) == (wl[0] == "c")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("eps", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("ignored", [0.0, 0.5, 1.0])
def test_xent_reductions_smoothing_and_ignored(dtype, reduction, eps, ignored):
    W, H, y = problem(333, 150, 48, dtype, seed=11, ignored=ignored)
    gout = (torch.randn(150, device=DEV) if reduction == "none" else torch.tensor(-3.5, device=DEV))
    loss, lse, dW, dH = check(W, H, y, dtype, eps, reduction, gout)
    if ignored == 1.0:
        for t in (loss, lse, dW, dH):
            assert (t == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 6, 200])
def test_xent_nothing_of_an_ignored_column_is_read(dtype, n):
    W, H, y = problem(300, 2 * n, 64, dtype, seed=1)
    y[::2] = 7777
    clean = nmfx.softmax_xent_grad(W, H, y, ignore_index=7777)
    H[:, 0::4] = float("nan")
    H[:, 2::4] = float("inf")
    for a, b in zip(clean, nmfx.softmax_xent_grad(W, H, y, ignore_index=7777)):
        assert torch.equal(a, b)
    near("loss", nmfx.softmax_xent(W, H, y, ignore_index=7777)[0], clean[0].double(), torch.tensor(1e-6, device=DEV))


@pytest.mark.parametrize("n", [1, 5, 100])
def test_xent_a_label_that_is_no_class_shows(n):
    W, H, y = problem(50, n, 32, "f32")
    for bad in (50, -1, 2 ** 40):
        y2 = y.clone()
        y2[n // 2] = bad
        loss, lse = nmfx.softmax_xent(W, H, y2, reduction="none")
        want = torch.zeros(n, dtype=torch.bool, device=DEV)
        want[n // 2] = True
        assert torch.equal(loss.isnan(), want) and torch.equal(lse.isnan(), want)
        l2, _, dW, dH = nmfx.softmax_xent_grad(W, H, y2)
        assert l2.isnan() and dW.isnan().all() and torch.equal(dH.isnan().all(0), want) and torch.equal(dH.isnan().any(0), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3, 70])
def test_xent_nan_and_infinite_inputs_stay_in_their_column(dtype, n):
    W, H, y = problem(200, n, 40, dtype, seed=2)
    H[3, 1] = float("nan")
    loss, lse = nmfx.softmax_xent(W, H, y, reduction="none")
    bad = torch.zeros(n, dtype=torch.bool, device=DEV)
    bad[1] = True
    assert torch.equal(loss.isnan(), bad) and torch.equal(lse.isnan(), bad)
    dH = nmfx.softmax_xent_grad(W, H, y, reduction="none")[3]
    assert torch.equal(dH.isnan().any(0), bad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 80])
def test_xent_large_logits(dtype, n):
    """Logits of +-10^4 and a class whose logits are minus infinity: exp must neither overflow nor meet inf - inf."""
    p, k = 400, 32
    W, H, y = problem(p, n, k, dtype, seed=4)
    W.zero_()
    H[0] = 100.0
    W[:, 0] = torch.linspace(-100, 100, p, device=DEV).to(W.dtype)
    check(W, H, y, dtype, reduction="none")
    W[:, 0] = -100.0                    # all logits of a tile equal and far below 0
    check(W, H, y, dtype, reduction="none")
    W, H, y = problem(p, n, k, dtype, seed=4)
    H[0] = 1.0
    clean, _ = nmfx.softmax_xent(W, H, torch.full_like(y, 399), reduction="none")
    W[:390, 0] = -float("inf")          # whole tiles of it
    loss, lse = nmfx.softmax_xent(W, H, torch.full_like(y, 399), reduction="none")
    want = oracle(W[390:], H, torch.full_like(y, 9), reduction="none", dtype=dtype)
    near("loss", loss, want["loss"], want["eloss"])


def test_xent_no_columns():
    W, H, y = problem(20, 0, 8, "bf16")
    loss, lse, dW, dH = nmfx.softmax_xent_grad(W, H, y)
    assert loss == 0 and lse.shape == (0,) and (dW == 0).all() and dH.shape == (8, 0)
    assert nmfx.softmax_xent(W, H, y, reduction="none")[0].shape == (0,)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_xent_several_pieces_of_the_classes(dtype):
    """600,001 classes: dz of all of them at 700 columns has over 2^28 entries, so the gradients go in pieces."""
    check(*problem(600001, 700, 9, dtype, seed=6, ignored=0.1), dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_xent_gradient_is_the_loss_s_slope(dtype):
    """Differences of the loss in Float64 along a random direction against <gradient, direction>."""
    p, n, k = 150, 60, 24
    W, H, y = problem(p, n, k, dtype, seed=8, ignored=0.3)
    _, _, dW, dH = nmfx.softmax_xent_grad(W, H, y, label_smoothing=0.1)
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    A, B = torch.randn(p, k, generator=g, device=DEV, dtype=torch.float64), torch.randn(k, n, generator=g, device=DEV, dtype=torch.float64)
    t = 1e-4
    up, down = (oracle(W.double() + s * A, H.double() + s * B, y, 0.1)["loss"] for s in (t, -t))
    slope = float((up - down) / (2 * t))
    bound = oracle(W, H, y, 0.1, dtype=dtype)
    tol = float((bound["edW"] * A.abs()).sum() + (bound["edH"] * B.abs()).sum()) + 1e-5     # 1e-5: the difference's own error, of order t^2
    assert abs(float((dW.double() * A).sum() + (dH.double() * B).sum()) - slope) <= tol


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_xent_float16_range(dtype):
    """Factors g_j / n far below Float16's smallest step, and one 2^20 times the others."""
    W, H, y = problem(500, 300, 64, dtype, seed=9)
    gout = torch.full((300,), 2.0 ** 20, device=DEV)
    check(W, H, y, dtype, reduction="none", gout=gout / 2.0 ** 18)
    gout = torch.rand(300, device=DEV) + 0.5
    gout[7] = 4096.0
    check(W, H, y, dtype, reduction="none", gout=gout)


@pytest.mark.parametrize("n", [1, 2048, 2049, 5000, 9000])
def test_xent_factors_of_many_columns(n):
    """A factor of its own for every column, the largest (which sets Float16's scale) in the last: found over one round and over several."""
    for dtype in TYPES:
        W, H, y = problem(130, n, 16, dtype, seed=n, ignored=0.3)
        y[-1] = 5
        gout = torch.rand(n, device=DEV) - 0.5
        gout[-1] = -512.0
        check(W, H, y, dtype, reduction="none", gout=gout)


# sizes that form the logits once
ONCE = [("f32", 400001, 600, 9), ("f32", 1024, 300, 300), ("f32", 5000, 1000, 100), ("f32", 1537, 2500, 129), ("f32", 4097, 1100, 520)]


@pytest.mark.parametrize("dtype,p,n,k", ONCE)
@pytest.mark.parametrize("wl,ignored,reduction", [("r", 0.0, "mean"), ("c", 0.4, "none"), ("r+o", 0.95, "sum"), ("r", 1.0, "mean")])
def test_xent_logits_formed_once(dtype, p, n, k, wl, ignored, reduction):
    W, H, y = problem(p, n, k, dtype, seed=p + n, ignored=ignored, wl=wl)
    gout = torch.linspace(-2, 2, n, device=DEV) if reduction == "none" else None
    check(W, H, y, dtype, reduction=reduction, gout=gout)


@pytest.mark.parametrize("p,n,k", [(1024, 300, 300), (5001, 1000, 256), (4097, 1100, 520), (160001, 2000, 257)])
@pytest.mark.parametrize("eps,ignored", [(0.1, 0.0), (0.7, 0.3), (1.0, 0.95), (0.1, 1.0)])
def test_xent_logits_formed_once_with_smoothing(p, n, k, eps, ignored):
    W, H, y = problem(p, n, k, "f32", seed=p + n, ignored=ignored, wl="r" if p % 2 else "c")
    check(W, H, y, "f32", eps=eps, reduction="none", gout=torch.linspace(-2, 2, n, device=DEV))


@pytest.mark.parametrize("dtype,p,n,k", [ONCE[0], ONCE[2], ONCE[4]])
def test_xent_losses_beyond_any_exponential(dtype, p, n, k):
    """Columns whose losses are near and far beyond where exp() of them leaves Float32 (88.7), among ordinary ones, in some column tiles."""
    W, H, y = problem(p, n, k, dtype, seed=k)
    cols = torch.tensor([3, 4, 5, 6, n // 2, n - 1], device=DEV)
    z = W.double() @ H[:, cols].double()
    y[cols] = z.argmin(0)
    spread = z.max(0).values - z.min(0).values
    H = H.clone()
    H[:, cols] = (H[:, cols].double() * (torch.tensor([50.0, 68.0, 75.0, 87.0, 200.0, 1000.0], device=DEV, dtype=torch.float64) / spread)).to(H.dtype)
    check(W, H, y, dtype, reduction="none", gout=torch.linspace(-1, 1, n, device=DEV))
    check(W, H, y, dtype, eps=0.2, reduction="none", gout=torch.linspace(-1, 1, n, device=DEV))


@pytest.mark.parametrize("dtype,p,n,k", ONCE[2:4])
def test_xent_formed_once_keeps_nan_and_no_classes_to_their_columns(dtype, p, n, k):
    W, H, y = problem(p, n, k, dtype, seed=1, ignored=0.3)
    good = nmfx.softmax_xent_grad(W, H, y, reduction="none")
    on = torch.nonzero(y != -100).flatten()
    H2, y2 = H.clone(), y.clone()
    H2[1, on[0]] = float("nan")
    H2[0, on[7]] = float("inf")
    y2[on[9]] = p
    y2[on[11]] = -1
    loss, lse, dW, dH = nmfx.softmax_xent_grad(W, H2, y2, reduction="none")
    bad = torch.zeros(n, dtype=torch.bool, device=DEV)
    bad[on[[0, 7, 9, 11]]] = True
    assert loss[bad].isnan().all() and lse[bad][[0, 2, 3]].isnan().all() and dH[:, bad].isnan().all(0).all() and dW.isnan().all()
    for name, a, b, t in (("loss", loss, good[0], 2.0 ** -20), ("lse", lse, good[1], 2.0 ** -20), ("dH", dH, good[3], 4 * HALF_STEP[dtype])):
        a, b = a[..., ~bad].double(), b[..., ~bad].double()
        assert ((a - b).abs() <= t * b.abs().max()).all(), name


def test_xent_formed_once_in_a_graph():
    W, H, y = problem(4000, 900, 120, "f32", ignored=0.2)
    kw = dict(reduction="sum", dW=torch.empty_like(W), dH=torch.empty_like(H.t()).t())
    nmfx.softmax_xent_grad(W, H, y, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, lse, dW, dH = nmfx.softmax_xent_grad(W, H, y, **kw)
    for r in range(4):
        H.copy_(torch.randn_like(H))
        if r == 2:
            H[:, 5] *= 300
            y[5] = (W @ H[:, 5]).argmin()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (loss, lse, dW, dH)]
        for a, b in zip(got, nmfx.softmax_xent_grad(W, H, y, reduction="sum")):
            assert torch.equal(a, b), r


def test_xent_same_bits_twice_and_given_outputs():
    W, H, y = problem(3000, 500, 136, "bf16", ignored=0.2)
    a = nmfx.softmax_xent_grad(W, H, y)
    dW, dH = torch.full((3000, 150), 7.0, dtype=W.dtype, device=DEV), torch.full((136, 501), 7.0, dtype=W.dtype, device=DEV)
    b = nmfx.softmax_xent_grad(W, H, y, dW=dW[:, 3:139], dH=dH[:, 1:])
    for x, z in zip(a, b):
        assert torch.equal(x, z)
    assert (dW[:, :3] == 7).all() and (dW[:, 139:] == 7).all() and (dH[:, 0] == 7).all()


@pytest.mark.parametrize("p,n,k,wl", [(1000, 1, 64, "r"), (1000, 12, 64, "c"), (3000, 300, 72, "r")])
def test_xent_and_clip_in_a_graph(p, n, k, wl):
    """A captured training step, replayed with other inputs between eager work, against the eager call each time."""
    W, H, y = problem(p, n, k, "bf16", seed=1, ignored=0.2, wl=wl)
    y[0] = 3
    s = torch.cuda.Stream()

    def step():
        loss, lse, dW, dH = nmfx.softmax_xent_grad(W, H, y)
        norm = nmfx.clip_grad_norm([dW, dH], 0.01)
        return loss, lse, dW, dH, norm, nmfx.softmax_xent(W, H, y, reduction="none")[0]

    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        W2, H2, y2 = problem(p, n, k, "bf16", seed=10 + seed, ignored=0.3 * seed)
        W.copy_(W2), H.copy_(H2), y.copy_(y2)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    args = [problem(2000, 300, 128, "bf16", seed=i) for i in range(2)]
    want = [nmfx.softmax_xent_grad(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(nmfx.softmax_xent_grad(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for a, b in zip(g, want[i]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_xent_many_components(dtype):
    for n in (1, 5, 40):
        check(*problem(300, n, 9000, dtype, seed=n), dtype)


def _guarded(nbytes, guard=4096):
    """nbytes of 0xff (NaN in every type) between guards, 256-byte aligned; and the check that the guards are as they were."""
    room = (nbytes + 255) // 256 * 256
    buf = torch.full((room + 2 * guard,), 0xff, dtype=torch.uint8, device=DEV)
    buf[:guard] = buf[guard + room:] = 0x5a

    def untouched():
        assert (buf[:guard] == 0x5a).all() and (buf[guard + room:] == 0x5a).all() and (buf[guard + nbytes:guard + room] == 0xff).all()

    return buf[guard:guard + nbytes], untouched


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p,n,k,wl,ignored", [(1, 1, 1, "r", 0.0), (70, 3, 8, "r", 0.0), (70, 3, 9, "c", 0.5), (777, 65, 40, "c", 0.3), (5000, 300, 64, "r", 0.9), (257, 2100, 33, "r", 0.5), (300, 5000, 24, "r", 0.4),
                                              (20000, 4200, 40, "r", 0.2)])
def test_xent_stays_in_its_buffers_and_takes_nothing_from_them(dtype, p, n, k, wl, ignored):
    """Workspace and outputs full of NaN beforehand and between guards: same bits as with torch's memory, guards untouched."""
    L = nmfx._lib
    lib = L.load()
    W, H, y = problem(p, n, k, dtype, seed=p, ignored=ignored, wl=wl)
    code = {"f32": L.F32, "bf16": L.BF16, "f16": L.F16}[dtype]
    es = W.element_size()

    def mat(t, rows, cols, rs, cs):
        return L.DMat(t.data_ptr(), rows, cols, rs, cs, code, 0)

    w, h = mat(W, p, k, *W.stride()), mat(H, k, n, *H.stride())
    import ctypes as C
    for eps in (0.0, 0.1):
        o, size = L.XentOpts(eps, -100, L.REDUCE_MEAN, 0), C.c_int64()
        for grad in (0, 1):
            assert lib.nmfx_xent_workspace(w, h, o, grad, size) == L.OK
            bufs = [_guarded(b) for b in (size.value, 4, 4 * n, p * k * es, k * n * es)]
            ws, loss, lse, dW, dH = (b[0] for b in bufs)
            stream = torch.cuda.current_stream().cuda_stream
            if grad:
                st = lib.nmfx_xent_grad(w, h, y.data_ptr(), o, None, 0, loss.data_ptr(), lse.data_ptr(), mat(dW, p, k, k, 1), mat(dH, k, n, 1, k), ws.data_ptr(), size.value, 0, stream)
                got = (loss.view(torch.float32)[0], lse.view(torch.float32), dW.view(W.dtype).view(p, k), dH.view(W.dtype).view(n, k).t())
                want = nmfx.softmax_xent_grad(W, H, y, label_smoothing=eps, dW=torch.empty(p, k, dtype=W.dtype, device=DEV))
            else:
                st = lib.nmfx_xent(w, h, y.data_ptr(), o, loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), size.value, 0, stream)
                got, want = (loss.view(torch.float32)[0], lse.view(torch.float32)), nmfx.softmax_xent(W, H, y, label_smoothing=eps)
            assert st == L.OK, lib.nmfx_last_op_error()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
            for _, untouched in bufs:
                untouched()


def test_norm_stays_in_its_buffers():
    L = nmfx._lib
    lib = L.load()
    import ctypes as C
    sizes = [1, 7, 8191, 40000, 3] * 40
    flat, flat_ok = _guarded(4 * sum(sizes))
    flat.view(torch.float32).copy_(torch.randn(sum(sizes), device=DEV))
    views = flat.view(torch.float32).split(sizes)
    want = [v.clone() for v in views]
    norm = nmfx.clip_grad_norm(want, 0.5)
    for count in (5, 200):
        data = [v.clone() for v in views[:count]]
        out, out_ok = _guarded(4 * sum(sizes[:count]))
        outs = out.view(torch.float32).split(sizes[:count])
        a = (L.DMat * count)(*[L.DMat(t.data_ptr(), 1, t.numel(), t.numel(), 1, L.F32, 0) for t in data])
        b = (L.DMat * count)(*[L.DMat(t.data_ptr(), 1, t.numel(), t.numel(), 1, L.F32, 0) for t in outs])
        size = C.c_int64()
        assert lib.nmfx_grad_norm_workspace(count, size) == L.OK
        ws, ws_ok = _guarded(size.value)
        got, got_ok = _guarded(4)
        assert lib.nmfx_clip_grad_norm(count, C.addressof(a), C.addressof(b), 0.5, L.NORM_2, got.data_ptr(), ws.data_ptr(), size.value, 0, torch.cuda.current_stream().cuda_stream) == L.OK
        if count == 200:
            assert torch.equal(got.view(torch.float32)[0], norm) and all(torch.equal(x, y) for x, y in zip(outs, want))
        assert not out.view(torch.float32).isnan().any()
        out_ok(), ws_ok(), got_ok(), flat_ok()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p,n,k", [(70, 3, 9), (300, 40, 64), (900, 300, 129), (5000, 1000, 100)])
@pytest.mark.parametrize("gw,gh", [("c", "r"), ("r+o", "c+"), ("c+", "r+o")])
def test_xent_outputs_in_any_order(dtype, p, n, k, gw, gh):
    """Outputs of another contiguous index than their inputs, padded, off by an element: the values of dense ones, nothing beside them."""
    W, H, y = problem(p, n, k, dtype, seed=p, ignored=0.2)
    want = nmfx.softmax_xent_grad(W, H, y)
    dW, dH = lay(torch.zeros_like(W), gw), lay(torch.zeros_like(H), gh)

    def around(t):
        buf = torch.as_strided(t, (t.untyped_storage().nbytes() // t.element_size(),), (1,), 0)
        return int(buf.isnan().sum())

    pads = around(dW), around(dH)
    loss, lse, a, b = nmfx.softmax_xent_grad(W, H, y, dW=dW, dH=dH)
    assert a is dW and b is dH and (around(dW), around(dH)) == pads
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    for name, got, dense in (("dW", dW, want[2]), ("dH", dH, want[3])):      # (the order decides the tiles: sums may differ in their last bits)
        u = (4 * HALF_STEP[dtype] + n * V + p * V) * dense.abs().max().double()
        assert ((got.double() - dense.double()).abs() <= u).all(), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 60])
def test_xent_ignored_label_that_is_a_class(dtype, n):
    W, H, y = problem(40, n, 24, dtype, seed=n)
    y[::3] = 7
    check(W, H, y, dtype, ignore=7)


@pytest.mark.parametrize("p,n,k", [(2 ** 21 - 1024, 3, 4), (2 ** 21 - 1024, 20, 4), (5, 2 ** 21 - 1024, 4), (2, 3, 2 ** 20 - 512)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_xent_largest_extents(dtype, p, n, k):
    W, H, y = problem(p, n, k, dtype, seed=1, ignored=0.1 if n > 3 else 0.0)
    check(W, H, y, dtype)


@pytest.mark.parametrize("wl", ["r", "c"])
@pytest.mark.parametrize("n", [4, 30])
def test_xent_wide_strides_of_w(wl, n):
    W, H, y = problem(300, n, 40, "bf16", seed=n)
    ld = 2 ** 21 - 1024
    buf = torch.full(((300 if wl == "r" else 40) * ld,), float("nan"), dtype=W.dtype, device=DEV).view(-1, ld)
    v = buf[:, :40] if wl == "r" else buf[:, :300].t()
    v.copy_(W)
    check(v, H, y, "bf16")


def test_an_error_left_behind_is_not_reported():
    set_device = nmfx._lib.load().hipSetDevice                   # of the runtime that the library is linked to
    W, H, y = problem(50, 4, 8, "f32")
    for call in (lambda: nmfx.softmax_xent(W, H, y), lambda: nmfx.softmax_xent_grad(W, H, y), lambda: nmfx.grad_norm([W, H])):
        call()
        assert set_device(99) != 0
        call()
    torch.cuda.synchronize()


# ---- norm and clipping ---------------------------------------------------------------------------------------------------------------
def tensors(shapes, dtypes, seed=0, scale=0.1):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    ts = [(torch.randn(s, generator=g, device=DEV, dtype=torch.float64) * scale).to(d) for s, d in zip(shapes, dtypes)]
    return ts


def total(ts, kind=2):
    if kind == 2:
        return math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in ts))
    return max((float(t.double().abs().max()) for t in ts if t.numel()), default=0.0)


ALL = [torch.float32, torch.float64, torch.bfloat16, torch.float16]


def clip_check(ts, max_norm, kind=2, out=None):
    norm, before = total(ts, kind), [t.clone() for t in ts]
    got = nmfx.grad_norm(ts, kind)
    # the sum of squares in Float64 is off by 2^-53 per addition of a tree: far below the Float32 it is rounded to
    assert got.dtype == torch.float32 and got.dim() == 0 and abs(float(got) - norm) <= 2 * V * norm
    back = nmfx.clip_grad_norm(ts, max_norm, kind, out=out)
    assert torch.equal(back, got)
    coef = min(1.0, max_norm / (norm + 1e-6))
    for b, t in zip(before, ts if out is None else out):
        u = {torch.float32: V, torch.float64: 2.0 ** -50, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[t.dtype]
        # the coefficient in Float32, the product, and the rounding to the type (Float16: subnormals too)
        slack = 3 * V if t.dtype != torch.float64 else 0.0
        want = b.double() * coef
        tiny = 2.0 ** -25 if t.dtype == torch.float16 else 0.0
        assert ((t.double() - want).abs() <= (u + slack) * want.abs() + tiny).all()
    if out is not None:
        for b, t in zip(before, ts):
            assert torch.equal(b, t)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shapes", [[(1,)], [(7,), (3, 5)], [(8191,), (8192,), (8193,)], [(300, 301), (1,), (65536,)], [(2000, 3000), (17, 9, 5)]])
@pytest.mark.parametrize("kind", [2, float("inf")])
def test_norm_and_clip(dtype, shapes, kind):
    for max_norm in (0.05, 1e6, 0.0):
        clip_check(tensors(shapes, [dtype] * len(shapes)), max_norm, kind)
        ts = tensors(shapes, [dtype] * len(shapes), seed=1)
        clip_check(ts, max_norm, kind, out=[torch.full_like(t, 3.0) for t in ts])


def test_norm_many_mixed_tensors():
    rng = np.random.default_rng(0)
    shapes = [(int(rng.integers(1, 40000)),) for _ in range(331)] + [(0,), (5, 0), ()]
    clip_check(tensors(shapes, [ALL[i % 4] for i in range(len(shapes))]), 1.0)


def test_clip_into_a_flat_buffer_at_odd_offsets():
    shapes = [(333, 5), (7,), (40001,), (1, 1), (99, 1000)]
    for d in ALL:
        ts = tensors(shapes, [d] * 5)
        sizes = [t.numel() for t in ts]
        flat = torch.zeros(sum(sizes) + 3, dtype=d, device=DEV)
        clip_check(ts, 0.5, out=[v.view(s) for v, s in zip(flat[1:-2].split(sizes), shapes)])
        assert flat[0] == 0 and (flat[-2:] == 0).all()


@pytest.mark.parametrize("dtype", ALL)
def test_clip_strided(dtype):
    big = tensors([(300, 500)], [dtype])[0]
    keep = big.clone()
    a, b = big[:, :200], big[:, 207:499]                # interleaved rows of one buffer, disjoint
    c = tensors([(64, 33)], [dtype], seed=2)[0].t()     # transposed
    d = tensors([(500,)], [dtype], seed=3)[0][::3]
    clip_check([a, b, c, d], 0.5)
    assert torch.equal(big[:, 200:207], keep[:, 200:207]) and torch.equal(big[:, 499:], keep[:, 499:])
    ts = tensors([(300, 200), (77,)], [dtype] * 2)
    clip_check(ts, 0.5, out=[big[:, 11:211], tensors([(154,)], [dtype])[0][::2]])   # dense into strided
    clip_check([big[:, 5:105]], 0.5, out=[torch.empty(300, 100, dtype=dtype, device=DEV)])


def test_norm_range():
    """Squares beyond Float32's range, on both sides."""
    for value in (1e30, 1e-30):
        t = torch.full((5000,), value, device=DEV)
        assert abs(float(nmfx.grad_norm([t])) / (value * math.sqrt(5000)) - 1) < 1e-6
    for value in (1e30, 1e-30, 1e-18, 2e19, 3e38):        # bf16, in whole groups and beside others
        t = torch.full((50001,), value, device=DEV).bfloat16()
        norm = float(t[0].double()) * math.sqrt(50001)
        got = float(nmfx.grad_norm([t]))
        assert abs(got / norm - 1) < 1e-6 if norm < 3e38 else math.isinf(got)
        t[::7] = 0
        assert abs(float(nmfx.grad_norm([t])) / (float(t[1].double()) * math.sqrt(50001 - 7143)) - 1) < 1e-6 or norm > 1e38
    for value in (65504.0, 2.0 ** -24):
        t = torch.full((50001,), value, device=DEV).half()
        assert abs(float(nmfx.grad_norm([t])) / (value * math.sqrt(50001)) - 1) < 1e-6
    t = torch.full((3,), 3e38, device=DEV)
    nmfx.clip_grad_norm([t], 1.0)
    assert abs(float(t[0]) * math.sqrt(3) - 1) < 1e-6          # the norm is beyond Float32, the coefficient is not
    z = torch.zeros(40000, device=DEV)
    assert float(nmfx.clip_grad_norm([z], 1.0)) == 0 and (z == 0).all()


@pytest.mark.parametrize("size", [100, 300000])
def test_clip_not_finite(size):
    a, b = tensors([(size,), (50,)], [torch.float32] * 2)
    a[size // 2] = float("nan")
    for kind in (2, float("inf")):
        x, y = a.clone(), b.clone()
        assert nmfx.clip_grad_norm([x, y], 1.0, kind).isnan() and x.isnan().all() and y.isnan().all()
    a[size // 2] = float("inf")
    assert nmfx.clip_grad_norm([a, b], 1.0).isinf() and (b == 0).all() and a[size // 2].isnan() and a.isnan().sum() == 1


def test_norm_of_one_large_tensor_and_of_thousands():
    big = torch.full((2 ** 31 + 2 ** 20 + 3,), 0.5, dtype=torch.bfloat16, device=DEV)
    big[-1] = 3.0
    want = math.sqrt((big.numel() - 1) * 0.25 + 9.0)
    assert abs(float(nmfx.grad_norm(big)) - want) <= 2 * V * want
    assert float(nmfx.grad_norm(big, norm_type=float("inf"))) == 3.0
    norm = nmfx.clip_grad_norm([big], want / 2)
    assert abs(float(norm) - want) <= 2 * V * want and float(big[-1]) == 1.5 and float(big[0]) == 0.25 and float(big[2 ** 31 + 7]) == 0.25
    del big
    many = [torch.full((i % 7 + 1,), 1.0, device=DEV) for i in range(3000)] + [torch.ones(5, 8, device=DEV)[:, :3] for _ in range(50)]
    count = sum(t.numel() for t in many)
    assert abs(float(nmfx.clip_grad_norm(many, 1.0)) - math.sqrt(count)) <= 2 * V * math.sqrt(count)
    assert all(((t * math.sqrt(count) - 1).abs() <= 8 * V + 2e-6).all() for t in many[::97] + many[-3:])


def test_clip_on_another_stream():
    t = tensors([(1 << 20,)], [torch.float32])[0]
    want = t.clone()
    nmfx.clip_grad_norm([want], 0.5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        t.mul_(1.0)
        nmfx.clip_grad_norm(t, 0.5)
    s.synchronize()
    assert torch.equal(t, want)


# ---- together ------------------------------------------------------------------------------------------------------------------------
def test_training_steps_follow_float64():
    """Ten clipped gradient steps on W and H, against the same steps in Float64: a step's error is the gradients' (Float32, about 1e-5 of
    their size, see the bounds above) and steps of a convex-ish loss do not amplify it."""
    p, n, k = 600, 400, 32
    W, H, y = problem(p, n, k, "f32", seed=21, ignored=0.25)
    Wd, Hd = W.double(), H.double()
    for _ in range(10):
        loss, _, dW, dH = nmfx.softmax_xent_grad(W, H, y, label_smoothing=0.1)
        norm = nmfx.clip_grad_norm([dW, dH], 0.02)
        want = oracle(Wd, Hd, y, 0.1)
        gn = math.sqrt(float((want["dW"] ** 2).sum() + (want["dH"] ** 2).sum()))
        assert abs(float(norm) - gn) <= 1e-4 * gn and abs(float(loss - want["loss"])) <= 1e-4 * float(want["loss"])
        c = min(1.0, 0.02 / (gn + 1e-6))
        W -= 5.0 * dW
        H -= 5.0 * dH
        Wd = Wd - 5.0 * c * want["dW"]
        Hd = Hd - 5.0 * c * want["dH"]
    assert float((W.double() - Wd).norm() / Wd.norm()) < 1e-4 and float((H.double() - Hd).norm() / Hd.norm()) < 1e-4


def test_xent_refuses_on_the_gpu():
    W, H, y = problem(30, 10, 16, "f32")
    with pytest.raises(nmfx.ArgumentError):
        nmfx.softmax_xent(W.double(), H, y)
    with pytest.raises(nmfx.NMFXError):
        nmfx.softmax_xent(W.double(), H.double(), y)
    with pytest.raises(nmfx.DimensionMismatch):
        nmfx.softmax_xent(W, H[:15], y)
    with pytest.raises(nmfx.DimensionMismatch):
        nmfx.softmax_xent(W, H, y[:9])
    with pytest.raises(nmfx.ArgumentError):
        nmfx.softmax_xent(W, H, y.int())
    with pytest.raises(nmfx.ArgumentError):
        nmfx.softmax_xent(W, H, y, label_smoothing=1.5)
    with pytest.raises(nmfx.ArgumentError):
        nmfx.softmax_xent(W, H, y, reduction="median")
    with pytest.raises(nmfx.ArgumentError):
        nmfx.softmax_xent(W[::2, ::2], H[::2], y)
    with pytest.raises(nmfx.ArgumentError):
        nmfx.softmax_xent(W.cpu(), H, y)
    with pytest.raises(nmfx.DimensionMismatch):
        nmfx.softmax_xent_grad(W, H, y, dW=torch.empty(30, 15, device=DEV))
    with pytest.raises(nmfx.ArgumentError):
        nmfx.softmax_xent_grad(W, H, y, dH=torch.empty(16, 10, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(nmfx.ArgumentError):
        nmfx.softmax_xent_grad(W, H, y, dH=torch.empty(16, 1, device=DEV).expand(16, 10))
    with pytest.raises(nmfx.ArgumentError):
        nmfx.softmax_xent_backward(W, H, y, None)


def test_clip_refuses_on_the_gpu():
    t = torch.randn(100, 30, device=DEV)
    for bad in ([t, t], [t, t[5:]], [t[:, :20], t[:, 19:]]):
        keep = t.clone()
        with pytest.raises(nmfx.ArgumentError):
            nmfx.clip_grad_norm(bad, 1.0)
        assert torch.equal(t, keep)
    assert abs(float(nmfx.grad_norm([t, t])) - float(t.norm()) * math.sqrt(2)) < 1e-2      # reading one twice is no fault
    u = torch.empty(100, 30, device=DEV)
    with pytest.raises(nmfx.ArgumentError):
        nmfx.clip_grad_norm([t, u], 1.0, out=[u, torch.empty_like(u)])                     # a result over another's gradient
    with pytest.raises(nmfx.DimensionMismatch):
        nmfx.clip_grad_norm([t], 1.0, out=[u[:99]])
    with pytest.raises(nmfx.ArgumentError):
        nmfx.clip_grad_norm([t], 1.0, out=[torch.empty(30, 100, device=DEV).t()])
    with pytest.raises(nmfx.ArgumentError):
        nmfx.clip_grad_norm([t], 1.0, out=[u.half()])
    with pytest.raises(nmfx.ArgumentError):
        nmfx.clip_grad_norm([t], -1.0)
    with pytest.raises(nmfx.ArgumentError):
        nmfx.grad_norm([t], 1)
    with pytest.raises(nmfx.ArgumentError):
        nmfx.grad_norm([])
    with pytest.raises(nmfx.ArgumentError):
        nmfx.grad_norm([t.cpu()])
    with pytest.raises(nmfx.ArgumentError):
        nmfx.grad_norm([t.int()])
