"""Softmax cross entropy of a factor model's logits W*H with its gradients, and the norm over many gradients with clipping:
cases that stand for their use, their plain forms, and the framework's calls."""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
IGNORED = -100
MAX_NORM = 1.0


def _lib():
    path = os.path.join(os.getcwd(), "nmf.jl_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import nmfx
    return nmfx


def _xent(name, dtype, p, n, k, grad, layout="k", ignored=0.0, smoothing=0.0):
    """W is p x k (classes by components), H is k x n (components by observations, a column's components contiguous).
    layout: which index of W is contiguous ("k": a class's row, "p": column-major, as the framework's host matrices are)."""
    c = {"op": "xent", "dtype": dtype, "p": p, "n": n, "k": k, "grad": grad, "layout": layout, "ignored": ignored, "smoothing": smoothing}
    return c | {"name": name} if name else c


def _norm(name, dtype, layers, d, p, n, clip):
    """Gradients of `layers` blocks of width d, of a p x d output matrix and of its d x n states."""
    c = {"op": "norm", "dtype": dtype, "layers": layers, "d": d, "p": p, "n": n, "clip": clip}
    return c | {"name": name} if name else c


def listed():
    return [
        # serving: the log-probability of one token, where latency counts
        _xent("score-one", "bf16", 32768, 1, 512, False),
        # serving: a few candidates over an odd vocabulary
        _xent("score-few", "f16", 100003, 7, 1000, False),
        # evaluation of a long text under a factor model: the framework's 131072 x 16384, k = 256 problem
        _xent("evaluate-long", "bf16", 131072, 16384, 256, False),
        # a small training step in the framework's own type and order: 4096 x 4096, k = 64, W column-major
        _xent("train-f32", "f32", 4096, 4096, 64, True, layout="p"),
        # fine-tuning on answers only: ragged sizes, two tokens in five ignored, smoothed labels
        _xent("train-ragged", "bf16", 50021, 1021, 777, True, ignored=0.4, smoothing=0.1),
        # an ordinary training step
        _xent("train", "bf16", 32768, 4096, 1024, True),
        # the framework's headline shape, 16384 x 16384, k = 256, W column-major
        _xent("train-columns", "f16", 16384, 16384, 256, True, layout="p"),
        # the largest: a large vocabulary and a long batch
        _xent("train-large", "bf16", 131072, 8192, 2048, True),
        # clipping the two factors of a small model: latency
        _norm("clip-factors", "f32", 0, 16, 512, 300, True),
        # many tensors of odd sizes
        _norm("clip-ragged", "f16", 12, 333, 5003, 77, True),
        # the gradients of a deep model
        _norm("clip-layers", "bf16", 24, 1024, 32768, 4096, True),
        # only the norm, as a monitor takes it, of single-precision gradients of a large model
        _norm("norm-large", "f32", 24, 2048, 32768, 8192, False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.3:
        return _norm(None, rng.choice(["f32", "bf16", "f16"]), rng.randint(0, 24), _log(rng, 16, 1024), _log(rng, 300, 32768), _log(rng, 1, 4096), rng.random() < 0.7)
    grad = rng.random() < 0.6
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    n, k = _log(rng, 1, 8192), _log(rng, 32, 2048)
    p = _log(rng, 300, 131072 if dtype != "f32" else 32768)
    if rng.random() < 0.5:
        k = (k + 31) // 32 * 32
    return _xent(None, dtype, p, n, k, grad, layout=rng.choice(["k", "k", "p"]), ignored=rng.choice([0.0, 0.0, 0.3, 0.8]), smoothing=rng.choice([0.0, 0.0, 0.1]))


def _shapes(case):
    d = case["d"]
    block = [(d, d)] * 4 + [(4 * d, d), (d, 4 * d), (d,), (d,)]
    return block * case["layers"] + [(case["p"], d), (d, case["n"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["dtype"]]
    if case["op"] == "norm":
        grads = [(torch.randn(s, generator=g, device="cuda") * 0.02).to(t) for s in _shapes(case)]
        state = {"case": case, "grads": grads}
        if case["clip"]:  # the clipped gradients go into one flat buffer, as a sharded optimizer keeps them
            state["flat"] = torch.empty(sum(x.numel() for x in grads), dtype=t, device="cuda")
            state["clipped"] = [v.view(x.shape) for v, x in zip(state["flat"].split([x.numel() for x in grads]), grads)]
        return state
    p, n, k = case["p"], case["n"], case["k"]
    H = torch.randn((n, k), generator=g, device="cuda").to(t)
    scale = 2.0 / math.sqrt(k)  # logits of deviation 2
    W = torch.randn((p, k) if case["layout"] == "k" else (k, p), generator=g, device="cuda").mul_(scale).to(t)
    # a few classes are frequent and most are rare, as words are
    labels = (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) ** 3 * p).long().clamp_(0, p - 1)
    off = int(n * case["ignored"])
    labels[torch.randperm(n, generator=g, device="cuda")[:off]] = IGNORED
    return {"case": case, "W": W if case["layout"] == "k" else W.t(), "H": H.t(), "labels": labels}


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        grads = state["grads"]
        if own:
            lib = _lib()
            if case["clip"]:
                return {"norm": lib.clip_grad_norm(grads, MAX_NORM, out=state["clipped"]), "grads": state["flat"]}
            return {"norm": lib.grad_norm(grads)}
        norm = torch.sqrt(torch.stack([x.float().square().sum() for x in grads]).sum())
        if not case["clip"]:
            return {"norm": norm}
        coef = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
        [o.copy_(x.float() * coef) for o, x in zip(state["clipped"], grads)]
        return {"norm": norm, "grads": state["flat"]}
    W, H, labels, eps = state["W"], state["H"], state["labels"], case["smoothing"]
    if own:
        lib = _lib()
        if not case["grad"]:
            loss, lse = lib.softmax_xent(W, H, labels, ignore_index=IGNORED, label_smoothing=eps, reduction="none")
            return {"loss": loss, "lse": lse}
        loss, lse, dW, dH = lib.softmax_xent_grad(W, H, labels, ignore_index=IGNORED, label_smoothing=eps, reduction="mean")
        return {"loss": loss, "lse": lse, "dW": dW, "dH": dH}
    p = W.shape[0]
    Wf, Hf = W.float(), H.float()
    z = Hf.t() @ Wf.t()  # n x p
    valid = labels != IGNORED
    y = labels.clamp(min=0)
    top = z.max(1, keepdim=True).values
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    loss = lse[:, 0] - (1 - eps) * z.gather(1, y[:, None])[:, 0]
    if eps:
        loss = loss - eps * z.mean(1)
    loss = torch.where(valid, loss, 0.0)
    lse_out = torch.where(valid, lse[:, 0], 0.0)
    if not case["grad"]:
        return {"loss": loss, "lse": lse_out}
    count = valid.sum().clamp(min=1)
    g = torch.where(valid, 1.0 / count, 0.0)
    dz = torch.exp(z - lse)
    if eps:
        dz -= eps / p
    dz.scatter_add_(1, y[:, None], torch.full_like(lse, eps - 1.0))
    dz *= g[:, None]
    return {"loss": loss.sum() / count, "lse": lse_out, "dW": (dz.t() @ Hf.t()).to(W.dtype), "dH": (dz @ Wf).t().to(H.dtype)}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        grads = state["grads"]
        norm = math.sqrt(math.fsum(float((x.double() ** 2).sum()) for x in grads))
        out = {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda")}
        if case["clip"]:
            out["grads"] = torch.cat([x.reshape(-1) for x in grads]).double() * min(1.0, MAX_NORM / (norm + 1e-6))
        return out
    W, X, labels, eps = state["W"].double(), state["H"].t().double(), state["labels"], case["smoothing"]
    n, p = X.shape[0], W.shape[0]
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    lse = torch.zeros_like(loss)
    dX, dW = torch.zeros_like(X), torch.zeros(p, X.shape[1], dtype=torch.float64, device="cuda")
    rows = torch.nonzero(labels != IGNORED)[:, 0]
    for r in torch.split(rows, 2048):
        if not len(r):
            continue
        z, y, i = X[r] @ W.t(), labels[r], torch.arange(len(r), device="cuda")
        lse[r] = torch.logsumexp(z, 1)
        target = torch.full((1, p), eps / p, dtype=torch.float64, device="cuda").expand(len(r), p).clone()
        target[i, y] += 1 - eps
        loss[r] = lse[r] - (target * z).sum(1)
        if case["grad"]:
            dz = (torch.softmax(z, 1) - target) / len(rows)
            dX[r] = dz @ W
            dW += dz.t() @ X[r]
    if not case["grad"]:
        return {"loss": loss, "lse": lse}
    return {"loss": loss.sum() / max(1, len(rows)), "lse": lse, "dW": dW, "dH": dX.t()}


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "norm":
        count = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": e * count * (2 if case["clip"] else 1) + 4, "flops": count * (3 if case["clip"] else 2)}
    p, n, k = case["p"], case["n"], case["k"]
    valid = n - int(n * case["ignored"])
    times = 2 if case["grad"] else 1
    return {"bytes": times * e * k * (p + n) + 16 * n, "flops": 2 * p * valid * k * (3 if case["grad"] else 1)}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(s)) for s in range(6)]:
        print(c, work(c))
