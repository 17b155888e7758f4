"""Operators on matrices that are in device memory (torch tensors): softmax cross entropy of W*H with its gradients, the norm over many
gradients, clipping by it.

They run on torch's current stream of the tensors' device, take their workspace from torch's allocator, wait for nothing and can be captured
into a graph.  The reference has no counterpart; the arithmetic is stated at the entry points in include/nmfx.h.  The rest of the package
works without torch: it is imported with the first call."""
from __future__ import annotations

import ctypes as C
from operator import attrgetter

import numpy as np

from . import _lib as L
from .api import ArgumentError, DimensionMismatch, _raise

_DMAT = np.dtype([("data", "u8"), ("rows", "i8"), ("cols", "i8"), ("rs", "i8"), ("cs", "i8"), ("dtype", "i4"), ("reserved", "i4")])
_REDUCTIONS = {"none": L.REDUCE_NONE, "sum": L.REDUCE_SUM, "mean": L.REDUCE_MEAN}
_state = {}
_dtype_of = attrgetter("dtype")


def _torch():
    if not _state:
        import torch
        _state.update(raw=getattr(torch._C, "_cuda_getCurrentRawStream", None), torch=torch, bytes=torch.uint8, written=torch.autograd.graph.increment_version, dtypes={torch.float32: L.F32, torch.float64: L.F64, torch.bfloat16: L.BF16, torch.float16: L.F16})
    return _state["torch"]


def _ck(status):
    if status != L.OK:
        _raise(status, L.load().nmfx_last_op_error().decode())


def _matrix(t, name, index=None):
    """The descriptor of a matrix; index: the device that it has to be on."""
    try:
        rows, cols = t.shape
        rs, cs = t.stride()
        d = L.DMat(t.data_ptr(), rows, cols, rs, cs, _state["dtypes"][t.dtype], 0)
        on = t.get_device()
    except (TypeError, ValueError, AttributeError, KeyError):
        on = None
    if on is None or on < 0 or (index is not None and on != index):
        _refuse_matrix(t, name, index)
    return d


def _refuse_matrix(t, name, index):
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise ArgumentError(f"{name} must be a torch tensor")
    if t.dim() != 2:
        raise DimensionMismatch(f"{name} must be a matrix, not {t.dim()}-dimensional")
    if t.dtype not in _state["dtypes"]:
        raise ArgumentError(f"{name} has dtype {t.dtype}: float32, float64, bfloat16 and float16 are taken")
    if not t.is_cuda:
        raise ArgumentError(f"{name} must be in device memory: there is no CPU path")
    raise ArgumentError(f"{name} is on {t.device}, not on cuda:{index}")


def _vector(t, name, n, dtype, index):
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise ArgumentError(f"{name} must be a torch tensor")
    if t.dtype != dtype:
        raise ArgumentError(f"{name} must be {dtype}, not {t.dtype}")
    if t.numel() != n or t.dim() > 1:
        raise DimensionMismatch(f"{name} must have {n} value(s), not the shape {tuple(t.shape)}")
    if t.get_device() != index:
        raise ArgumentError(f"{name} is on {t.device}, not on cuda:{index}")
    return t if t.is_contiguous() else t.contiguous()


def _xent_args(W, H, labels, ignore_index, label_smoothing, reduction):
    torch = _torch()
    if reduction not in _REDUCTIONS:
        raise ArgumentError(f"reduction must be 'none', 'sum' or 'mean', not {reduction!r}")
    w = _matrix(W, "W")
    index = W.get_device()
    h = _matrix(H, "H", index)
    return w, h, _vector(labels, "labels", h.cols, torch.int64, index), L.XentOpts(label_smoothing, ignore_index, _REDUCTIONS[reduction], 0), index


def _workspace(lib, w, h, o, grad, device):
    size = C.c_int64()
    status = lib.nmfx_xent_workspace(w, h, o, grad, size)
    if status:
        _ck(status)
    return _state["torch"].empty(size.value, dtype=_state["bytes"], device=device), size.value


def _stream(index):
    raw = _state["raw"]
    return raw(index) if raw else _torch().cuda.current_stream(index).cuda_stream


def _no_graph():
    """Outputs that torch's autograd takes for a function of W and H, and whose gradient it is refused: left out, it would be missing from a sum of
    losses without a word."""
    if "no_graph" not in _state:
        torch = _torch()

        class NoGraph(torch.autograd.Function):
            @staticmethod
            def forward(ctx, W, H, call):
                return call()

            @staticmethod
            def backward(ctx, *grads):
                raise ArgumentError("softmax_xent has no autograd graph: its gradients come from softmax_xent_grad or softmax_xent_backward "
                                    "(detach() its results where they are to be constants)")

        _state["no_graph"] = NoGraph
    return _state["no_graph"]


def softmax_xent(W, H, labels, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
    """Softmax cross entropy of the logits W @ H against one class per column, without keeping the logits: (loss, lse).

    W (p x k) and H (k x n) are float32, bfloat16 or float16 with one contiguous index each; labels has n int64 values, classes 0..p-1 or
    ignore_index.  loss is float32: n values for reduction 'none' (-loss is the label's log-probability), else one, the sum or the mean over
    the columns that are not ignored (0 where there is none).  lse, the log-sum-exp of every column's logits, has n values; both are 0 in
    ignored columns.  A label that is no class makes its column's loss NaN.

    There is no autograd graph behind them: a backward pass that reaches W or H through them (both count as functions of W and H while torch
    records gradients) is refused.  softmax_xent_grad gives the gradients."""
    torch = _torch()
    if (getattr(W, "requires_grad", False) or getattr(H, "requires_grad", False)) and torch.is_grad_enabled():
        return _no_graph().apply(W, H, lambda: _forward(W, H, labels, ignore_index, label_smoothing, reduction))
    return _forward(W, H, labels, ignore_index, label_smoothing, reduction)


def _forward(W, H, labels, ignore_index, label_smoothing, reduction):
    torch = _state["torch"]
    w, h, labels, o, index = _xent_args(W, H, labels, ignore_index, label_smoothing, reduction)
    lib, dev, n = L.load(), W.device, h.cols
    ws, size = _workspace(lib, w, h, o, 0, dev)
    loss = torch.empty((n,) if reduction == "none" else (), dtype=torch.float32, device=dev)
    lse = torch.empty(n, dtype=torch.float32, device=dev)
    status = lib.nmfx_xent(w, h, labels.data_ptr(), o, loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), size, index, _stream(index))
    if status:
        _ck(status)
    return loss, lse


def _like(t, d, device):
    """An empty matrix of t's shape, type and contiguous index, dense (d: t's descriptor)."""
    if d.cs == 1 or d.rs != 1:
        return _state["torch"].empty((d.rows, d.cols), dtype=t.dtype, device=device)
    return _state["torch"].empty((d.cols, d.rows), dtype=t.dtype, device=device).t()


def _grad(W, H, labels, ignore_index, label_smoothing, reduction, gout, lse, dW, dH):
    torch = _torch()
    w, h, labels, o, index = _xent_args(W, H, labels, ignore_index, label_smoothing, reduction)
    lib, dev, n = L.load(), W.device, h.cols
    if gout is not None:
        gout = _vector(gout, "gout", n if reduction == "none" else 1, torch.float32, index)
    given = lse is not None
    if given:
        lse, loss = _vector(lse, "lse", n, torch.float32, index), None
    else:
        lse = torch.empty(n, dtype=torch.float32, device=dev)
        loss = torch.empty((n,) if reduction == "none" else (), dtype=torch.float32, device=dev)
    theirs = [t for t in (dW, dH) if t is not None]
    dW = _like(W, w, dev) if dW is None else dW
    dH = _like(H, h, dev) if dH is None else dH
    gw, gh = _matrix(dW, "dW", index), _matrix(dH, "dH", index)
    ws, size = _workspace(lib, w, h, o, 1, dev)
    status = lib.nmfx_xent_grad(w, h, labels.data_ptr(), o, None if gout is None else gout.data_ptr(), given, None if given else loss.data_ptr(), lse.data_ptr(), gw, gh,
                                ws.data_ptr(), size, index, _stream(index))
    if status:
        _ck(status)
    if theirs:
        _state["written"](theirs)
    return loss, lse, dW, dH


def softmax_xent_grad(W, H, labels, ignore_index=-100, label_smoothing=0.0, reduction="mean", gout=None, dW=None, dH=None):
    """softmax_xent with its gradients: (loss, lse, dW, dH).

    gout is the gradient with respect to the loss (float32; n values for reduction 'none', else one; None: 1; with float16 gradients a loss
    scale belongs here).  dW and dH have the types of W and H and their contiguous index; matrices to write them to can be given.

    The results are constants to torch's autograd: dW and dH are the gradients, and go on from there as `H.backward(dH)` or into W.grad."""
    return _grad(W, H, labels, ignore_index, label_smoothing, reduction, gout, None, dW, dH)


def softmax_xent_backward(W, H, labels, lse, gout=None, ignore_index=-100, label_smoothing=0.0, reduction="mean", dW=None, dH=None):
    """The gradients alone, (dW, dH), from the lse that softmax_xent returned for the same arguments: for a gout that depends on the loss."""
    if lse is None:
        raise ArgumentError("lse must be what softmax_xent returned")
    return _grad(W, H, labels, ignore_index, label_smoothing, reduction, gout, lse, dW, dH)[2:]


def _list(ts, name, device):
    """The descriptors of a list of tensors, as an array of nmfx_dmat: contiguous ones as one row.  (A call over hundreds of small tensors
    takes as long as this does: a few passes over the list, each in C.)"""
    torch = _torch()
    T = torch.Tensor
    try:
        devices = set(map(T.get_device, ts))
        dtypes = list(map(_dtype_of, ts))
    except (TypeError, AttributeError):
        raise ArgumentError(f"{name} must be torch tensors") from None
    if devices != {device.index} or device.type != "cuda":
        if not all(t.is_cuda for t in ts):
            raise ArgumentError(f"{name} must be in device memory: there is no CPU path")
        raise ArgumentError(f"{name} are on several devices")
    codes = _state["dtypes"]
    kinds = set(dtypes)
    if not kinds <= codes.keys():
        raise ArgumentError(f"one of {name} has dtype {next(d for d in dtypes if d not in codes)}: float32, float64, bfloat16 and float16 are taken")
    a = np.zeros(len(ts), _DMAT)
    sizes = list(map(T.numel, ts))
    a["data"] = list(map(T.data_ptr, ts))
    a["cols"] = a["rs"] = sizes
    a["rows"] = a["cs"] = 1
    a["dtype"] = codes[dtypes[0]] if len(kinds) == 1 else [codes[d] for d in dtypes]
    dense = list(map(T.is_contiguous, ts))
    plain = all(dense)
    if not plain:
        for i in range(len(ts)):
            if not dense[i]:
                _strided(a, i, ts[i], name)
    return a, sizes, plain


def _few(ts, index):
    """The descriptors of a short list (2 us for two tensors; _list, made for hundreds, takes 6), or None where a tensor is not contiguous or
    not what it should be: _list then says what."""
    codes, sizes = _state["dtypes"], []
    a = (L.DMat * len(ts))()
    try:
        for d, t in zip(a, ts):
            if t.get_device() != index or not t.is_contiguous():
                return None
            n = t.numel()
            sizes.append(n)
            d.data, d.rows, d.cols, d.rs, d.cs, d.dtype = t.data_ptr(), 1, n, n, 1, codes[t.dtype]
    except (TypeError, AttributeError, KeyError):
        return None
    return a, sizes


def _strided(a, i, t, name):
    if t.dim() == 1:
        a[i] = (t.data_ptr(), t.shape[0], 1, t.stride(0), 1, a[i]["dtype"], 0)
    elif t.dim() == 2:
        a[i] = (t.data_ptr(), *t.shape, *t.stride(), a[i]["dtype"], 0)
    else:
        raise ArgumentError(f"one of {name} has more than two indices and is not contiguous")


def _norm_type(norm_type):
    if norm_type == 2:
        return L.NORM_2
    if norm_type == float("inf"):
        return L.NORM_INF
    raise ArgumentError(f"norm_type must be 2 or inf, not {norm_type!r}")


def _lists(grads, out, dev):
    """The descriptors of grads and of out (or None), as pointers to arrays that live as long as they do."""
    a, sizes, plain = _list(grads, "grads", dev)
    if out is None:
        return _pointer(a), None
    b, counts, plain_too = _list(out, "out", dev)
    if sizes != counts:
        raise DimensionMismatch("one of out has another number of elements than its gradient")
    # where one of the two is not contiguous both go by the strides of their matrix
    if not (plain and plain_too):
        for i in np.nonzero((a["rows"] != 1) | (b["rows"] != 1))[0]:
            if grads[i].shape != out[i].shape:
                raise DimensionMismatch("one of out has another shape than its gradient")
            _strided(a, i, grads[i], "grads")
            _strided(b, i, out[i], "out")
    return _pointer(a), _pointer(b)


def _pointer(a):
    return (L.DMat * len(a)).from_buffer(a)


def _norm(grads, max_norm, norm_type, out):
    torch = _torch()
    kind = _norm_type(norm_type)
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if not grads:
        raise ArgumentError("grads is empty")
    if not isinstance(grads[0], torch.Tensor):
        raise ArgumentError("grads must be torch tensors")
    dev = grads[0].device
    if out is not None:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(out) != len(grads):
            raise DimensionMismatch(f"out has {len(out)} tensors, grads {len(grads)}")
    few = len(grads) <= 8
    a = few and _few(grads, dev.index)
    b = few and out is not None and _few(out, dev.index)
    if a and (b or out is None):
        a, sizes = a
        if b:
            b, counts = b
            if sizes != counts:
                raise DimensionMismatch("one of out has another number of elements than its gradient")
    else:
        a, b = _lists(grads, out, dev)
    lib = L.load()
    size = C.c_int64()
    status = lib.nmfx_grad_norm_workspace(len(grads), size)
    if status:
        _ck(status)
    ws = torch.empty(size.value, dtype=torch.uint8, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    common = (norm.data_ptr(), ws.data_ptr(), size.value, dev.index, _stream(dev.index))
    if max_norm is None:
        _ck(lib.nmfx_grad_norm(len(grads), a, kind, *common))
    else:
        status = lib.nmfx_clip_grad_norm(len(grads), a, b or None, float(max_norm), kind, *common)
        if status:
            _ck(status)
        # autograd is told what was written in place: a graph that has saved it refuses its backward pass then (0.05 us a tensor)
        _state["written"](grads if out is None else out)
    return norm


def grad_norm(grads, norm_type=2):
    """The norm over all elements of a list of tensors (or of one), as a float32 tensor on their device: sqrt(sum g^2), or max |g| for
    norm_type inf.  float32, float64, bfloat16 and float16 may be mixed; squares are summed in float64."""
    return _norm(grads, None, norm_type, None)


def clip_grad_norm(grads, max_norm, norm_type=2, out=None):
    """Scales a list of tensors by min(1, max_norm / (norm + 1e-6)), in place or into `out`, and returns the norm that they had.

    Tensors are contiguous, or matrices and vectors with a stride; out's have as many elements as their gradients (where one of the two is
    strided, the same shape), and no two that are written may share elements."""
    if max_norm is None:
        raise ArgumentError("max_norm is None")
    return _norm(grads, max_norm, norm_type, out)
