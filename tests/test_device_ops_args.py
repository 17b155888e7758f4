"""The checks that the operators on device matrices make on the host, without a GPU: addresses are numbers here, nothing is read."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib(built):
    import nmfx
    if torch.cuda.is_available():
        pytest.skip("addresses here are made up: only where no GPU could read them")
    return nmfx._lib


def mat(L, rows=64, cols=32, rs=32, cs=1, dtype=0, data=0x10000, reserved=0):
    return L.DMat(data, rows, cols, rs, cs, dtype, reserved)


def opts(L, s=0.0, reduction=2, reserved=0):
    return L.XentOpts(s, -100, reduction, reserved)


def xent(L, W=None, H=None, o=None, labels=0x20000, loss=0x30000, ws=0x40000, size=1 << 40):
    lib = L.load()
    return lib.nmfx_xent(W or mat(L), H or mat(L, 32, 8, 1, 32), labels, o or opts(L), loss, None, ws, size, 0, None)


def test_struct_layouts(lib):
    assert C.sizeof(lib.DMat) == 48 and C.sizeof(lib.XentOpts) == 24


def test_xent_arguments(lib):
    L = lib
    assert xent(L) == L.ERR_NO_DEVICE                     # everything else is in order
    assert b"no CPU fallback" in L.load().nmfx_last_op_error()
    bad, dim, uns = L.ERR_BAD_ARG, L.ERR_DIM_MISMATCH, L.ERR_UNSUPPORTED
    assert xent(L, W=mat(L, dtype=7)) == bad
    assert xent(L, W=mat(L, dtype=2)) == bad              # H is Float32
    assert xent(L, W=mat(L, dtype=1), H=mat(L, 32, 8, 1, 32, 1)) == uns
    assert xent(L, W=mat(L, data=None)) == bad
    assert xent(L, W=mat(L, data=0x10002)) == bad
    assert xent(L, W=mat(L, reserved=1)) == bad
    assert xent(L, W=mat(L, rs=31)) == bad                # rows overlap
    assert xent(L, W=mat(L, rs=-32)) == bad
    assert xent(L, W=mat(L, rs=64, cs=2)) == bad
    assert xent(L, W=mat(L, rows=-1)) == dim
    assert xent(L, W=mat(L, rows=0)) == dim
    assert xent(L, W=mat(L, rows=(1 << 21) + 1)) == uns
    assert xent(L, W=mat(L, rs=(1 << 21) + 16)) == uns
    assert xent(L, H=mat(L, 31, 8, 1, 32)) == dim
    assert xent(L, o=opts(L, -0.1)) == bad and xent(L, o=opts(L, 1.1)) == bad and xent(L, o=opts(L, float("nan"))) == bad
    assert xent(L, o=opts(L, reduction=3)) == bad and xent(L, o=opts(L, reserved=1)) == bad
    assert xent(L, labels=None) == bad and xent(L, loss=None) == bad and xent(L, ws=None) == bad and xent(L, ws=0x40010) == bad
    size = C.c_int64()
    assert L.load().nmfx_xent_workspace(mat(L), mat(L, 32, 8, 1, 32), opts(L), 0, size) == L.OK
    assert xent(L, size=size.value - 1) == bad and xent(L, size=size.value) == L.ERR_NO_DEVICE
    assert L.load().nmfx_xent_workspace(mat(L), mat(L, 32, 8, 1, 32), None, 0, size) == bad
    assert L.load().nmfx_xent_workspace(mat(L), mat(L, 32, 8, 1, 32), opts(L), 0, None) == bad


def test_xent_grad_arguments(lib):
    L = lib

    def grad(dW=None, dH=None, lse=0x50000, given=0):
        return L.load().nmfx_xent_grad(mat(L), mat(L, 32, 8, 1, 32, data=0x60000), 0x20000, opts(L), None, given, None, lse, dW or mat(L, data=0x70000),
                                       dH or mat(L, 32, 8, 1, 32, data=0x80000), 0x40000, 1 << 40, 0, None)

    assert grad() == L.ERR_NO_DEVICE and grad(lse=None) == L.ERR_NO_DEVICE
    assert grad(lse=None, given=1) == L.ERR_BAD_ARG
    assert grad(dW=mat(L, rows=63)) == L.ERR_DIM_MISMATCH and grad(dH=mat(L, 32, 9, 1, 32)) == L.ERR_DIM_MISMATCH
    assert grad(dW=mat(L, dtype=2)) == L.ERR_BAD_ARG and grad(dH=mat(L, 32, 8, 0, 1)) == L.ERR_BAD_ARG
    # W: 64 x 32 at 0x10000, H: 32 x 8 at 0x60000, Float32
    assert grad(dW=mat(L)) == L.ERR_BAD_ARG and grad(dW=mat(L, data=0x60000 - 64 * 32 * 4 + 4)) == L.ERR_BAD_ARG
    assert grad(dW=mat(L, data=0x60000 - 64 * 32 * 4)) == L.ERR_NO_DEVICE and grad(dW=mat(L, data=0x60000 + 8 * 32 * 4)) == L.ERR_NO_DEVICE
    assert grad(dH=mat(L, 32, 8, 1, 32, data=0x60000)) == L.ERR_BAD_ARG and grad(dH=mat(L, 32, 8, 1, 32, data=0x70000 + 512)) == L.ERR_BAD_ARG
    assert grad(dH=mat(L, 32, 8, 1, 32, data=0x10000 + 64 * 32 * 4 - 4)) == L.ERR_BAD_ARG
    # side by side in one buffer's rows of 64
    side = mat(L, rs=64, data=0x70000)
    assert grad(dW=side, dH=mat(L, 32, 8, 8, 1, data=0x70000 + 32 * 4)) == L.ERR_BAD_ARG       # longer than the gap
    assert grad(dW=side, dH=mat(L, 32, 8, 64, 1, data=0x70000 + 32 * 4)) == L.ERR_NO_DEVICE
    assert grad(dW=side, dH=mat(L, 32, 8, 64, 1, data=0x70000 + 31 * 4)) == L.ERR_BAD_ARG


def test_workspace_is_bounded(lib):
    """Pieces keep dz's two images at 512 MiB each whatever the sizes; the rest grows with W and H, not with their product."""
    L = lib
    size = C.c_int64()
    for p, n, k in ((131072, 8192, 2048), (1 << 20, 65536, 64)):
        assert L.load().nmfx_xent_workspace(mat(L, p, k, k, 1, 2), mat(L, k, n, 1, k, 2), opts(L), 1, size) == L.OK
        assert size.value < (3 << 30) + 2 * (p * k * 2 + 16 * n * k * 4) + p * n // 8, (p, n, k, size.value)
        assert size.value < p * n * 4 or p * n < 1 << 28


def test_norm_arguments(lib):
    L = lib
    lib_ = L.load()

    def clip(grads, out=None, max_norm=1.0, kind=2, count=None, norm=0x90000, ws=0xa0000, size=1 << 30):
        a = (L.DMat * max(1, len(grads)))(*grads)
        b = (L.DMat * len(out))(*out) if out else None
        return lib_.nmfx_clip_grad_norm(len(grads) if count is None else count, C.addressof(a), C.addressof(b) if b else None, max_norm, kind, norm, ws, size, 0, None)

    bad, dim = L.ERR_BAD_ARG, L.ERR_DIM_MISMATCH
    one = mat(L)
    assert clip([one]) == L.ERR_NO_DEVICE
    assert clip([]) == L.ERR_NO_DEVICE
    assert clip([one], max_norm=-1.0) == bad and clip([one], max_norm=float("nan")) == bad
    assert clip([one], kind=1) == bad and clip([one], count=-1) == bad and clip([one], norm=None) == bad
    assert clip([one], ws=None) == bad and clip([one], ws=0xa0004) == bad and clip([one], size=100) == bad
    assert clip([mat(L, dtype=9)]) == bad and clip([mat(L, reserved=2)]) == bad and clip([mat(L, data=None)]) == bad
    assert clip([mat(L, data=0x10001)]) == bad and clip([mat(L, rows=-1)]) == dim and clip([mat(L, rs=5)]) == bad
    assert clip([one, one]) == bad                                        # one tensor twice
    assert clip([one, mat(L, data=0x10000 + 64 * 32 * 4 - 4)]) == bad     # the last element
    assert clip([one, mat(L, data=0x10000 + 64 * 32 * 4)]) == L.ERR_NO_DEVICE
    left, right = mat(L, 64, 16, 32, 1), mat(L, 64, 16, 32, 1, data=0x10000 + 64)
    assert clip([left, right]) == L.ERR_NO_DEVICE                         # two halves of one buffer's rows
    assert clip([left, mat(L, 64, 16, 32, 1, data=0x10000 + 60)]) == bad
    assert clip([mat(L, 64, 17, 32, 1), right]) == bad
    gap = mat(L, 1, 16, 16, 1, data=0x10000 + 5 * 128 + 64)               # 16 elements behind a row's left half, dense
    assert clip([left, gap]) == L.ERR_NO_DEVICE and clip([right, gap]) == bad and clip([left, mat(L, 1, 17, 17, 1, data=0x10000 + 5 * 128 + 64)]) == bad
    assert clip([left, mat(L, 1, 16, 16, 1, data=0x10000 - 64)]) == L.ERR_NO_DEVICE and clip([left, mat(L, 1, 17, 17, 1, data=0x10000 - 64)]) == bad
    other = mat(L, data=0x80000)
    assert clip([one], [other]) == L.ERR_NO_DEVICE and clip([one], [one]) == L.ERR_NO_DEVICE
    assert clip([one, other], [other, one]) == bad                        # exchanged: one's result is another's gradient
    assert clip([one], [mat(L, data=0x10004)]) == bad
    assert clip([one], [mat(L, rows=63, data=0x80000)]) == dim
    assert clip([one], [mat(L, dtype=2, data=0x80000)]) == bad
    assert clip([one], [mat(L, 64, 32, 1, 64, data=0x80000)]) == bad      # another contiguous index


def test_norm_of_nothing_shares_nothing(lib):
    L = lib
    empty = mat(L, rows=0, data=None)
    a = (L.DMat * 3)(empty, empty, mat(L))
    assert L.load().nmfx_clip_grad_norm(3, C.addressof(a), None, 1.0, 2, 0x90000, 0xa0000, 1 << 30, 0, None) == L.ERR_NO_DEVICE


def test_messages_are_per_thread(lib):
    import threading
    L = lib
    assert xent(L, W=mat(L, dtype=7)) == L.ERR_BAD_ARG
    seen = []
    t = threading.Thread(target=lambda: seen.append(L.load().nmfx_last_op_error()))
    t.start()
    t.join()
    assert seen == [b""] and b"dtype" in L.load().nmfx_last_op_error()


def test_python_refuses_host_tensors(built):
    import nmfx
    W, H, y = torch.zeros(4, 2), torch.zeros(2, 3), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: nmfx.softmax_xent(W, H, y), lambda: nmfx.softmax_xent_grad(W, H, y), lambda: nmfx.grad_norm([W]), lambda: nmfx.clip_grad_norm(W, 1.0)):
        with pytest.raises(nmfx.ArgumentError, match="no CPU path"):
            call()
    with pytest.raises(nmfx.ArgumentError):
        nmfx.grad_norm([3.0])
