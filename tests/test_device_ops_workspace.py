"""The workspace of the softmax cross entropy against what is said of it, without a GPU."""
import ctypes as C

import pytest


def workspace(L, p, n, k, dtype, grad, s=0.0, by="r"):
    size = C.c_int64()
    w = L.DMat(0x100000, p, k, *((k, 1) if by == "r" else (1, p)), dtype, 0)
    assert L.load().nmfx_xent_workspace(w, L.DMat(0x100000, k, n, 1, k, dtype, 0), L.XentOpts(s, -100, L.REDUCE_MEAN, 0), grad, size) == L.OK
    return size.value


@pytest.mark.parametrize("dtype", [0, 2, 3])          # Float32, BFloat16, Float16
@pytest.mark.parametrize("p,n,k", [(4096, 4096, 64), (32768, 8192, 1024), (131072, 8192, 2048), (50021, 1021, 777), (1 << 20, 65536, 64), (2 ** 21 - 1024, 2 ** 21 - 1024, 4)])
@pytest.mark.parametrize("s", [0.0, 0.1])
@pytest.mark.parametrize("by", ["r", "c"])
def test_workspace_is_what_the_header_says(built, dtype, p, n, k, s, by):
    import nmfx
    L = nmfx._lib
    es = 4 if dtype == 0 else 2
    n1, p1, k1 = -(-n // 256) * 256 + 128, -(-p // 256) * 256 + 128, -(-k // 64) * 64
    copies = es * k1 * (n1 + p1)
    lists = 64 * n1 + 65536                            # what there is of a column: indexes, labels, factors, losses
    tile = 256 if p * n >= 1 << 28 else 64
    statistics = (12 if s else 8) * max(-(-p // tile) * n1, 16384)
    forward = workspace(L, p, n, k, dtype, 0, s, by)
    assert forward <= copies + statistics + lists
    images = 2 * es * max(1 << 28, 256 * n1)
    sums = 4 * (k + 4) * (n1 + p1) + (1 << 28)         # dH, dW in Float32; parts of them only where they are small: 512 tiles of 256 x 256 floats each
    grad = workspace(L, p, n, k, dtype, 1, s, by)
    assert forward < grad <= 2 * copies + statistics + lists + images + sums
    if p * n >= 1 << 30 and n <= 65536:                # the logits of a large problem are never there as a whole
        assert grad < 4 * p * n
