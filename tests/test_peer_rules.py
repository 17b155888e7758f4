"""The peer transport's decisions that need no device (csrc/peer_rules.hpp), compiled for the host by themselves."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("peer_rules") / "rules.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", os.path.join(ROOT, "tests", "native", "peer_rules.cpp"), "-o", so], check=True, timeout=120)
    lib = C.CDLL(so)
    lib.pool_new.restype = C.c_void_p
    lib.pool_take.restype = C.c_uint64
    return lib


class Pool:
    def __init__(self, lib):
        self.lib, self.p = lib, C.c_void_p(lib.pool_new())

    def give(self, window, size, held, dev=0, flags=1):
        self.lib.pool_give(self.p, dev, flags, C.c_uint64(size), C.c_uint64(window), held)

    def take(self, size, dev=0, flags=1):
        b = C.c_uint64(size)
        w = self.lib.pool_take(self.p, dev, flags, C.byref(b))
        return (w, b.value) if w else None

    def end(self, window, rank):
        self.lib.window_end(C.c_uint64(window), rank)


@pytest.fixture
def pool(rules):
    p = Pool(rules)
    yield p
    rules.pool_delete(p.p)


def test_a_window_is_not_used_again_while_a_peer_may_store_into_it(pool):
    """Rank 0 of 4 leaves (no time-out has been seen: nothing in the window says that anything is wrong) while 1, 2 and 3 still solve."""
    pool.give(0x1000, 512, held=0b1110)
    assert pool.take(512) is None
    for rank in (2, 1):
        pool.end(0x1000, rank)
        assert pool.take(512) is None
    pool.end(0x1000, 3)
    assert pool.take(512) == (0x1000, 512)
    assert pool.take(512) is None                         # it is somebody's now


def test_a_rank_that_never_lets_go_keeps_the_window_out_of_use(pool):
    pool.give(0x1000, 512, held=0b0110)
    pool.end(0x1000, 1)
    for _ in range(3):
        assert pool.take(512) is None
    pool.give(0x2000, 512, held=0)                        # its handle never went out
    assert pool.take(512) == (0x2000, 512) and pool.take(512) is None


def test_the_smallest_window_that_serves_is_taken(pool):
    pool.give(0x1000, 4096, held=0)
    pool.give(0x2000, 1024, held=0)
    pool.give(0x3000, 512, held=0)
    pool.give(0x4000, 768, held=0b10)                     # would fit best, but is held
    assert pool.take(600) == (0x2000, 1024)
    assert pool.take(600) == (0x1000, 4096)
    assert pool.take(600) is None
    pool.end(0x4000, 1)
    assert pool.take(600) == (0x4000, 768)


def test_a_window_of_another_device_or_kind_of_memory_does_not_serve(pool):
    pool.give(0x1000, 512, held=0, dev=1, flags=1)
    pool.give(0x2000, 512, held=0, dev=0, flags=2)
    assert pool.take(512, dev=0, flags=1) is None
    assert pool.take(512, dev=1, flags=1) == (0x1000, 512) and pool.take(512, dev=0, flags=2) == (0x2000, 512)
