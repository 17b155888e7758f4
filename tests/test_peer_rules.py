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
    lib.layout_refusal.restype = C.c_char_p
    lib.place_of.restype = C.c_uint64
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


def refusal(lib, ranks):
    """ranks: (process, hardware queues, device); every rank has a window of its own."""
    flat = [v for i, (pid, queues, device) in enumerate(ranks) for v in (pid, queues, device, 0x1000 * (i + 1))]
    why = lib.layout_refusal((C.c_uint64 * len(flat))(*flat), len(ranks))
    return why.decode() if why else None


def test_one_process_per_device_is_fine(rules):
    for n in (1, 2, 8, 16):
        assert refusal(rules, [(100 + r, 4, 7000 + r) for r in range(n)]) is None


def test_two_processes_share_a_device_and_more_are_refused(rules):
    assert refusal(rules, [(1, 4, 7), (2, 4, 7)]) is None
    assert refusal(rules, [(1, 24, 7), (2, 24, 7), (3, 4, 8), (4, 4, 8)]) is None          # two each on two devices
    for queues in (1, 4, 24):
        for n in (3, 4, 8):
            assert "two processes" in refusal(rules, [(r, queues, 7) for r in range(n)])
    crowd = [(1, 4, 8), (2, 4, 7), (3, 4, 7), (4, 4, 7)]                                  # the rank on device 8 answers as the others do
    assert all("two processes" in refusal(rules, crowd[i:] + crowd[:i]) for i in range(4))


def test_ranks_of_one_process_on_one_device_need_queues(rules):
    assert refusal(rules, [(1, 4, 7)] * 2) is None and "GPU_MAX_HW_QUEUES" in refusal(rules, [(1, 3, 7)] * 2)
    for n, enough in ((3, 10), (4, 13), (8, 25)):
        assert refusal(rules, [(1, enough, 7)] * n) is None
        for queues in (1, 4, enough - 1):
            assert "GPU_MAX_HW_QUEUES" in refusal(rules, [(1, queues, 7)] * n)
    assert refusal(rules, [(1, 4, 7 + r) for r in range(8)]) is None                      # a device each: a queue each
    mixed = [(1, 24, 7)] * 4 + [(2, 4, 7)] * 3
    assert "GPU_MAX_HW_QUEUES" in refusal(rules, mixed) and "GPU_MAX_HW_QUEUES" in refusal(rules, mixed[::-1])


def test_the_timing_stand_in_is_its_own_peer(rules):
    """One rank's handle for all of them: one window, one stream that never waits."""
    flat = [1, 4, 7, 0x1000] * 8
    assert rules.layout_refusal((C.c_uint64 * len(flat))(*flat), 8) is None


def test_the_runtime_s_number_of_queues(rules):
    assert [rules.queues_of(s) for s in (None, b"", b"4", b"24", b"x", b"-1", b"0")] == [4, 4, 4, 24, 4, 4, 4]


def test_partitions_of_a_card_are_devices_of_their_own(rules):
    """One PCI address, numbers or visible devices of their own: eight processes, one on each, are one process per device."""
    pci = b"0000:05:00.0"
    by_number = [rules.place_of(pci, r, None, None) for r in range(8)]
    by_hip = [rules.place_of(pci, 0, b"%d" % r, None) for r in range(8)]
    by_rocr = [rules.place_of(pci, 0, None, b"%d" % r) for r in range(8)]
    assert len(set(by_number + by_hip + by_rocr)) >= 22 and len(set(by_number)) == len(set(by_hip)) == len(set(by_rocr)) == 8
    for places in (by_number, by_hip, by_rocr):
        assert refusal(rules, [(100 + r, 4, d) for r, d in enumerate(places)]) is None
    assert rules.place_of(pci, 0, None, None) == rules.place_of(pci, 0, None, None) != rules.place_of(b"0000:06:00.0", 0, None, None)
    assert rules.place_of(pci, 1, b"2", None) != rules.place_of(pci, 1, None, b"2") != rules.place_of(pci, 12, None, None)
