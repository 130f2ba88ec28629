"""The order in which b2_pages_move reads and writes pages (csrc/page_plan.h), run on the host as the kernel runs it: every
destination holds what its source held before, whatever the moves, the lanes and the steps that a launch takes."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def emul(tmp_path_factory):
    so = tmp_path_factory.mktemp("page_plan") / "emul.so"
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-o", str(so), os.path.join(HERE, "page_plan_emul.cpp")])
    lib = ctypes.CDLL(str(so))
    lib.emul_pages.restype = ctypes.c_long
    sz, vp = ctypes.c_size_t, ctypes.c_void_p
    lib.emul_pages.argtypes = [sz, vp, vp, ctypes.c_int, sz, sz, sz, vp, sz, vp]

    def run(pages, dst, src, cap=480, lanes=64, batch=8, other=None):
        pool = np.arange(100, 100 + pages, dtype=np.int64)
        want = pool.copy()
        for d, s in zip(dst, src):
            want[d] = 0 if s < 0 else (pool if other is None else other)[s]
        d, s = np.array(dst, dtype=np.int64), np.array(src, dtype=np.int64)
        o = np.zeros(1, dtype=np.int64) if other is None else other
        reads = lib.emul_pages(len(d), d.ctypes.data, s.ctypes.data, other is not None, cap, lanes, batch, pool.ctypes.data, pages, o.ctypes.data)
        assert reads >= 0, {-1: "two lanes touch one page", -2: "a launch is too large"}[reads]
        assert np.array_equal(pool, want)
        return reads

    return run


def test_nothing_and_moves_onto_themselves(emul):
    assert emul(4, [], []) == 0
    assert emul(4, [0, 1, 2, 3], [0, 1, 2, 3]) == 0


def test_a_source_of_many_is_read_once_a_batch(emul):
    assert emul(20, list(range(1, 9)), [0] * 8, lanes=1) == 1
    assert emul(20, [5, 1, 7, 3], [2, 0, 2, 0], lanes=1) == 2


@pytest.mark.parametrize("cap", [3, 4, 5, 7, 480])
@pytest.mark.parametrize("length", [2, 3, 4, 8, 9, 17, 40])
def test_cycles_of_every_length(emul, cap, length):
    """one page is read more for each time that a cycle is closed early; a cycle that fits reads each page once"""
    pages = list(range(length))
    reads = emul(length, pages, pages[1:] + pages[:1], cap=cap)
    assert reads == length if length + 1 <= cap else reads > length


@pytest.mark.parametrize("cap,lanes,batch", [(480, 64, 8), (480, 1, 4), (5, 3, 1), (3, 2, 8), (16, 64, 4)])
def test_random_moves(emul, cap, lanes, batch):
    rng = random.Random(100 * cap + lanes)
    for _ in range(400):
        pages = rng.randint(1, 60)
        n = rng.randint(0, pages)
        dst = rng.sample(range(pages), n)
        kind = rng.randrange(4)
        if kind == 0:    # a permutation among the destinations
            src = rng.sample(dst, n)
        elif kind == 1:  # anything, zeros among it
            src = [rng.randint(-1, pages - 1) for _ in range(n)]
        elif kind == 2:  # few sources
            src = [rng.choice([0, pages - 1, pages // 2]) for _ in range(n)]
        else:            # to the front, in order: compaction
            dst, src = list(range(n)), sorted(rng.sample(range(pages), n))
        emul(pages, dst, src, cap=cap, lanes=lanes, batch=batch)
        other = np.array([rng.randrange(1 << 40) for _ in range(pages)], dtype=np.int64)
        emul(pages, dst, src, cap=cap, lanes=lanes, batch=batch, other=other)


def test_many_moves(emul):
    """several launches: more moves than one launch's parameters hold, and a cycle that no launch holds"""
    rng = random.Random(3)
    pages = 5000
    perm = rng.sample(range(pages), pages)
    emul(pages, list(range(pages)), perm)
    emul(pages, list(range(pages)), list(range(1, pages)) + [0])
    emul(pages, rng.sample(range(pages), 3000), [rng.randint(-1, pages - 1) for _ in range(3000)])
    emul(pages, list(range(1, pages)), [0] * (pages - 1))


# ---- at the batch of the kernel ---------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def kernel_batch(emul, tmp_path_factory):
    so = tmp_path_factory.mktemp("page_batch") / "batch.so"
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-o", str(so), os.path.join(HERE, "page_plan_emul.cpp")])
    return ctypes.CDLL(str(so)).kernel_batch()


def test_reads_of_one_source_in_the_kernel(emul, kernel_batch):
    """once for every batch that its steps take in a lane"""
    for copies in range(1, 20):
        assert emul(20, list(range(1, copies + 1)), [0] * copies, lanes=1, batch=kernel_batch) == -(-copies // kernel_batch)
    assert emul(20, [5, 1, 7, 3], [2, 0, 2, 0], lanes=1, batch=kernel_batch) == 2


@pytest.mark.parametrize("cap", [3, 4, 5, 7, 480])
@pytest.mark.parametrize("length", [2, 3, 4, 5, 8, 9, 17, 40, 481, 1200])
def test_cycles_in_the_kernel(emul, kernel_batch, cap, length):
    pages = list(range(length))
    reads = emul(length, pages, pages[1:] + pages[:1], cap=cap, batch=kernel_batch)
    assert reads == length if length + 1 <= cap else reads > length


@pytest.mark.parametrize("lanes", [1, 2, 7, 64])
def test_random_moves_in_the_kernel(emul, kernel_batch, lanes):
    rng = random.Random(lanes)
    for _ in range(400):
        pages = rng.randint(1, 90)
        n = rng.randint(0, pages)
        dst = rng.sample(range(pages), n)
        for src in (rng.sample(dst, n), [rng.randint(-1, pages - 1) for _ in range(n)], [rng.choice([0, pages - 1]) for _ in range(n)]):
            emul(pages, dst, src, lanes=lanes, batch=kernel_batch)
            other = np.array([rng.randrange(1 << 40) for _ in range(pages)], dtype=np.int64)
            emul(pages, dst, src, lanes=lanes, batch=kernel_batch, other=other)
    emul(5000, list(range(5000)), rng.sample(range(5000), 5000), lanes=lanes, batch=kernel_batch)
