"""A batch of queries alone in the paged caches' book: it takes no position and no
page, and is over when one of its sequences changes.  CPU only."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
INVALID = -1


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("ask") / "ask.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", os.path.join(HERE, "kv_ask_shim.cpp"), "-o", so],
                   check=True)
    lib = C.CDLL(so)
    lib.ask_new.restype = C.c_void_p
    return lib


class Book:
    def __init__(self, lib):
        self.lib, self.p = lib, C.c_void_p(lib.ask_new(64, 8, 4, 256))

    def __del__(self):
        self.lib.ask_free(self.p)

    def do(self, name, seqs, rows):
        s, r = (np.array(x, np.int32) for x in (seqs, rows))
        return getattr(self.lib, "ask_" + name)(self.p, s.ctypes.data_as(C.c_void_p), r.ctypes.data_as(C.c_void_p), len(seqs))

    def batch(self):
        s, r = np.full(8, -1, np.int32), np.full(9, -1, np.int32)
        n = self.lib.ask_batch(self.p, s.ctypes.data_as(C.c_void_p), r.ctypes.data_as(C.c_void_p))
        return s[:n].tolist(), r[:n + 1].tolist()

    def lens(self, seqs):
        return [self.lib.ask_len(self.p, s) for s in seqs]


def test_no_position_and_no_page(lib):
    b = Book(lib)
    s = [lib.ask_seq(b.p) for _ in range(3)]
    assert b.do("extend", s, [70, 5, 0]) == 0
    free = lib.ask_pages(b.p)
    assert b.do("ask", [s[2], s[0]], [4, 300]) == 0
    assert b.batch() == ([s[2], s[0]], [0, 4, 304])
    assert b.lens(s) == [70, 5, 0] and lib.ask_pages(b.p) == free
    assert b.do("ask", s, [0, 0, 0]) == 0 and b.batch() == (s, [0, 0, 0, 0])
    assert b.do("ask", [], []) == 0 and b.batch() == ([], [0])
    # rows of its own again
    assert b.do("extend", [s[1]], [1]) == 0 and b.batch() == ([s[1]], [0, 1]) and b.lens(s) == [70, 6, 0]


def test_refusals_leave_the_batch(lib):
    b = Book(lib)
    s = [lib.ask_seq(b.p) for _ in range(2)]
    assert b.do("extend", s, [3, 4]) == 0
    was = b.batch()
    for seqs, rows in (([s[0], s[0]], [1, 1]), ([s[0], 3], [1, 1]), ([-1], [1]), ([4], [1]), ([s[1]], [-1]), (s, [2 ** 31 - 1, 1])):
        assert b.do("ask", seqs, rows) == INVALID
        assert b.batch() == was and b.lens(s) == [3, 4]


def test_a_batch_is_over_when_its_sequences_change(lib):
    for change in ("truncate", "drop"):
        b = Book(lib)
        s = [lib.ask_seq(b.p) for _ in range(2)]
        assert b.do("extend", s, [100, 4]) == 0 and b.do("ask", [s[0]], [7]) == 0
        if change == "truncate":
            assert lib.ask_truncate(b.p, s[0], 60) == 0
        else:
            assert lib.ask_drop(b.p, s[0]) == 0
        assert b.batch() == ([], [0])
