"""The 4-bit cache's page book against lists: every operation in random order,
the pages' contents followed through copies and moves, the counts of holders
and the free pages checked after each.  CPU only."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def book(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("book") / "book.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC",
                    os.path.join(HERE, "kv4_book_shim.cpp"), "-o", so], check=True)
    lib = C.CDLL(so)
    lib.book_new.restype = C.c_void_p
    for name in ("free_seq", "fork", "truncate", "free_pages", "len", "table", "refs", "batch", "copy", "extend",
                 "compact", "new_seq", "free"):
        getattr(lib, "book_" + name).argtypes = None
    return lib


class Book:
    def __init__(self, lib, page, pages, seqs, cap):
        self.lib, self.page, self.n_pages = lib, page, pages
        self.p = C.c_void_p(lib.book_new(page, pages, seqs, cap))
        self.pool = {}  # (page, slot) -> value

    def ints(self, v):
        return np.ascontiguousarray(v, dtype=np.int32)

    def table(self, s):
        out = np.zeros(self.n_pages + 8, np.int32)
        n = self.lib.book_table(self.p, s, out.ctypes.data_as(C.c_void_p))
        return out[:n].tolist()

    def contents(self, s):
        t = self.table(s)
        return [self.pool.get((t[i // self.page], i % self.page)) for i in range(self.lib.book_len(self.p, s))]

    def copy_pages(self, pairs):
        for a, z in pairs:
            for i in range(self.page):
                self.pool[z, i] = self.pool.get((a, i))

    def extend(self, seqs, rows):
        s, r, pairs = self.ints(seqs), self.ints(rows), np.zeros(2 * len(seqs) + 2, np.int32)
        n = self.lib.book_extend(self.p, s.ctypes.data_as(C.c_void_p), r.ctypes.data_as(C.c_void_p), len(seqs),
                                 pairs.ctypes.data_as(C.c_void_p))
        if n > 0:
            self.copy_pages(pairs[:2 * n].reshape(-1, 2).tolist())
        return n

    def copy(self, s):
        to, pairs = C.c_int(-1), np.zeros(2 * self.n_pages, np.int32)
        n = self.lib.book_copy(self.p, s, C.byref(to), pairs.ctypes.data_as(C.c_void_p))
        if n < 0:
            return n
        self.copy_pages(pairs[:2 * n].reshape(-1, 2).tolist())
        return to.value

    def compact(self, seqs, ranges):
        s, counts = self.ints(seqs), self.ints([len(r) for r in ranges])
        flat = self.ints([x for r in ranges for pair in r for x in pair] or [0])
        total = sum(max(0, e - a) for r in ranges for a, e in r)
        moves = np.zeros(4 * total + 4, np.int32)
        n = self.lib.book_compact(self.p, s.ctypes.data_as(C.c_void_p), len(seqs), counts.ctypes.data_as(C.c_void_p),
                                  flat.ctypes.data_as(C.c_void_p), moves.ctypes.data_as(C.c_void_p))
        if n > 0:
            # all reads before all writes: fresh pages hold nothing yet
            got = [(tuple(m[2:]), self.pool.get(tuple(m[:2]))) for m in moves[:4 * n].reshape(-1, 4).tolist()]
            self.pool.update(got)
        return n

    def check(self, model):
        """Pages held as often as the tables say, the others free, contents as the model has them."""
        held = {}
        for s, want in model.items():
            assert self.lib.book_len(self.p, s) == len(want)
            t = self.table(s)
            assert len(t) == -(-len(want) // self.page) and len(set(t)) == len(t)
            assert self.contents(s) == want
            for p in t:
                held[p] = held.get(p, 0) + 1
        for p in range(self.n_pages):
            assert self.lib.book_refs(self.p, p) == held.get(p, 0), p
        assert self.lib.book_free_pages(self.p) == self.n_pages - len(held)


@pytest.mark.parametrize("seed", range(12))
def test_random_operations(book, seed):
    rng = random.Random(seed)
    page = rng.choice((4, 8, 32))
    b = Book(book, page, rng.choice((6, 20, 60)), 9, 12 * page)
    model, tag = {}, 0
    for _ in range(250):
        op = rng.choice(("new", "free", "fork", "copy", "truncate", "extend", "extend", "extend", "compact"))
        live = sorted(model)
        if op == "new":
            s = book.book_new_seq(b.p)
            if s >= 0:
                assert s not in model
                model[s] = []
            else:
                assert s == -4 and len(model) == 9
        elif not live:
            continue
        elif op == "free":
            s = rng.choice(live)
            assert book.book_free_seq(b.p, s) == 0
            del model[s]
        elif op == "fork":
            s, n = rng.choice(live), rng.randrange(0, 4)
            out = np.zeros(4, np.int32)
            rc = book.book_fork(b.p, s, n, out.ctypes.data_as(C.c_void_p))
            if rc == 0:
                for c in out[:n].tolist():
                    assert c not in model
                    model[c] = list(model[s])
            else:
                assert rc == -4 and len(model) + n > 9
        elif op == "copy":
            s = rng.choice(live)
            before = book.book_free_pages(b.p)
            c = b.copy(s)
            if c >= 0:
                assert c not in model
                model[c] = list(model[s])
            else:
                assert c == -4 and (len(model) == 9 or before < -(-len(model[s]) // page))
        elif op == "truncate":
            s = rng.choice(live)
            n = rng.randrange(0, len(model[s]) + 1)
            assert book.book_truncate(b.p, s, n) == 0
            model[s] = model[s][:n]
        elif op == "extend":
            seqs = rng.sample(live, rng.randrange(0, len(live) + 1))
            rows = [rng.choice((0, 1, 2, page, rng.randrange(0, 2 * page))) for _ in seqs]
            rc = b.extend(seqs, rows)
            if rc >= 0:
                bs, br = np.zeros(16, np.int32), np.zeros(17, np.int32)
                assert book.book_batch(b.p, bs.ctypes.data_as(C.c_void_p), br.ctypes.data_as(C.c_void_p)) == len(seqs)
                assert bs[:len(seqs)].tolist() == seqs
                assert np.diff(br[:len(seqs) + 1]).tolist() == rows and br[0] == 0
                for s, r in zip(seqs, rows):
                    t = b.table(s)
                    for i in range(len(model[s]), len(model[s]) + r):
                        p = t[i // page]
                        assert book.book_refs(b.p, p) == 1, "a written page is its writer's alone"
                        tag += 1
                        b.pool[p, i % page] = tag
                        model[s].append(tag)
            else:
                assert rc in (-1, -4)
                if rc == -1:
                    assert any(len(model[s]) + r > 12 * page for s, r in zip(seqs, rows))
        else:
            seqs = rng.sample(live, rng.randrange(1, min(3, len(live)) + 1))
            ranges = []
            for s in seqs:
                cuts = sorted(rng.randrange(0, len(model[s]) + 1) for _ in range(2 * rng.randrange(0, 4)))
                if cuts and rng.random() < 0.5:
                    cuts[0] = 0
                ranges.append(list(zip(cuts[::2], cuts[1::2])))
            rc = b.compact(seqs, ranges)
            if rc >= 0:
                for s, r in zip(seqs, ranges):
                    model[s] = [x for a, e in r for x in model[s][a:e]]
            else:
                assert rc == -4
        b.check(model)
    book.book_free(b.p)


def test_refusals_change_nothing(book):
    b = Book(book, 32, 4, 3, 96)
    s = book.book_new_seq(b.p)
    assert b.extend([s], [40]) == 0
    for i in range(40):
        b.pool[b.table(s)[i // 32], i % 32] = i
    model = {s: list(range(40))}
    b.check(model)
    assert b.extend([s], [57]) == -1          # past the capacity
    assert b.extend([s, s], [1, 1]) == -1     # named twice
    assert b.extend([2], [1]) == -1           # not a sequence
    assert b.extend([-1], [1]) == -1
    assert b.extend([s], [-1]) == -1
    assert book.book_truncate(b.p, s, 41) == -1
    assert book.book_truncate(b.p, s, -1) == -1
    assert book.book_free_seq(b.p, 7) == -1
    assert b.compact([s], [[(5, 4)]]) == -1
    assert b.compact([s], [[(0, 8), (7, 9)]]) == -1
    assert b.compact([s], [[(0, 41)]]) == -1
    assert b.compact([s], [[(-1, 4)]]) == -1
    assert b.compact([s, s], [[(0, 4)], [(0, 4)]]) == -1
    out = np.zeros(8, np.int32)
    assert book.book_fork(b.p, s, 3, out.ctypes.data_as(C.c_void_p)) == -4
    assert book.book_fork(b.p, s, -1, out.ctypes.data_as(C.c_void_p)) == -1
    b.check(model)
    # three holders of one part-filled page: two of them need a copy, one page is left
    assert book.book_fork(b.p, s, 2, out.ctypes.data_as(C.c_void_p)) == 0
    kids = out[:2].tolist()
    t = b.copy(s)
    assert t == -4
    model |= {k: list(range(40)) for k in kids}
    b.check(model)
    assert b.extend([s, *kids], [1, 1, 1]) == 2
    assert book.book_free_pages(b.p) == 0
    assert b.extend([s], [30]) == -4
    # what fills a page exactly is shared without a copy
    assert book.book_truncate(b.p, s, 32) == 0
    assert book.book_free_pages(b.p) == 1


def test_a_changed_sequence_ends_the_batch(book):
    b = Book(book, 32, 16, 6, 96)
    s, o = book.book_new_seq(b.p), book.book_new_seq(b.p)
    batch, row0 = np.zeros(8, np.int32), np.zeros(8, np.int32)

    def size():
        return book.book_batch(b.p, batch.ctypes.data_as(C.c_void_p), row0.ctypes.data_as(C.c_void_p))
    out = np.zeros(4, np.int32)
    for change in (lambda: book.book_truncate(b.p, s, 1), lambda: book.book_fork(b.p, s, 1, out.ctypes.data_as(C.c_void_p)),
                   lambda: b.copy(s), lambda: b.compact([s], [[(1, 2)]]), lambda: book.book_free_seq(b.p, s)):
        assert b.extend([s], [3]) >= 0 and size() == 1
        book.book_truncate(b.p, o, 0)
        assert size() == 1
        assert change() >= 0
        assert size() == 0
