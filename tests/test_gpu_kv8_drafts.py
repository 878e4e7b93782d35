"""Refused drafts in the 8-bit cache: what the rows that are kept hold after a cut, and drafts fed to a branch."""
import numpy as np
import pytest
import torch

import kv8_ref as ref
from test_gpu_kv8 import plain, rows_of

pytestmark = pytest.mark.gpu


def cache(nh):
    c = nh.KvCache8(1, 2, 64, 64, pages=6, seqs=3, cap=128)
    return c, c.new_seq()


def store(c, s, x):
    c.extend([s], [len(x)])
    c.append(0, x.cuda(), x.cuda())


def held(c, s, a=0):
    n = c.length(s) - a
    k, v = c.read(0, [s], [a], [n])
    assert torch.equal(k, v)
    return plain(k)


@pytest.mark.parametrize("size", [0.5, 3.0, 300.0, 1e6])
def test_a_refused_draft_leaves_its_step(nh, size):
    """The kept rows of its block are rounded to the step that the draft grew, off by a step in all, and later rows join
    that step; a block that begins anew is as if there had been no draft."""
    rng = np.random.default_rng(7)
    kept, draft, next_ = (rows_of(rng, n, 2, 64, "f32", s) for n, s in ((21, 1.0), (3, size), (20, 1.0)))
    c, s = cache(nh)
    store(c, s, kept)
    store(c, s, draft)
    c.truncate(s, 21)
    side = ref.Side(2, 64)
    side.store(plain(kept))
    before = side.held32()
    side.store(plain(draft))
    side.cut(21)
    now = held(c, s)
    assert np.array_equal(now, side.held32())
    assert np.array_equal(now[:16], before[:16]), "a whole block stays"
    grown = side.steps[1]
    for h in (0, 1):
        # (4 eps: the f32 roundings of x (1 / step) and code x step)
        assert np.abs(now[16:, h] - plain(kept)[16:, h]).max() <= grown[h] + 4 * 2.0 ** -23 * np.abs(plain(kept)).max()
    store(c, s, next_)
    side.store(plain(next_))
    now = held(c, s)
    assert np.array_equal(now, side.held32())
    assert np.array_equal(now[32:], ref.quantize(plain(next_)[11:])), "the next block has a step of its own"
    # cut back to the block's first position: nothing of the draft is left
    c.truncate(s, 16)
    store(c, s, kept[16:])
    assert np.array_equal(held(c, s), ref.quantize(plain(kept), (16,)))


def test_drafts_fed_to_a_branch_leave_no_trace(nh):
    rng = np.random.default_rng(8)
    kept, draft, next_ = (rows_of(rng, n, 2, 64, "f32", s) for n, s in ((21, 1.0), (3, 1e3), (4, 1.0)))
    c, s = cache(nh)
    store(c, s, kept)
    was = held(c, s)
    b, = c.fork(s)
    store(c, b, draft)
    c.free(b)
    assert np.array_equal(held(c, s), was)
    side = ref.Side(2, 64)
    side.store(plain(kept))
    for i in range(4):
        store(c, s, next_[i:i + 1])
        side.store(plain(next_[i:i + 1]))
    assert np.array_equal(held(c, s), side.held32())
