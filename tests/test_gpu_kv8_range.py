"""Attention over the 8-bit cache where blocks of values differ in size by more than any exponent of the kernels' own
spans: steps up to 2^110, zeros before them, large blocks that a window hides."""
import numpy as np
import pytest
import torch

import kv8_ref as ref
from test_gpu_kv8 import check_attend, plain, rows_of

pytestmark = pytest.mark.gpu


def held_of(nh, k, v, page=64):
    """A cache of one sequence with the rows k, v, which are its batch: (cache, id, k and v as held)."""
    c = nh.KvCache8(1, k.shape[1], k.shape[2], v.shape[2], pages=-(-len(k) // page), seqs=1, cap=len(k), page=page)
    s = c.new_seq()
    c.extend([s], [len(k)])
    c.append(0, k.cuda(), v.cuda())
    return c, s, ref.quantize(plain(k)), ref.quantize(plain(v))


# a factor for each 64 positions, the last one on to the end
SIZES = {"zeros then 1e20": (0, 1e20), "zeros then 1e25": (0, 1e25), "zeros then 1e30": (0, 1e30), "zeros then 1e34": (0, 1e34),
         "zeros then 1e-33": (0, 1e-33), "1e-30 then 1e10": (1e-30, 1e10), "1e30 then 1e-30": (1e30, 1e-30),
         "up by 1e8 a chunk": [10.0 ** (8 * i - 34) for i in range(9)], "up and down": (1.0, 1e30, 1e-25, 0, 1e33, 1.0)}


def sized(v, sizes):
    v = v.float()
    for i in range(-(-len(v) // 64)):
        v[64 * i:64 * i + 64] *= sizes[min(i, len(sizes) - 1)]
    return v.to(torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sizes", SIZES)
def test_rows_that_see_all_sizes(nh, sizes, dim):
    """The bound is of the largest value; a row that sees it all is far from 0 beside it."""
    rng = np.random.default_rng(dim)
    n, rows = 700, 300
    v = sized(rows_of(rng, n, 2, dim, "bf16"), SIZES[sizes])
    c, s, hk, hv = held_of(nh, rows_of(rng, n, 2, dim, "bf16"), v)
    q = rows_of(rng, rows, 4, dim, "bf16")
    o, _ = ref.attend(plain(q), hk, hv, dim ** -0.5, ask=True)
    assert np.abs(o).max() > 20 * 2.0 ** -10 * np.abs(hv).max()
    c.ask([s], [rows])
    for kernel in (0, 1, 2):
        c.debug_kernel(kernel)
        check_attend(c, 0, q, [hk], [hv], [rows], "bf16", ask=True, many=True)


def test_ranges_of_all_sizes(nh):
    """Few tiles of many keys: each range of keys begins with another size, and the ranges are joined."""
    rng = np.random.default_rng(3)
    n, rows = 9000, 260
    v = sized(rows_of(rng, n, 1, 64, "bf16"), [0, 0, 1e-30, 1e20, 0, 1e30, 1.0] * 20)
    c, s, hk, hv = held_of(nh, rows_of(rng, n, 1, 64, "bf16"), v, 256)
    q = rows_of(rng, rows, 1, 64, "bf16")
    c.ask([s], [rows])
    for kernel in (1, 2):
        c.debug_kernel(kernel)
        check_attend(c, 0, q, [hk], [hv], [rows], "bf16", ask=True, many=True)


@pytest.mark.parametrize("sizes", SIZES)
def test_rows_of_their_own_beside_all_sizes(nh, sizes):
    """Causal: rows of the first 64 positions are held to the size of what they see, whatever comes after them."""
    rng = np.random.default_rng(11)
    n = 300
    k, v = rows_of(rng, n, 2, 64, "bf16"), sized(rows_of(rng, n, 2, 64, "bf16"), SIZES[sizes])
    c, s, hk, hv = held_of(nh, k, v)
    q = rows_of(rng, n, 2, 64, "bf16")
    o, l = ref.attend(plain(q), hk, hv, 0.125)
    for kernel in (0, 1, 2):
        c.debug_kernel(kernel)
        lse = torch.empty(n, 2, dtype=torch.float32, device="cuda")
        got = plain(c.attend(0, q.cuda(), lse=lse)).astype(np.float64)
        for a, z in ((0, 64), (64, 128), (128, n)):
            limit = ref.attend_bound(plain(q), hk[:z], hv[:z], o[a:z], 0.125, "bf16", True)
            assert (np.abs(got[a:z] - o[a:z]) <= limit).all(), (kernel, a)
            # the scores' error alone: the bound of a value of 1
            score = ref.attend_bound(plain(q), hk[:z], np.ones_like(hv[:z]), 0 * o[a:z], 0.125, "bf16", True).max()
            assert np.abs(plain(lse[a:z]) - l[a:z]).max() <= score + 2.0 ** -20, (kernel, a)


@pytest.mark.parametrize("size", [1e6, 1e13, 1e20, 1e30])
@pytest.mark.parametrize("rows,heads,dim", [(1, 2, 64), (5, 2, 128), (300, 4, 64), (3, 2, 256)])
def test_large_blocks_that_a_window_hides(nh, rows, heads, dim, size):
    """Blocks that no row of the call sees, in chunks of which it sees other blocks, are as if they were not there."""
    rng = np.random.default_rng(rows + dim)
    n, sink, ring = 400, 20, 40
    v = rows_of(rng, n, 2, dim, "bf16").float()
    v[32:n - 48] *= size  # (positions 360 .. 399 and the sink's 0 .. 19 are seen; blocks from 32 to 351 are not)
    k, v = rows_of(rng, n, 2, dim, "bf16"), v.to(torch.bfloat16)
    c, s, hk, hv = held_of(nh, k, v)
    q = rows_of(rng, rows, heads, dim, "bf16")
    hidden = hv.copy()
    hidden[32:n - 48] = 0
    c.ask([s], [rows])
    for kernel in (0, 1, 2):
        c.debug_kernel(kernel)
        check_attend(c, 0, q, [hk], [hidden], [rows], "bf16", sink, ring, ask=True, many=True)


@pytest.mark.parametrize("kernel", [1, 2])
def test_rows_beside_large_values_of_later_rows(nh, kernel):
    """A border of blocks 10^6 times as large inside a tile of rows: rows in tiles before it keep the bound of what they
    see, rows of its own tile lose what is finer than 2^-40 of the largest step (2^-60, many rows)."""
    rng = np.random.default_rng(12)
    n, last = 200, 100
    k, v = rows_of(rng, n, 1, 64, "bf16"), rows_of(rng, n, 1, 64, "bf16")
    v[:32] *= 1e-6
    v[160:] *= 1e6
    c = nh.KvCache8(1, 1, 64, 64, pages=4, seqs=1, cap=256)
    c.debug_kernel(kernel)
    s = c.new_seq()
    q = rows_of(rng, n, 1, 64, "bf16")
    hk, hv = (ref.quantize(plain(x), (n - last,)) for x in (k, v))
    o, _ = ref.attend(plain(q), hk, hv, 0.125)
    for a, z in ((0, n - last), (n - last, n)):
        c.extend([s], [z - a])
        c.append(0, k[a:z].cuda(), v[a:z].cuda())
        got = plain(c.attend(0, q[a:z].cuda())).astype(np.float64)
        tile = 256 if kernel == 2 else 16
        for r in range(a, z):
            end = min(a + ((r - a) // tile + 1) * tile, z)  # of the row's tile
            steps = np.abs(hv[:end]).max() / 127
            limit = ref.attend_bound(plain(q), hk[:r + 1], hv[:r + 1], o[r], 0.125, "bf16", True)
            assert (np.abs(got[r - a] - o[r]) <= limit + 127 * steps * 2.0 ** -(60 if kernel == 2 else 40)).all(), r
