"""Attention over keys and values of very different size: what a row does not see, and groups far larger than others,
must not coarsen what it does see.  With a window of one position the output is the row's own value and the log-sum its
own score, so both are held to the rounding of one key."""
import numpy as np
import pytest
import torch

import kv4_ref as ref
from test_gpu_kv4 import T, plain, rows_of

pytestmark = pytest.mark.gpu

H = 2.0 ** -11  # half a step of 11 bits


def ranges(x, group):
    """15 steps of each value's group (what step x code reaches) and the group's largest size, as rows have them."""
    r, big = np.zeros(x.shape), np.zeros(x.shape)
    for a in range(0, x.shape[-1], group):
        y = x[..., a:a + group]
        step = ((y.max(-1) - y.min(-1)).astype(np.float32) * ref.THIRD).astype(np.float16).astype(np.float64)
        r[..., a:a + group] = 15 * step[..., None]
        big[..., a:a + group] = np.abs(y).max(-1)[..., None]
    return r, big


def build(nh, k, v, group, kernel):
    n, kv, d = k.shape
    c = nh.KvCache4(1, kv, d, v.shape[-1], pages=-(-n // 64), seqs=1, cap=n, group=group)
    c.debug_kernel(kernel)
    s = c.new_seq()
    c.extend([s], [n])
    c.append(0, k.cuda(), v.cuda())
    return c


def check_own(nh, k, v, q, group, dtype, kernel):
    """A window of one: out = v_i to its roundings, lse = scale q . k_i to its own."""
    n, kv, d = k.shape
    c = build(nh, k, v, group, kernel)
    lse = torch.empty((n, kv), device="cuda")
    out = plain(c.attend(0, q.cuda(), ring=1, lse=lse)).astype(np.float64)
    kk, vv = (ref.quantize(plain(x), group) for x in (k, v))
    kr, kbig = ranges(plain(k), group)
    vr, _ = ranges(plain(v), group)
    # step x code to 11 bits (below 2^-20 of the call's largest step: to 2^-26 of that), the weight of the low
    # and of the sum it is divided by alike (both the same rounded number), the output's rounding
    bound = ref.half_step(dtype) * np.abs(vv) + H * vr + 2.0 ** -26 * vr.max() / 15 + 2.0 ** -20 * np.abs(vv) + 1e-30
    bad = np.abs(out - vv) > bound
    assert not bad.any(), (np.argwhere(bad)[:4].tolist(), float((np.abs(out - vv) / bound).max()))
    x = plain(q).astype(np.float64)
    want = (x * kk).sum(-1) * d ** -0.5
    size, most = np.abs(x), np.abs(x).max(-1, keepdims=True)
    # of the score: each dim's step x code as above, a query's element to 2^-20 of the row's largest, the lows' sums
    # to 22 bits, each product cut off at 2^-20 of its largest term (measured; a lows' term is up to a group's sum),
    # f32 sums; of the log-sum: its own weight to 11 bits, f32 arithmetic
    off = (size * (H * kr + 2.0 ** -26 * kr.max() / 15)).sum(-1) + 2.0 ** -20 * (most * kr).sum(-1)
    off += 2.0 ** -22 * (size * kbig).sum(-1) + (d / 16 + 2) * 2.0 ** -20 * (most[..., 0] * kr.max(-1) + (size * kbig).sum(-1))
    off = (off + (d + 16) * 2.0 ** -24 * (size * np.abs(kk)).sum(-1)) * d ** -0.5 + H + 2.0 ** -21 * np.abs(want) + 2.0 ** -20
    got = plain(lse).astype(np.float64)
    bad = np.abs(got - want) > off
    assert not bad.any(), (np.argwhere(bad)[:4].tolist(), float((np.abs(got - want) / off).max()))
    return c


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (51, 32), (128, 32)])
@pytest.mark.parametrize("base,factor", [(1.0, 300.0), (1.0, 1e4), (0.3, 6e4), (1e-3, 2e4), (300.0, 50.0)])
def test_one_large_row(nh, base, factor, d, group, dtype, kernel):
    """One key and one value, a later one among the tile's rows, `factor` times the others."""
    rng = np.random.default_rng(d + group)
    n = 300
    k, v, q = (rows_of(rng, n, 2, d, "f32", spread) for spread in (base, base, min(1.0, 1.0 / base)))
    for x, at in ((k, 77), (v, 120)):
        x[at] = (x[at] * factor).clamp(-6e4, 6e4)
    check_own(nh, *(x.to(T[dtype]) for x in (k, v, q)), group, dtype, kernel)


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_one_large_group(nh, dtype, kernel):
    """Channels of one group 10,000 times the others in every row: the others keep their own bits."""
    rng = np.random.default_rng(5)
    k, v, q = (rows_of(rng, 280, 2, 128, "f32") for _ in range(3))
    k[..., 32:64] *= 2000.0
    q[..., 32:64] /= 2000.0
    v[..., 96:] *= 10000.0
    check_own(nh, *(x.clamp(-6e4, 6e4).to(T[dtype]) for x in (k, v, q)), 32, dtype, kernel)


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("spread", [1e-7, 1e-5, 1e-2, 2e4])
def test_keys_and_values_of_any_size(nh, spread, kernel):
    """All of a size, from f16's subnormals to its end (bf16 rows), the queries the inverse of it."""
    rng = np.random.default_rng(6)
    k, v, q = (rows_of(rng, 270, 1, 64, "bf16", s) for s in (spread, spread, 1.0 / spread))
    check_own(nh, k, v, q, 32, "bf16", kernel)


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_large_row_out_of_the_window(nh, dtype, kernel):
    """Even weights (queries of zero) over a window: the mean of its values, to a value's roundings, where the window
    does not hold the large one; one range of keys and several."""
    rng = np.random.default_rng(7)
    for n, rows in ((320, 320), (5000, 16)):
        k, v = rows_of(rng, n, 1, 64, "f32"), rows_of(rng, n, 1, 64, "f32")
        v[n - 200] *= 15000.0
        k[n - 201] *= 15000.0
        k, v = (x.clamp(-6e4, 6e4).to(T[dtype]) for x in (k, v))
        c = nh.KvCache4(1, 1, 64, 64, pages=-(-n // 64), seqs=1, cap=n)
        c.debug_kernel(kernel)
        s = c.new_seq()
        for a, e in ((0, n - rows), (n - rows, n)):
            c.extend([s], [e - a])
            c.append(0, k[a:e].cuda(), v[a:e].cuda())
        ring = 60 if n == 320 else 150
        out = plain(c.attend(0, torch.zeros((rows, 2, 64), dtype=T[dtype], device="cuda"), ring=ring)).astype(np.float64)
        vv = ref.quantize(plain(v), 32)[:, 0]
        vr = ranges(plain(v), 32)[0][:, 0]
        for r in range(rows):
            i = n - rows + r
            seen = slice(max(0, i - ring + 1), i + 1)
            want, size = vv[seen].mean(0), np.abs(vv[seen]).mean(0)
            bound = ref.half_step(dtype) * np.abs(want) + H * vr[seen].mean(0) + 2.0 ** -26 * vr.max() / 15
            bound = bound + (ring + 64) * 2.0 ** -23 * size
            assert np.all(np.abs(out[r] - want) <= bound), (n, r, float((np.abs(out[r] - want) / bound).max()))
