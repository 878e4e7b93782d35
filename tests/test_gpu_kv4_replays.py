"""Captured steps of the 4-bit cache replayed when the cache holds another batch: nothing is read or written."""
import numpy as np
import pytest
import torch

from test_gpu_kv4 import filled, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("was,now", [([4], [4, 4]), ([4], [4, 0]), ([4, 4], [4]), ([4, 4], [8]), ([3, 3], [2, 4]),
                                     ([2, 4], [3, 3]), ([2, 4], [4, 2]), ([5, 1, 2], [5, 1]), ([4], [3])])
def test_a_replay_of_another_shape_touches_nothing(nh, was, now, kernel):
    """A step captured for the rows `was`, replayed after an extend of `now`: as many rows in all, or the same rows of the
    first sequences, among them."""
    rng = np.random.default_rng(7)
    c, ids, _, _ = filled(nh, rng, [40, 33, 70], 2, 64, 64, 32, 32, "bf16", extra_pages=12)
    c.debug_kernel(kernel)
    n = sum(was)
    x, q = rows_of(rng, n, 2, 64, "bf16").cuda(), rows_of(rng, n, 4, 64, "bf16").cuda()
    out = torch.zeros(n, 4, 64, device="cuda", dtype=torch.bfloat16)
    a = ids[:len(was)]
    c.extend(a, was)
    c.append(0, x, x)
    c.attend(0, q, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(0, x, x)
        c.attend(0, q, out=out)
    b = ids[::-1][:len(now)]
    c.extend(b, now)
    m = sum(now)
    y = rows_of(rng, m, 2, 64, "bf16").cuda()
    c.append(0, y, y)
    before = c.read(0, ids, [0] * 3, [c.length(s) for s in ids])
    for _ in range(2):
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert bool((out == 3.0).all())
        for s, t in zip(before, c.read(0, ids, [0] * 3, [c.length(s) for s in ids])):
            assert torch.equal(s, t)
    # the same rows again, of other sequences: the replay is the eager step
    c.extend(b[:1] + [s for s in ids if s != b[0]][:len(was) - 1], was)
    out.fill_(3.0)
    g.replay()
    torch.cuda.synchronize()
    got = out.clone()
    c.append(0, x, x)
    c.attend(0, q, out=out)
    assert torch.allclose(got.float(), out.float(), rtol=2.0 ** -7, atol=2.0 ** -8 * float(x.float().abs().max()))


def test_a_replay_after_the_batch_is_over_touches_nothing(nh):
    """A compaction, a cut and a freed sequence end the batch; what is dealt afterwards stays as it is."""
    rng = np.random.default_rng(8)
    c, ids, _, _ = filled(nh, rng, [64, 50, 40], 1, 64, 64, 32, 32, "bf16", extra_pages=8)
    x, q = rows_of(rng, 2, 1, 64, "bf16").cuda(), rows_of(rng, 2, 2, 64, "bf16").cuda()
    out = torch.zeros(2, 2, 64, device="cuda", dtype=torch.bfloat16)

    def step():
        c.extend(ids[:2], [1, 1])
        c.append(0, x, x)
    step()
    c.attend(0, q, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(0, x, x)
        c.attend(0, q, out=out)
    for change in ("compact", "truncate and copy", "extend another"):
        if change == "compact":
            step()
            c.compact([ids[0]], [[(0, 20), (40, 60)]])
        elif change == "truncate and copy":
            step()
            c.truncate(ids[0], 10)
            c.free(c.copy(ids[2]))
        else:
            step()
            c.extend([ids[2]], [1])
            c.append(0, x[:1], x[:1])
        before = c.read(0, ids, [0] * 3, [c.length(s) for s in ids])
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert bool((out == 3.0).all()), change
        for s, t in zip(before, c.read(0, ids, [0] * 3, [c.length(s) for s in ids])):
            assert torch.equal(s, t), change
