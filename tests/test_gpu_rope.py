"""Rotary positions on the GPU against plain numpy in 80 bits."""
import numpy as np
import pytest
import torch

import rope_ref as ref

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def plain(t):
    return t.float().cpu().numpy()


def rows_of(rng, n, heads, dim, dtype):
    return torch.from_numpy(rng.standard_normal((n, heads, dim)).astype(np.float32)).to(T[dtype]).cuda()


def bound(x, want, plan, dtype):
    """Cosine and sine are off by half a step of at most the amplitude, the products and the sum round once each, and
    the result to its type: (1/2 + 1 + 1 + ..) steps of |xa| + |xb|, held to 4 half steps of f32."""
    a, b = ref.halves(plan.dim, plan.layout)
    size = np.zeros(x.shape)
    size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return 4 * 2.0 ** -24 * abs(plan.amplitude) * size + HALF[dtype] * np.abs(want.astype(np.float64)) * 1.001 + 1e-30


def check(got, x, positions, plan, dtype, transposed=False):
    x = plain(x)
    want = ref.turn(x, positions, plan.freqs, plan.amplitude, plan.layout, transposed)
    off = np.abs(plain(got).astype(ref.LD) - want).astype(np.float64)
    tail = x[..., plan.dim:]
    assert np.array_equal(plain(got)[..., plan.dim:], tail), "dims that do not turn"
    # (f16: a result below its smallest normal number is off by half its smallest step)
    least = 2.0 ** -25 if dtype == "f16" else 0.0
    assert (off <= bound(x, want, plan, dtype) + least).all(), off.max()


SHAPES = [(1, 1, 0, 2, 2), (8, 12, 2, 48, 48), (5, 3, 1, 45, 44), (7, 4, 4, 64, 32), (33, 8, 2, 128, 128), (3, 2, 2, 96, 24),
          (2, 40, 8, 256, 256), (300, 5, 1, 51, 2), (19, 1, 1, 80, 80), (4, 7, 3, 300, 64)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,heads,kv,dim,turned", SHAPES)
def test_rows_turn(nh, rows, heads, kv, dim, turned, layout, dtype):
    rng = np.random.default_rng(rows * 100 + dim)
    plan = nh.Rope(turned, theta=10000.0, layout=layout, scaling=("parts", 8.0, 8192.0) if rows % 2 else None)
    positions = rng.integers(0, 9000, rows).astype(np.int32)
    pos = torch.from_numpy(positions).cuda()
    q, k = rows_of(rng, rows, heads, dim, dtype), rows_of(rng, rows, max(kv, 1), dim, dtype)
    for back in (False, True):
        if kv:
            got = plan.apply(pos, q, k, transposed=back)
            check(got[1], k, positions, plan, dtype, back)
        else:
            got = (plan.apply(pos, q, transposed=back),)
        check(got[0], q, positions, plan, dtype, back)
        # in place: the same numbers
        mine = q.clone()
        assert plan.apply(pos, mine, out=mine, transposed=back) is mine
        assert torch.equal(mine, got[0])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_and_negative_positions(nh, layout):
    rng = np.random.default_rng(11)
    positions = np.array([0, 1, -1, -5, 10 ** 6, 999983, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, -123456789], np.int32)
    plan = nh.Rope(128, theta=500000.0, layout=layout, scaling=("bands", 8.0, 8192.0))
    x = rows_of(rng, len(positions), 3, 128, "f32")
    got = plan.apply(torch.from_numpy(positions).cuda(), x)
    # the angle is off by 2^-65 of a turn a position more: at most 2^-34 turns, 2^-31 of the values
    want = ref.turn(plain(x), positions, plan.freqs, 1.0, layout)
    off = np.abs(plain(got).astype(ref.LD) - want).astype(np.float64)
    assert (off <= bound(plain(x), want, plan, "f32") + 2.0 ** -30 * np.abs(plain(x)).max()).all(), off.max()


def test_f32_rows_are_the_rules_numbers(nh):
    """Cosines rounded to f32, then one rounding a product and a sum: the numbers themselves."""
    rng = np.random.default_rng(12)
    positions = rng.integers(0, 100000, 500).astype(np.int32)
    plan = nh.Rope(64, scaling=("parts", 4.0, 4096.0))
    x = rows_of(rng, 500, 2, 64, "f32")
    got = plain(plan.apply(torch.from_numpy(positions).cuda(), x))
    want = ref.turn32(plain(x), positions, plan.freqs, plan.amplitude)
    # a cosine within 2^-20 of its half step may round the other way: 32,000 cosines and sines, two numbers each
    assert (got != want).sum() <= 8


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("turned", [6, 8])
def test_transposed_is_the_gradient(nh, layout, turned):
    """The rotation's matrix from unit rows; the gradient by it, and by differences of the rotation itself."""
    plan = nh.Rope(turned, theta=100.0, layout=layout, scaling=("parts", 8.0, 64.0, 0.5, 3.0))
    dim, pos = 9, torch.full((9,), 37, dtype=torch.int32, device="cuda")
    eye = torch.eye(dim, device="cuda").view(dim, 1, dim)
    m = plan.apply(pos, eye)[:, 0].double()      # row i: what unit vector i becomes
    g = torch.randn(dim, 1, dim, generator=torch.Generator().manual_seed(3)).cuda()
    got = plan.apply(pos, g, transposed=True)[:, 0].double()
    want = g[:, 0].double() @ m.t()
    # (the matrix's entries are rounded to f32, as are the gradient's products and sums)
    assert (got - want).abs().max() <= 4 * 2.0 ** -24 * plan.amplitude * 2 * g.abs().max()
    x = torch.randn(dim, 1, dim, generator=torch.Generator().manual_seed(4)).cuda()
    step = 2.0 ** -3
    for d in range(dim):
        e = torch.zeros_like(x)
        e[..., d] = step
        up, down = (plan.apply(pos, x + w * e).double() for w in (1, -1))
        slope = ((up - down) * g.double()).sum(-1)[:, 0] / (2 * step)
        # each of the difference's 2 dim numbers is off by a few roundings of values below 8, over 2 step
        assert (slope - got[:, d]).abs().max() <= dim * 8 * 2.0 ** -22 * g.abs().max() / step


def test_rows_of_a_wider_matrix(nh):
    """q and k as columns of a fused product's rows, turned in place: their neighbours stay."""
    rng = np.random.default_rng(5)
    y = torch.from_numpy(rng.standard_normal((7, 577 + 576 + 96 + 64)).astype(np.float32)).cuda()
    was = y.clone()
    q, k = y[:, 577:577 + 576].view(7, 12, 48), y[:, 1153:1249].view(7, 2, 48)
    positions = np.arange(7, dtype=np.int32) + 40
    pos = torch.from_numpy(positions).cuda()
    plan = nh.Rope(48)
    a, b = plan.apply(pos, q.contiguous(), k.contiguous())
    plan.apply(pos, q, k, out=(q, k))
    assert torch.equal(q, a) and torch.equal(k, b)
    assert torch.equal(y[:, :577], was[:, :577]) and torch.equal(y[:, 1249:], was[:, 1249:])
    # one in place, the other apart
    q2, k2 = a.clone(), b.clone()
    o = torch.full_like(k2, 3.0)
    plan.apply(pos, q2, k2, out=(q2, o), transposed=True)
    assert torch.equal(k2, b)
    check(q2, a, positions, plan, "f32", True)
    check(o, b, positions, plan, "f32", True)


def test_values_that_are_not_finite_stay_in_their_pair(nh):
    plan = nh.Rope(8, layout="half")
    x = torch.ones(3, 2, 10, device="cuda")
    x[1, 0, 2], x[2, 1, 9] = float("nan"), float("inf")
    y = plan.apply(torch.arange(3, dtype=torch.int32, device="cuda"), x)
    bad = ~torch.isfinite(y)
    assert bad[1, 0, 2] and bad[1, 0, 6] and bad[2, 1, 9] and int(bad.sum()) == 3


def test_other_stream_and_graph(nh):
    rng = np.random.default_rng(8)
    plan = nh.Rope(64)
    q, k = rows_of(rng, 9, 4, 64, "bf16"), rows_of(rng, 9, 2, 64, "bf16")
    pos = torch.arange(9, dtype=torch.int32, device="cuda")
    want = plan.apply(pos, q, k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = plan.apply(pos, q, k, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out = (torch.empty_like(q), torch.empty_like(k))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.apply(pos, q, k, out=out)
    for shift in (0, 5, 1000):
        pos.copy_(torch.arange(9, dtype=torch.int32) + shift)
        want = plan.apply(pos, q, k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), shift


def test_no_rows(nh):
    plan = nh.Rope(64)
    pos = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert plan.apply(pos, torch.zeros(0, 4, 64, device="cuda")).shape == (0, 4, 64)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert plan.apply(one, torch.zeros(1, 0, 64, device="cuda")).shape == (1, 0, 64)


def test_refusals(nh):
    plan = nh.Rope(64)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.zeros(4, 2, 64, device="cuda")
    for bad in (dict(q=x[:3]), dict(q=x.double()), dict(q=x.cpu()), dict(q=x.transpose(0, 1)), dict(q=x[0]),
                dict(q=torch.zeros(4, 64, 2, device="cuda").transpose(1, 2)), dict(q=x, k=x.half()),
                dict(q=x, k=torch.zeros(4, 2, 48, device="cuda")), dict(q=x, out=x.half()), dict(q=x, k=x, out=x[:1]),
                dict(q=x, out=torch.zeros(4, 3, 64, device="cuda")), dict(positions=pos.long(), q=x),
                dict(positions=pos[:3], q=x), dict(positions=pos.cpu(), q=x)):
        with pytest.raises(ValueError):
            plan.apply(**{"positions": pos, **bad})
    for bad in (dict(q=torch.zeros(4, 2, 62, device="cuda")), dict(q=x[:1].expand(4, 2, 64)),
                dict(q=x, out=torch.zeros(1, 2, 64, device="cuda").expand(4, 2, 64))):
        with pytest.raises(nh.NeedleHipError):
            plan.apply(**{"positions": pos, **bad})
    # rows in place whose outputs would lie elsewhere in the same memory
    wide = torch.zeros(4, 256, device="cuda")
    with pytest.raises(nh.NeedleHipError):
        plan.apply(pos, wide[:, :128].view(4, 2, 64), out=wide.view(-1)[:512].view(4, 2, 64))
