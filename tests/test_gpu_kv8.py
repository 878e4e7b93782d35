"""The 8-bit key/value cache on the GPU: what it holds, its pages, keys turned on
the way in, and its attention, against plain numpy in 64 bits."""
import random

import numpy as np
import pytest
import torch

import kv8_ref as ref
import rope_ref

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EINVAL, ESMALL, ENOMEM = -1, -2, -4


def rows_of(rng, n, heads, dim, dtype, spread=1.0):
    """Rows as projections give them: channels of different size and offset, as the type holds them."""
    x = rng.standard_normal((n, heads, dim)) * np.exp(0.5 * rng.standard_normal(dim)) + 0.5 * rng.standard_normal(dim)
    return torch.from_numpy((x * spread).astype(np.float32)).to(T[dtype])


def plain(t):
    return t.float().cpu().numpy()


def typed(x, dtype):
    return plain(torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(T[dtype]))


def filled(nh, rng, lens, kv, qk, v, page, dtype, layers=1, extra_pages=0, last=None, seqs=None):
    """A cache whose sequences hold `lens` rows, the last `last[i]` as the batch: (cache, ids, k, v held, [layer][sequence])."""
    pages = sum(-(-n // page) for n in lens) + extra_pages
    c = nh.KvCache8(layers, kv, qk, v, pages=max(pages, 1), seqs=seqs or len(lens) + 8, cap=max(max(lens), 1) + 64, page=page)
    ids = [c.new_seq() for _ in lens]
    last = last or [0] * len(lens)
    ks = [[rows_of(rng, n, kv, qk, dtype) for n in lens] for _ in range(layers)]
    vs = [[rows_of(rng, n, kv, v, dtype) for n in lens] for _ in range(layers)]
    cuts = [n - r for n, r in zip(lens, last)]
    for a, z in (([0] * len(lens), cuts), (cuts, list(lens))):
        c.extend(ids, [e - b for b, e in zip(a, z)])
        for layer in range(layers):
            c.append(layer, torch.cat([x[b:e] for x, b, e in zip(ks[layer], a, z)]).cuda(),
                     torch.cat([x[b:e] for x, b, e in zip(vs[layer], a, z)]).cuda())
    held = [[[ref.quantize(plain(x), (cut,)) for x, cut in zip(side[layer], cuts)] for layer in range(layers)] for side in (ks, vs)]
    return c, ids, *held


SHAPES = [(2, 48, 64, 64), (1, 64, 64, 128), (3, 45, 51, 64), (8, 128, 128, 64), (5, 80, 96, 64), (2, 256, 256, 64),
          (1, 200, 129, 256), (4, 1, 3, 64), (2, 192, 128, 128), (2, 64, 128, 64)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,qk,v,page", SHAPES)
def test_rows_hold_the_formats_values(nh, kv, qk, v, page, dtype):
    rng = np.random.default_rng(qk * 7 + v)
    lens = [1, 70, page, 0, 2 * page + 1]
    c, ids, ks, vs = filled(nh, rng, lens, kv, qk, v, page, dtype, layers=2, last=[1, 3, 0, 0, page + 5])
    for layer in (0, 1):
        k, w = c.read(layer, ids, [0] * 5, lens)
        # f32 rounds code x step once, as numpy does
        assert np.array_equal(plain(k), np.concatenate(ks[layer]))
        assert np.array_equal(plain(w), np.concatenate(vs[layer]))
    k, w = c.read(None, [ids[4], ids[1]], [page - 1, 5], [3, 60], T[dtype])
    assert k.shape == (2, 63, kv, qk) and k.dtype == T[dtype]
    for layer in (0, 1):
        for got, want in ((k, ks), (w, vs)):
            want = np.concatenate([want[layer][4][page - 1:page + 2], want[layer][1][5:65]])
            assert np.array_equal(plain(got[layer]), typed(want, dtype))


def test_values_at_the_borders(nh):
    """Zeros, tiny and huge values; a row with a NaN or an infinity reads as NaN and leaves its block alone."""
    d = 96
    rng = np.random.default_rng(3)
    x = np.zeros((7 * 16, 2, d), np.float32)
    x[16:32] = rng.standard_normal((16, 2, d)) * 1e-38       # below the smallest step: zeros
    x[32:48] = rng.standard_normal((16, 2, d)) * 1e-33
    x[48:64] = rng.standard_normal((16, 2, d)).clip(-3, 3) * 1e38
    x[64:96] = rng.standard_normal((32, 2, d))
    x[64 + 3, 0, 40], x[64 + 4, 1, 95], x[80, 0, 0] = np.nan, np.inf, -np.inf
    x[96:] = -0.0
    c = nh.KvCache8(1, 2, d, d, pages=2, seqs=1, cap=128)
    s = c.new_seq()
    c.extend([s], [len(x)])
    t = torch.from_numpy(x).cuda()
    c.append(0, t, t)
    k, v = c.read(0, [s], [0], [len(x)])
    want = ref.quantize(x)
    assert np.isnan(want).sum() == 3 * d and (want[16:32] == 0).all() and np.isfinite(want[48:64]).all()
    assert np.array_equal(plain(k), want, equal_nan=True)
    assert np.array_equal(plain(v), want, equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_steps_grow_as_rows_join(nh, dim, dtype):
    """Rows one at a time, each some times larger or smaller than the last, zeros, marked rows; cut back and stored anew."""
    rng, pick = np.random.default_rng(dim), random.Random(dim)
    c = nh.KvCache8(1, 2, dim, dim, pages=2, seqs=1, cap=128)
    s = c.new_seq()
    sides = [ref.Side(2, dim), ref.Side(2, dim)]
    for step in range(150):
        n = len(sides[0].codes)
        if n > 100 or (n and pick.random() < 0.12):
            n = pick.randrange(n)
            c.truncate(s, n)
            for side in sides:
                side.cut(n)
        rows = pick.choice((1, 1, 1, 2, 5, 17))
        c.extend([s], [rows])
        size = pick.choice((0.0, 1e-3, 0.5, 1.0, 1.99, 2.0, 2.01, 7.0, 300.0, 1e6))
        k, v = (rows_of(rng, rows, 2, dim, dtype, size) for _ in range(2))
        if pick.random() < 0.1:
            k[pick.randrange(rows), 0, 3] = float("nan")
            v[pick.randrange(rows), 1, dim - 1] = float("-inf")
        c.append(0, k.cuda(), v.cuda())
        for side, x in zip(sides, (k, v)):
            side.store(plain(x))
        got = c.read(0, [s], [0], [len(sides[0].codes)])
        for side, x in zip(sides, got):
            assert np.array_equal(plain(x), side.held32(), equal_nan=True), step


def test_appending_the_same_rows_again_changes_nothing(nh):
    rng = np.random.default_rng(4)
    c = nh.KvCache8(1, 2, 48, 64, pages=2, seqs=1, cap=100)
    s = c.new_seq()
    c.extend([s], [5])
    c.append(0, rows_of(rng, 5, 2, 48, "f32", 0.1).cuda(), rows_of(rng, 5, 2, 64, "f32", 0.1).cuda())
    c.extend([s], [20])
    k, v = rows_of(rng, 20, 2, 48, "f32", 3.0).cuda(), rows_of(rng, 20, 2, 64, "f32", 3.0).cuda()
    c.append(0, k, v)
    was = c.read(0, [s], [0], [25])
    c.append(0, k, v)
    now = c.read(0, [s], [0], [25])
    assert torch.equal(was[0], now[0]) and torch.equal(was[1], now[1])


@pytest.mark.parametrize("seed", range(3))
def test_pages_in_random_order(nh, seed):
    """Forks, copies and cuts in random order; every sequence reads as the lists have it."""
    rng, pick = np.random.default_rng(seed), random.Random(seed)
    layers, kv, qk, v, page = 2, 2, (48, 128, 70)[seed], (64, 96, 200)[seed], 64
    c = nh.KvCache8(layers, kv, qk, v, pages=30, seqs=7, cap=500, page=page)
    model = {}

    def check():
        live = sorted(model)
        lens = [len(model[s][0].codes) for s in live]
        k, w = c.read(None, live, [0] * len(live), lens)
        at = 0
        for s, n in zip(live, lens):
            assert c.length(s) == n
            for layer in range(layers):
                for got, side in ((k, model[s][2 * layer]), (w, model[s][2 * layer + 1])):
                    assert np.array_equal(plain(got[layer, at:at + n]), side.held32()), (s, n)
            at += n
    for _ in range(70):
        op = pick.choice(("new", "free", "fork", "copy", "cut", "extend", "extend", "extend", "extend"))
        live = sorted(model)
        try:
            if op == "new":
                model[c.new_seq()] = [ref.Side(kv, d) for _ in range(layers) for d in (qk, v)]
            elif not live:
                continue
            elif op == "free":
                s = pick.choice(live)
                c.free(s)
                del model[s]
            elif op == "fork":
                s = pick.choice(live)
                for made in c.fork(s, pick.randrange(3)):
                    model[made] = [x.fork() for x in model[s]]
            elif op == "copy":
                s = pick.choice(live)
                model[c.copy(s)] = [x.fork() for x in model[s]]
            elif op == "cut":
                s = pick.choice(live)
                n = pick.randrange(len(model[s][0].codes) + 1)
                c.truncate(s, n)
                for x in model[s]:
                    x.cut(n)
            else:
                some = pick.sample(live, pick.randrange(1, len(live) + 1))
                rows = [pick.choice((0, 1, 1, 2, 7, 40)) for _ in some]
                c.extend(some, rows)
                for layer in range(layers):
                    ks, vs = ([rows_of(rng, r, kv, d, "f32", pick.choice((0.2, 1.0, 5.0))) for r in rows] for d in (qk, v))
                    c.append(layer, torch.cat(ks).cuda(), torch.cat(vs).cuda())
                    for s, k, w in zip(some, ks, vs):
                        model[s][2 * layer].store(plain(k))
                        model[s][2 * layer + 1].store(plain(w))
        except nh.NeedleHipError as e:
            assert e.code in (ENOMEM, EINVAL), e
        check()


# ------------------------------------------------------------------ turned
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("qk,v,turned,heads", [(48, 64, 48, 12), (128, 128, 128, 4), (128, 64, 24, 2), (45, 51, 44, 3), (256, 256, 256, 2),
                                               (192, 128, 64, 2), (80, 80, 6, 1), (2, 2, 2, 5)])
def test_keys_and_queries_turned(nh, qk, v, turned, heads, layout, dtype):
    rng = np.random.default_rng(qk + turned)
    kv, lens, last = 1 + heads % 2, [70, 1, 133, 0], [3, 1, 130, 0]
    plan = nh.Rope(turned, layout=layout, scaling=("bands", 4.0, 64.0))
    c = nh.KvCache8(1, kv, qk, v, pages=8, seqs=4, cap=200)
    ids = [c.new_seq() for _ in lens]
    ks, vs = ([rows_of(rng, n, kv, d, dtype) for n in lens] for d in (qk, v))
    cuts = [n - r for n, r in zip(lens, last)]
    for a, z in (([0] * 4, cuts), (cuts, lens)):
        rows = [e - b for b, e in zip(a, z)]
        c.extend(ids, rows)
        q = rows_of(rng, sum(rows), heads, qk, dtype).cuda()
        k, w = (torch.cat([x[b:e] for x, b, e in zip(side, a, z)]).cuda() for side in (ks, vs))
        got = c.append(0, k, w, rope=plan, q=q)
        pos = torch.from_numpy(np.concatenate([np.arange(b, e) for b, e in zip(a, z)]).astype(np.int32)).cuda()
        assert torch.equal(got, plan.apply(pos, q)), "queries as the rotation alone turns them"
        mine = q.clone()
        assert c.append(0, k, w, rope=plan, q=mine, out=mine) is mine and torch.equal(mine, got)
    k, w = c.read(0, ids, [0] * 4, lens)
    want = [rope_ref.turn32(plain(x), np.arange(len(x)), plan.freqs, plan.amplitude, layout) for x in ks]
    want = np.concatenate([ref.quantize(x, (cut,)) for x, cut in zip(want, cuts)])
    # a cosine that rounds the other way (one in 2^20) moves a key by 2^-24 of it, and its code only beside a border
    assert (plain(k) != want).sum() <= 1
    assert np.array_equal(plain(w), np.concatenate([ref.quantize(plain(x), (cut,)) for x, cut in zip(vs, cuts)]))


def test_keys_turned_to_given_positions(nh):
    rng = np.random.default_rng(9)
    plan = nh.Rope(64)
    c = nh.KvCache8(1, 2, 64, 64, pages=2, seqs=2, cap=64)
    ids = [c.new_seq(), c.new_seq()]
    c.extend(ids, [5, 9])
    x = rows_of(rng, 14, 2, 64, "f32")
    q = rows_of(rng, 14, 4, 64, "f32").cuda()
    positions = rng.integers(-100, 5000, 14).astype(np.int32)
    pos = torch.from_numpy(positions).cuda()
    got = c.append(0, x.cuda(), x.cuda(), rope=plan, positions=pos, q=q)
    assert torch.equal(got, plan.apply(pos, q))
    k, _ = c.read(0, ids, [0, 0], [5, 9])
    turned = rope_ref.turn32(plain(x), positions, plan.freqs)
    assert np.array_equal(plain(k), np.concatenate([ref.quantize(turned[:5]), ref.quantize(turned[5:])]))
    # keys alone
    assert c.append(0, x.cuda(), x.cuda(), rope=plan, positions=pos) is None
    assert torch.equal(c.read(0, ids, [0, 0], [5, 9])[0], k)


def test_rows_of_a_wider_matrix(nh):
    """k, v and q as columns of the fused projection's rows, at an odd offset; the output's neighbours stay."""
    rng = np.random.default_rng(5)
    y = torch.from_numpy(rng.standard_normal((7, 577 + 96 + 128 + 768)).astype(np.float32)).cuda()
    k, v, q = y[:, 577:673].view(7, 2, 48), y[:, 673:801].view(7, 2, 64), y[:, :576].view(7, 12, 48)
    c = nh.KvCache8(1, 2, 48, 64, pages=2, seqs=2, cap=64)
    s = [c.new_seq(), c.new_seq()]
    c.extend(s, [3, 4])
    plan, was = nh.Rope(48), y.clone()
    turned = c.append(0, k, v, rope=plan, q=q, out=q)
    assert torch.equal(y[:, 576:], was[:, 576:])
    pos = torch.tensor([0, 1, 2, 0, 1, 2, 3], dtype=torch.int32, device="cuda")
    assert torch.equal(turned, plan.apply(pos, was[:, :576].contiguous().view(7, 12, 48)))
    b = c.read(0, s, [0, 0], [3, 4])[1]
    assert np.array_equal(plain(b), np.concatenate([ref.quantize(plain(v[:3])), ref.quantize(plain(v[3:]))]))
    out = torch.full((7, 2, 12 * 64), 7.0, device="cuda")
    o = out[:, 1].view(7, 12, 64)
    c.attend(0, q, out=o)
    assert torch.equal(o, c.attend(0, q.contiguous()))
    assert bool((out[:, 0] == 7.0).all()), "the rows' neighbours are left as they were"


# --------------------------------------------------------------- attention
def check_attend(c, layer, q, ks, vs, rows, dtype, sink=0, ring=0, ask=False, kernel=0, scale=None, many=False):
    """attend of the batch against 64 bits, lse too; ks, vs: the sequences' held keys and values."""
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
    out = c.attend(layer, q.cuda(), scale=scale, sink=sink, ring=ring, lse=lse)
    assert torch.equal(out, c.attend(layer, q.cuda(), scale=scale, sink=sink, ring=ring)) or bool(torch.isnan(out).any())
    at = 0
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    for n, k, v in zip(rows, ks, vs):
        if not n:
            continue
        x = plain(q[at:at + n])
        o, l = ref.attend(x, k, v, scale, sink, ring, ask)
        got, gl = plain(out[at:at + n]).astype(np.float64), plain(lse[at:at + n])
        nan = np.isnan(o)
        assert np.array_equal(np.isnan(got), nan)
        limit = ref.attend_bound(x, k, v, np.nan_to_num(o), scale, dtype, many)
        off = np.abs(np.where(nan, 0, got - np.nan_to_num(o)))
        assert (off <= limit).all(), (off.max(), limit.min(), len(k))
        fine = np.isfinite(l)
        assert np.array_equal(np.isneginf(gl), np.isneginf(l))
        if fine.any():
            # the scores' error, and f32 roundings of a logarithm and of a sum a key long
            vmax = max(np.abs(np.nan_to_num(v)).max(), 1e-30)
            assert np.abs(gl - l)[fine].max() <= limit.max() / vmax + 2.0 ** -22 * (np.abs(l[fine]).max() + 1) + 2.0 ** -20
        at += n


ATTEND = [  # kv heads, query heads, dims, lengths, rows
    (2, 12, 48, 64, [700], [1]),
    (1, 1, 64, 64, [1], [1]),
    (3, 3, 45, 51, [65, 64, 63], [1, 64, 5]),
    (8, 32, 128, 128, [300, 17, 129], [5, 17, 2]),
    (2, 8, 192, 128, [200, 90], [3, 90]),
    (2, 4, 256, 256, [130, 40], [2, 9]),
    (1, 6, 80, 96, [500, 31], [70, 31]),
    (4, 4, 1, 3, [33, 100], [33, 1]),
    (2, 2, 64, 64, [5000], [3]),
    (1, 8, 128, 128, [3000, 2], [1, 2]),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,heads,qk,v,lens,rows", ATTEND)
def test_attention(nh, kv, heads, qk, v, lens, rows, dtype):
    rng = np.random.default_rng(qk * 3 + lens[0])
    c, ids, ks, vs = filled(nh, rng, lens, kv, qk, v, 64, dtype, layers=2, last=rows)
    q = rows_of(rng, sum(rows), heads, qk, dtype)
    for kernel in (0, 1, 2):
        c.debug_kernel(kernel)
        check_attend(c, 1, q, ks[1], vs[1], rows, dtype, kernel=kernel, many=dtype != "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sink,ring", [(0, 1), (4, 1), (118, 256), (1, 64), (1000, 3), (64, 64), (0, 130), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_attention_under_a_span(nh, sink, ring, dtype):
    rng = np.random.default_rng(sink % 1000 + ring % 1000)
    lens, rows = [700, 64, 300], [5, 64, 70]
    c, ids, ks, vs = filled(nh, rng, lens, 2, 64, 64, 64, dtype, last=rows)
    q = rows_of(rng, sum(rows), 4, 64, dtype)
    for kernel in (0, 1, 2):
        c.debug_kernel(kernel)
        check_attend(c, 0, q, ks[0], vs[0], rows, dtype, sink, ring, kernel=kernel, many=dtype != "f32")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,heads,qk,v,lens,rows", [
    (16, 16, 64, 64, [1500, 1, 0, 64, 63], [4, 4, 4, 4, 4]), (2, 4, 128, 128, [0], [3]), (1, 8, 80, 80, [129, 500], [1, 300]),
    (2, 2, 256, 192, [77, 0, 300], [0, 2, 5]), (2, 6, 48, 64, [4000], [1]), (1, 1, 64, 64, [30, 0], [500, 40])])
def test_rows_that_ask(nh, kv, heads, qk, v, lens, rows, dtype):
    """Cross attention: every row sees the whole of its sequence, whatever their numbers; none: 0 and -inf."""
    rng = np.random.default_rng(sum(lens) + qk)
    c, ids, ks, vs = filled(nh, rng, lens, kv, qk, v, 64, dtype, extra_pages=len(lens))
    c.ask(ids, rows)
    assert c.rows == sum(rows) and [c.length(s) for s in ids] == lens
    q = rows_of(rng, sum(rows), heads, qk, dtype)
    for kernel in (0, 1, 2):
        c.debug_kernel(kernel)
        for sink, ring in ((0, 0), (3, 70)):
            check_attend(c, 0, q, ks[0], vs[0], rows, dtype, sink, ring, ask=True, kernel=kernel, many=dtype != "f32")
    with pytest.raises(nh.NeedleHipError):
        c.append(0, torch.zeros(sum(rows), kv, qk, device="cuda"), torch.zeros(sum(rows), kv, v, device="cuda"))
    # back to a step of its own
    c.extend(ids, [1] * len(ids))
    c.append(0, rows_of(rng, len(ids), kv, qk, dtype).cuda(), rows_of(rng, len(ids), kv, v, dtype).cuda())
    assert [c.length(s) for s in ids] == [n + 1 for n in lens]


def test_f32_attention_beside_a_plain_f32_evaluation(nh):
    """Few and many keys: the error's norm against 64 bits is of the size of a plain f32 evaluation's."""
    rng = np.random.default_rng(21)
    for n, heads in ((20, 4), (700, 12), (6000, 4)):
        c, ids, ks, vs = filled(nh, rng, [n], 2, 64, 64, 64, "f32", last=[2])
        q = rows_of(rng, 2, heads, 64, "f32")
        want, _ = ref.attend(plain(q), ks[0][0], vs[0][0], 0.125)
        got = plain(c.attend(0, q.cuda()))
        k, v = (torch.from_numpy(np.repeat(x[0][0], heads // 2, 1)).transpose(0, 1) for x in (ks, vs))
        s = torch.matmul(q.transpose(0, 1), k.transpose(1, 2)) * 0.125
        s[:, 0, n - 1] = float("-inf")
        p = torch.exp(s - s.amax(-1, keepdim=True))
        other = plain((torch.matmul(p, v) / p.sum(-1, keepdim=True)).transpose(0, 1))
        size = np.linalg.norm(want)
        mine, plain32 = (np.linalg.norm(x - want) / size for x in (got, other))
        # f32 sums of n keys: both within a few of the other; an MFMA's cut at 2^-20 of a product, over many, 2^-21
        assert mine <= 4 * plain32 + 2.0 ** -21, (n, mine, plain32)


def test_nan_rows_spoil_their_readers_alone(nh):
    rng = np.random.default_rng(6)
    for dtype in ("f32", "bf16"):
        c = nh.KvCache8(1, 2, 64, 64, pages=12, seqs=2, cap=400)
        ids = [c.new_seq(), c.new_seq()]
        c.extend(ids, [300, 90])
        k, v = rows_of(rng, 390, 2, 64, dtype), rows_of(rng, 390, 2, 64, dtype)
        k[280, 0, 5], v[100, 1, 63], k[300 + 80, 1, 0] = float("nan"), float("inf"), float("-inf")
        c.append(0, k.cuda(), v.cuda())
        hk, hv = ([ref.quantize(plain(x[:300])), ref.quantize(plain(x[300:]))] for x in (k, v))
        q = rows_of(rng, 390, 4, 64, dtype)
        for kernel in (0, 1, 2):
            c.debug_kernel(kernel)
            for sink, ring in ((0, 0), (2, 50)):
                check_attend(c, 0, q, hk, hv, [300, 90], dtype, sink, ring, kernel=kernel, many=dtype != "f32")


def test_queries_that_are_not_finite_spoil_their_own_rows(nh):
    rng = np.random.default_rng(7)
    for dtype in ("f32", "f16", "bf16"):
        c, ids, ks, vs = filled(nh, rng, [90], 2, 64, 64, 64, dtype, last=[40])
        q = rows_of(rng, 40, 4, 64, dtype).cuda()
        want = [None] * 3
        for kernel in (0, 1, 2):
            c.debug_kernel(kernel)
            want[kernel] = c.attend(0, q)
        q[3, 1, 7], q[20, 2, 0] = float("nan"), float("inf")
        for kernel in (0, 1, 2):
            c.debug_kernel(kernel)
            got = c.attend(0, q)
            spoilt = torch.isnan(got).all(-1)
            assert spoilt[3, 1] and spoilt[20, 2] and int(spoilt.sum()) == 2
            assert torch.equal(got[~spoilt], want[kernel][~spoilt])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_values_of_very_different_size(nh, dtype):
    """Blocks of values 10^6 times the others, seen or hidden: each row's result keeps its own precision."""
    rng = np.random.default_rng(8)
    n = 200
    k, v = rows_of(rng, n, 1, 64, dtype), rows_of(rng, n, 1, 64, dtype)
    v[:32] *= 1e-6
    v[160:] *= 1e6
    c = nh.KvCache8(1, 1, 64, 64, pages=4, seqs=1, cap=256)
    s = c.new_seq()
    c.extend([s], [n])
    c.append(0, k.cuda(), v.cuda())
    hk, hv = ref.quantize(plain(k)), ref.quantize(plain(v))
    q = rows_of(rng, n, 2, 64, dtype)
    for kernel in (0, 1):
        c.debug_kernel(kernel)
        got = plain(c.attend(0, q.cuda())).astype(np.float64)
        o, _ = ref.attend(plain(q), hk, hv, 0.125)
        for r in range(0, 160):
            limit = ref.attend_bound(plain(q), hk[:r + 1], hv[:r + 1], o[r], 0.125, dtype)
            # (weights x steps finer than 2^-40 of the tile's largest step are dropped: 1e6 hidden in the row's own tile)
            assert (np.abs(got[r] - o[r]) <= limit + 2.0 ** -38 * np.abs(hv).max()).all(), (kernel, r)
    with pytest.raises(nh.NeedleHipError):
        c.debug_kernel(3)


# ------------------------------------------------- streams, graphs, refusals
def test_other_stream(nh):
    rng = np.random.default_rng(13)
    plan = nh.Rope(64)
    c, ids, ks, vs = filled(nh, rng, [100, 7], 2, 64, 64, 64, "bf16", extra_pages=2)
    d, jds, _, _ = filled(nh, np.random.default_rng(13), [100, 7], 2, 64, 64, 64, "bf16", extra_pages=2)
    k, q = rows_of(rng, 6, 2, 64, "bf16").cuda(), rows_of(rng, 6, 4, 64, "bf16").cuda()
    c.extend(ids, [2, 4])
    want = c.attend(0, c.append(0, k, k, rope=plan, q=q))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    d.extend(jds, [2, 4], stream=side)
    got = d.attend(0, d.append(0, k, k, rope=plan, q=q, stream=side), stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_a_captured_step_follows_the_batch(nh):
    """append (turned) and attend captured once, replayed after every extend; under a batch of another shape, or of rows
    that ask, a replay touches no page."""
    rng = np.random.default_rng(14)
    plan = nh.Rope(48)
    lens = [60, 5]
    made = [filled(nh, np.random.default_rng(14), lens, 2, 48, 64, 64, "f32", extra_pages=6) for _ in range(2)]
    (c, ids, _, _), (d, jds, _, _) = made
    k, v, q = (torch.zeros(2, h, n, device="cuda") for h, n in ((2, 48), (2, 64), (12, 48)))
    out, turned = torch.zeros(2, 12, 64, device="cuda"), torch.zeros(2, 12, 48, device="cuda")
    c.extend(ids, [1, 1])
    d.extend(jds, [1, 1])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c.append(0, k, v, rope=plan, q=q, out=turned)
        c.attend(0, turned, out=out)
    for step in range(40):
        if step:
            c.extend(ids, [1, 1])
            d.extend(jds, [1, 1])
        for t, n in ((k, 48), (v, 64), (q, 48)):
            t.copy_(torch.from_numpy(rng.standard_normal(tuple(t.shape)).astype(np.float32) * (1 + step % 5)))
        torch.cuda.synchronize()
        graph.replay()
        want = d.attend(0, d.append(0, k, v, rope=plan, q=q))
        assert torch.equal(out, want), step
    n = [c.length(s) for s in ids]
    held = c.read(0, ids, [0, 0], n)
    for form in ("other rows", "asks", "over"):
        if form == "other rows":
            c.extend(ids, [2, 0])
            n = [c.length(s) for s in ids]
            c.append(0, torch.ones(2, 2, 48, device="cuda"), torch.ones(2, 2, 64, device="cuda"))
            held = c.read(0, ids, [0, 0], n)
        elif form == "asks":
            c.ask(ids, [1, 1])
        else:
            c.truncate(ids[0], n[0] - 2)
            n[0] -= 2
            held = [x[list(range(n[0])) + list(range(n[0] + 2, sum(n) + 2))] for x in held]
            c.copy(ids[1])
        k.fill_(50.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        now = c.read(0, ids, [0, 0], n)
        assert torch.equal(now[0], held[0]) and torch.equal(now[1], held[1]), form


def test_captured_rows_that_ask(nh):
    rng = np.random.default_rng(15)
    c, ids, ks, vs = filled(nh, rng, [300, 40, 0, 9], 2, 64, 64, 64, "bf16", extra_pages=4)
    q, out = torch.zeros(6, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(6, 4, 64, dtype=torch.bfloat16, device="cuda")
    c.ask(ids[:2], [2, 4])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(0, q, out=out)
    for pair in (ids[:2], ids[2:], [ids[3], ids[0]], ids[:2]):
        c.ask(pair, [2, 4])
        q.copy_(rows_of(rng, 6, 4, 64, "bf16"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = c.attend(0, q)
        at = 0
        for s, n in zip(pair, (2, 4)):
            o, _ = ref.attend(plain(q[at:at + n]), ks[0][ids.index(s)], vs[0][ids.index(s)], 0.125, ask=True)
            limit = ref.attend_bound(plain(q), ks[0][ids.index(s)], vs[0][ids.index(s)], o, 0.125, "bf16", True)
            for x in (out, want):
                assert (np.abs(plain(x[at:at + n]) - o) <= limit).all()
            at += n
    # a step of rows of its own, of the same numbers: the captured attention is of rows that ask, and does nothing
    c.extend(ids[:2], [2, 4])
    c.append(0, rows_of(rng, 6, 2, 64, "bf16").cuda(), rows_of(rng, 6, 2, 64, "bf16").cuda())
    out.fill_(3.0)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert bool((out == 3.0).all())


def test_changes_are_refused_in_a_capture(nh):
    c = nh.KvCache8(1, 1, 64, 64, pages=4, seqs=2, cap=128)
    s = c.new_seq()
    c.extend([s], [1])
    x = torch.zeros(1, 1, 64, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: c.extend([s], [1]), lambda: c.ask([s], [1]), lambda: c.copy(s), lambda: c.read(0, [s], [0], [1])):
            with pytest.raises(nh.NeedleHipError):
                call()
        c.append(0, x, x)
    graph.replay()
    assert c.length(s) == 1


def test_refusals(nh):
    c = nh.KvCache8(2, 2, 64, 48, pages=3, seqs=3, cap=128)
    s = c.new_seq()
    plan, wide = nh.Rope(64), nh.Rope(96)
    k, v, q = (torch.zeros(4, h, d, device="cuda") for h, d in ((2, 64), (2, 48), (4, 64)))
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    for call, code in ((lambda: c.extend([s], [129]), EINVAL), (lambda: c.extend([s, s], [1, 1]), EINVAL),
                       (lambda: c.extend([s], [-1]), EINVAL), (lambda: c.extend([2], [1]), EINVAL),
                       (lambda: c.ask([s, s], [1, 1]), EINVAL), (lambda: c.ask([s], [-1]), EINVAL), (lambda: c.ask([1], [1]), EINVAL),
                       (lambda: c.truncate(s, 1), EINVAL), (lambda: c.fork(s, 3), ENOMEM)):
        with pytest.raises(nh.NeedleHipError) as e:
            call()
        assert e.value.code == code
    c.extend([s], [4])
    for bad in (dict(k=k[:3]), dict(v=k), dict(v=v.half()), dict(q=q), dict(positions=pos), dict(out=q), dict(rope=plan, q=q.half()),
                dict(rope=plan, q=q, out=k), dict(rope=plan, out=q), dict(rope=plan, positions=pos.long()),
                dict(rope=plan, positions=pos[:2]), dict(k=k.cpu(), v=v.cpu())):
        with pytest.raises(ValueError):
            c.append(0, **{"k": k, "v": v, **bad})
    for call in (lambda: c.append(2, k, v), lambda: c.append(-1, k, v), lambda: c.append(0, k, v, rope=wide),
                 lambda: c.append(0, k[:1].expand(4, 2, 64), v), lambda: c.attend(0, torch.zeros(4, 3, 64, device="cuda")),
                 lambda: c.attend(0, q, scale=float("nan")), lambda: c.attend(0, q, ring=-1), lambda: c.attend(5, q)):
        with pytest.raises(nh.NeedleHipError):
            call()
    for call in (lambda: c.attend(0, q, lse=torch.zeros(4, 4)), lambda: c.attend(0, q, out=q), lambda: c.attend(0, q[:2])):
        with pytest.raises(ValueError):
            call()
    c.append(0, k, v, rope=plan, q=q)
    assert c.free_pages == 2 and c.bytes() > 0
    other = c.new_seq()
    c.extend([s, other], [2, 0])
    c.free(other)
    # (the batch is over: it has no rows)
    with pytest.raises(ValueError):
        c.append(0, k[:2], v[:2])
    with pytest.raises(nh.NeedleHipError):
        c.append(0, k[:0], v[:0])


def test_no_rows(nh):
    c = nh.KvCache8(1, 2, 64, 64, pages=2, seqs=2, cap=64)
    s = c.new_seq()
    x, q = torch.zeros(0, 2, 64, device="cuda"), torch.zeros(0, 4, 64, device="cuda")
    for batch in (c.extend, c.ask):
        for seqs in ([], [s]):
            batch(seqs, [0] * len(seqs))
            assert c.attend(0, q).shape == (0, 4, 64)
            if batch == c.extend:
                c.append(0, x, x, rope=nh.Rope(64), q=q)
    assert c.read(0, [s], [0], [0])[0].shape == (0, 2, 64)
