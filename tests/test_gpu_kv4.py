"""The 4-bit key/value cache on the GPU: what it holds, its pages, and its
attention, against plain numpy in 64 bits."""
import random

import numpy as np
import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EINVAL, ESMALL, ENOMEM = -1, -2, -4


def rows_of(rng, n, heads, dim, dtype, spread=1.0):
    """Rows as projections give them: channels of different size and offset; as the type holds them, f32 numpy."""
    x = rng.standard_normal((n, heads, dim)) * np.exp(0.5 * rng.standard_normal(dim)) + 0.5 * rng.standard_normal(dim)
    return torch.from_numpy((x * spread).astype(np.float32)).to(T[dtype])


def plain(t):
    return t.float().cpu().numpy()


def filled(nh, rng, lens, kv, qk, v, group, page, dtype, layers=1, extra_pages=0, last=None, spread=1.0, seqs=None):
    """A cache whose sequences hold `lens` rows, the last `last[i]` as the batch: (cache, ids, k, v per sequence [layer])."""
    pages = sum(-(-n // page) for n in lens) + extra_pages
    c = nh.KvCache4(layers, kv, qk, v, pages=max(pages, 1), seqs=seqs or len(lens) + 8, cap=max(max(lens), 1) + 64, group=group,
                    page=page)
    ids = [c.new_seq() for _ in lens]
    last = last or [0] * len(lens)
    ks = [[rows_of(rng, n, kv, qk, dtype, spread) for n in lens] for _ in range(layers)]
    vs = [[rows_of(rng, n, kv, v, dtype, spread) for n in lens] for _ in range(layers)]
    for a, z in (([0] * len(lens), [n - r for n, r in zip(lens, last)]), ([n - r for n, r in zip(lens, last)], list(lens))):
        c.extend(ids, [e - b for b, e in zip(a, z)])
        for layer in range(layers):
            c.append(layer, torch.cat([x[b:e] for x, b, e in zip(ks[layer], a, z)]).cuda(),
                     torch.cat([x[b:e] for x, b, e in zip(vs[layer], a, z)]).cuda())
    return c, ids, ks, vs


SHAPES = [(2, 48, 64, 32, 32), (1, 64, 64, 64, 64), (3, 45, 51, 32, 64), (8, 128, 128, 32, 128), (5, 80, 96, 64, 32),
          (2, 256, 256, 32, 64), (1, 200, 129, 64, 256), (4, 1, 3, 32, 32)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,qk,v,group,page", SHAPES)
def test_rows_hold_the_formats_values(nh, kv, qk, v, group, page, dtype):
    rng = np.random.default_rng(qk * 7 + v)
    lens = [1, 70, page, 0, 2 * page + 1]
    c, ids, ks, vs = filled(nh, rng, lens, kv, qk, v, group, page, dtype, layers=2, last=[1, 3, 0, 0, page + 5])
    for layer in (0, 1):
        k, w = c.read(layer, ids, [0] * 5, lens)
        want_k = ref.quantize(np.concatenate([plain(x) for x in ks[layer]]), group)
        want_v = ref.quantize(np.concatenate([plain(x) for x in vs[layer]]), group)
        # f32 rounds the value once: half a step of it
        assert np.array_equal(plain(k), want_k.astype(np.float32))
        assert np.array_equal(plain(w), want_v.astype(np.float32))
    k, w = c.read(None, [ids[4], ids[1]], [page - 1, 5], [3, 60], T[dtype])
    assert k.shape == (2, 63, kv, qk) and k.dtype == T[dtype]
    for layer in (0, 1):
        want = np.concatenate([ref.quantize(plain(ks[layer][4]), group)[page - 1:page + 2],
                               ref.quantize(plain(ks[layer][1]), group)[5:65]]).astype(np.float32)
        assert np.array_equal(plain(k[layer]), plain(torch.from_numpy(want).to(T[dtype])))


def test_values_at_the_borders(nh):
    """Constant groups, values past f16's range, tiny ranges, NaN and infinities: the group alone reads as NaN."""
    group, d = 32, 96
    x = np.zeros((9, 1, d), np.float32)
    rng = np.random.default_rng(3)
    x[0] = 0.37
    x[1] = rng.standard_normal(d) * 1e5
    x[2] = rng.standard_normal(d) * 1e-9
    x[3] = -0.0
    x[4] = rng.standard_normal(d)
    x[4, 0, 40] = np.nan
    x[5] = rng.standard_normal(d)
    x[5, 0, 95] = np.inf
    x[6] = rng.standard_normal(d)
    x[6, 0, 0] = -np.inf
    x[7] = np.linspace(-65504, 65504, d)
    x[8] = 3.4e38
    c = nh.KvCache4(1, 1, d, d, pages=1, seqs=1, cap=32, group=group, page=32)
    s = c.new_seq()
    c.extend([s], [9])
    t = torch.from_numpy(x).cuda()
    c.append(0, t, t)
    k, v = c.read(0, [s], [0], [9])
    want = ref.quantize(x, group).astype(np.float32)
    assert np.isnan(want).sum() == 3 * group
    assert np.array_equal(plain(k), want, equal_nan=True)
    assert np.array_equal(plain(v), want, equal_nan=True)


def test_rows_of_a_wider_matrix(nh):
    """k and v as columns of the fused projection's rows, at an odd offset."""
    rng = np.random.default_rng(5)
    y = torch.from_numpy(rng.standard_normal((7, 577 + 96 + 128 + 768)).astype(np.float32)).cuda()
    k, v = y[:, 577:577 + 96].view(7, 2, 48), y[:, 577 + 96:577 + 224].view(7, 2, 64)
    c = nh.KvCache4(1, 2, 48, 64, pages=2, seqs=2, cap=64, page=32)
    s = [c.new_seq(), c.new_seq()]
    c.extend(s, [3, 4])
    c.append(0, k, v)
    a, b = c.read(0, s, [0, 0], [3, 4])
    assert np.array_equal(plain(a), ref.quantize(plain(k), 32).astype(np.float32))
    assert np.array_equal(plain(b), ref.quantize(plain(v), 32).astype(np.float32))
    q, out = y[:, :576].view(7, 12, 48), torch.full((7, 2, 12 * 64), 7.0, device="cuda")
    o = out[:, 1].view(7, 12, 64)
    c.attend(0, q, out=o)
    assert torch.equal(o, c.attend(0, q.contiguous()))
    assert bool((out[:, 0] == 7.0).all()), "the rows' neighbours are left as they were"


@pytest.mark.parametrize("seed", range(3))
def test_pages_in_random_order(nh, seed):
    """Forks, copies, cuts and compaction in random order; every sequence reads as the lists have it."""
    rng, pick = np.random.default_rng(seed), random.Random(seed)
    layers, kv, qk, v, group, page = 2, 2, (48, 128, 70)[seed], (64, 96, 200)[seed], 32, 32
    c = nh.KvCache4(layers, kv, qk, v, pages=40, seqs=7, cap=500, group=group, page=page)
    model = {}

    def check():
        live = sorted(model)
        k, w = c.read(None, live, [0] * len(live), [len(model[s][0]) for s in live])
        at = 0
        for s in live:
            n = len(model[s][0])
            assert c.length(s) == n
            for got, want in ((k, model[s][0]), (w, model[s][1])):
                assert np.array_equal(plain(got[:, at:at + n]).transpose(1, 0, 2, 3), want), (s, n)
            at += n

    def held(t):  # [layers][rows].. -> [rows][layers].. as held
        return ref.quantize(plain(t), group).astype(np.float32).transpose(1, 0, 2, 3)
    for _ in range(60):
        op = pick.choice(("new", "free", "fork", "copy", "cut", "extend", "extend", "extend", "compact"))
        live = sorted(model)
        try:
            if op == "new" or not live:
                s = c.new_seq()
                model[s] = (np.zeros((0, layers, kv, qk), np.float32), np.zeros((0, layers, kv, v), np.float32))
            elif op == "free":
                s = pick.choice(live)
                c.free(s)
                del model[s]
            elif op == "fork":
                s = pick.choice(live)
                for b in c.fork(s, pick.randrange(1, 3)):
                    model[b] = model[s]
            elif op == "copy":
                s = pick.choice(live)
                model[c.copy(s)] = model[s]
            elif op == "cut":
                s = pick.choice(live)
                n = pick.randrange(0, len(model[s][0]) + 1)
                c.truncate(s, n)
                model[s] = (model[s][0][:n], model[s][1][:n])
            elif op == "extend":
                seqs = pick.sample(live, pick.randrange(1, len(live) + 1))
                rows = [pick.choice((0, 1, 5, 40, 90)) for _ in seqs]
                c.extend(seqs, rows)
                n = sum(rows)
                k = torch.stack([rows_of(rng, n, kv, qk, "f32") for _ in range(layers)])
                w = torch.stack([rows_of(rng, n, kv, v, "f32") for _ in range(layers)])
                for layer in range(layers):
                    c.append(layer, k[layer].cuda(), w[layer].cuda())
                at = 0
                for s, r in zip(seqs, rows):
                    model[s] = tuple(np.concatenate((old, held(new[:, at:at + r]))) for old, new in zip(model[s], (k, w)))
                    at += r
            else:
                seqs = pick.sample(live, pick.randrange(1, min(2, len(live)) + 1))
                ranges = []
                for s in seqs:
                    cuts = sorted(pick.randrange(0, len(model[s][0]) + 1) for _ in range(2 * pick.randrange(0, 5)))
                    ranges.append(list(zip(cuts[::2], cuts[1::2])))
                c.compact(seqs, ranges)
                for s, r in zip(seqs, ranges):
                    at = [i for a, e in r for i in range(a, e)]
                    model[s] = (model[s][0][at], model[s][1][at])
        except nh.NeedleHipError as e:
            assert e.code == ENOMEM, e
        check()


def test_many_single_positions_compact(nh):
    """More kept runs than one launch takes: every third position of two sequences."""
    rng = np.random.default_rng(11)
    c, ids, ks, vs = filled(nh, rng, [1000, 777], 2, 64, 64, 64, 64, "f32", layers=2, extra_pages=20)
    ranges = [[(i, i + 1) for i in range(1, 1000, 3)], [(i, i + 2) for i in range(0, 776, 3)]]
    c.compact(ids, ranges)
    for layer in (0, 1):
        k, v = c.read(layer, ids, [0, 0], [c.length(s) for s in ids])
        at = [[i for a, e in r for i in range(a, e)] for r in ranges]
        want = np.concatenate([ref.quantize(plain(x), 64)[i] for x, i in zip(ks[layer], at)]).astype(np.float32)
        assert np.array_equal(plain(k), want)
        want = np.concatenate([ref.quantize(plain(x), 64)[i] for x, i in zip(vs[layer], at)]).astype(np.float32)
        assert np.array_equal(plain(v), want)


def attend_case(nh, lens, rows, kv, per, qk, v, group, page, dtype, sink=0, ring=0, scale=None, spread=1.0, seed=0,
                kernel=0):
    rng = np.random.default_rng(seed + 100 * qk + v)
    c, ids, ks, vs = filled(nh, rng, lens, kv, qk, v, group, page, dtype, last=rows, spread=spread)
    q = rows_of(rng, sum(rows), kv * per, qk, dtype)
    lse = torch.full((sum(rows), kv * per), 9.0, device="cuda")
    c.debug_kernel(kernel)
    o = c.attend(0, q.cuda(), scale=scale, sink=sink, ring=ring, lse=lse)
    assert o.dtype == T[dtype] and o.shape == (sum(rows), kv * per, v)
    s = qk ** -0.5 if scale is None else scale
    at = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        if not r:
            continue
        k, w = ref.quantize(plain(ks[0][b]), group), ref.quantize(plain(vs[0][b]), group)
        x = plain(q[at:at + r])
        want, want_lse = ref.attend(x, k, w, s, sink, ring)
        bound = ref.attend_bound(x, k, w, want, s, dtype)
        got = plain(o[at:at + r]).astype(np.float64)
        assert np.all(np.abs(got - want) <= bound), (b, n, r, float(np.max(np.abs(got - want) / bound)))
        # the log of a sum of weights that are each off by the scores' bound
        size = np.abs(x).sum(-1).max() * np.abs(k).max() * abs(s)
        off = (qk + 16) * 2.0 ** -24 * size * 2 + (n + 64) * 2.0 ** -23 + 2.0 ** -22 * np.abs(want_lse)
        if dtype != "f32" and max(qk, v) <= 128 and kernel != 1:
            # Calls of many rows round step x code of a key to 11 bits, half a step 2^-12 of at most
            # the group's range, 2 max |k|: a score moves by scale sum |q| 2^-11 max |k| at most, and so
            # the log of the sum; each weight, rounded to 11 bits and summed so, by 2^-12 of itself.
            off = off + 2.0 ** -11 * size + 2.0 ** -12
        assert np.all(np.abs(plain(lse[at:at + r]) - want_lse) <= off)
        at += r
    return c, ids, o


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,qk,v,group,page", SHAPES)
def test_attend_shapes(nh, kv, qk, v, group, page, dtype):
    attend_case(nh, [1, 33, 200, 64, 31], [1, 2, 7, 0, 31], kv, 2, qk, v, group, page, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("per", [1, 3, 6, 8, 17])
def test_attend_shared_heads(nh, per, dtype):
    attend_case(nh, [500, 77], [1, 1], 2, per, 48, 64, 32, 32, dtype, seed=per)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("sink,ring", [(0, 1), (1, 1), (118, 256), (4, 100), (0, 64), (64, 32), (2000, 5), (3, 5000), (37, 31)])
def test_attend_spans(nh, sink, ring, dtype):
    attend_case(nh, [600, 1, 130, 290], [5, 1, 130, 3], 2, 2, 64, 64, 32, 64, dtype, sink, ring)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 5, 16, 33, 150])
def test_attend_rows(nh, rows, dtype):
    attend_case(nh, [rows + 700], [rows], 1, 4, 128, 128, 32, 64, dtype, seed=rows)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_long(nh, dtype):
    attend_case(nh, [20000, 300, 9000], [1, 1, 1], 1, 4, 128, 128, 64, 64, dtype)


def test_attend_long_prompt_rows(nh):
    attend_case(nh, [1500, 700], [800, 300], 2, 2, 128, 128, 32, 64, "bf16")
    attend_case(nh, [1500, 700], [800, 300], 2, 2, 64, 64, 64, 64, "f32", sink=10, ring=200)


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kv,per,qk,v,group,page", [(1, 1, 64, 64, 32, 32), (2, 4, 48, 64, 64, 32), (2, 3, 45, 51, 32, 64),
                                                    (2, 4, 128, 128, 64, 64), (1, 8, 80, 96, 32, 128), (1, 2, 128, 72, 32, 64)])
def test_attend_prompts(nh, kv, per, qk, v, group, page, dtype, kernel):
    """Rows by the hundred, ragged, from the first position on and after others, with and without a span, by
    either kernel."""
    attend_case(nh, [300, 517, 33, 260], [300, 129, 33, 200], kv, per, qk, v, group, page, dtype, kernel=kernel)
    attend_case(nh, [410], [257], kv, per, qk, v, group, page, dtype, sink=5, ring=70, kernel=kernel)
    attend_case(nh, [900, 900], [256, 256], kv, per, qk, v, group, page, dtype, sink=130, ring=300, kernel=kernel)
    attend_case(nh, [1700, 3], [12, 1], kv, per, qk, v, group, page, dtype, kernel=kernel)


def test_the_rule_takes_either_kernel(nh):
    """Few rows, or short ones, go to the one kernel, long prompts to the other."""
    rng = np.random.default_rng(41)
    for n, rows, which in ((700, 100, 1), (4000, 16, 1), (2100, 1700, 2)):
        c, _, _, _ = filled(nh, rng, [n], 8, 128, 128, 32, 64, "bf16", last=[rows])
        q = rows_of(rng, rows, 32, 128, "bf16").cuda()
        outs = []
        for kernel in (0, 1, 2):
            c.debug_kernel(kernel)
            outs.append(c.attend(0, q))
        assert torch.equal(outs[0], outs[which]) and not torch.equal(outs[0], outs[3 - which])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_prompt_scales(nh, dtype):
    for spread, scale in ((1e-3, None), (50.0, 0.01), (1.0, -0.2), (1.0, 0.0), (3.0, 1.0)):
        attend_case(nh, [350], [290], 2, 2, 64, 64, 32, 32, dtype, scale=scale, spread=spread, kernel=2)


def test_prompt_nan_reaches_its_readers_only(nh):
    rng = np.random.default_rng(19)
    n = 400
    k, v, q = (rows_of(rng, n, 2, 64, "bf16") for _ in range(3))
    v2, k2, q2 = v.clone(), k.clone(), q.clone()
    v2[140, 1, 40] = float("nan")
    k2[300, 0, 3] = float("inf")
    q2[10, 0, 5] = float("nan")
    outs = []
    for kk, vv, qq in ((k, v, q), (k, v2, q), (k2, v, q), (k, v, q2)):
        c = nh.KvCache4(1, 2, 64, 64, pages=14, seqs=1, cap=n, page=32)
        c.debug_kernel(2)
        s = c.new_seq()
        c.extend([s], [n])
        c.append(0, kk.cuda(), vv.cuda())
        outs.append(plain(c.attend(0, qq.cuda(), ring=50)))
    assert not np.isnan(outs[0]).any()
    for got, seen in ((outs[1], (slice(140, 190), 1, slice(32, 64))), (outs[2], (slice(300, 350), 0, slice(0, 64))),
                      (outs[3], (10, 0, slice(0, 64)))):
        spoiled = np.zeros((n, 2, 64), bool)
        spoiled[seen] = True
        assert np.array_equal(np.isnan(got), spoiled)
        assert np.array_equal(got[~spoiled], outs[0][~spoiled])


def test_prompt_rows_do_not_depend_on_hidden_rows(nh):
    """Rows of a page that were written after this sequence's end (another's, larger, or NaN) change no bit."""
    rng = np.random.default_rng(23)
    k, v, q = (rows_of(rng, 161, 1, 128, "bf16").cuda() for _ in range(3))
    outs = []
    for stale in (None, 3000.0, float("nan")):
        c = nh.KvCache4(1, 1, 128, 128, pages=3, seqs=1, cap=192, page=64)
        c.debug_kernel(2)
        if stale is not None:
            s = c.new_seq()
            c.extend([s], [192])
            x = torch.full((192, 1, 128), stale, device="cuda") * torch.randn(192, 1, 128, device="cuda")
            c.append(0, x, x)
            c.free(s)
        s = c.new_seq()
        c.extend([s], [161])
        c.append(0, k, v)
        outs.append(c.attend(0, q))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_scales(nh, dtype):
    """Keys and values far from one in size, a negative and a zero scale, peaked scores."""
    for spread, scale in ((1e-3, None), (50.0, 0.01), (1.0, -0.2), (1.0, 0.0), (3.0, 1.0)):
        attend_case(nh, [150, 40], [3, 1], 2, 2, 64, 64, 32, 32, dtype, scale=scale, spread=spread)


@pytest.mark.parametrize("qk,v,group,n", [(48, 64, 32, 300), (128, 128, 32, 1000), (128, 128, 64, 90), (256, 256, 64, 200)])
def test_f32_calls_carry_22_bits(nh, qk, v, group, n):
    """f32 results to 1e-5 of their size.  A score is a sum of some ten matrix products, each cut off at 2^-20.6 of its
    largest term (measured; a term here is up to some 40, over the scale of 1 / sqrt(qk) some 4), so off by a few
    2^-19 at random, and weights and parts carry 2^-22: 1e-5 is five times that.  Codes taken as subnormals gave 4e-5."""
    rng = np.random.default_rng(qk + n)
    c, ids, ks, vs = filled(nh, rng, [n], 2, qk, v, group, 32, "f32", last=[1])
    q = rows_of(rng, 1, 12, qk, "f32")
    o = plain(c.attend(0, q.cuda())).astype(np.float64)
    want, _ = ref.attend(plain(q), ref.quantize(plain(ks[0][0]), group), ref.quantize(plain(vs[0][0]), group), qk ** -0.5)
    assert np.linalg.norm(o - want) <= 1e-5 * np.linalg.norm(want)


def test_attend_does_not_depend_on_the_batch(nh):
    """A sequence's result is the same bits beside other sequences whose values are larger."""
    rng = np.random.default_rng(2)
    k, v, q = (rows_of(rng, n, 2, 64, "bf16").cuda() for n in (300, 300, 1))
    out = []
    for others in (0, 3):
        c = nh.KvCache4(1, 2, 64, 64, pages=60, seqs=8, cap=400)
        ids = [c.new_seq() for _ in range(1 + others)]
        c.extend(ids, [300] * len(ids))
        c.append(0, torch.cat([k] + [100 * k] * others), torch.cat([v] + [1000 * v] * others))
        c.extend(ids, [1] * len(ids))
        c.append(0, torch.cat([k[:1]] * len(ids)), torch.cat([v[:1]] * len(ids)))
        out.append(c.attend(0, torch.cat([q] * len(ids)))[0].cpu())
    assert torch.equal(out[0], out[1])


def test_stale_pages_are_not_seen(nh):
    """A page that held NaN and infinity, freed and dealt again: its old rows past the new length do not matter."""
    rng = np.random.default_rng(8)
    c = nh.KvCache4(1, 1, 64, 64, pages=2, seqs=2, cap=64, page=32)
    s = c.new_seq()
    c.extend([s], [64])
    bad = torch.full((64, 1, 64), float("nan"), device="cuda")
    c.append(0, bad, bad)
    c.free(s)
    s = c.new_seq()
    k, v, q = (rows_of(rng, n, 1, 64, "f32") for n in (37, 37, 37))
    c.extend([s], [37])
    c.append(0, k.cuda(), v.cuda())
    o = plain(c.attend(0, q.cuda()))
    a, b = ref.quantize(plain(k), 32), ref.quantize(plain(v), 32)
    want, _ = ref.attend(plain(q), a, b, 0.125)
    assert np.all(np.abs(o - want) <= ref.attend_bound(plain(q), a, b, want, 0.125, "f32"))


@pytest.mark.parametrize("rows,kernel", [(1, 1), (160, 1), (160, 2), (1, 2)])
def test_nan_reaches_its_readers_over_ranges_of_keys(nh, rows, kernel):
    """A long sequence's keys are attended in ranges.  A NaN key spoils the rows that see it, a NaN value its group
    of them, a NaN query its own row, also where that range's other weights vanish beside another one's."""
    rng = np.random.default_rng(12)
    n, at = 6000, 300
    k, v = (rows_of(rng, n, 1, 64, "bf16") for _ in range(2))
    q = rows_of(rng, rows, 2, 64, "bf16")
    k[5000] = 60.0 * torch.sign(q[-1, 0])  # takes all of the weight of the last row's first head
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    k2[at, 0, 7] = float("nan")
    v2[at, 0, 40] = float("nan")
    q2[0, 1, 5] = float("nan")
    outs = []
    for kk, vv, qq in ((k, v, q), (k2, v, q), (k, v2, q), (k, v, q2)):
        c = nh.KvCache4(1, 1, 64, 64, pages=200, seqs=1, cap=8192, page=64)
        c.debug_kernel(kernel)
        s = c.new_seq()
        c.extend([s], [n - rows])
        c.append(0, kk[: n - rows].cuda(), vv[: n - rows].cuda())
        c.extend([s], [rows])
        c.append(0, kk[n - rows :].cuda(), vv[n - rows :].cuda())
        lse = torch.empty((rows, 2), device="cuda")
        outs.append([plain(x) for x in (c.attend(0, qq.cuda(), scale=1.0, lse=lse), lse)])
    assert not np.isnan(outs[0][0]).any() and not np.isnan(outs[0][1]).any()
    assert np.isnan(outs[1][0]).all() and np.isnan(outs[1][1]).all()
    assert np.isnan(outs[2][0][..., 32:]).all() and not np.isnan(outs[2][0][..., :32]).any()
    assert np.array_equal(outs[2][1], outs[0][1])
    spoiled = np.zeros((rows, 2), bool)
    spoiled[0, 1] = True
    assert np.array_equal(np.isnan(outs[3][1]), spoiled)
    assert np.array_equal(np.isnan(outs[3][0]).all(-1), spoiled) and np.array_equal(np.isnan(outs[3][0]).any(-1), spoiled)


def test_nan_reaches_its_readers_only(nh):
    """A NaN value in a row: outputs of the rows that see it are NaN in its group, all others are as without it;
    the window hides it from later rows.  A NaN query spoils its own row and head."""
    rng = np.random.default_rng(9)
    k, v, q = (rows_of(rng, 90, 2, 64, "f32") for _ in range(3))
    v2, q2 = v.clone(), q.clone()
    v2[40, 1, 3] = float("nan")
    q2[10, 0, 5] = float("nan")
    outs = []
    for vv, qq in ((v, q), (v2, q), (v, q2)):
        c = nh.KvCache4(1, 2, 64, 64, pages=4, seqs=1, cap=96, page=32)
        s = c.new_seq()
        c.extend([s], [90])
        c.append(0, k.cuda(), vv.cuda())
        outs.append(plain(c.attend(0, qq.cuda(), ring=20)))
    seen = np.zeros((90, 2, 64), bool)
    seen[40:60, 1, :32] = True
    assert np.array_equal(np.isnan(outs[1]), seen)
    assert np.array_equal(outs[1][~seen], outs[0][~seen])
    spoiled = np.zeros((90, 2, 64), bool)
    spoiled[10, 0] = True
    assert np.array_equal(np.isnan(outs[2]), spoiled)
    assert np.array_equal(outs[2][~spoiled], outs[0][~spoiled])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_ragged_sequences(nh, dtype):
    """More sequences than a wavefront has lanes, of 0 to 9 rows each; more spans than one launch reads."""
    rng = np.random.default_rng(31)
    lens = [int(x) for x in rng.integers(0, 90, 150)]
    rows = [int(min(n, x)) for n, x in zip(lens, rng.integers(0, 10, 150))]
    c, ids, _ = attend_case(nh, lens, rows, 1, 2, 64, 64, 32, 32, dtype)
    pick = [int(x) for x in rng.integers(0, 150, 400)]
    begin = [int(rng.integers(0, lens[i] + 1)) for i in pick]
    count = [int(rng.integers(0, lens[i] - b + 1)) for i, b in zip(pick, begin)]
    k, v = c.read(0, [ids[i] for i in pick], begin, count)
    whole_k, whole_v = c.read(0, ids, [0] * 150, lens)
    first = np.concatenate(([0], np.cumsum(lens)))
    at = [first[i] + b + j for i, b, n in zip(pick, begin, count) for j in range(n)]
    assert torch.equal(k, whole_k[at]) and torch.equal(v, whole_v[at])


def test_a_long_sequence_is_copied_and_closed_up(nh):
    """More pages than one launch's arguments name: tables, copies, compaction of 40,000 positions."""
    rng = np.random.default_rng(37)
    n = 40000
    c, ids, ks, vs = filled(nh, rng, [n], 1, 64, 64, 64, 32, "f16", extra_pages=2600, seqs=3, last=[2])
    t = c.copy(ids[0])
    c.compact([t], [[(3, 20000), (20001, n)]])
    keep = [i for i in range(3, n) if i != 20000]
    k, v = c.read(0, [t], [0], [n - 4])
    a, b = c.read(0, ids, [0], [n])
    assert torch.equal(k, a[keep]) and torch.equal(v, b[keep])
    assert np.array_equal(plain(a), ref.quantize(plain(ks[0][0]), 64).astype(np.float32))
    c.extend([t], [1])
    x = rows_of(rng, 1, 1, 64, "f16")
    c.append(0, x.cuda(), x.cuda())
    q = rows_of(rng, 1, 4, 64, "f16")
    o = plain(c.attend(0, q.cuda()))
    kk, vv = (np.concatenate((plain(y), ref.quantize(plain(x), 64))) for y in (k, v))
    want, _ = ref.attend(plain(q), kk, vv, 0.125)
    assert np.all(np.abs(o - want) <= ref.attend_bound(plain(q), kk, vv, want, 0.125, "f16"))


def test_a_replay_of_another_shape_does_nothing(nh):
    """A step captured for two rows, replayed after an extend of five: neither the rows nor the cache are touched."""
    rng = np.random.default_rng(41)
    c, ids, _, _ = filled(nh, rng, [40], 1, 64, 64, 32, 32, "bf16", extra_pages=4, last=[2])
    x, q = rows_of(rng, 2, 1, 64, "bf16").cuda(), rows_of(rng, 2, 2, 64, "bf16").cuda()
    out = torch.zeros(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    c.attend(0, q, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(0, x, x)
        c.attend(0, q, out=out)
    c.extend(ids, [5])
    y = rows_of(rng, 5, 1, 64, "bf16").cuda()
    c.append(0, y, y)
    before = c.read(0, ids, [0], [45])
    out.fill_(3.0)
    g.replay()
    torch.cuda.synchronize()
    assert bool((out == 3.0).all())
    for a, b in zip(before, c.read(0, ids, [0], [45])):
        assert torch.equal(a, b)


def test_a_replay_after_pages_changed_hands_does_nothing(nh):
    """A captured step whose sequences are gone, and one whose second sequence is: what took their pages stays as it is."""
    rng = np.random.default_rng(43)
    c, ids, _, _ = filled(nh, rng, [64, 64, 50], 1, 64, 64, 32, 32, "bf16", extra_pages=2, last=[1, 1, 0])
    x, q = rows_of(rng, 3, 1, 64, "bf16").cuda(), rows_of(rng, 3, 2, 64, "bf16").cuda()
    out = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    c.extend(ids, [1, 1, 1])
    c.append(0, x, x)
    c.attend(0, q, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(0, x, x)
        c.attend(0, q, out=out)
    for change in ("extend", "copy", "compact"):
        if change == "extend":
            c.free(ids[1])
            c.extend([ids[0]], [0])
            t = ids[2]
        else:
            c.extend([i for i in ids if i != ids[1]], [1, 1])
            c.append(0, x[:2], x[:2])
            c.truncate(ids[0], 33)
            t = c.copy(ids[2])
            if change == "compact":
                c.compact([t], [[(7, 40)]])
        before = c.read(0, [ids[0], t], [0, 0], [c.length(ids[0]), c.length(t)])
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(before, c.read(0, [ids[0], t], [0, 0], [c.length(ids[0]), c.length(t)])):
            assert torch.equal(a, b), change
        if change != "extend":
            c.free(t)


def test_refusals(nh):
    c = nh.KvCache4(2, 2, 48, 64, pages=3, seqs=2, cap=90, page=32)
    k, v = torch.zeros(4, 2, 48, device="cuda"), torch.zeros(4, 2, 64, device="cuda")
    q = torch.zeros(4, 12, 48, device="cuda")
    s = c.new_seq()
    c.extend([s], [4])

    def refused(code, f, *a, **kw):
        with pytest.raises(nh.NeedleHipError) as e:
            f(*a, **kw)
        assert e.value.code == code, e.value
    refused(EINVAL, c.append, 2, k, v)
    refused(EINVAL, c.append, -1, k, v)
    refused(EINVAL, c.attend, 2, q)
    refused(EINVAL, c.attend, 0, q, sink=-1, ring=3)
    refused(EINVAL, c.attend, 0, q, ring=-2)
    refused(EINVAL, c.attend, 0, q, scale=float("nan"))
    refused(EINVAL, c.attend, 0, q, scale=float("inf"))
    refused(EINVAL, c.attend, 0, torch.zeros(4, 3, 48, device="cuda"))  # 3 heads over 2
    refused(EINVAL, c.read, 0, [s], [2], [3])
    refused(EINVAL, c.read, 0, [s], [-1], [3])
    refused(EINVAL, c.read, 0, [1], [0], [0])
    refused(EINVAL, c.read, 5, [s], [0], [1])
    refused(EINVAL, c.extend, [s], [93])
    refused(EINVAL, c.extend, [s, s], [1, 1])
    refused(EINVAL, c.truncate, s, 9)
    refused(EINVAL, c.free, 1)
    refused(EINVAL, c.copy, 1)
    refused(ENOMEM, c.fork, s, 2)
    for bad in (k[:3], k[:, :1], k[:, :, :47], k.double(), k.cpu(), k.transpose(0, 1).contiguous().transpose(0, 1)):
        with pytest.raises(ValueError):
            c.append(0, bad, v)
    with pytest.raises(ValueError):
        c.append(0, k.half(), v)
    with pytest.raises(ValueError):
        c.attend(0, q, out=torch.zeros(4, 12, 64, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError):
        c.attend(0, q, lse=torch.zeros(4, 12))
    c.append(0, k, v)  # the batch is as it was
    c.truncate(s, 2)
    refused(EINVAL, c.append, 0, k[:0], v[:0])
    refused(EINVAL, c.attend, 0, q[:0])
    # a workspace that is missing, small or unaligned
    c.extend([s], [2])
    lib = nh._lib
    need = lib.nh_kv4_attend_ws_bytes(c.h, 12, 0, 0)
    assert need >= 0
    if need:
        out, ws = torch.zeros(2, 12, 64, device="cuda"), torch.zeros(need + 16, dtype=torch.uint8, device="cuda")
        args = (c.h, 0, q.data_ptr(), 576, 12, 0.1, 0, 0, out.data_ptr(), 768, None, 0)
        assert lib.nh_kv4_attend(*args, None, need, None) == EINVAL
        assert lib.nh_kv4_attend(*args, ws.data_ptr() + 4, need, None) == EINVAL
        assert lib.nh_kv4_attend(*args, ws.data_ptr(), need - 1, None) == ESMALL
    # rows that overlap, an unknown type, null pointers
    assert lib.nh_kv4_append(c.h, 0, k.data_ptr(), v.data_ptr(), 95, 128, 0, None) == EINVAL
    assert lib.nh_kv4_append(c.h, 0, k.data_ptr(), v.data_ptr(), 96, 128, 3, None) == EINVAL
    assert lib.nh_kv4_append(c.h, 0, None, v.data_ptr(), 96, 128, 0, None) == EINVAL
    torch.cuda.synchronize()


def test_empty_batches(nh):
    c = nh.KvCache4(1, 1, 64, 64, pages=2, seqs=2, cap=64)
    k, q = torch.zeros(0, 1, 64, device="cuda"), torch.zeros(0, 4, 64, device="cuda")
    c.append(0, k, k)
    assert c.attend(0, q).shape == (0, 4, 64)
    s = c.new_seq()
    c.extend([s], [0])
    c.append(0, k, k)
    assert c.attend(0, q).shape == (0, 4, 64)
    c.extend([], [])
    c.append(0, k, k)
    a, b = c.read(0, [s], [0], [0])
    assert a.shape == (0, 1, 64) and b.shape == (0, 1, 64)
    c.compact([s], [[]])
    assert c.fork(s, 0) == []


def test_changes_are_refused_under_capture(nh):
    c = nh.KvCache4(1, 1, 64, 64, pages=4, seqs=3, cap=64)
    s = c.new_seq()
    k = torch.ones(2, 1, 64, device="cuda")
    c.extend([s], [2])
    c.append(0, k, k)
    torch.cuda.synchronize()
    errors = []
    x = torch.zeros(4, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x.add_(1)
        for f in (lambda: c.extend([s], [1]), lambda: c.copy(s), lambda: c.compact([s], [[(0, 1)]])):
            try:
                f()
            except nh.NeedleHipError as e:
                errors.append(e.code)
    assert errors == [EINVAL] * 3
    assert c.length(s) == 2
    g.replay()
    torch.cuda.synchronize()


def test_a_cache_is_freed_during_a_capture(nh):
    """The collector may run inside a capture: a cache that goes there leaves the graph whole."""
    c = nh.KvCache4(1, 1, 64, 64, pages=4, seqs=3, cap=64)
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x.add_(1)
        del c
        x.add_(2)
    for i in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert x.tolist() == [3.0 * (i + 1)] * 4


def test_a_captured_step_follows_the_cache(nh):
    """append and attention of a step captured once, replayed after each extend (other lengths, a page border,
    a fork's copied page), with eager work between; every replay against the eager call."""
    rng = np.random.default_rng(4)
    lens = [90, 31]
    c, ids, ks, vs = filled(nh, rng, lens, 2, 64, 64, 32, 32, "bf16", extra_pages=10)
    k, v = (torch.zeros(2, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q = torch.zeros(2, 8, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.zeros(2, 8, 64, device="cuda", dtype=torch.bfloat16)
    c.extend(ids, [1, 1])
    c.append(0, k, v)
    c.attend(0, q, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(0, k, v)
        c.attend(0, q, out=out, sink=3, ring=64)
    for step in range(5):
        if step:
            if step == 3:
                c.fork(ids[1], 1)  # the tail page is shared now: the extend copies it
            c.extend(ids, [1, 1])
        for t in (k, v, q):
            t.copy_(torch.from_numpy(rng.standard_normal(tuple(t.shape)).astype(np.float32)))
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = c.attend(0, q, sink=3, ring=64)
        # (the captured call may split the keys another way: both are within the bound of the exact result)
        kk, vv = c.read(0, ids, [0, 0], [c.length(s) for s in ids])
        at = 0
        for b, s in enumerate(ids):
            n = c.length(s)
            x = plain(q[b:b + 1])
            w, _ = ref.attend(x, plain(kk[at:at + n]), plain(vv[at:at + n]), 0.125, 3, 64)
            bound = ref.attend_bound(x, plain(kk[at:at + n]), plain(vv[at:at + n]), w, 0.125, "bf16")
            for o in (got, want):
                assert np.all(np.abs(plain(o[b:b + 1]) - w) <= bound), step
            at += n


def test_other_streams(nh):
    """Every call on a stream that is not the current one, its inputs made there."""
    rng = np.random.default_rng(6)
    st = torch.cuda.Stream()
    c = nh.KvCache4(1, 2, 64, 64, pages=20, seqs=4, cap=300)
    s = c.new_seq()
    k, v = rows_of(rng, 200, 2, 64, "f32"), rows_of(rng, 200, 2, 64, "f32")
    q = rows_of(rng, 200, 4, 64, "f32")
    with torch.cuda.stream(st):
        kd, vd, qd = (t.cuda() for t in (k, v, q))
    c.extend([s], [200], stream=st)
    c.append(0, kd, vd, stream=st)
    o = c.attend(0, qd, stream=st)
    t = c.copy(s, stream=st)
    c.compact([t], [[(0, 5), (150, 200)]], stream=st)
    a, b = c.read(0, [t], [0], [55], stream=st)
    st.synchronize()
    kk, vv = ref.quantize(plain(k), 32), ref.quantize(plain(v), 32)
    want, _ = ref.attend(plain(q), kk, vv, 0.125)
    assert np.all(np.abs(plain(o) - want) <= ref.attend_bound(plain(q), kk, vv, want, 0.125, "f32"))
    at = list(range(5)) + list(range(150, 200))
    assert np.array_equal(plain(a), kk[at].astype(np.float32)) and np.array_equal(plain(b), vv[at].astype(np.float32))


def test_offsets_past_32_bits(nh):
    """A cache of more than 4 GiB: pages at its end are written, copied and attended to."""
    layers, kv, d, page = 64, 8, 128, 256
    per_page = layers * kv * page * 160
    pages = (1 << 32) // per_page + 12
    c = nh.KvCache4(layers, kv, d, d, pages=pages, seqs=4, cap=pages * page, page=page)
    assert c.bytes() > 1 << 32
    a, s = c.new_seq(), c.new_seq()
    c.extend([a], [(pages - 6) * page])  # holds the first pages; its rows are not read
    rng = np.random.default_rng(1)
    n, layer = 2 * page + 3, layers - 1
    k, v, q = rows_of(rng, n, kv, d, "f32"), rows_of(rng, n, kv, d, "f32"), rows_of(rng, n, kv, d, "f32")[-3:]
    c.extend([s], [n - 3])
    c.append(layer, k[:-3].cuda(), v[:-3].cuda())
    c.extend([s], [3])
    c.append(layer, k[-3:].cuda(), v[-3:].cuda())
    o = plain(c.attend(layer, q.cuda()))
    kk, vv = ref.quantize(plain(k), 32), ref.quantize(plain(v), 32)
    want, _ = ref.attend(plain(q), kk, vv, d ** -0.5)
    assert np.all(np.abs(o - want) <= ref.attend_bound(plain(q), kk, vv, want, d ** -0.5, "f32"))
    t = c.copy(s)
    x, y = c.read(layer, [t], [0], [n])
    assert np.array_equal(plain(x), kk.astype(np.float32)) and np.array_equal(plain(y), vv.astype(np.float32))
