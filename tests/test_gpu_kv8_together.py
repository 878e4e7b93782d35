"""The 8-bit cache as a program uses it: prompts, branches, steps, drafts and their
states of an encoder, keys turned on the way in; many rows and splits in captured
graphs; uneven batches; pages beyond 4 GiB.  The turn alone at sizes beyond 2^32."""
import random

import numpy as np
import pytest
import torch

import kv8_ref as ref
import rope_ref
from test_gpu_kv8 import T, check_attend, filled, plain, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,kv,heads,qk,v,layout", [("f32", 2, 12, 48, 64, "half"), ("f16", 4, 4, 64, 64, "half"),
                                                        ("bf16", 2, 8, 128, 128, "half"), ("bf16", 1, 4, 80, 96, "interleaved")])
def test_a_conversation(nh, dtype, kv, heads, qk, v, layout):
    """Two prompts against two encoded inputs, three branches of the first, steps, drafts in a window and their cuts."""
    rng, pick = np.random.default_rng(qk + heads), random.Random(qk)
    layers, turned = 2, min(qk, 64)
    plan = nh.Rope(turned, layout=layout)
    enc, eids, ek, ev = filled(nh, rng, [150, 33], kv, qk, v, 64, dtype, layers=layers)
    c = nh.KvCache8(layers, kv, qk, v, pages=24, seqs=6, cap=256)
    ids = [c.new_seq(), c.new_seq()]
    home = {ids[0]: 0, ids[1]: 1}  # each sequence's input
    model = {s: [ref.Side(kv, d) for _ in range(layers) for d in (qk, v)] for s in ids}
    turned_over = 0

    def step(seqs, rows, sink=0, ring=0):
        nonlocal turned_over
        c.extend(seqs, rows)
        lens = [c.length(s) for s in seqs]
        pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)])
        for layer in range(layers):
            k, w = rows_of(rng, len(pos), kv, qk, dtype), rows_of(rng, len(pos), kv, v, dtype)
            q = c.append(layer, k.cuda(), w.cuda(), rope=plan, q=rows_of(rng, len(pos), heads, qk, dtype).cuda())
            keys = rope_ref.turn32(plain(k), pos, plan.freqs, plan.amplitude, layout)
            at = 0
            for s, r in zip(seqs, rows):
                model[s][2 * layer].store(keys[at:at + r])
                model[s][2 * layer + 1].store(plain(w[at:at + r]))
                at += r
            got = c.read(layer, seqs, [0] * len(seqs), lens)
            want = [np.concatenate([model[s][2 * layer + side].held32() for s in seqs]) for side in (0, 1)]
            # (a cosine that rounds the other way moves a code only beside a border)
            turned_over += (plain(got[0]) != want[0]).sum()
            assert np.array_equal(plain(got[1]), want[1])
            cuts = np.cumsum([0] + lens)
            held = [[plain(x[a:z]) for a, z in zip(cuts, cuts[1:])] for x in c.read(layer, seqs, [0] * len(seqs), lens, torch.float32)]
            check_attend(c, layer, q, *held, rows, dtype, sink, ring, many=dtype != "f32")
        # each input's rows, all of its branches' together
        inputs = sorted({home[s] for s in seqs})
        asked = [sum(r for s, r in zip(seqs, rows) if home[s] == i) for i in inputs]
        enc.ask([eids[i] for i in inputs], asked)
        for layer in range(layers):
            check_attend(enc, layer, rows_of(rng, sum(asked), heads, qk, dtype), [ek[layer][i] for i in inputs],
                         [ev[layer][i] for i in inputs], asked, dtype, ask=True, many=dtype != "f32")

    step(ids, [70, 5])
    for s in c.fork(ids[0], 2):
        home[s], model[s] = 0, [x.fork() for x in model[ids[0]]]
        ids.append(s)
    for _ in range(4):
        step(ids, [1] * 4)
    for _ in range(3):
        some = pick.sample(ids, 3)
        step(some, [5, 1, 5], 4, 40)
        for s in some:
            n = c.length(s) - pick.randrange(5)
            if n < c.length(s) and n > 6:
                c.truncate(s, n)
                for x in model[s]:
                    x.cut(n)
    c.free(ids.pop(2))
    step(ids, [1, 1, 1])
    assert turned_over <= 4


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_uneven_rows(nh, dtype):
    rng, pick = np.random.default_rng(31), random.Random(31)
    lens = [pick.choice((0, 1, 15, 16, 63, 64, 65, pick.randrange(300))) for _ in range(70)]
    rows = [pick.choice((0, 1, n, n // 2)) if n else 0 for n in lens]
    c, ids, ks, vs = filled(nh, rng, lens, 2, 64, 64, 64, dtype, last=rows)
    q = rows_of(rng, sum(rows), 6, 64, dtype)
    for kernel in (0, 1, 2):
        c.debug_kernel(kernel)
        check_attend(c, 0, q, ks[0], vs[0], rows, dtype, kernel=kernel, many=dtype != "f32")
        check_attend(c, 0, q, ks[0], vs[0], rows, dtype, 3, 33, kernel=kernel, many=dtype != "f32")


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64)])
def test_many_rows_of_many_keys(nh, dtype, dim):
    """Few tiles of 256 rows: their keys in ranges that are joined."""
    rng = np.random.default_rng(dim)
    c, ids, ks, vs = filled(nh, rng, [9000], 1, dim, dim, 256, dtype, last=[260])
    q = rows_of(rng, 260, 2, dim, dtype)
    for kernel in (1, 2):
        c.debug_kernel(kernel)
        for sink, ring in ((0, 0), (100, 4000)):
            check_attend(c, 0, q, ks[0], vs[0], [260], dtype, sink, ring, kernel=kernel, many=True)


def test_many_rows_in_a_graph(nh):
    """The kernel of many rows with ranges of keys and their join, captured; every replay beside the program's own calls."""
    rng = np.random.default_rng(33)
    rows, room = [130, 200], 2600
    c = nh.KvCache8(1, 1, 128, 128, pages=90, seqs=2, cap=room)
    c.debug_kernel(2)
    ids = [c.new_seq(), c.new_seq()]
    sides = [[ref.Side(1, 128), ref.Side(1, 128)] for _ in ids]

    def grow(n):
        c.extend(ids, n)
        k, v = rows_of(rng, sum(n), 1, 128, "bf16"), rows_of(rng, sum(n), 1, 128, "bf16")
        c.append(0, k.cuda(), v.cuda())
        for (a, b), x, y in zip(sides, k.split(n), v.split(n)):
            a.store(plain(x))
            b.store(plain(y))

    grow([900, 1500])
    grow(rows)
    q = torch.zeros(sum(rows), 4, 128, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(0, q, out=out)
    for turn in range(4):
        if turn:
            for i, cut in enumerate(((500, 1600), (600, 3), (64, 150))[turn - 1]):
                c.truncate(ids[i], cut)
                for x in sides[i]:
                    x.cut(cut)
            if turn == 3:
                grow([300, 2200])  # further than at the capture
            grow(rows)
        q.copy_(rows_of(rng, sum(rows), 4, 128, "bf16"))
        out.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = c.attend(0, q)
        at = 0
        for (k, v), n in zip(sides, rows):
            x, hk, hv = plain(q[at:at + n]), k.held32(), v.held32()
            o, _ = ref.attend(x, hk, hv, 128 ** -0.5)
            limit = ref.attend_bound(x, hk, hv, o, 128 ** -0.5, "bf16", True)
            for y in (out, eager):
                assert (np.abs(plain(y[at:at + n]) - o) <= limit).all(), turn
            at += n


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("qk,v,turned,layout", [(64, 64, 48, "half"), (128, 128, 128, "half"), (128, 96, 64, "interleaved"),
                                                (256, 256, 32, "half"), (45, 51, 44, "half")])
def test_rows_at_odd_addresses(nh, qk, v, turned, layout, dtype):
    """k, v, q and every output an element behind an aligned address, rows of an odd stride: the bits of contiguous rows."""
    rng = np.random.default_rng(qk + v)
    kv, heads, rows = 2, 4, [5, 70]
    plan, n = nh.Rope(turned, layout=layout), sum(rows)

    def odd(x):
        wide = torch.full((n, x.shape[1] * x.shape[2] + 3), 5.0, dtype=x.dtype, device="cuda")
        view = wide[:, 1:1 + x.shape[1] * x.shape[2]].unflatten(1, x.shape[1:])
        view.copy_(x)
        return wide, view

    k, w, q = (rows_of(rng, n, h, d, dtype).cuda() for h, d in ((kv, qk), (kv, v), (heads, qk)))
    got = []
    for move in (lambda x: (None, x), odd):
        c = nh.KvCache8(1, kv, qk, v, pages=4, seqs=2, cap=128)
        ids = [c.new_seq(), c.new_seq()]
        c.extend(ids, rows)
        turned_to, out = move(torch.zeros_like(q)), move(torch.zeros(n, heads, v, dtype=T[dtype], device="cuda"))
        c.append(0, move(k)[1], move(w)[1], rope=plan, q=move(q)[1], out=turned_to[1])
        result = [*c.read(0, ids, [0, 0], rows), turned_to[1].clone()]
        for kernel in (1, 2):
            c.debug_kernel(kernel)
            c.attend(0, turned_to[1], out=out[1])
            result.append(out[1].clone())
        got.append(result)
        for wide, view in (turned_to, out):
            if wide is not None:
                assert bool((wide[:, 0] == 5.0).all()) and bool((wide[:, -2:] == 5.0).all())
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size_k,size_v", [(1.0, 1e-25), (1.0, 1e30), (1e28, 1.0), (1e-28, 1e-20)])
def test_attention_over_small_and_large_numbers(nh, size_k, size_v, dtype):
    rng = np.random.default_rng(70)
    n, rows = 700, 300
    k, v = rows_of(rng, n, 2, 64, dtype, size_k), rows_of(rng, n, 2, 64, dtype, size_v)
    q = rows_of(rng, rows, 4, 64, dtype, 1 / size_k)
    c = nh.KvCache8(1, 2, 64, 64, pages=12, seqs=1, cap=n)
    s = c.new_seq()
    for m, a in ((n - rows, 0), (rows, n - rows)):
        c.extend([s], [m])
        c.append(0, k[a:a + m].cuda(), v[a:a + m].cuda())
    held = [ref.quantize(plain(x), (n - rows,)) for x in (k, v)]
    for kernel in (0, 1, 2):
        c.debug_kernel(kernel)
        check_attend(c, 0, q, [held[0]], [held[1]], [rows], dtype, kernel=kernel, many=dtype != "f32")


def test_reads_of_many_spans(nh):
    """Spans by the hundred, of the same sequences again and again, some empty, over one another."""
    rng, pick = np.random.default_rng(60), random.Random(60)
    lens = [300, 64, 1, 129]
    c, ids, ks, vs = filled(nh, rng, lens, 2, 48, 64, 64, "f32", layers=2, last=[5, 0, 1, 100])
    for count in (1, 15, 16, 17, 100, 700):
        which = [pick.randrange(4) for _ in range(count)]
        first = [pick.randrange(lens[i]) for i in which]
        rows = [pick.randrange(min(lens[i] - a, 40) + 1) for i, a in zip(which, first)]
        k, v = c.read(None, [ids[i] for i in which], first, rows, torch.float32)
        for got, side in ((k, ks), (v, vs)):
            for layer in (0, 1):
                want = np.concatenate([side[layer][i][a:a + r] for i, a, r in zip(which, first, rows)])
                assert np.array_equal(plain(got[layer]), want), count


def test_two_graphs_on_two_streams(nh):
    """Steps of two caches captured apart and replayed at once: neither's workspace is the other's."""
    made = []
    for i in range(2):
        rng = np.random.default_rng(40 + i)
        c, ids, ks, vs = filled(nh, rng, [5000], 1, 64, 64, 64, "bf16", last=[1])
        q = rows_of(rng, 1, 8, 64, "bf16").cuda()
        out, stream, graph = torch.zeros_like(q), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            c.attend(0, q, out=out)
        made.append((c, q, out, stream, graph))
    want = [c.attend(0, q) for c, q, *_ in made]
    for _ in range(5):
        torch.cuda.synchronize()
        for c, q, out, stream, graph in made:
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for (c, q, out, *_), w in zip(made, want):
            assert torch.equal(out, w) and torch.equal(c.attend(0, q), w)


def test_many_rows_keep_their_own_precision(nh):
    """Blocks of values 10^6 times the others, hidden in a row's own tile or seen."""
    rng = np.random.default_rng(8)
    n = 200
    k, v = rows_of(rng, n, 1, 64, "bf16"), rows_of(rng, n, 1, 64, "bf16")
    v[:32] *= 1e-6
    v[160:] *= 1e6
    c = nh.KvCache8(1, 1, 64, 64, pages=4, seqs=1, cap=256)
    s = c.new_seq()
    c.extend([s], [n])
    c.append(0, k.cuda(), v.cuda())
    hk, hv = ref.quantize(plain(k)), ref.quantize(plain(v))
    q = rows_of(rng, n, 2, 64, "bf16")
    c.debug_kernel(2)
    got = plain(c.attend(0, q.cuda())).astype(np.float64)
    o, _ = ref.attend(plain(q), hk, hv, 0.125)
    for r in range(n):
        limit = ref.attend_bound(plain(q), hk[:r + 1], hv[:r + 1], o[r], 0.125, "bf16", True)
        assert (np.abs(got[r] - o[r]) <= limit).all(), r


@pytest.mark.parametrize("kv,dim", [(16, 256), (64, 64)])
def test_pages_beyond_4_gib(nh, kv, dim):
    """Sequences whose pages lie at both ends of more than 4 GiB."""
    rng = np.random.default_rng(dim)
    c = nh.KvCache8(1, kv, dim, dim, pages=2200, seqs=3, cap=2200 * 256, page=256)
    assert c.bytes() > 2 ** 32 + 2 ** 28
    ids = [c.new_seq() for _ in range(3)]
    held = {}
    for s, rows in ((ids[0], 270), (ids[1], 2190 * 256), (ids[2], 270)):
        c.extend([s], [rows])
        if s == ids[1]:
            continue  # (claimed, never read)
        k, v = rows_of(rng, rows, kv, dim, "bf16"), rows_of(rng, rows, kv, dim, "bf16")
        c.append(0, k.cuda(), v.cuda())
        held[s] = ref.quantize(plain(k)), ref.quantize(plain(v))
    for s in (ids[0], ids[2]):
        k, v = c.read(0, [s], [0], [270], torch.float32)
        assert np.array_equal(plain(k), held[s][0]) and np.array_equal(plain(v), held[s][1])
        c.ask([s], [40])
        q = rows_of(rng, 40, kv, dim, "bf16")
        for kernel in (1, 2):
            c.debug_kernel(kernel)
            check_attend(c, 0, q, [held[s][0]], [held[s][1]], [40], "bf16", ask=True, kernel=kernel, many=True)


def test_pages_of_more_than_4_gib_each(nh):
    rng = np.random.default_rng(50)
    layers, kv, some = 128, 1024, [0, 1, 511, 1022, 1023]
    c = nh.KvCache8(layers, kv, 64, 64, pages=2, seqs=1, cap=512, page=256)
    assert c.bytes() > 2 ** 33
    s = c.new_seq()
    c.extend([s], [300])
    k, v = (torch.randn(300, kv, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    c.append(layers - 1, k, v)
    got = c.read(layers - 1, [s], [0], [300], torch.float32)
    held = [ref.quantize(plain(x[:, some])) for x in (k, v)]
    assert all(np.array_equal(plain(x[:, some]), y) for x, y in zip(got, held))
    c.ask([s], [20])
    q = torch.randn(20, kv, 64, device="cuda", dtype=torch.bfloat16)
    for kernel in (1, 2):
        c.debug_kernel(kernel)
        out = plain(c.attend(layers - 1, q)[:, some])
        x = plain(q[:, some])
        o, _ = ref.attend(x, *held, 0.125, ask=True)
        assert (np.abs(out - o) <= ref.attend_bound(x, *held, o, 0.125, "bf16", True)).all()


def test_rows_beyond_the_threads_of_a_launch(nh):
    """More than 2^30 threads' rows of 63 pairs, a pair a thread, 2^31 elements: turned in place as a few of them alone."""
    border = (1 << 30) // 63  # the row where a launch's blocks go on in another dimension
    rows, plan = border + 2000, nh.Rope(126)
    some = [0, 1, border - 1, border, border + 1, 1 << 23, rows - 1001, rows - 1]
    assert 0 <= min(some) and max(some) < rows and 125 * rows < 2 ** 31
    x = torch.empty(rows, 1, 128, dtype=torch.bfloat16, device="cuda").normal_()
    pos = torch.arange(rows, dtype=torch.int32, device="cuda") * 125 - 5
    want = plan.apply(torch.cat([pos[i:i + 1] for i in some]), torch.cat([x[i:i + 1] for i in some]))
    plan.apply(pos, x, out=x)
    assert torch.equal(torch.cat([x[i:i + 1] for i in some]), want)


def test_more_heads_than_a_grid_has_shares(nh):
    plan, heads = nh.Rope(2), 1 << 20
    q, k = torch.randn(1, heads, 2, device="cuda"), torch.randn(1, heads, 2, device="cuda")
    pos = torch.tensor([77], dtype=torch.int32, device="cuda")
    got = plan.apply(pos, q, k)
    for x, y in zip((q, k), got):
        assert torch.equal(y.view(heads, 1, 2), plan.apply(pos.expand(heads).contiguous(), x.view(heads, 1, 2)))
