"""The pieces together: drafted decoding on a session, and a run of the 4-bit
cache's calls as a server makes them (prefix, branches, drafts, check, cut,
compaction)."""
import numpy as np
import pytest
import torch

import kv4_ref as ref
import oracle as o
from oracle import cact

pytestmark = pytest.mark.gpu

SMALL = dict(vocab=300, num_layers=3, engram_slots=64, engram_sites=(1,), global_layers=(1,), sliding_window=8)


def archive(seed):
    g = cact.Geometry(**SMALL)
    ts, _ = cact.needle3_tensors(g, seed=seed, kind=lambda n: ("cq", 4) if n == "embedding" else ("random", 4))
    return cact.pack(ts, g.header())


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_session_drafts(nh, temperature):
    """Each step against a clone that is fed the drafts, checked in numpy, rolled back and fed the next token."""
    rng = np.random.default_rng(5)
    m = nh.Model.from_archive(archive(71))
    s = m.session(256)
    s.forward(o.random_tokens(40, 300, seed=72))
    total, kept_all = 40, 0
    for step in range(12):
        n = int(rng.integers(0, 9))
        c = s.clone()
        if rng.random() < 0.7:  # a drafter that is right for a while
            guess = s.clone().generate_greedy(n)[0] if n else np.zeros(0, np.uint32)
            drafts = guess.astype(np.int64)
            if n > 2:
                drafts[int(rng.integers(0, n))] = int(rng.integers(0, 300))
        else:
            drafts = rng.integers(0, 300, n)
        u = rng.random(n + 1).astype(np.float32)
        first = c.forward([]).cpu().numpy()
        rows = c.forward(drafts, nh.OUT_ALL_LOGITS).cpu().numpy() if n else np.zeros((0, m.out_rows), np.float32)
        accepted, tokens = ref.verify(np.concatenate((first[None], rows))[None], drafts[None].astype(np.int32), u[None],
                                      temperature=temperature)
        kept = int(accepted[0])
        want = tokens[0, :kept + 1].tolist()
        c.rollback(n - kept)
        logits = c.forward(want[-1:])
        got = s.verify_drafts(drafts, u, temperature)
        assert got == want, (step, got, want)
        total += len(got)
        kept_all += kept
        assert len(s) == len(c) == total
        assert torch.equal(s.forward([]), logits)
    assert kept_all > (5 if temperature == 0 else 0)  # some were kept, so both ways were taken


def test_session_drafts_refusals(nh):
    m = nh.Model.from_archive(archive(73))
    s = m.session(64)
    with pytest.raises(nh.NeedleHipError):
        s.verify_drafts([1, 2])  # nothing fed yet
    assert len(s) == 0
    s.forward([5, 6, 7])
    for bad in ([1] * 33, [1] * 61):
        with pytest.raises(ValueError):
            s.verify_drafts(bad)
    with pytest.raises(nh.NeedleHipError):
        s.verify_drafts([300])  # not a token
    with pytest.raises(nh.NeedleHipError):
        s.verify_drafts([1], temperature=0.5)  # no uniforms
    assert len(s.verify_drafts([])) == 1 and len(s) == 4


def test_a_servers_run(nh):
    """Two layers, a shared prefix, three branches; every step adds 1 + drafts rows to each, attends, takes logits
    from the last layer's output, checks the drafts, cuts the refused rows, and closes long branches up to their sink
    and ring.  The cache's contents and every attention result follow a numpy model of the same program."""
    rng = np.random.default_rng(17)
    layers, kv, heads, d, group, page, vocab = 2, 2, 8, 64, 32, 32, 50
    sink, ring, most = 20, 30, 62
    c = nh.KvCache4(layers, kv, d, d, pages=24, seqs=5, cap=160, group=group, page=page)
    wo = rng.standard_normal((heads * d, vocab)).astype(np.float32) * 0.4
    emb = rng.standard_normal((vocab, layers, 3, heads, d)).astype(np.float32)

    def rows_of(tokens):  # k, v, q of each layer
        x = emb[np.asarray(tokens)] + 0.1 * rng.standard_normal((len(tokens), layers, 3, heads, d)).astype(np.float32)
        return x[:, :, 0, :kv], x[:, :, 1, :kv], x[:, :, 2]

    def cuda(x):
        return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda()

    prefix = rng.integers(0, vocab, 45)
    k, v, _ = rows_of(prefix)
    s = c.new_seq()
    c.extend([s], [45])
    for layer in range(layers):
        c.append(layer, cuda(k[:, layer]), cuda(v[:, layer]))
    held = (ref.quantize(k, group), ref.quantize(v, group))
    ids = c.fork(s, 3)
    c.free(s)
    model = {i: held for i in ids}
    last = {i: int(rng.integers(0, vocab)) for i in ids}
    free = c.free_pages
    compacted = cut = 0
    for step in range(14):
        n = int(rng.integers(0, 5))
        drafts = {i: rng.integers(0, vocab, n) for i in ids}
        tokens = [t for i in ids for t in (last[i], *drafts[i])]
        k, v, q = rows_of(tokens)
        c.extend(ids, [n + 1] * 3)
        out = None
        for layer in range(layers):
            c.append(layer, cuda(k[:, layer]), cuda(v[:, layer]))
            out = c.attend(layer, cuda(q[:, layer]), sink=sink, ring=ring)
            for b, i in enumerate(ids):
                r = slice(b * (n + 1), (b + 1) * (n + 1))
                kk = np.concatenate((model[i][0][:, layer], ref.quantize(k[r, layer], group)))
                vv = np.concatenate((model[i][1][:, layer], ref.quantize(v[r, layer], group)))
                want, _ = ref.attend(q[r, layer], kk, vv, d ** -0.5, sink, ring)
                bound = ref.attend_bound(q[r, layer], kk, vv, want, d ** -0.5, "f32")
                assert np.all(np.abs(out[r].cpu().numpy() - want) <= bound), (step, layer, i)
        logits = torch.matmul(out.reshape(3 * (n + 1), heads * d), cuda(wo)).view(3, n + 1, vocab)
        u = rng.random((3, n + 1)).astype(np.float32)
        x = np.stack([drafts[i] for i in ids]).astype(np.int32).reshape(3, n)
        if n and step % 2:  # drafts that are the likeliest
            x[:, 0] = logits[:, 0].argmax(-1).cpu().numpy()
        kept, new = nh.verify_drafts(logits, torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), temperature=0.7)
        want_kept, want_new = ref.verify(logits.cpu().numpy(), x, u, temperature=0.7)
        assert np.array_equal(kept.cpu().numpy(), want_kept) and np.array_equal(new.cpu().numpy(), want_new)
        for b, i in enumerate(ids):
            r = slice(b * (n + 1), b * (n + 1) + 1 + int(want_kept[b]))
            model[i] = tuple(np.concatenate((old, ref.quantize(x2[r], group))) for old, x2 in zip(model[i], (k, v)))
            c.truncate(i, len(model[i][0]))
            cut += n - int(want_kept[b])
            last[i] = int(want_new[b, want_kept[b]])
        long = [i for i in ids if len(model[i][0]) > most]
        if long:
            c.compact(long, [[(0, sink), (c.length(i) - ring, c.length(i))] for i in long])
            for i in long:
                model[i] = tuple(np.concatenate((old[:sink], old[len(old) - ring:])) for old in model[i])
            compacted += len(long)
        if step == 6:  # one branch is given up for a copy of another
            c.free(ids[0])
            ids[0] = c.copy(ids[1])
            model[ids[0]], last[ids[0]] = model[ids[1]], last[ids[1]]
        kk, vv = c.read(None, ids, [0] * 3, [c.length(i) for i in ids])
        for got, part in ((kk, 0), (vv, 1)):
            want = np.concatenate([model[i][part] for i in ids]).astype(np.float32).transpose(1, 0, 2, 3)
            assert np.array_equal(got.cpu().numpy(), want), step
    assert cut > 5 and compacted > 1
    for i in ids:
        c.free(i)
    assert c.free_pages == 24 and free < 24
