"""The check of drafted tokens on the GPU against plain numpy in 64 bits."""
import numpy as np
import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def softmax(x, t):
    y = np.exp((x - x.max(-1, keepdims=True)) / t)
    return y / y.sum(-1, keepdims=True)


def case(seed, b, n, vocab, temperature, with_probs, peak=3.0):
    rng = np.random.default_rng(seed)
    logits = (peak * rng.standard_normal((b, n + 1, vocab))).astype(np.float32)
    q = softmax(logits[:, :n].astype(np.float64) + 0.5 * rng.standard_normal((b, n, vocab)), max(temperature, 0.5))
    drafts = np.zeros((b, n), np.int32)
    for s in range(b):
        for i in range(n):
            drafts[s, i] = rng.choice(vocab, p=q[s, i]) if rng.random() < 0.6 or temperature else logits[s, i].argmax()
            if not with_probs and rng.random() < 0.7:
                drafts[s, i] = logits[s, i].argmax()
    u = rng.random((b, n + 1)).astype(np.float32)
    return logits, drafts, u, q.astype(np.float32) if with_probs else None


def check(nh, logits, drafts, u, probs=None, counts=None, temperature=1.0, dtype="f32", ptype="f32"):
    cuda = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    lg = cuda(logits).to(T[dtype])
    pr = None if probs is None else cuda(probs).to(T[ptype])
    a, t = nh.verify_drafts(lg, cuda(drafts), cuda(u), probs=pr, counts=cuda(counts), temperature=temperature)
    want_a, want_t = ref.verify(lg.float().cpu().numpy(), drafts, u, None if pr is None else pr.float().cpu().numpy(), counts,
                                temperature)
    assert np.array_equal(a.cpu().numpy(), want_a), (a.tolist(), want_a.tolist())
    assert np.array_equal(t.cpu().numpy(), want_t), (t.tolist(), want_t.tolist())
    return want_a, want_t


@pytest.mark.parametrize("with_probs", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("b,n,vocab", [(1, 4, 8192), (3, 0, 1000), (5, 1, 1), (7, 3, 2), (4, 8, 4097), (2, 17, 255),
                                       (33, 2, 513), (1, 1, 131072)])
def test_sampled(nh, b, n, vocab, dtype, with_probs):
    for seed, t in ((b * n + vocab, 1.0), (7 * vocab + n, 0.6)):
        check(nh, *case(seed, b, n, vocab, t, with_probs), temperature=t, dtype=dtype, ptype=dtype)


@pytest.mark.parametrize("ptype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_types_mixed(nh, dtype, ptype):
    kept = [check(nh, *case(s, 6, 5, 2000, 1.0, True), dtype=dtype, ptype=ptype)[0] for s in range(4)]
    assert 0 < np.concatenate(kept).mean() < 5


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 3, 1000, 32768])
def test_greedy(nh, vocab, dtype):
    logits, drafts, u, _ = case(vocab, 5, 4, vocab, 0.0, False)
    check(nh, logits, drafts, u, temperature=0.0, dtype=dtype)
    # ties go to the lowest index
    logits = np.round(logits)
    drafts = logits[:, :-1].argmax(-1).astype(np.int32)
    a, t = check(nh, logits, drafts, u, temperature=0.0, dtype=dtype)
    assert (a == 4).all()


def test_counts_and_bad_drafts(nh):
    logits, drafts, u, q = case(1, 9, 4, 700, 1.0, True)
    drafts[:, :] = logits[:, :4].argmax(-1)
    u[:, :4] = 0.0
    counts = np.array([0, 1, 2, 3, 4, 5, -3, 4, 4], np.int32)
    drafts[7, 2], drafts[8, 0] = 700, -1
    for probs in (None, q):
        a, _ = check(nh, logits, drafts, u, probs, counts)
        assert a.tolist() == [0, 1, 2, 3, 4, 4, 0, 2, 0]
    check(nh, logits, drafts, u, None, counts, temperature=0.0)


def test_edges_of_the_uniform(nh):
    """u = 0 takes the first token that weighs anything, u near (or past) 1 the last."""
    logits, drafts, u, q = case(2, 4, 0, 5000, 1.0, False)
    logits[:, :, :7] = -np.inf
    logits[:, :, 4990:] = -np.inf
    u[:, 0] = [0.0, np.float32(1) - np.float32(2) ** -24, 1.0, 2.0]
    _, t = check(nh, logits, drafts, u)
    assert t[:, 0].tolist() == [7, 4989, 4989, 4989]


def test_rows_without_a_distribution(nh):
    logits, drafts, u, q = case(3, 6, 2, 300, 1.0, True)
    logits[0, 0] = -np.inf
    logits[1, 0] = np.nan
    logits[2, 0, 5:9] = np.inf
    drafts[2, 0] = 6
    logits[3, 0, ::2] = np.nan
    logits[4, 0] = np.float32(-3.4028235e38)   # masked by the type's lowest value: even weights
    logits[5, 0, 0] = np.nan
    for probs in (None, q):
        a, t = check(nh, logits, drafts, u, probs)
        assert a[0] == 0 and a[1] == 0 and t[0, 0] == 0 and t[1, 0] == 0
        assert t[3, 0] % 2 == 1 or a[3] > 0
    check(nh, logits, drafts, u, temperature=0.0)
    nans = q.copy()
    nans[:, :, ::3] = np.nan
    check(nh, logits, drafts, u, nans)


def test_a_drafter_equal_to_the_target_keeps_all(nh):
    logits, drafts, u, _ = case(4, 16, 6, 900, 1.0, False)
    q = (softmax(logits[:, :6].astype(np.float64), 1.0) * (1 - 1e-6)).astype(np.float32)
    u = np.minimum(u, np.float32(0.999999))
    a, _ = check(nh, logits, drafts, u, q)
    assert (a == 6).all()


def test_nothing_left_of_the_target(nh):
    """A refused draft whose q covers p everywhere: the token is drawn from p itself."""
    logits, drafts, u, _ = case(5, 8, 1, 64, 1.0, False)
    q = np.ones((8, 1, 64), np.float32)
    u[:, 0] = 0.9999
    logits = np.minimum(logits, 0.5 * logits)
    a, t = check(nh, logits, drafts, u, q)
    assert (a == 0).any()


def test_padded_rows_and_streams(nh):
    logits, drafts, u, q = case(6, 3, 2, 1001, 1.0, True)
    want_a, want_t = ref.verify(logits, drafts, u, q)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        wide = torch.full((3, 3, 1030), 50.0, device="cuda")
        wide[..., 3:1004] = torch.from_numpy(logits)
        pw = torch.full((3, 2, 1009), 9.0, device="cuda")
        pw[..., 1:1002] = torch.from_numpy(q)
        d, uu = torch.from_numpy(drafts).cuda(), torch.from_numpy(u).cuda()
    a, t = nh.verify_drafts(wide[..., 3:1004], d, uu, probs=pw[..., 1:1002], stream=st)
    st.synchronize()
    assert np.array_equal(a.cpu().numpy(), want_a) and np.array_equal(t.cpu().numpy(), want_t)


def test_captured(nh):
    logits, drafts, u, q = case(7, 4, 3, 5000, 1.0, True)
    lg, d, uu, pr = (torch.from_numpy(x).cuda() for x in (logits, drafts, u, q))
    nh.verify_drafts(lg, d, uu, probs=pr)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, t = nh.verify_drafts(lg, d, uu, probs=pr)
    for seed in range(8, 12):
        fresh = case(seed, 4, 3, 5000, 1.0, True)
        for x, y in zip((lg, d, uu, pr), fresh):
            x.copy_(torch.from_numpy(y))
        a.fill_(77)
        t.fill_(77)
        g.replay()
        torch.cuda.synchronize()
        want_a, want_t = ref.verify(*fresh)
        assert np.array_equal(a.cpu().numpy(), want_a) and np.array_equal(t.cpu().numpy(), want_t)
        ea, et = nh.verify_drafts(lg, d, uu, probs=pr)
        assert torch.equal(ea, a) and torch.equal(et, t)


def test_distribution(nh):
    """Drafts checked with many uniforms: the first token's frequencies are the target's (chi-square, 5 sigma)."""
    rng = np.random.default_rng(12)
    vocab, b = 6, 20000
    row, qrow = 1.2 * rng.standard_normal((2, vocab)).astype(np.float32), softmax(rng.standard_normal(vocab), 1.0)
    drafts = rng.choice(vocab, p=qrow, size=(b, 1)).astype(np.int32)
    u = rng.random((b, 2)).astype(np.float32)
    lg = torch.from_numpy(np.broadcast_to(row, (b, 2, vocab)).copy()).cuda()
    pr = torch.from_numpy(np.broadcast_to(qrow.astype(np.float32), (b, 1, vocab)).copy()).cuda()
    _, t = nh.verify_drafts(lg, torch.from_numpy(drafts).cuda(), torch.from_numpy(u).cuda(), probs=pr)
    got = np.bincount(t[:, 0].cpu().numpy(), minlength=vocab)
    want = softmax(row[0].astype(np.float64), 1.0) * b
    assert np.all(np.abs(got - want) <= 5 * np.sqrt(want))


def test_python_refusals(nh):
    lg, d, u = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda"), \
        torch.zeros(2, 3, device="cuda")
    for bad in (dict(drafts=d.long()), dict(drafts=d[:1]), dict(u=u.double()), dict(u=u[:, :2]), dict(logits=lg[0]),
                dict(logits=lg.double()), dict(logits=lg.transpose(0, 1)), dict(probs=torch.zeros(2, 2, 9, device="cuda")),
                dict(counts=d[:, 0]), dict(u=u.cpu())):
        with pytest.raises(ValueError):
            nh.verify_drafts(**{"logits": lg, "drafts": d, "u": u, **bad})
    with pytest.raises(nh.NeedleHipError):
        nh.verify_drafts(lg, d, u, temperature=-1.0)
    with pytest.raises(nh.NeedleHipError):
        nh.verify_drafts(lg, d, None)
    a, t = nh.verify_drafts(lg[:0].contiguous(), d[:0].contiguous(), u[:0].contiguous())
    assert a.shape == (0,) and t.shape == (0, 3)
