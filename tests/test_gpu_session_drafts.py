"""Drafted decoding on a session: what is refused leaves the session as it was; a drafter's probabilities; other streams."""
import numpy as np
import pytest
import torch

import kv4_ref as ref
import oracle as o
from test_gpu_drafts import archive

pytestmark = pytest.mark.gpu


def test_refused_probabilities_leave_the_session(nh):
    """Another type, the CPU, a wrong size, a temperature past f32: refused before the drafts are fed."""
    m = nh.Model.from_archive(archive(81))
    s = m.session(96)
    s.forward(o.random_tokens(20, 300, seed=82))
    before = s.forward([]).clone()
    width = m.out_rows
    q = torch.full((3, width), 1.0 / width, device="cuda")
    u = np.full(4, 0.5, np.float32)
    for bad in (dict(probs=q.double()), dict(probs=q.cpu()), dict(probs=q[:2]), dict(probs=q[:, 1:]),
                dict(probs=q.cpu().numpy()), dict(probs=q, temperature=1e39), dict(probs=q, temperature=float("nan")),
                dict(probs=q, u=None), dict(probs=q, u=u[:3])):
        with pytest.raises((ValueError, RuntimeError)):
            s.verify_drafts([1, 2, 3], **{"u": u, "temperature": 1.0, **bad})
        assert len(s) == 20, bad
        assert torch.equal(s.forward([]), before)


@pytest.mark.parametrize("sure", [False, True])
@pytest.mark.parametrize("other_stream", [False, True])
def test_session_drafts_with_probabilities(nh, other_stream, sure):
    """Each step against a clone that is fed the drafts, checked in numpy with the drafter's probabilities, rolled back
    and fed the next token; on the current stream or another one; by a drafter that gives every token little, or is
    sure of its own."""
    rng = np.random.default_rng(6)
    m = nh.Model.from_archive(archive(83))
    s = m.session(200)
    st = torch.cuda.Stream() if other_stream else None
    s.forward(o.random_tokens(30, 300, seed=84))
    torch.cuda.synchronize()
    kept_all = refused = 0
    for step in range(10):
        n = int(rng.integers(1, 7))
        drafts = rng.integers(0, 300, n)
        c = s.clone()
        first = c.forward([]).cpu().numpy()
        rows = c.forward(drafts, nh.OUT_ALL_LOGITS).cpu().numpy()
        logits = np.concatenate((first[None], rows))[None]
        width = m.out_rows
        q = np.full((1, n, width), 0.5 / width, np.float32)
        if step % 3 == 0:  # (a drafter that gives its own drafts little: they are kept)
            q[0, np.arange(n), drafts] = 1e-7
        elif sure:
            q[0, np.arange(n), drafts] = 0.9
        u = rng.random(n + 1).astype(np.float32)
        accepted, tokens = ref.verify(logits, drafts[None].astype(np.int32), u[None], q, temperature=0.9)
        kept = int(accepted[0])
        want = tokens[0, :kept + 1].tolist()
        c.rollback(n - kept)
        want_logits = c.forward(want[-1:])
        probs = torch.from_numpy(q[0]).cuda()
        torch.cuda.synchronize()
        got = s.verify_drafts(drafts, u, 0.9, probs=probs, stream=st)
        assert got == want, step
        torch.cuda.synchronize()
        assert torch.equal(s.forward([]), want_logits)
        kept_all += kept
        refused += n - kept
    assert kept_all > 3 and (refused > 3) == sure


@pytest.mark.parametrize("sink,ring,fed", [(6, 40, 100), (0, 33, 40), (10, 64, 50), (118, 256, 60)])
def test_refused_drafts_under_a_span_leave_no_trace(nh, sink, ring, fed):
    """Drafts that are all refused, before and after the ring is full: the session goes on bit by bit as one that was
    only ever fed the picked tokens, one at a time."""
    rng = np.random.default_rng(9)
    m = nh.Model.from_archive(archive(85))
    s = m.session(256)
    s.set_attend(sink, ring)
    s.forward(o.random_tokens(fed, 300, seed=86))
    plain = s.clone()
    for step in range(16):
        best = int(plain.forward([]).argmax())
        n = int(rng.integers(1, 21))
        drafts = rng.integers(0, 300, n)
        drafts[0] = (best + 1 + int(rng.integers(0, 298))) % 300
        assert s.verify_drafts(drafts) == [best]
        plain.forward([best])
        assert torch.equal(s.forward([]), plain.forward([])), step
    assert len(s) == len(plain) == fed + 16


def test_kept_drafts_under_a_span(nh):
    """Some kept, some refused, by greedy picks: each step as a clone that is fed the kept drafts and the next token."""
    rng = np.random.default_rng(10)
    m = nh.Model.from_archive(archive(87))
    s = m.session(256)
    s.set_attend(5, 48)
    s.forward(o.random_tokens(70, 300, seed=88))
    kept_all = 0
    for step in range(12):
        n = int(rng.integers(1, 9))
        c, like = s.clone(), s.clone()
        drafts = s.clone().generate_greedy(n)[0].astype(np.int64)
        if n > 2:
            drafts[int(rng.integers(1, n))] = int(rng.integers(0, 300))
        first = c.forward([]).cpu().numpy()
        rows = c.forward(drafts, nh.OUT_ALL_LOGITS).cpu().numpy()
        accepted, tokens = ref.verify(np.concatenate((first[None], rows))[None], drafts[None].astype(np.int32), None,
                                      temperature=0.0)
        want = tokens[0, :int(accepted[0]) + 1].tolist()
        assert s.verify_drafts(drafts) == want
        if n == 1:  # its slot is the next token's, so it is fed in place, and kept as it was fed
            like.forward(drafts, nh.OUT_ALL_LOGITS)
            like.rollback(2 - len(want))
        elif len(want) > 1:
            like.forward(want[:-1], nh.OUT_NONE)
        like.forward(want[-1:])
        assert len(s) == len(like)
        assert torch.equal(s.forward([]), like.forward([])), step
        kept_all += len(want) - 1
    assert kept_all > 5
