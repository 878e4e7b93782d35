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
