"""The picked token where the wavefronts of a workgroup use the same words of LDS one after the other: many sequences,
several slices of the vocabulary, every call against numpy in 64 bits."""
import numpy as np
import pytest

from test_gpu_verify import case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [5000, 40000])
def test_all_drafts_kept_with_probabilities(nh, vocab):
    """Nothing is refused, so the token is drawn from p, whose slices' sums are at hand: no load stands between the
    workgroup's question whether it was the last and the next use of that word."""
    logits, drafts, u, q = case(vocab, 24, 2, vocab, 1.0, True)
    u[:, :2] = 0.0
    for k in range(4):
        u[:, 2] = np.random.default_rng(vocab + k).random(24).astype(np.float32)
        kept, _ = check(nh, logits, drafts, u, q)
        assert (kept == 2).all()


@pytest.mark.parametrize("with_probs", [False, True])
@pytest.mark.parametrize("vocab", [300, 5000, 20000])
def test_uniforms_past_the_whole(nh, vocab, with_probs):
    """No cumulative weight passes the goal: the last token that weighs anything, wherever its slice begins."""
    logits, drafts, u, q = case(vocab, 24, 1, vocab, 1.0, with_probs)
    last = np.random.default_rng(vocab).integers(vocab // 2, vocab, 24)
    for b in range(24):
        logits[b, :, last[b] + 1:] = -np.inf
        if with_probs:
            q[b, 0, last[b]] = 0.0  # (so that it is left of the target when the draft is refused)
    drafts[:, 0] = 0
    u[:, 0] = np.where(np.arange(24) % 2, 0.0, 1.0)  # kept and refused in turn
    for past in (1.0, 1.5, 4.0):
        u[:, 1] = past
        kept, tokens = check(nh, logits, drafts, u, q)
        assert np.array_equal(tokens[np.arange(24), kept], last)


@pytest.mark.parametrize("with_probs", [False, True])
@pytest.mark.parametrize("temperature", [1e-45, 1e-40, 4e-39, 5e-39, 1e-20, 1e30, 3e38])
def test_temperatures_of_any_size(nh, temperature, with_probs):
    """From the smallest f32 to its end: next to greedy, then next to even."""
    logits, drafts, u, q = case(11, 6, 3, 5000, 1.0, with_probs)
    drafts[::2] = logits[::2, :3].argmax(-1)
    kept, tokens = check(nh, logits, drafts, u, q, temperature=float(np.float32(temperature)))
    if temperature < 1:
        assert (kept[::2] == 3).all() and np.array_equal(tokens[::2, 3], logits[::2, 3].argmax(-1))
