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
