"""Views that the check of drafts takes and refuses: rows may be padded, but not repeat or overlap, which the kernels,
stepping a row of the vocabulary at a time, would read past the end of."""
import pytest
import torch

import needle_hip as nh
from needle_hip import kv4


class View:
    """What the check looks at of a tensor of the GPU."""

    def __init__(self, shape, stride, dtype=torch.float32, index=0):
        self.shape, self.dtype, self._stride, self._index = torch.Size(shape), dtype, stride, index

    def stride(self):
        return self._stride

    def get_device(self):
        return self._index


@pytest.mark.parametrize("shape,stride", [
    ((1, 4, 1000), (0, 0, 1)),       # one row for every draft
    ((3, 4, 1000), (0, 0, 1)),       # .. of every sequence
    ((3, 1, 1000), (0, 1000, 1)),    # one sequence's row for all
    ((3, 4, 1000), (4000, 0, 1)),
    ((3, 4, 1000), (0, 1000, 1)),
    ((1, 4, 1000), (0, 500, 1)),     # rows that overlap
    ((3, 4, 1000), (2000, 500, 1)),
    ((1, 2, 1000), (1998, 999, 1)),
    ((2, 3, 1), (0, 0, 1)),
    ((2, 3, 1000), (6000, 2000, 2)),
    ((2, 3, 1000), (1000, 2000, 1)),
])
def test_rows_that_repeat_or_overlap_are_refused(shape, stride):
    with pytest.raises(ValueError):
        kv4._row_stride(View(shape, stride), 0, "probs")


@pytest.mark.parametrize("shape,stride,ld", [
    ((3, 4, 1000), (4000, 1000, 1), 1000),
    ((3, 4, 1000), (4400, 1100, 1), 1100),
    ((1, 4, 1000), (7, 1100, 1), 1100),
    ((3, 1, 1000), (1100, 3, 1), 1100),
    ((1, 1, 1000), (0, 0, 1), 1000),
    ((0, 4, 1000), (0, 0, 1), 1000),
    ((2, 3, 1), (3, 1, 9), 1),
])
def test_rows_that_are_taken(shape, stride, ld):
    assert kv4._row_stride(View(shape, stride), 0, "probs") == ld


@pytest.mark.parametrize("batch,n,vocab", [(1 << 22, 0, 5), (1 << 21, 7, 5), (1 << 14, 1023, 5), (1 << 18, 1, 1 << 17)])
def test_batches_that_no_launch_takes_are_refused(batch, n, vocab):
    """2^32 threads and more: a workgroup of 256 for each 4,096 logits of a row, one of 1,024 for each sequence."""
    f = nh.load_library().nh_verify_drafts_ws_bytes
    assert f(batch, n, vocab) == -1
    assert f(batch - 1, n, vocab) > 0


@pytest.mark.gpu
def test_an_expanded_row_is_refused(nh):  # noqa: F811
    """A uniform drafter as one expanded row, and a target's row for every position."""
    b, n, v = 2, 3, 1000
    logits = torch.zeros(b, n + 1, v, device="cuda")
    drafts = torch.zeros(b, n, dtype=torch.int32, device="cuda")
    u = torch.full((b, n + 1), 0.5, device="cuda")
    even = torch.full((1, 1, v), 1.0 / v, device="cuda")
    for bad in (dict(probs=even.expand(b, n, v)), dict(logits=logits[:1, :1].expand(b, n + 1, v)),
                dict(logits=torch.zeros(v + 3, device="cuda").as_strided((1, 4, v), (0, 1, 1)), drafts=drafts[:1], u=u[:1])):
        with pytest.raises(ValueError):
            nh.verify_drafts(**{"logits": logits, "drafts": drafts, "u": u, **bad})
    kept, _ = nh.verify_drafts(logits, drafts, u, probs=even.expand(b, n, v).contiguous())
    assert kept.tolist() == [n] * b  # u q < p for equal p and q
