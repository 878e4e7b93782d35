"""The 8-bit cache's append beyond the threads that a launch has in one dimension."""
import numpy as np
import pytest
import torch

import kv8_ref as ref
from test_gpu_kv8 import plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("each", [True, False])
def test_more_workgroups_than_a_dimension_has(nh, each):
    """Few rows of 2^20 query heads: 131,072 workgroups a block of the queries, 2^24 and more in all."""
    rows = [1] * 129 if each else [1] * 128 + [2]
    n, heads = sum(rows), 1 << 20
    assert 2 ** 24 < (len(rows) if each else len(rows) + 1) * heads // 8 < 2 ** 26
    c = nh.KvCache8(1, 3, 2, 2, pages=len(rows), seqs=len(rows), cap=64)
    ids = [c.new_seq() for _ in rows]
    plan = nh.Rope(2)
    c.extend(ids, rows)
    k = torch.randn(n, 3, 2, dtype=torch.bfloat16, device="cuda")
    q = torch.empty(n, heads, 2, dtype=torch.bfloat16, device="cuda").normal_()
    pos = torch.arange(n, dtype=torch.int32, device="cuda") * 13 + 1
    got = c.append(0, k, k, rope=plan, positions=pos, q=q)
    assert torch.equal(got, plan.apply(pos, q))
    turned = plain(plan.apply(pos, k.float()))
    x, y = c.read(0, ids, [0] * len(ids), rows)
    at = 0
    for r in rows:
        assert np.array_equal(plain(y[at:at + r]), ref.quantize(plain(k[at:at + r])))
        assert np.array_equal(plain(x[at:at + r]), ref.quantize(turned[at:at + r]))
        at += r
