"""Rotary positions under autograd: rows that need gradients are refused rather than returned without their history;
inside a function of a caller's own, forwards and transposed, their gradients are the formula's."""
import numpy as np
import pytest
import torch

import rope_ref as ref

pytestmark = pytest.mark.gpu


def test_rows_that_need_gradients_are_refused(nh):
    plan = nh.Rope(16)
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    q, k = (torch.randn(5, h, 16, device="cuda") for h in (3, 2))
    plain = plan.apply(pos, q, k)
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    for call in (lambda: plan.apply(pos, a), lambda: plan.apply(pos, q, b), lambda: plan.apply(pos, a, b, transposed=True),
                 lambda: plan.apply(pos, 2.0 * a, k), lambda: plan.apply(pos, a, out=torch.empty_like(q))):
        with pytest.raises(ValueError, match="gradients"):
            call()
    # what needs none, and what asked for none
    for got in (plan.apply(pos, a.detach(), b.detach()), plan.apply(pos, q, k)):
        assert all(torch.equal(x, y) for x, y in zip(got, plain))
    with torch.no_grad():
        assert all(torch.equal(x, y) for x, y in zip(plan.apply(pos, a, b), plain))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_a_function_of_a_callers_own(nh, layout):
    rng = np.random.default_rng(5)
    plan = nh.Rope(24, layout=layout, scaling=("parts", 4.0, 64.0))
    positions = rng.integers(0, 5000, 7).astype(np.int32)

    class Turn(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, pos):
            ctx.save_for_backward(pos)
            return plan.apply(pos, x)

        @staticmethod
        def backward(ctx, g):
            return plan.apply(ctx.saved_tensors[0], g.contiguous(), transposed=True), None

    pos = torch.from_numpy(positions).cuda()
    x = torch.from_numpy(rng.standard_normal((7, 2, 40)).astype(np.float32)).cuda().requires_grad_()
    g = rng.standard_normal((7, 2, 40)).astype(np.float32)
    (Turn.apply(x, pos) * torch.from_numpy(g).cuda()).sum().backward()
    want = ref.turn(g, positions, plan.freqs, plan.amplitude, layout, True)
    # a cosine and a sine off by half a step of f32 each, two products and a sum: 4 half steps of |a| + |b|
    limit = 4 * 2.0 ** -24 * abs(plan.amplitude) * 2 * np.abs(g).max()
    assert np.abs(x.grad.cpu().numpy() - want.astype(np.float64)).max() <= limit
