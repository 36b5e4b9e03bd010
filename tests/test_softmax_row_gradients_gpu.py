"""Gradients per query that are not finite, or zero: they reach what they meet by
the formula (their own row of dQ, all of dC) and nothing else."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [(6, 40, 16), (70, 130, 33), (300, 700, 40)]


def step(t, v, d, dtype, grad, ignore=()):
    """(dq, dc) of sum(grad * loss); ignore: queries without a target."""
    import surfface_hip as S
    g = torch.Generator().manual_seed(t + v + d)
    q, c = torch.randn(t, d, generator=g).to(dtype).cuda(), torch.randn(v, d, generator=g).to(dtype).cuda()
    at = torch.randint(0, v, (t,), generator=g)
    for i in ignore:
        at[i] = -1
    qg, cg = q.requires_grad_(), c.requires_grad_()
    loss = S.softmax_loss(qg, cg, at.cuda(), scale=0.5, reduction="none")
    return [x.cpu() for x in torch.autograd.grad(loss, (qg, cg), grad.cuda())]


@pytest.mark.parametrize("t,v,d", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_every_gradient_not_finite(t, v, d, dtype, bad):
    dq, dc = step(t, v, d, dtype, torch.full((t,), bad), ignore=(1,))
    assert not dq[1].any()
    dq[1] = math.nan
    assert torch.isnan(dq).all() and torch.isnan(dc).all()


@pytest.mark.parametrize("t,v,d", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_one_gradient_not_finite_among_zeros(t, v, d, dtype, bad):
    grad = torch.zeros(t)
    grad[2] = bad
    dq, dc = step(t, v, d, dtype, grad)
    assert torch.isnan(dq[2]).all() and torch.isnan(dc).all()
    dq[2] = 0
    assert not dq.any()


@pytest.mark.parametrize("t,v,d", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_one_gradient_not_finite_among_others(t, v, d, dtype, bad):
    """The other rows of dQ: the bits that they have where the bad row takes no part."""
    grad = torch.linspace(-2, 3, t)
    grad[4] = bad
    dq, dc = step(t, v, d, dtype, grad)
    assert torch.isnan(dq[4]).all() and torch.isnan(dc).all()
    want, rest = step(t, v, d, dtype, grad, ignore=(4,))
    assert torch.isfinite(want).all() and torch.isfinite(rest).all() and want.any()
    dq[4] = 0
    assert torch.equal(dq, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_query_on_its_own(dtype):
    """One value for all queries, one query, one item (whose gradient is 0 times the value)."""
    for bad in (math.nan, math.inf):
        for t, v in ((1, 9), (1, 1), (3, 1)):
            dq, dc = step(t, v, 8, dtype, torch.full((t,), bad))
            assert torch.isnan(dq).all() and torch.isnan(dc).all()
    dq, dc = step(3, 9, 8, dtype, torch.zeros(3))
    assert not dq.any() and not dc.any()
