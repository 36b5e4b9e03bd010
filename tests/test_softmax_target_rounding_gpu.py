"""dC of the softmax loss in bf16: the entry of a query's target, the largest of its
item by far, is not rounded to bf16.

With D = p - [j = t(i)] cut into the targets' entries and the others, b = 2^-8
and the terms of test_softmax_gpu.py, an entry of dC is off by at most (2 delta +
(t + 64) u) sum |D_ij q_i|, b of the others' part of that sum, b^2 of the targets'
(a rounding's rest is rounded itself) and half a step of its own type.  Where the
others weigh little (fewer queries than a third of the items) and enough queries
are there for a large rounding (one a query), it is checked too that the formula
with the targets' entries rounded to bf16 is outside the bound."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, B = 2.0 ** -24, 2.0 ** -8
CHUNK = 16384


def data(t, v, d, seed):
    """Queries near their target's item, of different lengths, so that its probability is anything; some without a target."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = torch.empty(v, d, device="cuda", dtype=torch.bfloat16)
    for j in range(0, v, CHUNK):
        x = torch.randn(min(CHUNK, v - j), d, device="cuda", generator=g)
        c[j:j + CHUNK] = (x / x.norm(dim=1, keepdim=True)).bfloat16()
    at = torch.randint(0, v, (t,), device="cuda", generator=g)
    at[0], at[1] = v - 1, 0
    q = c[at].float() + 0.2 * torch.randn(t, d, device="cuda", generator=g) / math.sqrt(d)
    q = (q * (0.6 + torch.rand(t, 1, device="cuda", generator=g))).bfloat16()
    at[3::7] = -1
    return q, c, at


def check(q, c, at, dc, scale, lo=0, hi=None):
    """dc: gradient of the mean loss, rows lo .. hi - 1 of the items."""
    t, v = len(at), c.shape[0]
    has = at >= 0
    n = int(has.sum())
    x = torch.where(has[:, None], q.double(), 0.0)
    lse = torch.full((t,), -math.inf, dtype=torch.float64, device="cuda")
    most = 0.0
    for j in range(0, v, CHUNK):
        y = c[j:j + CHUNK].double().t().contiguous()
        lse = torch.logaddexp(lse, torch.logsumexp(scale * (x @ y), 1))
        most = max(most, scale * float((x.abs() @ y.abs()).max()))
    delta = 2 * (6 * q.shape[1] + 8) * U * most + 16 * U * (1 + float(lse[has].abs().max()) + math.log2(v + 1))
    told = False
    hi = v if hi is None else hi
    assert len(dc) == hi - lo
    for j in range(lo, hi, CHUNK):
        y = c[j:min(j + CHUNK, hi)].double()
        D = torch.exp(scale * (x @ y.t().contiguous()) - lse[:, None]) * (has / n)[:, None]
        here = ((at >= j) & (at < j + len(y))).nonzero()[:, 0]
        T = torch.zeros_like(D)
        T[here, at[here] - j] = D[here, at[here] - j] - 1.0 / n
        D[here, at[here] - j] = 0.0
        others, targets = scale * (D.t().contiguous() @ x.abs()), scale * (T.abs().t().contiguous() @ x.abs())
        want = scale * ((D + T).t().contiguous() @ x)
        tol = (2 * delta + (t + 64) * U) * (others + targets) + B * others + B * B * targets + B * want.abs() + 1e-30
        got = dc[j - lo:j - lo + len(y)].double()
        assert ((got - want).abs() <= tol).all(), f"items from {j}"
        bad = (want + scale * (((T * n).bfloat16().double() / n - T).t().contiguous() @ x)).bfloat16().double()
        told = told or bool(((bad - want).abs() > tol).any())
    assert told or t < 300 or 3 * t > v


@pytest.mark.parametrize("t,v,d", [(700, 1500, 33), (64, 64, 96), (33, 300, 260), (1000, 40, 100), (5, 7, 3), (3000, 500, 200),
                                   (300, 530001, 16),    # two pieces
                                   (9001, 33500, 64),    # more queries in a block than are looked at together
                                   (70001, 40, 2100)])   # the same, and every one's target is in the tile
def test_targets_in_full_precision(t, v, d):
    import surfface_hip as S
    q, c, at = data(t, v, d, t + v + d)
    cg = c.clone().requires_grad_()
    scale = math.log(v) + 1.0
    dc, = torch.autograd.grad(S.softmax_loss(q, cg, at, scale=scale), cg)
    check(q, c, at, dc, scale)


def test_ranges_and_one_target_for_all():
    import surfface_hip as S
    q, c, at = data(200, 900, 48, 5)
    st = S.softmax_stats(q, c, at, 3.0)
    one = torch.ones(1, device="cuda")
    for lo, hi in ((0, 300), (300, 301), (301, 900)):
        _, dc = S.softmax_backward(q, c[lo:hi], at, st.rest, st.target, one, 3.0, c_offset=lo, grad_scale=st.share)
        check(q, c, at, dc, 3.0, lo, hi)
    c = c[:500].clone()
    at[:] = 450
    st = S.softmax_stats(q, c, at, 3.0)
    _, dc = S.softmax_backward(q, c, at, st.rest, st.target, one, 3.0, grad_scale=st.share)
    check(q, c, at, dc, 3.0)
    again = S.softmax_backward(q, c, at, st.rest, st.target, one, 3.0, grad_scale=st.share)[1]
    assert torch.equal(dc, again)
