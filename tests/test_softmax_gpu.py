"""Softmax cross entropy over an item table and its gradients
(mn_softmax_stats, mn_softmax_merge, mn_softmax_backward) against the
definition in 64 bits.

Tolerances.  Half a step: u = 2^-24 (f32 sums, whose worst case over n terms is
n u of the sum of magnitudes), b = 2^-8 (a rounding to bf16).  With A = scale
max_ij sum_k |q_ik c_jk|, a logit is off by at most e = (6 d + 8) u A (6 d
products in the f32 form, none of which is rounded), and log-sum-exp by e and
the roundings of its own, 16 u (|lse| + log2 v): delta = 2 e + 16 u (1 + |lse|
+ log2 v) bounds what an exponent z - lse is off by, e^delta - 1 <= 2 delta an
entry of D relative to itself.  A gradient, sum_j D_ij c_jk, is off by at most
(2 delta + n u [+ b for D in bf16]) sum |D_ij c_jk|, and half a step of its own
type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, B = 2.0 ** -24, 2.0 ** -8


def data(t, v, d, dtype, seed, ignore=True):
    g = torch.Generator().manual_seed(seed)
    c = torch.randn(v, d, generator=g)
    c = c / c.norm(dim=1, keepdim=True)
    at = torch.randint(0, v, (t,), generator=g)
    q = c[at] + 0.7 * torch.randn(t, d, generator=g) / math.sqrt(d)
    if ignore:
        at[1::5] = -1
    return q.to(dtype), c.to(dtype), at


def formula(q, c, at, scale, grad=None):
    """(loss, dq, dc, sum |D c|, sum |D q|, delta) in f64; grad [t] f64 (mean where None)."""
    q, c = q.double(), c.double()
    d = q.shape[1]
    has = at >= 0
    z = scale * (q @ c.T)
    z[~has] = 0
    lse = torch.logsumexp(z, 1)
    rows = torch.arange(len(at))
    one = torch.zeros_like(z)
    one[rows[has], at[has]] = 1
    loss = torch.where(has, lse - (z * one).sum(1), 0.0)
    if grad is None:
        grad = torch.full((len(at),), 1.0 / max(1, int(has.sum())), dtype=torch.float64)
    D = (torch.exp(z - lse[:, None]) - one) * torch.where(has, grad, 0.0)[:, None]
    D[~has] = 0
    qz = torch.where(has[:, None], q, 0.0)
    A = scale * float((qz.abs() @ c.abs().T).max()) if len(at) else 0.0
    lmax = float(lse[has].abs().max()) if has.any() else 0.0
    delta = 2 * (6 * d + 8) * U * A + 16 * U * (1 + lmax + math.log2(c.shape[0] + 1))
    return (loss, scale * D @ c, scale * D.T @ qz, scale * D.abs() @ c.abs(), scale * D.abs().T @ qz.abs(), delta)


def close(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((err / tol.clamp(min=1e-300)).max()):.3g} times the bound"


def check_step(q, c, at, scale, dtype, loss, dq, dc, grad=None, mean=False):
    w_loss, w_dq, w_dc, s_dq, s_dc, delta = formula(q, c, at, scale, grad)
    has = at >= 0
    b = B if dtype == torch.bfloat16 else 0.0
    if mean:
        n = max(1, int(has.sum()))
        close(loss, w_loss.sum() / n, torch.tensor(2 * delta + (len(at) + 4) * U * float(w_loss.sum()) / n), "loss")
    else:
        close(loss, w_loss, 2 * delta + 4 * U * w_loss, "loss")
    out = b or U
    for got, want, mag, n, name in ((dq, w_dq, s_dq, c.shape[0], "dq"), (dc, w_dc, s_dc, len(at), "dc")):
        if got is not None:
            assert got.dtype == dtype and torch.isfinite(got).all()
            close(got, want, (2 * delta + (6 * n + 64) * U + b) * mag + out * want.abs() + 1e-40, name)


SIZES = [(1, 1, 1), (1, 2, 3), (2, 1, 5), (3, 130, 8), (16, 100, 64), (17, 257, 33), (64, 64, 96), (65, 300, 100),
         (130, 129, 40), (257, 700, 65), (300, 1500, 32), (5, 3000, 768), (70, 513, 257), (520, 260, 520)]


@pytest.mark.parametrize("t,v,d", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step(t, v, d, dtype):
    import surfface_hip as S
    q, c, at = data(t, v, d, dtype, t * 7 + v * 3 + d)
    qg, cg = q.cuda().requires_grad_(), c.cuda().requires_grad_()
    loss = S.softmax_loss(qg, cg, at.cuda(), scale=12.0)
    dq, dc = torch.autograd.grad(loss, (qg, cg))
    assert loss.dtype == torch.float32 and loss.dim() == 0
    check_step(q, c, at, 12.0, dtype, loss.detach(), dq, dc, mean=True)
    assert not dq.cpu()[at < 0].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_per_query_losses_and_gradients(dtype):
    """reduction none with a gradient per query (signs, a zero, sizes apart), and sum."""
    import surfface_hip as S
    q, c, at = data(37, 301, 48, dtype, 5)
    g = torch.linspace(-2, 3, 37)
    g[7] = 0
    g[8] = 1e-6
    qg, cg = q.cuda().requires_grad_(), c.cuda().requires_grad_()
    loss = S.softmax_loss(qg, cg, at.cuda(), scale=7.0, reduction="none")
    dq, dc = torch.autograd.grad(loss, (qg, cg), g.cuda())
    check_step(q, c, at, 7.0, dtype, loss.detach(), dq, dc, grad=g.double())
    loss = S.softmax_loss(qg, cg, at.cuda(), scale=7.0, reduction="sum")
    dq, dc = torch.autograd.grad(loss, (qg, cg))
    check_step(q, c, at, 7.0, dtype, S.softmax_loss(q.cuda(), c.cuda(), at.cuda(), 7.0, "none"), dq, dc,
               grad=torch.ones(37, dtype=torch.float64))


def test_gradient_against_differences():
    """Central differences of the loss itself along random directions (f32).

    The step h = 1/64 leaves a truncation of h^2 / 6 of the third derivative,
    which softmax bounds by (scale |direction| max|c|)^3 <= (2 * 1 * 1.2)^3, and
    two losses off by their bound (below 2e-5 here) over 2 h."""
    import surfface_hip as S
    q, c, at = data(9, 40, 16, torch.float32, 3, ignore=False)
    q, c, at = q.cuda(), c.cuda(), at.cuda()
    qg, cg = q.clone().requires_grad_(), c.clone().requires_grad_()
    dq, dc = torch.autograd.grad(S.softmax_loss(qg, cg, at, scale=2.0), (qg, cg))
    g = torch.Generator().manual_seed(1)
    h = 1 / 64
    for k in range(4):
        p = torch.randn(q.shape, generator=g)
        p = (p / p.norm()).cuda()
        diff = (S.softmax_loss(q + h * p, c, at, scale=2.0) - S.softmax_loss(q - h * p, c, at, scale=2.0)) / (2 * h)
        assert abs(float(diff) - float((dq * p).sum())) <= h * h / 6 * 2.4 ** 3 + 2e-5 / h
        p = torch.randn(c.shape, generator=g)
        p = (p / p.norm()).cuda()
        diff = (S.softmax_loss(q, c + h * p, at, scale=2.0) - S.softmax_loss(q, c - h * p, at, scale=2.0)) / (2 * h)
        assert abs(float(diff) - float((dc * p).sum())) <= h * h / 6 * (2 * 1 * 3) ** 3 + 2e-5 / h


@pytest.mark.parametrize("t,v,d", [(37, 300, 40), (100, 700, 64), (261, 1030, 20)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_logits(t, v, d, dtype):
    """Logits of several hundred, the last query's largest: exp of them, unlike
    exp of their distance to the log-sum-exp, is infinite.  (Terms below 2^-126
    may be flushed: n of them, times at most scale and 4.)"""
    import surfface_hip as S
    q, c, at = data(t, v, d, torch.float32, 31)
    q, at[-1] = q.abs() + 0.2, v - 1
    c[: v // 2] = c[: v // 2].abs()
    q[-1] *= 4
    q, c = q.to(dtype), c.to(dtype)
    qg, cg = q.cuda().requires_grad_(), c.cuda().requires_grad_()
    loss = S.softmax_loss(qg, cg, at.cuda(), scale=60.0)
    dq, dc = torch.autograd.grad(loss, (qg, cg))
    w_loss, w_dq, w_dc, s_dq, s_dc, delta = formula(q, c, at, 60.0)
    assert float((60 * q[-1].double() @ c.double().T).max()) > 300
    n = int((at >= 0).sum())
    close(loss.detach(), w_loss.sum() / n, torch.tensor(2 * delta + (t + 4) * U * float(w_loss.sum()) / n), "loss")
    b = B if dtype == torch.bfloat16 else 0.0
    for got, want, mag, k in ((dq, w_dq, s_dq, v), (dc, w_dc, s_dc, t)):
        close(got, want, (2 * delta + (6 * k + 64) * U + b) * mag + (b or U) * want.abs() + k * 240 * 2.0 ** -126, "gradient")


def test_small_losses_keep_their_precision():
    """Targets whose probability is nearly 1: loss and gradients relative to
    themselves, not to the logits: 1 - p = sum exp(z_j - z_t) is off by the
    exponents' delta only."""
    import surfface_hip as S
    v, d = 40, 48
    c = torch.eye(v, d)
    at = torch.arange(30)
    q = c[at] * 1.25
    q, c, scale = q.float(), c.float(), 16.0  # z: 20 at the target, 0 elsewhere
    qg, cg = q.cuda().requires_grad_(), c.cuda().requires_grad_()
    loss = S.softmax_loss(qg, cg, at.cuda(), scale=scale, reduction="none")
    dq, dc = torch.autograd.grad(loss.sum(), (qg, cg))
    want = math.log1p((v - 1) * math.exp(-20.0))
    assert (loss.detach().double().cpu() / want - 1).abs().max() <= 64 * U * 20
    w = formula(q, c, at, scale, torch.ones(30, dtype=torch.float64))
    assert ((dq.double().cpu() - w[1]).abs() <= 64 * U * 20 * w[3]).all()
    assert ((dc.double().cpu() - w[2]).abs() <= 64 * U * 20 * w[4]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_without_a_target_reach_nothing(dtype):
    """NaN and infinities in queries whose target is negative; a batch of only such."""
    import surfface_hip as S
    q, c, at = data(40, 200, 36, dtype, 9)
    out = []
    for bad in (False, True):
        x = q.clone()
        if bad:
            x[at < 0] = float("nan")
            x[6] = float("inf")
        xg, cg = x.cuda().requires_grad_(), c.cuda().requires_grad_()
        assert at[6] < 0
        loss = S.softmax_loss(xg, cg, at.cuda(), scale=5.0)
        out.append([loss.detach(), *torch.autograd.grad(loss, (xg, cg))])
    for a, b in zip(*out):
        assert torch.isfinite(b).all() and torch.equal(a, b)
    none = torch.full((40,), -100)
    xg, cg = q.cuda().requires_grad_(), c.cuda().requires_grad_()
    loss = S.softmax_loss(xg, cg, none.cuda(), scale=5.0)
    dq, dc = torch.autograd.grad(loss, (xg, cg))
    assert loss.item() == 0 and not dq.any() and not dc.any()


def test_masked_items_extreme_logits_and_missing_targets():
    """Items at the lowest value of the type, logits of 1e4, a target outside the table, one item."""
    import surfface_hip as S
    q, c, at = data(6, 50, 8, torch.float32, 2, ignore=False)
    q[:, 0], c[:, 0] = 1.0, 0.0
    c[10:20, 0] = torch.finfo(torch.float32).min
    at[:] = torch.arange(6)
    loss = S.softmax_loss(q.cuda(), c.cuda(), at.cuda(), scale=1.0, reduction="none").cpu()
    keep = torch.cat([c[:10], c[20:]])
    w = formula(q, keep, at, 1.0)
    assert (loss.double() - w[0]).abs().max() <= 2 * w[5]
    big = S.softmax_loss((q * 1e4).cuda(), keep.cuda(), at.cuda(), reduction="none").cpu()
    wb = formula(q * 1e4, keep, at, 1.0)
    assert (big.double() - wb[0]).abs().max() <= 2 * wb[5]
    at[2] = 50
    assert torch.isinf(S.softmax_loss(q.cuda(), c.cuda(), at.cuda(), reduction="none"))[2]
    one = S.softmax_loss(q.cuda(), c[:1].cuda(), torch.zeros(6, dtype=torch.int64).cuda(), reduction="none")
    assert not one.any()
    bad = q.clone()
    bad[4, 3] = float("nan")
    assert torch.isnan(S.softmax_loss(bad.cuda(), keep.cuda(), torch.zeros(6).long().cuda(), reduction="none"))[4]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_row_ranges_of_a_table_join(dtype):
    """Stats of three ranges, merged; gradients of the ranges against the whole table's."""
    import surfface_hip as S
    q, c, at = data(50, 400, 40, dtype, 11)
    qd, cd, ad = q.cuda(), c.cuda(), at.cuda()
    cut = [0, 1, 150, 400]
    parts = [S.softmax_stats(qd, cd[a:b], ad, 6.0, c_offset=a) for a, b in zip(cut, cut[1:])]
    st = S.softmax_merge(torch.stack([p.rest for p in parts]), torch.stack([p.target for p in parts]), ad)
    one = torch.ones(1).cuda()
    got = [S.softmax_backward(qd, cd[a:b], ad, st.rest, st.target, one, 6.0, c_offset=a, grad_scale=st.share)
           for a, b in zip(cut, cut[1:])]
    dq = sum(g[0].double() for g in got).cpu()
    dc = torch.cat([g[1] for g in got])
    check_step(q, c, at, 6.0, dtype, st.mean, None, dc, mean=True)
    w = formula(q, c, at, 6.0)
    b = B if dtype == torch.bfloat16 else 0.0
    close(dq, w[1], (2 * w[5] + 3000 * U + b + 3 * (b or U)) * w[3] + 1e-40, "dq")
    only = S.softmax_backward(qd, cd, ad, st.rest, st.target, one, 6.0, grad_scale=st.share, need=(False, True))
    assert only[0] is None and torch.equal(only[1], S.softmax_backward(
        qd, cd, ad, st.rest, st.target, one, 6.0, grad_scale=st.share)[1])


def test_nan_in_the_target_s_row_survives_the_join():
    """A NaN in an item is in no other item's logit: the row's rest is finite, its loss NaN."""
    import surfface_hip as S
    q, c, at = data(9, 80, 12, torch.float32, 21, ignore=False)
    at[:] = torch.arange(9) * 8
    c[at[4], 5] = float("nan")
    qd, cd, ad = q.cuda(), c.cuda(), at.cuda()
    parts = [S.softmax_stats(qd, cd[a:b], ad, 2.0, c_offset=a) for a, b in ((0, 40), (40, 80))]
    st = S.softmax_merge(torch.stack([p.rest for p in parts]), torch.stack([p.target for p in parts]), ad)
    for x in (st, S.softmax_stats(qd, cd, ad, 2.0)):
        assert torch.isfinite(x.rest[4]) and torch.isnan(x.target[4]) and torch.isnan(x.loss).all() and torch.isnan(x.mean)
    one = qd.clone()
    one[3] = float("nan")
    alone = S.softmax_stats(one, cd[:1], torch.zeros(9, dtype=torch.int64).cuda())
    assert torch.isnan(alone.loss[3]) and not alone.loss[:3].any()


def test_calls_by_name_and_streams_of_another_device():
    import surfface_hip as S
    q, c, at = (x.cuda() for x in data(20, 60, 16, torch.float32, 27))
    a = S.softmax_stats(queries=q, items=c, targets=at, scale=2.0)
    b = S.softmax_stats(q, c, at, 2.0)
    assert torch.equal(a.loss, b.loss)
    rows = S.quantize_rows(X=q)
    assert torch.equal(S.scores_i8(queries=rows, items=rows), S.scores_i8(rows, rows))

    class Elsewhere:
        device = torch.device("cuda", 1)
    for bad in (lambda: S.softmax_loss(q, c, at, stream=Elsewhere()), lambda: S.quantize_rows(X=q, stream=Elsewhere()),
                lambda: S.scores_i8(rows, rows, stream=Elsewhere())):
        with pytest.raises(ValueError, match="stream is on"):
            bad()


def test_same_target_many_times_and_int32_targets():
    import surfface_hip as S
    q, c, at = data(200, 90, 24, torch.float32, 13, ignore=False)
    at[:] = 17
    qg, cg = q.cuda().requires_grad_(), c.cuda().requires_grad_()
    loss = S.softmax_loss(qg, cg, at.int().cuda(), scale=3.0)
    dq, dc = torch.autograd.grad(loss, (qg, cg))
    check_step(q, c, at, 3.0, torch.float32, loss.detach(), dq, dc, mean=True)


def test_views_streams_and_repeats():
    """Rows off a border, strided inputs, another stream; the same bits every time."""
    import surfface_hip as S
    q, c, at = data(70, 310, 30, torch.bfloat16, 17)
    wide = torch.zeros(310, 50, dtype=torch.bfloat16, device="cuda")
    wide[:, 11:41] = c.cuda()
    more = torch.zeros(71, 30, dtype=torch.bfloat16, device="cuda")
    more[1:] = q.cuda()
    runs = []
    for qq, cc in ((q.cuda(), c.cuda()), (more[1:], wide[:, 11:41]), (q.cuda(), c.cuda())):
        st = S.softmax_stats(qq, cc, at.cuda(), 9.0)
        runs.append([st.loss, st.mean, *S.softmax_backward(qq, cc, at.cuda(), st.rest, st.target,
                                                           torch.ones(1).cuda(), 9.0, grad_scale=st.share)])
    s = torch.cuda.Stream()
    qd, cd, ad, one = q.cuda(), c.cuda(), at.cuda(), torch.ones(1).cuda()
    s.wait_stream(torch.cuda.current_stream())
    st = S.softmax_stats(qd, cd, ad, 9.0, stream=s)
    dq, dc = S.softmax_backward(qd, cd, ad, st.rest, st.target, one, 9.0, grad_scale=st.share, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    runs.append([st.loss, st.mean, dq, dc])
    for r in runs[1:]:
        for a, b in zip(runs[0], r):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_steps(dtype):
    """Two graphs of a step (each with its own workspace), replayed in turn with eager work between."""
    import surfface_hip as S
    q, c, at = data(48, 500, 64, dtype, 19)
    cd, one = c.cuda(), torch.ones(1).cuda()

    def step(x, a):
        st = S.softmax_stats(x, cd, a, 8.0)
        return [st.mean, *S.softmax_backward(x, cd, a, st.rest, st.target, one, 8.0, grad_scale=st.share)]

    step(q.cuda(), at.cuda())
    graphs = []
    for k in range(2):
        x, a = q.cuda(), at.cuda()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(x, a)
        graphs.append((g, x, a, out))
    for k in range(3):
        for n, (g, x, a, out) in enumerate(graphs):
            x.copy_((q.float() * (1 + k + n)).to(dtype))
            a.copy_(at.roll(k + 2 * n))
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, x, a, out in graphs:
            for got, want in zip(out, step(x, a)):
                assert torch.equal(got, want)


def test_capture_of_the_loss():
    """Without gradients: replays equal the eager call, each reduction; with: refused."""
    import surfface_hip as S
    q, c, at = data(300, 500, 32, torch.float32, 29)
    x, cd, a = q.cuda(), c.cuda(), at.cuda()
    kinds = ("mean", "sum", "none")
    want = [S.softmax_loss(x, cd, a, 5.0, k) for k in kinds]
    # a sum over t f32 losses, a product and a quotient
    close(want[1], want[2].double().sum().cpu(), (len(at) + 4) * U * want[2].double().sum().cpu(), "sum")
    cg = cd.clone().requires_grad_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="graph capture"):
            S.softmax_loss(x, cg, a)
        with torch.no_grad():
            out = [S.softmax_loss(x, cg, a, 5.0, k) for k in kinds]
    for k in range(3):
        x.copy_((q * (1 + k)).cuda())
        want = [S.softmax_loss(x, cd, a, 5.0, k) for k in kinds]
        g.replay()
        torch.cuda.synchronize()
        for o, w in zip(out, want):
            assert torch.equal(o, w)


def test_autograd_rules():
    """Gradients add up, a kept graph gives the same bits, what torch forbids is refused, a table that is its
    own queries, views (strided, expanded)."""
    import surfface_hip as S
    q, c, at = (x.cuda() for x in data(100, 300, 40, torch.float32, 33))
    q.requires_grad_(), c.requires_grad_()
    S.softmax_loss(q, c, at).backward()
    once = c.grad.clone()
    S.softmax_loss(q, c, at).backward()
    assert torch.equal(c.grad, 2 * once)
    loss = S.softmax_loss(q, c, at)
    a = torch.autograd.grad(loss, c, retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(loss, c)[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, c)
    first = torch.autograd.grad(S.softmax_loss(q, c, at), c, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), c)
    loss = S.softmax_loss(q, c, at)
    with torch.no_grad():
        c.mul_(2)
    with pytest.raises(RuntimeError):
        loss.backward()

    g = torch.Generator().manual_seed(34)
    x, t = torch.randn(200, 32, generator=g), torch.arange(200)
    xg = x.cuda().requires_grad_()
    got = torch.autograd.grad(S.softmax_loss(xg, xg, t.cuda(), 0.5), xg)[0]
    _, w_dq, w_dc, s_dq, s_dc, delta = formula(x, x, t, 0.5)
    close(got, w_dq + w_dc, (2 * delta + (6 * 200 + 64) * U) * (s_dq + s_dc) + 3 * U * (w_dq.abs() + w_dc.abs()), "own queries")

    wide = torch.randn(200, 64, generator=g)
    wg = wide.cuda().requires_grad_()
    dq, = torch.autograd.grad(S.softmax_loss(wg[:, ::2], xg.detach(), t.cuda(), 0.5), wg)
    _, w_dq, _, s_dq, _, delta = formula(wide[:, ::2].contiguous(), x, t, 0.5)
    assert not dq[:, 1::2].any()
    close(dq[:, ::2], w_dq, (2 * delta + (6 * 200 + 64) * U) * s_dq + U * w_dq.abs(), "strided")
    e = torch.randn(5, 1, generator=g).cuda().expand(5, 32)
    assert torch.equal(S.softmax_loss(e, xg.detach(), t[:5].cuda()), S.softmax_loss(e.contiguous(), xg.detach(), t[:5].cuda()))


def test_empty_batch_and_refusals():
    import surfface_hip as S
    q, c, at = (x.cuda() for x in data(8, 30, 16, torch.float32, 1))
    e = q[:0].clone().requires_grad_()
    cg = c.clone().requires_grad_()
    loss = S.softmax_loss(e, cg, at[:0])
    dq, dc = torch.autograd.grad(loss, (e, cg))
    assert loss.item() == 0 and dq.shape == (0, 16) and not dc.any()
    for bad in (lambda: S.softmax_loss(q, c[:, :8], at), lambda: S.softmax_loss(q, c, at[:5]),
                lambda: S.softmax_loss(q, c[:0], at), lambda: S.softmax_loss(q, c, at, reduction="max"),
                lambda: S.softmax_backward(q, c, at, at.float()[:3], at.float(), at.float()),
                lambda: S.softmax_backward(q, c, at, at.float(), at.float(), at.float()[:3])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: S.softmax_loss(q, c.bfloat16(), at), lambda: S.softmax_loss(q.half(), c.half(), at),
                lambda: S.softmax_loss(q.cpu(), c, at), lambda: S.softmax_loss(q, c, at.float())):
        with pytest.raises(TypeError):
            bad()
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(S.MnError):
            S.softmax_loss(q, c, at, scale=scale)
    with pytest.raises(S.MnError):
        S.softmax_stats(q, c, at, c_offset=-1)


def test_train_quantize_serve():
    """The operators as they are used together: steps of training on a table, the
    table and the queries quantised, the scores of 8 bits against the formula's
    error bound of quantisation, and the same best item where it is ahead by
    more than that."""
    import surfface_hip as S
    q, c, at = data(256, 1000, 64, torch.float32, 23, ignore=False)
    table = c.cuda().requires_grad_()
    queries, ad = q.cuda(), at.cuda()
    for _ in range(5):
        loss = S.softmax_loss(queries, table, ad, scale=10.0)
        (dc,) = torch.autograd.grad(loss, (table,))
        with torch.no_grad():
            table -= 2.0 * dc
    t = table.detach()
    q8, c8 = S.quantize_rows(queries), S.quantize_rows(t)
    got = S.scores_i8(q8, c8).double().cpu()
    x, y = queries.double().cpu(), t.double().cpu()
    want = x @ y.T
    # a code is off by at most (1/2 + 127 * 2 u) of its scale
    sq, sc = 0.5001 * q8.scale.double().cpu()[:, None], 0.5001 * c8.scale.double().cpu()[None]
    tol = sq * y.abs().sum(1) + sc * x.abs().sum(1, keepdim=True) + 64 * sq * sc + 4 * U * want.abs()
    assert ((got - want).abs() <= tol).all()
    top = want.topk(2, 1)
    clear = (top.values[:, 0] - top.values[:, 1]) > 2 * tol.max(1).values
    assert clear.any() and torch.equal(got.argmax(1)[clear], top.indices[clear, 0])
