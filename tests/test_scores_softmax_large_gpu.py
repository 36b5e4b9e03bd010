"""Item scores and softmax loss where the sizes decide: tables in several pieces,
partial sums added up, every class of the kernels for few queries, offsets past
2^31 and 2^32, several threads at once.  References in 64 bits, in chunks on the
GPU; tolerances as in test_softmax_gpu.py."""
import math
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

U, B = 2.0 ** -24, 2.0 ** -8
CHUNK = 65536


def make(t, v, d, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = torch.empty(v, d, dtype=dtype, device="cuda")
    for j in range(0, v, CHUNK):
        x = torch.randn(min(CHUNK, v - j), d, generator=g, device="cuda")
        c[j:j + CHUNK] = (x / x.norm(dim=1, keepdim=True)).to(dtype)
    at = torch.randint(0, v, (t,), generator=g, device="cuda")
    q = (c[at].float() + 0.7 * torch.randn(t, d, generator=g, device="cuda") / math.sqrt(d)).to(dtype)
    at[0] = v - 1
    at[1::5] = -1
    return q, c, at


def worst(got, want, tol):
    return float(((got.double() - want).abs() / tol).nan_to_num(nan=math.inf).max())


def check(t, v, d, dtype, seed, scale=8.0):
    import surfface_hip as S
    q, c, at = make(t, v, d, dtype, seed)
    qg, cg = q.clone().requires_grad_(), c.requires_grad_()
    loss = S.softmax_loss(qg, cg, at, scale=scale, reduction="none")
    n = int((at >= 0).sum())
    dq, dc = torch.autograd.grad(loss, (qg, cg), torch.full((t,), 1.0 / n, device="cuda"))
    c = c.detach()
    has = at >= 0
    x = torch.where(has[:, None], q.double(), 0.0)
    zt = scale * (x * c[at.clamp(min=0)].double()).sum(1)
    rest, A = torch.full((t,), -math.inf, dtype=torch.float64, device="cuda"), 0.0
    rows = torch.arange(t, device="cuda")

    def logits(j):
        y = c[j:j + CHUNK].double()
        here = (at >= j) & (at < j + y.shape[0])
        return y, scale * (x @ y.T), rows[here], at[here] - j

    for j in range(0, v, CHUNK):
        y, z, r, k = logits(j)
        z[r, k] = -math.inf
        rest = torch.logaddexp(rest, torch.logsumexp(z, 1))
        A = max(A, scale * float((x.abs() @ y.abs().T).max()))
    lse = torch.logaddexp(rest, zt)
    want = torch.where(has, lse - zt, 0.0)
    delta = 2 * (6 * d + 8) * U * A + 16 * U * (1 + float(lse.abs().max()) + math.log2(v + 1))
    b = B if dtype == torch.bfloat16 else 0.0
    assert worst(loss.detach(), want, 2 * delta + 4 * U * want) <= 1
    w_dq, s_dq = torch.zeros(t, d, dtype=torch.float64, device="cuda"), 0
    for j in range(0, v, CHUNK):
        y, z, r, k = logits(j)
        D = torch.exp(z - lse[:, None])
        D[r, k] -= 1
        D *= torch.where(has, 1.0 / n, 0.0)[:, None]
        w_dq += scale * (D @ y)
        s_dq = s_dq + scale * (D.abs() @ y.abs())
        w, mag = scale * (D.T @ x), scale * (D.abs().T @ x.abs())
        tol = (2 * delta + (6 * t + 64) * U + b) * mag + (b or U) * w.abs() + t * 4 * scale * 2.0 ** -126
        assert worst(dc[j:j + CHUNK], w, tol) <= 1, f"items from {j}"
    tol = (2 * delta + (6 * v + 64) * U + b) * s_dq + (b or U) * w_dq.abs() + 1e-30
    assert worst(dq, w_dq, tol) <= 1
    assert not dq[~has].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pieces_of_a_table(dtype):
    """Three (bf16) and five (f32) pieces, the last one short and odd, many partial sums of dQ."""
    check(300, 530001, 16, dtype, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_partial_sums_added_up(dtype):
    """Partial sums of dQ above 256 MB in all: each piece adds to those before."""
    check(4096, 150001, 2048, dtype, 2)


@pytest.mark.parametrize("dtype,v", [(torch.float32, 1500001), (torch.bfloat16, 3000001)])
def test_tables_past_32_bits(dtype, v):
    """4.6 GB of items: targets and gradients at the far end among them."""
    check(70, v, 768, dtype, 3)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,t,d", [
    (torch.bfloat16, t, d) for t, d in ((1, 1288), (16, 4600), (16, 4616), (1, 65536), (17, 640), (32, 648), (33, 320), (64, 328),
                                        (64, 1152), (64, 1160), (50, 331))] + [
    (torch.float32, t, d) for t, d in ((1, 640), (16, 644), (16, 2304), (5, 2308), (17, 320), (32, 324), (31, 1152), (32, 1156),
                                       (33, 40), (20, 323))])
def test_stats_of_few_queries(dtype, t, d):
    """Both sides of every border between the kernels for few queries, loss against the formula."""
    check(t, 701, d, dtype, t + d, scale=4.0)


@pytest.mark.parametrize("t,v,d", [(33, 700, 580), (64, 300, 1160), (40, 901, 2304), (31, 129, 1200), (65, 500, 768),
                                   (130, 1003, 772), (500, 1500, 130), (700, 300, 1000), (1024, 500, 768), (1030, 40, 2048)])
def test_groups_of_queries_in_f32(t, v, d):
    """Queries that LDS does not hold at once, with both sides of the rules that choose the kernel."""
    check(t, v, d, torch.float32, t + v, scale=4.0)


@pytest.mark.parametrize("t,v,d", [(2049, 10001, 33), (2000, 10003, 64), (701, 30011, 40), (1025, 20001, 129), (300, 60001, 768),
                                   (4097, 6007, 16), (3000, 9001, 1), (2500, 8192, 1000), (70, 60001, 775)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tiles_with_odd_ends(t, v, d, dtype):
    """Enough tiles that both passes go to the kernels of 256 x 256 (128) tiles; ends inside a tile and a k-step."""
    check(t, v, d, dtype, t + v + d, scale=5.0)


@pytest.mark.parametrize("m,n,d", [(2049, 16001, 33), (1999, 16003, 64), (4097, 8200, 768), (513, 64001, 100), (70, 90001, 769),
                                   (3001, 20011, 1), (2050, 9003, 200), (256, 131072, 192), (65, 60001, 2000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_in_tiles_with_odd_ends(m, n, d, dtype):
    import surfface_hip as S
    g = torch.Generator(device="cuda").manual_seed(m + n + d)
    q, c = S.quantize_rows(torch.randn(m, d, generator=g, device="cuda")), S.quantize_rows(torch.randn(n, d, generator=g, device="cuda"))
    y = S.scores_i8(q, c, dtype)
    for j in range(0, n, CHUNK):
        exact = (q.codes[:, :d].double() @ c.codes[j:j + CHUNK, :d].double().T) * q.scale.double()[:, None] * \
            c.scale[j:j + CHUNK].double()
        tol = exact.abs() * (3.01 * U + (B if dtype == torch.bfloat16 else 0)) + 1e-44
        assert worst(y[:, j:j + CHUNK], exact, tol) <= 1


@pytest.mark.parametrize("m,n,d", [(65, 1500, 64), (700, 3001, 384), (1000, 1003, 1025), (130, 40001, 33), (2040, 50, 65),
                                   (100, 200, 9000), (300, 77, 40000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_of_groups_of_queries(m, n, d, dtype):
    test_scores_in_tiles_with_odd_ends(m, n, d, dtype)


@pytest.mark.parametrize("m,d", [(1, 2560), (16, 2561), (16, 9216), (3, 9217), (17, 1280), (32, 1281), (32, 4608), (20, 4609),
                                 (33, 640), (64, 641), (64, 2304), (64, 2305)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_of_few_queries(dtype, m, d):
    import surfface_hip as S
    g = torch.Generator(device="cuda").manual_seed(m + d)
    q, c = S.quantize_rows(torch.randn(m, d, generator=g, device="cuda")), S.quantize_rows(torch.randn(333, d, generator=g, device="cuda"))
    exact = (q.codes[:, :d].double() @ c.codes[:, :d].double().T) * q.scale.double()[:, None] * c.scale.double()
    tol = exact.abs() * (3.01 * U + (B if dtype == torch.bfloat16 else 0)) + 1e-44
    assert worst(S.scores_i8(q, c, dtype), exact, tol) <= 1


@pytest.mark.parametrize("m", [2, 70])
def test_scores_of_a_table_past_32_bits(m):
    """6M rows of 768 codes (4.6 GB) from bf16 rows of 9.2 GB; scores of 1.7 GB."""
    import surfface_hip as S
    n, d = 6_000_001, 768
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
    for j in range(0, n, 1 << 20):
        x[j:j + (1 << 20)] = torch.randn(min(1 << 20, n - j), d, generator=g, device="cuda").bfloat16()
    c, q = S.quantize_rows(x), S.quantize_rows(x[-m:])
    y = S.scores_i8(q, c)
    back = S.dequantize_rows(c, torch.bfloat16)
    for j in (0, (1 << 31) // d - 500, (1 << 32) // d - 500, n - 1000):
        part = S.quantize_rows(x[j:j + 1000])
        assert torch.equal(part.codes, c.codes[j:j + 1000]) and torch.equal(part.scale, c.scale[j:j + 1000])
        assert torch.equal(back[j:j + 1000], S.dequantize_rows(part, torch.bfloat16))
        exact = (q.codes.double() @ part.codes.double().T) * q.scale.double()[:, None] * part.scale.double()
        assert worst(y[:, j:j + 1000], exact, exact.abs() * 3.01 * U + 1e-44) <= 1
    del x, c, y, back
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_past_32_bits_of_output(dtype):
    """2100 x 1.1M scores: 2.3e9 of them."""
    import surfface_hip as S
    g = torch.Generator(device="cuda").manual_seed(5)
    q = S.quantize_rows(torch.randn(2100, 40, generator=g, device="cuda"))
    c = S.quantize_rows(torch.randn(1_100_003, 40, generator=g, device="cuda"))
    y = S.scores_i8(q, c, dtype)
    rows = torch.tensor([0, 1951, 1952, 1953, 2047, 2048, 2099], device="cuda")  # 1952 n: 2^31
    for j in (0, 500_000, 1_100_003 - 70_000):
        exact = (q.codes[rows].double() @ c.codes[j:j + 70_000].double().T) * q.scale[rows].double()[:, None] * \
            c.scale[j:j + 70_000].double()
        tol = exact.abs() * (3.01 * U + (B if dtype == torch.bfloat16 else 0)) + 1e-44
        assert worst(y[rows, j:j + 70_000], exact, tol) <= 1
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [20, 130])
def test_items_masked_with_the_lowest_value(dtype, t):
    """A column that gives masked items the type's lowest value: no loss, no gradient, no NaN from them."""
    import surfface_hip as S
    q, c, at = make(t, 900, 24, dtype, 8)
    q[:, 0] = 1.0
    c[:, 0] = 0.0
    keep = torch.ones(900, dtype=torch.bool, device="cuda")
    keep[at.clamp(min=0)] = False
    masked = keep & (torch.arange(900, device="cuda") % 3 == 0)
    full = c.clone()
    full[masked, 0] = torch.finfo(dtype).min
    new = torch.cumsum(~masked, 0) - 1  # an item's place in the table without the masked ones
    out = []
    for table, goal in ((full, at), (c[~masked].contiguous(), torch.where(at >= 0, new[at.clamp(min=0)], -1))):
        qg, cg = q.clone().requires_grad_(), table.requires_grad_()
        loss = S.softmax_loss(qg, cg, goal, 6.0, "none")
        out.append([loss.detach(), *torch.autograd.grad(loss.mean(), (qg, cg))])
    (l0, q0, c0), (l1, q1, c1) = out
    assert torch.isfinite(q0).all() and torch.isfinite(c0).all() and not c0[masked].any()
    # both within their bounds of the same formula; see test_softmax_gpu.py for the terms
    A = 6.0 * float((q.double().abs() @ c.double().abs().T).max())
    delta = 2 * (6 * 24 + 8) * U * A + 16 * U * (1 + A + 10)
    assert ((l0 - l1).abs().double() <= 4 * delta + 8 * U * l1).all()
    b = B if dtype == torch.bfloat16 else U
    for a, w, mag in ((q0, q1, 12.0 / t * c.double().abs().max(0).values), (c0[~masked], c1, 12.0 / t * q.double().abs().sum(0))):
        assert ((a.double() - w.double()).abs() <= 2 * (2 * delta + 6000 * U + 2 * b) * mag).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,v,d", [(70001, 50, 16), (20000, 3, 9), (3, 70001, 1), (9, 2, 4100), (4100, 700, 8), (1, 300, 65536), (262144, 1300, 20), (5003, 600, 200)])
def test_lopsided_shapes(t, v, d, dtype):
    check(t, v, d, dtype, t + 3 * v + d, scale=3.0)


GUARD = 1 << 16


def guarded(n, dtype):
    """n values between two guards, 16 bytes past a larger border; and the whole buffer."""
    size = torch.empty(0, dtype=dtype).element_size()
    whole = torch.full((2 * GUARD + 16 + n * size,), 0x5a, dtype=torch.uint8, device="cuda")
    at = GUARD + 16
    return whole[at:at + n * size].view(dtype), whole, at, n * size


def untouched(*buffers):
    for _, whole, at, n in buffers:
        assert (whole[:at] == 0x5a).all() and (whole[at + n:] == 0x5a).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,v,d", [(1, 1, 1), (5, 130, 7), (33, 700, 100), (70, 513, 65), (130, 1000, 260), (300, 40, 33), (2000, 40, 70)])
def test_nothing_but_the_outputs_and_the_workspace_is_written(t, v, d, dtype):
    """The C entries with a workspace of exactly the size asked for, 16-byte aligned and no more."""
    import ctypes as C

    from surfface_hip import _lib
    L, kind = _lib.lib(), {torch.float32: _lib.MN_F32, torch.bfloat16: _lib.MN_BF16}[dtype]
    q, c, at = make(t, v, d, dtype, 40)
    n = C.c_size_t()
    P = lambda g: C.c_void_p(g[0].data_ptr())
    D = lambda x: C.c_void_p(x.data_ptr())
    st = torch.cuda.current_stream().cuda_stream
    f = lambda k: guarded(k, torch.float32)
    rest, zt, loss, mean, share = f(t), f(t), f(t), f(1), f(1)
    _lib.check(L.mn_softmax_workspace(t, v, d, kind, 0, C.byref(n)))
    ws = guarded(n.value, torch.uint8)
    _lib.check(L.mn_softmax_stats(D(q), D(c), kind, t, v, d, D(at), 0, 2.0, P(rest), P(zt), P(loss), P(mean), P(share),
                                  P(ws), n.value, st))
    _lib.check(L.mn_softmax_workspace(t, v, d, kind, 1, C.byref(n)))
    wb = guarded(n.value, torch.uint8)
    dq, dc = guarded(t * d, dtype), guarded(v * d, dtype)
    one = torch.ones(1, device="cuda")
    _lib.check(L.mn_softmax_backward(D(q), D(c), kind, t, v, d, D(at), 0, 2.0, P(rest), P(zt), D(one), 1, P(share), P(dq),
                                     P(dc), P(wb), n.value, st))
    untouched(rest, zt, loss, mean, share, ws, wb, dq, dc)
    ld = (d + 15) // 16 * 16
    qc, qs, cc, cs = guarded(t * ld, torch.int8), f(t), guarded(v * ld, torch.int8), f(v)
    _lib.check(L.mn_quantize_rows_i8(D(q), kind, t, d, P(qc), ld, P(qs), st))
    _lib.check(L.mn_quantize_rows_i8(D(c), kind, v, d, P(cc), ld, P(cs), st))
    _lib.check(L.mn_scores_i8_workspace(t, d, C.byref(n)))
    wi, y, back = guarded(n.value, torch.uint8), guarded(t * v, dtype), guarded(v * d, dtype)
    _lib.check(L.mn_scores_i8(P(qc), ld, P(qs), t, P(cc), ld, P(cs), v, d, P(y), kind, P(wi), n.value, st))
    _lib.check(L.mn_dequantize_rows_i8(P(cc), ld, P(cs), v, d, P(back), kind, st))
    untouched(qc, qs, cc, cs, wi, y, back)


def test_merge_of_many_ranges():
    """200 ranges, one of them without any item but the target, against the sum in 64 bits."""
    import surfface_hip as S
    g = torch.Generator().manual_seed(50)
    rests = torch.randn(200, 77, generator=g) * 30
    rests[3] = -math.inf
    zts = torch.full((200, 77), -math.inf)
    zts[torch.randint(0, 200, (77,), generator=g), torch.arange(77)] = torch.randn(77, generator=g) * 30
    at = torch.arange(77)
    at[5], zts[:, 6] = -1, -math.inf
    st = S.softmax_merge(rests.cuda(), zts.cuda(), at.cuda())
    rest, zt = torch.logsumexp(rests.double(), 0), zts.max(0).values
    want = torch.nn.functional.softplus(rest - zt.double(), threshold=1000)
    want[5] = 0
    # rest: 200 exponents and sums, off by 2^-24 of up to 200 / ln 2 and of their sum
    tol = 2.0 ** -24 * (4 * rest.abs() + 800)
    assert ((st.rest.double().cpu() - rest).abs() <= tol).all()
    assert torch.equal(st.target.cpu(), zt) and torch.isinf(st.loss[6]) and st.loss[5] == 0 and torch.isinf(st.mean)
    ok = torch.ones(77, dtype=torch.bool)
    ok[6] = False
    assert ((st.loss.double().cpu() - want).abs()[ok] <= (2 * tol + 4 * U * want)[ok]).all()
    assert abs(float(st.share) * 76 - 1) <= 2 * U


def test_threads_on_streams_of_their_own():
    """Two threads, a stream each, steps and scores at the same time: the results of one after the other."""
    import surfface_hip as S
    jobs = [make(200 + 300 * k, 5000 + 999 * k, 48, torch.bfloat16, 20 + k) for k in range(2)]

    def run(q, c, at):
        qg, cg = q.clone().requires_grad_(), c.clone().requires_grad_()
        loss = S.softmax_loss(qg, cg, at, 5.0)
        return [loss.detach(), *torch.autograd.grad(loss, (qg, cg)), S.scores_i8(S.quantize_rows(q), S.quantize_rows(c))]

    want = [run(*j) for j in jobs]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(10):
                    got[k].append(run(*jobs[k]))
            s.synchronize()
        except Exception as e:  # shown by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors
    for k in range(2):
        for r in got[k]:
            for a, b in zip(r, want[k]):
                assert torch.equal(a, b)
