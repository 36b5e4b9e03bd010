"""Rows in 8 bits and the scores of quantised queries (mn_quantize_rows_i8,
mn_dequantize_rows_i8, mn_scores_i8) against numpy: codes and scales bit for
bit, scores within the three roundings of their formula (and one more for
bf16)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U32, UBF = 2.0 ** -24, 2.0 ** -8  # half a step of f32 and bf16, relative


def quantize_ref(x):
    """The formula in f32, as numpy rounds it; rows below 2^-100 (above 2^100) times 2^64 (2^-64) first."""
    x = np.asarray(x, np.float32)
    a = np.abs(x).max(1, initial=0.0).astype(np.float32)
    finite = np.isfinite(x).all(1)
    up = np.where(a < np.float32(2.0 ** -100), np.float32(2.0 ** 64), np.float32(1.0))
    up = np.where(a > np.float32(2.0 ** 100), np.float32(2.0 ** -64), up)
    with np.errstate(all="ignore"):
        inv = np.where(finite & (a != 0), (np.float32(1.0) / (a * up)) * np.float32(127.0), np.float32(0.0))
        v = np.rint((x * up[:, None]) * inv[:, None])
        v = np.where(finite[:, None], np.clip(v, -127, 127), 0.0)
        scale = np.where(finite, a / np.float32(127.0), np.float32(np.nan))
    return v.astype(np.int8), scale.astype(np.float32)


def rows(n, d, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g) * torch.logspace(-3, 3, n)[:, None]
    return x.to(dtype)


@pytest.mark.parametrize("n,d", [(1, 1), (3, 15), (5, 16), (7, 17), (64, 64), (33, 96), (130, 768), (5, 1025), (2, 4099), (3, 1536), (7, 2048),
                                 (2, 2064), (3, 4112), (2, 16400), (1, 40001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_is_the_formula_bit_for_bit(n, d, dtype):
    import surfface_hip as S
    x = rows(n, d, n * 1000 + d, dtype)
    r = S.quantize_rows(x.cuda())
    codes, scale = quantize_ref(x.float().numpy())
    assert r.d == d and r.codes.shape == (n, (d + 15) // 16 * 16)
    got = r.codes.cpu().numpy()
    np.testing.assert_array_equal(got[:, :d], codes)
    assert not got[:, d:].any()
    np.testing.assert_array_equal(r.scale.cpu().numpy().view(np.uint32), scale.view(np.uint32))
    back = S.dequantize_rows(r).cpu().numpy()
    np.testing.assert_array_equal(back, codes.astype(np.float32) * scale[:, None])
    half = S.dequantize_rows(r, torch.bfloat16).cpu()
    assert torch.equal(half, torch.from_numpy(back).to(torch.bfloat16))


def test_quantize_rows_at_the_borders():
    """Zeros, -0, one value, the largest and smallest f32, rows that are not finite."""
    import surfface_hip as S
    big, tiny = np.float32(3.4028235e38), np.float32(1e-45)
    x = np.zeros((10, 20), np.float32)
    x[1, :] = -0.0
    x[2, 7] = -3.0
    x[3, :] = (np.linspace(-1, 1, 20) * float(big)).astype(np.float32)
    x[4, :5] = [tiny, -tiny, 3 * tiny, 0, 100 * tiny]
    x[5, :3] = [1e-36, -5e-37, 2.0 ** -101]
    x[6, 3] = np.inf
    x[7, 19] = np.nan
    x[8, :] = 2.0 ** -100
    x[9, :4] = [0.5, 1.5, -2.5, 127.0]  # ties to even
    r = S.quantize_rows(torch.from_numpy(x).cuda())
    codes, scale = quantize_ref(x)
    np.testing.assert_array_equal(r.codes.cpu().numpy()[:, :20], codes)
    np.testing.assert_array_equal(r.scale.cpu().numpy(), scale)
    assert np.isnan(scale[6:8]).all() and codes[9, :4].tolist() == [0, 2, -2, 127]


@pytest.mark.parametrize("d", [1100, 2100, 5000, 33000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_rows_that_are_not_finite(d, dtype):
    """The largest value, an infinity and a NaN at either end of a row that several waves share."""
    import surfface_hip as S
    x = torch.randn(6, d, generator=torch.Generator().manual_seed(d)).to(dtype)
    x[0, -1], x[1, 0], x[2, -1], x[3, 0] = 300.0, -300.0, float("nan"), float("-inf")
    x[4] = 0
    r = S.quantize_rows(x.cuda())
    codes, scale = quantize_ref(x.float().numpy())
    np.testing.assert_array_equal(r.codes.cpu().numpy()[:, :d], codes)
    np.testing.assert_array_equal(r.scale.cpu().numpy(), scale)
    assert np.isnan(scale[2:4]).all() and codes[0, -1] == 127 and codes[1, 0] == -127


def check_scores(q, qs, c, cs, d, dtype, got):
    total = q[:, :d].astype(np.int64) @ c[:, :d].astype(np.int64).T
    want = total * qs.astype(np.float64)[:, None] * cs.astype(np.float64)
    tol = np.abs(want) * (3.01 * U32 + (UBF if dtype == torch.bfloat16 else 0)) + 1e-44
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), (err / np.maximum(tol, 1e-300)).max()


def codes_of(n, d, ld, seed, junk=True):
    """Random codes, -128 among them, and junk behind column d."""
    g = np.random.RandomState(seed)
    c = g.randint(-128, 128, (n, ld)).astype(np.int8)
    if not junk:
        c[:, d:] = 0
    return c, ((g.rand(n) + 0.5) / 100).astype(np.float32)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 257])
@pytest.mark.parametrize("n,d", [(1, 1), (15, 16), (63, 33), (300, 64), (257, 100), (1500, 768), (70, 1030)])
def test_scores_sizes(m, n, d):
    import surfface_hip as S
    ld = (d + 15) // 16 * 16
    q, qs = codes_of(m, d, ld, m + n)
    c, cs = codes_of(n, d, ld, m * n + d)
    for dtype in (torch.float32, torch.bfloat16):
        y = S.scores_i8(S.Int8Rows(torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda(), d),
                        S.Int8Rows(torch.from_numpy(c).cuda(), torch.from_numpy(cs).cuda(), d), dtype=dtype)
        assert y.shape == (m, n) and y.dtype == dtype
        check_scores(q, qs, c, cs, d, dtype, y)


@pytest.mark.parametrize("m", [3, 100])
def test_scores_wider_rows_and_long_sums(m):
    """Rows of codes wider than needed; sums next to the border of int32."""
    import surfface_hip as S
    q, qs = codes_of(m, 70, 160, 1)
    c, cs = codes_of(90, 70, 96, 2)
    y = S.scores_i8(S.Int8Rows(torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda(), 70),
                    S.Int8Rows(torch.from_numpy(c).cuda(), torch.from_numpy(cs).cuda(), 70))
    check_scores(q, qs, c, cs, 70, torch.float32, y)
    d, ld = 131071, 131072
    q = np.full((m, ld), -128, np.int8)
    c = np.full((20, ld), -128, np.int8)
    c[1] = 127
    one = np.ones(max(m, 20), np.float32)
    y = S.scores_i8(S.Int8Rows(torch.from_numpy(q).cuda(), torch.from_numpy(one[:m]).cuda(), d),
                    S.Int8Rows(torch.from_numpy(c).cuda(), torch.from_numpy(one[:20]).cuda(), d))
    check_scores(q, one[:m], c, one[:20], d, torch.float32, y)


def test_scores_empty_and_nan_rows():
    import surfface_hip as S
    items = S.quantize_rows(torch.randn(10, 24).cuda())
    assert S.scores_i8(S.quantize_rows(torch.randn(0, 24).cuda()), items).shape == (0, 10)
    assert S.scores_i8(items, S.quantize_rows(torch.randn(0, 24).cuda())).shape == (10, 0)
    x = torch.randn(3, 24)
    x[1, 5] = float("inf")
    x[2] = 0
    y = S.scores_i8(S.quantize_rows(x.cuda()), items).cpu()
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1]).all() and (y[2] == 0).all()


def test_scores_views_streams_and_graph():
    """Rows that start off a border, another stream, a captured and replayed call."""
    import surfface_hip as S
    x = torch.randn(41, 50).cuda()
    items = S.quantize_rows(torch.randn(200, 50).cuda())
    want = S.scores_i8(S.quantize_rows(x[1:]), items)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = S.scores_i8(S.quantize_rows(x[1:], stream=s), items, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    xin = x[1:].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = S.scores_i8(S.quantize_rows(xin), items)
    for k in range(3):
        xin.copy_(x[1:] * (k + 1))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, S.scores_i8(S.quantize_rows(xin), items)), k


def test_refusals():
    import surfface_hip as S
    r = S.quantize_rows(torch.randn(4, 20).cuda())
    with pytest.raises(TypeError):
        S.quantize_rows(torch.randn(4, 20).cuda().double())
    with pytest.raises(TypeError):
        S.quantize_rows(torch.randn(4, 20))
    with pytest.raises(ValueError):
        S.quantize_rows(torch.randn(20).cuda())
    with pytest.raises(ValueError):
        S.scores_i8(r, S.quantize_rows(torch.randn(4, 21).cuda()))
    with pytest.raises(TypeError):
        S.scores_i8(torch.randn(4, 20).cuda(), r)
    with pytest.raises(TypeError):
        S.scores_i8(r, r, dtype=torch.float16)
    with pytest.raises(ValueError):
        S.scores_i8(r, S.Int8Rows(r.codes[:, :24].contiguous(), r.scale, 20))
    with pytest.raises(ValueError):
        S.scores_i8(r, S.Int8Rows(r.codes, r.scale[:3], 20))
    wide = S.Int8Rows(torch.zeros(2, 131072, dtype=torch.int8).cuda(), torch.ones(2).cuda(), 131072)
    with pytest.raises(S.MnError):
        S.scores_i8(wide, wide)
