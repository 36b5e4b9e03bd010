"""Rows in 8 bits where one launch does not reach: more than 2^30 threads, and the 2^32 that
HIP refuses."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("n,d,dtype", [(2 ** 29 + 300, 1, BF16),   # 2 lanes a row
                                       (2 ** 29 + 1, 2, F32),
                                       (2 ** 27 + 130, 33, BF16),  # 8
                                       (2 ** 24 + 5, 257, BF16),   # a wave
                                       (2 ** 24 + 9, 260, F32),
                                       (2 ** 23 + 3, 1025, BF16),  # a block of 128
                                       (2 ** 22 + 2, 4100, BF16)])  # a block of 1024: 2^32 threads
def test_quantised_in_parts(n, d, dtype):
    """Rows around every power of two from 2^20 on and the last ones, others zero, against the same rows alone."""
    import surfface_hip as S
    x = torch.zeros(n, d, dtype=dtype, device="cuda")
    at = torch.cat([torch.arange(2 ** k - 3, 2 ** k + 3) for k in range(20, 31)] + [torch.arange(n - 5, n)]).unique()
    at = at[at < n].cuda()
    some = torch.randn(len(at), d, generator=torch.Generator().manual_seed(d)).to(dtype).cuda()
    x[at] = some
    rows, want = S.quantize_rows(x), S.quantize_rows(some)
    del x
    assert torch.equal(rows.codes[at], want.codes) and torch.equal(rows.scale[at], want.scale)
    assert int((rows.scale != 0).sum()) == int((want.scale != 0).sum())
    back = S.dequantize_rows(rows, dtype)
    assert torch.equal(back[at], S.dequantize_rows(want, dtype))
    del rows, back
    torch.cuda.empty_cache()
