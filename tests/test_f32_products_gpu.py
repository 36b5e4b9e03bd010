"""f32 products on the bf16 matrix cores: what the three parts of each value leave
out has no sign of its own.

With two items and every target the first one, rest is the second item's logit
alone: x y for rows of one value, off by a product's roundings (six parts added
up, of which the last addition counts: u = 2^-24), the rounding to base 2 and the
one back (u each), and the constants 1 / ln 2 and ln 2 of f32, whose product is
known.  The roundings of many x have no mean: over 2^17 of them 3 u / sqrt(3 * 2^17)
is 0.005 u; 0.35 u is allowed.  Cutting all parts off leaves out 2 u of this y
in the mean, always towards zero."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
N = 1 << 17


@pytest.mark.parametrize("bits", [0x3f80ffff, 0x3f807fff, 0x3f8080ff, 0x3fffffff, 0xbf80fffe])
def test_products_have_no_bias(bits):
    import surfface_hip as S
    y = float(np.array([bits], np.uint32).view(np.float32)[0])
    x = (torch.rand(N, generator=torch.Generator().manual_seed(bits % 1000)) + 1.0)[:, None]  # [1, 2)
    c = torch.tensor([[0.0], [y]])
    st = S.softmax_stats(x.cuda(), c.cuda(), torch.zeros(N, dtype=torch.int64, device="cuda"))
    exact = x.double()[:, 0] * y * (float(np.float32(1 / np.log(2))) * float(np.float32(np.log(2))))
    off = (st.rest.double().cpu() - exact) / exact.abs() / U
    if y < 0:
        off = -off
    assert off.abs().max() <= 3.1 + 4  # what is left out is below 2^-22
    assert abs(off.mean()) <= 0.35, float(off.mean())


def test_the_largest_values_stay_finite():
    """Values that rounding to bf16 would take to infinity, times powers of two: exact but for the roundings above."""
    import surfface_hip as S
    top = torch.finfo(torch.float32).max
    x = torch.full((3000, 4), 2.0 ** -20)
    c = torch.zeros(2, 4)
    c[1] = torch.tensor([top, -top, top, top * 2.0 ** -3])
    x[:, 1] = 0
    x[:, 2] = 0
    st = S.softmax_stats(x.cuda(), c.cuda(), torch.zeros(3000, dtype=torch.int64, device="cuda"), scale=2.0 ** -90)
    exact = float(top) * 2.0 ** -20 * (1 + 2.0 ** -3) * 2.0 ** -90
    assert ((st.rest.double().cpu() / exact - 1).abs() <= 8 * U).all()
