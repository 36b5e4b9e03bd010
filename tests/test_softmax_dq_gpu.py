"""dQ of the softmax loss over large tables: pieces, partial sums, offsets past
2^31 and 2^32.

Most columns of the table mark a range of its rows (1 there, 0 elsewhere), so
that dQ of such a column is the probability of its range, less 1 for the
target's: a part of the table that is lost, counted twice or read elsewhere
changes it by as much as the part weighs.  The logits come from the other
columns.

Tolerance, as in test_softmax_gpu.py but for the sum: products with zeros are
zeros and round nothing, so a logit has FREE terms, and a column's error is that
of its n nonzero entries in any order, n u, 6 n u in the f32 form; (2 delta + (6 n + 64) u [+ b for D in
bf16]) sum |D_ij c_jk| and half a step of the own type.  It is checked beside
each comparison that the formula itself fails it once a tenth of a range is left
out, or all of dQ."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, B = 2.0 ** -24, 2.0 ** -8
CHUNK = 65536
FREE = 8  # columns that make the logits


def table(t, v, d, dtype, seed):
    """(queries, items, targets, rows of a range)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = -(-v // (d - FREE))
    c = torch.zeros(v, d, dtype=dtype, device="cuda")
    for j in range(0, v, CHUNK):
        n = min(CHUNK, v - j)
        c[j:j + n, :FREE] = (torch.randn(n, FREE, generator=g, device="cuda") / 4).to(dtype)
        rows = torch.arange(j, j + n, device="cuda")
        c[rows, FREE + rows // width] = 1.0
    q = torch.zeros(t, d, dtype=dtype, device="cuda")
    q[:, :FREE] = torch.randn(t, FREE, generator=g, device="cuda").to(dtype)
    at = torch.randint(0, v, (t,), generator=g, device="cuda")
    at[0], at[1] = v - 1, 0
    at[2::5] = -1
    return q, c, at, width


@pytest.mark.parametrize("t,v,d", [(300, 530001, 264),     # pieces of a table, partial sums apart
                                   (4096, 150001, 2048),   # partial sums added up, piece by piece
                                   (70, 1500001, 768),     # f32: 4.6 GB of items
                                   (70, 3000001, 768),     # bf16: the same
                                   (33, 70001, 40)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_range_of_a_table_counts_once(t, v, d, dtype):
    import surfface_hip as S
    q, c, at, width = table(t, v, d, dtype, t + d)
    st = S.softmax_stats(q, c, at)
    dq, _ = S.softmax_backward(q, c, at, st.rest, st.target, torch.ones(1, device="cuda"), need=(True, False))
    has = at >= 0
    x = torch.where(has[:, None], q.double(), 0.0)[:, :FREE].contiguous()
    lse = torch.full((t,), -math.inf, dtype=torch.float64, device="cuda")
    most = 0.0
    for j in range(0, v, CHUNK):
        y = c[j:j + CHUNK, :FREE].double().t().contiguous()
        lse = torch.logaddexp(lse, torch.logsumexp(x @ y, 1))
        most = max(most, float((x.abs() @ y.abs()).max()))
    free, mag = torch.zeros(t, FREE, dtype=torch.float64, device="cuda"), torch.zeros(t, FREE, dtype=torch.float64, device="cuda")
    mass, tenth = torch.zeros(t, d - FREE, dtype=torch.float64, device="cuda"), torch.zeros(t, d - FREE, dtype=torch.float64, device="cuda")
    hits = torch.zeros(t, d - FREE, dtype=torch.float64, device="cuda")
    rows = torch.arange(t, device="cuda")
    for j in range(0, v, CHUNK):
        y = c[j:j + CHUNK, :FREE].double()
        D = torch.exp(x @ y.t().contiguous() - lse[:, None]) * has[:, None]
        items = torch.arange(j, j + len(y), device="cuda")
        mark = c[j:j + CHUNK, FREE:].double()
        mass += D @ mark
        tenth += (D * (items % width < width / 10)) @ mark
        here = (at >= j) & (at < j + len(y))
        D[rows[here], at[here] - j] -= 1.0
        free += D @ y
        mag += D.abs() @ y.abs()
    hits[rows[has], at[has] // width] = 1.0
    want = torch.cat([free, mass - hits], 1)
    size = torch.cat([mag, mass + hits], 1)
    n = torch.full((d,), float(width), device="cuda", dtype=torch.float64)
    n[:FREE] = v
    delta = 2 * (6 * FREE + 8) * U * most + 16 * U * (1 + float(lse[has].abs().max()) + math.log2(v + 1))
    b = B if dtype == torch.bfloat16 else 0.0
    tol = (2 * delta + (6 * n + 64) * U + b) * size + (b or U) * want.abs() + 1e-30
    assert ((dq.double() - want).abs() <= tol).all()
    assert not dq[~has].any()
    # the bound tells: a tenth of any range lost, or everything
    full = torch.arange(d - FREE, device="cuda") < v // width
    clear = has[:, None] & full & (hits == 0)
    assert clear.any() and (tenth > tol[:, FREE:])[clear].all()
    assert (want.abs() > tol)[:, FREE:][clear].all()
    del c
    torch.cuda.empty_cache()
