"""The softmax gradients where one launch does not reach: more than 2^30 threads, and the 2^32 that
HIP refuses."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_partial_sums_joined_in_parts(dtype):
    """dQ of 2^22 + 300 queries of 1024 values (more than 2^30 threads of four values), three items:
    with two equal logits and one far below, dQ = (c_other - c_target) / 2."""
    import surfface_hip as S
    t, d = 2 ** 22 + 300, 1024
    q = torch.zeros(t, d, dtype=dtype, device="cuda")
    c = torch.randn(3, d, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    q[:, 0], c[:, 0] = 1.0, torch.tensor([0.0, 0.0, -512.0], dtype=dtype)
    at = torch.arange(t, device="cuda") % 3 - 1
    st = S.softmax_stats(q, c, at)
    dq, dc = S.softmax_backward(q, c, at, st.rest, st.target, torch.ones(1, device="cuda"))
    half = (c[1].double() - c[0].double()) / 2
    # rest and zt are 0, the target's entry -1/2, the other's exp2(0 - lse2) / 2 off by a few roundings of f32
    tol = 2.0 ** -20 * (c[0].double().abs() + c[1].double().abs()) + half.abs() * torch.finfo(dtype).eps / 2
    for j in range(0, t, 2 ** 20):
        g, a = dq[j:j + 2 ** 20], at[j:j + 2 ** 20]
        assert not g[a < 0].any()
        assert ((g[a == 0].double() - half).abs() <= tol).all() and ((g[a == 1].double() + half).abs() <= tol).all()
    del q, dq, dc
    torch.cuda.empty_cache()
