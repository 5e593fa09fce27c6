"""The products in 8 bits at the largest numbers of rows that they take."""
import pytest
import torch

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def test_as_many_rows_as_an_index_holds(kernels):
    """2 ** 31 - 257 rows of one number, the form for any size: the walk over them steps beyond 32 bits behind the last ones. Products of two numbers of e4m3 and
    scales that are powers of two are exact in bfloat16."""
    m = 2 ** 31 - 257
    q = torch.arange(251, dtype=torch.uint8, device="cuda").clamp_max_(126).repeat(m // 251 + 1)[:m].view(E4M3)[:, None]
    q_scale = torch.tensor([0.5, 1.0, 2.0], device="cuda").repeat(m // 3 + 1)[:m]
    w, w_scale = torch.tensor([[1.5]], device="cuda").to(E4M3), torch.tensor([0.25], device="cuda")
    out = kernels.gemm_e4m3(q, q_scale, w, w_scale)
    assert out.shape == (m, 1)
    for lo in range(0, m, 1 << 28):
        part = slice(lo, min(lo + (1 << 28), m))
        assert torch.equal(out[part, 0], (q[part, 0].float() * 0.375 * q_scale[part]).to(torch.bfloat16)), lo


def test_more_rows_than_an_index_holds_are_refused(kernels):
    from roost_b200.kernels.library import KernelError
    q, w, one = torch.zeros((2 ** 31 - 256, 1), dtype=torch.uint8, device="cuda").view(E4M3), torch.zeros((1, 1), dtype=torch.uint8, device="cuda").view(E4M3), torch.ones(1, device="cuda")
    scales = torch.ones(2 ** 31 - 256, device="cuda")
    with pytest.raises(KernelError, match="more rows"):
        kernels.gemm_e4m3(q, scales, w, one)
    with pytest.raises(KernelError, match="more rows"):
        kernels.gemm_e4m3(w, one, q, scales)
