"""Rows in 8 bits of prompts: many long rows, which blocks that stay walk out of a ring of bulk copies, and the sizes next to where that form ends."""
import pytest
import torch

from tests.test_e4m3_gpu import HALF, check_rows, norm64, norm_rel, rand

pytestmark = pytest.mark.gpu


def silu_of(x, block=0):
    """silu(gate) * up in float64."""
    inter = x.shape[1] // 2
    at = torch.arange(inter, device=x.device)
    gate_at = at // block * 2 * block + at % block if block else at
    gate, up = x.double()[:, gate_at], x.double()[:, gate_at + (block or inter)]
    return gate * torch.sigmoid(gate) * up


# two rows of inputs take 220 KB of shared memory at 28,160 numbers of 16 bits (gate and up) and 14,080 of 32: the longest rows that are walked
@pytest.mark.parametrize("dtype,edge", [(torch.bfloat16, 28160), (torch.float32, 14080)])
@pytest.mark.parametrize("beyond", [0, 8, 128, 248, 256, 264])
def test_gates_next_to_the_longest_row_that_is_walked(kernels, dtype, edge, beyond):
    inter = edge + beyond if dtype == torch.bfloat16 else edge + beyond // 16 * 8
    x = rand((300, 2 * inter), dtype, 3, 3.0)
    q, scale = kernels.silu_mul_e4m3(x)
    check_rows(q, scale, silu_of(x), 9 * HALF, f"silu_mul of {inter}")
    few, few_scale = kernels.silu_mul_e4m3(x[200:].contiguous())          # a block a row
    assert torch.equal(q[200:].view(torch.uint8), few.view(torch.uint8)) and torch.equal(scale[200:], few_scale)


@pytest.mark.parametrize("hidden", [14080, 14088, 14200, 14208, 14216])
def test_norms_next_to_the_longest_row_that_is_walked(kernels, hidden):
    x, res, w = rand((300, hidden), torch.float32, 1, 3.0), rand((300, hidden), torch.float32, 2), 1 + rand((hidden,), torch.float32, 3, 0.1)
    s = x + res
    q, scale = kernels.add_rms_norm_e4m3(x, res, w, 1e-5)
    assert torch.equal(res, s)
    check_rows(q, scale, norm64(s, w, 1e-5), norm_rel(hidden), f"add_norm of {hidden}")
