"""Which operands of the 8-bit products and of the adapters are read ahead of the wait for the kernel in front: what the header says of them, and the kernel that
may write one."""
import re

import pytest
import torch

from tests.test_kernel_launch_order import CSRC, _kernels

HEADER = (CSRC / "roost_kernels.h").read_text()
CONTRACT = re.search(r"/\* Programmatic dependent launch.*?\*/", HEADER, re.S).group(0)


def ahead(name, body):
    """A kernel's text up to its own wait (waits on the way out of a block without work left out)."""
    body = re.sub(r"pdl_wait\(\)\s*;\s*return\s*;", "", body)
    return body[: re.search(r"pdl_wait\(", body).start()]


def test_the_header_names_what_the_adapters_read_ahead():
    src = re.sub(r"//[^\n]*", "", (CSRC / "adapters.cu").read_text())
    found = set()
    for name, body in _kernels(CSRC / "adapters.cu"):
        head = src[: src.index(body)][-2000:]
        for table in re.findall(r"const (?:int32_t|float|T|__nv_bfloat16)\*\s*(?:__restrict__\s*)?(\w+)", head[head.rindex(name):]):
            if re.search(rf"\b{table}\b", ahead(name, body)):
                found.add(table)
    assert {"tiles", "rows", "ranks", "scales", "a", "b"} <= found
    for table in found - {"x", "a", "b"}:      # x: only the addresses are formed
        assert f"`{table}`" in CONTRACT, table
    assert "adapters' a, b and `scales`" in CONTRACT


def test_only_the_kernel_that_makes_weights_holds_the_next_one_back():
    """All others let it begin first of all; that one when its rows are written, for ordinary loads and for tensor copies."""
    held = {name for name, body in _kernels(CSRC / "rows_e4m3.cu") if "rows_are_written()" in body}
    assert held == {"quantise_e4m3_vec_kernel", "quantise_e4m3_kernel"}
    text = re.sub(r"//[^\n]*", "", (CSRC / "rows_e4m3.cu").read_text())
    body = text[text.index("void rows_are_written()"):]
    order = [body.index(s) for s in ("__threadfence()", "fence.proxy.async", "__syncthreads()", "pdl_launch_dependents()")]
    assert order == sorted(order)
    assert "but roost_quantise_e4m3 lets the next begin at once" in CONTRACT
    gemm = HEADER[HEADER.index("/* ---- gemm_e4m3.cu"):HEADER.index("int roost_gemm_e4m3(")]
    assert "roost_quantise_e4m3" in gemm and "after a copy" in gemm


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 48, 300])
def test_rows_of_the_norm_and_of_the_gate_as_a_weight(kernels, m):
    """As the documentation allows it: a copy of them stands between. Another weight every time: what was read too early would be the one before."""
    from tests.test_e4m3_gpu import rand
    q, q_scale = kernels.quantise_e4m3(rand((m, 2048), torch.float32, 1))
    ones = torch.ones(2048, dtype=torch.bfloat16, device="cuda")
    stored = [rand((4096, 4096), torch.bfloat16, 10 + i) for i in range(3)]
    calls = [lambda w: kernels.silu_mul_e4m3(w), lambda w: kernels.rms_norm_e4m3(w[:, :2048].contiguous(), ones, 1e-6)]
    wants = {}
    for c, call in enumerate(calls):
        for i, w in enumerate(stored):
            made = call(w)
            torch.cuda.synchronize()
            wants[c, i] = kernels.gemm_e4m3(q, q_scale, *made)
            torch.cuda.synchronize()
            del made
    for _ in range(3):
        for i, w in enumerate(stored):
            for c, call in enumerate(calls):
                rows, scale = call(w)
                assert torch.equal(kernels.gemm_e4m3(q, q_scale, rows.clone(), scale), wants[c, i])
