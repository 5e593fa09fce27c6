"""A request without an adapter computes the same bits whether a neighbour in its steps has one or not; and the gate's rows that the adapters read."""
import pytest
import torch

from roost_b200.engine.executor import StepEntry, StepExecutor
from roost_b200.engine.model import load_model
from tests.fake_kernels import FakeKernels
from tests.helpers import random_ids
from tests.test_adapter_models import write_adapter


@pytest.fixture(scope="module")
def adapter(tiny_model_dirs, tmp_path_factory):
    folder = tmp_path_factory.mktemp("neighbours") / "one"
    write_adapter(folder, tiny_model_dirs["D"], 4, 8.0, 1)
    return folder


def logits_beside(model, with_adapter, **kw):
    """Logits of request b, which has no adapter, beside request a in the same steps."""
    ids = {r: random_ids(20, 130, i) for i, r in enumerate("ab")}
    ex = StepExecutor(model, max_tokens=64, **kw)
    if with_adapter:
        ex.adapter_of["a"] = model.rt.adapters.names["x"]
    outs = {r: [] for r in "ab"}
    for lo, hi in [(0, 17), (17, 18), (18, 19), (19, 20)]:
        logits = ex.step([StepEntry(r, ids[r][lo:hi], list(range(hi - lo))) for r in "ab"])
        for i, r in enumerate("ab"):
            outs[r].append(logits[i * (hi - lo):(i + 1) * (hi - lo)].clone())
    return {r: torch.cat(v) for r, v in outs.items()}


def check(model, adapter, **kw):
    model.load_adapter("x", adapter)
    beside, alone = logits_beside(model, True, **kw), logits_beside(model, False, **kw)
    assert torch.equal(beside["b"], alone["b"])
    assert not torch.equal(beside["a"], alone["a"])


@pytest.mark.parametrize("weights", ["stored", "e4m3"])
def test_on_the_plain_kernels(tiny_model_dirs, adapter, weights):
    check(load_model(tiny_model_dirs["D"], torch.bfloat16, "cpu", FakeKernels(), weights, (2, 8)), adapter)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("weights", ["stored", "e4m3"])
def test_on_the_device(kernels, tiny_model_dirs, adapter, weights, graphs):
    check(load_model(tiny_model_dirs["D"], torch.bfloat16, "cuda", kernels, weights, (2, 8)), adapter, use_graphs=graphs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,inter,block", [(1, 1, 0), (5, 1111, 0), (16, 12288, 0), (3, 12288, 128), (600, 12288, 0), (4200, 4096, 128), (2, 32768, 0), (2, 40000, 0)])
def test_the_gates_rows_as_they_are(kernels, dtype, tokens, inter, block):
    """The 8 bits are those without ``keep``; the rows beside them are within the formula's 32-bit roundings (9 half steps) and one half step of their type."""
    from tests.test_e4m3_gpu import HALF, rand
    from tests.test_e4m3_walk_gpu import silu_of
    x = rand((tokens, 2 * inter), dtype, 5, 3.0)
    q, scale = kernels.silu_mul_e4m3(x, block)
    q2, scale2, kept = kernels.silu_mul_e4m3(x, block, keep=True)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(scale, scale2)
    want = silu_of(x, block)
    assert kept.dtype == dtype and kept.shape == want.shape
    assert bool(((kept.double() - want).abs() <= (9 * HALF + torch.finfo(dtype).eps / 2) * want.abs()).all())
    few = kernels.silu_mul_e4m3(x[-1:].contiguous(), block, keep=True)
    assert torch.equal(few[2], kept[-1:])
