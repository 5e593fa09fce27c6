"""Models whose layers' projections hold their weights in 8 bits: the parts on the plain kernels (CPU), the engine on the device."""
import pytest
import torch

from roost_b200.engine.executor import StepExecutor
from roost_b200.engine.model import load_model
from roost_b200.parts import Runtime, linear
from roost_b200.parts.linear import E4m3Linear, E4m3Rows
from tests.fake_kernels import FakeKernels
from tests.helpers import random_ids, rms_error, run_mixed, run_whole

# What rounding to e4m3 adds to a model's logits. A number is off by at most 2^-4 of itself, 2^-4 / sqrt(3) in the root mean square over a
# binade; both operands of a product are, so a product's outputs are off by 2^-4 sqrt(2 / 3) = 0.051 of theirs in the root mean square. The tiny models'
# two or three layers have four products each: twelve such errors in quadrature are 0.18, were each output to reach the logits alone; they reach them
# beside the stream that carries what earlier layers made.
E4M3_RMS = 0.18


def build(model_dir, weights, device="cpu", kernels=None):
    return load_model(model_dir, torch.bfloat16, device, kernels if kernels is not None else FakeKernels(), weights)


def test_linear_multiplies_rows_in_8_bits_by_weights_in_8_bits():
    rt = Runtime(torch.bfloat16, "cpu", FakeKernels(), "e4m3")
    g = torch.Generator().manual_seed(1)
    w, x = torch.randn(48, 64, generator=g).to(torch.bfloat16), torch.randn(5, 64, generator=g).to(torch.bfloat16)
    proj = E4m3Linear(rt, 48, 64)
    proj.load(w)
    y = proj(x, torch.float32)
    assert torch.equal(y, proj(E4m3Rows(*rt.kernels.quantise_e4m3(x)), torch.float32))
    assert torch.equal(proj.first_rows(16)(x), proj(x)[:, :16])
    # each operand within 2^-4 of itself, or of half the least step (2^-10 of the row's scale) near zero
    xs, ws = x.double().abs(), w.double().abs()
    bound = (xs @ ws.T) * (2 * 2.0 ** -4 + 2.0 ** -8) + (xs.amax(1) / 448 * 2.0 ** -10)[:, None] * ws.sum(1) * 1.1 + xs.sum(1)[:, None] * (ws.amax(1) / 448 * 2.0 ** -10) * 1.1
    assert bool(((y.double() - x.double() @ w.double().T).abs() <= bound + 1e-5).all())


@pytest.mark.parametrize("name", ["A", "D"])
def test_a_models_logits_on_the_plain_kernels(tiny_model_dirs, name):
    ids = random_ids(40, 250, 3)
    got = run_whole(StepExecutor(build(tiny_model_dirs[name], "e4m3"), max_tokens=64), "r", ids)
    want = run_whole(StepExecutor(build(tiny_model_dirs[name], "stored"), max_tokens=64), "r", ids)
    err = rms_error(got, want)
    print(f"MEASURED {name}: {err:.3f}")
    assert 0 < err < E4M3_RMS


def test_refusals(tiny_model_dirs):
    with pytest.raises(ValueError, match="weights"):
        Runtime(torch.bfloat16, "cpu", None, "int4")
    with pytest.raises(ValueError, match="bfloat16"):
        Runtime(torch.float32, "cpu", None, "e4m3")
    rt = Runtime(torch.bfloat16, "cpu", FakeKernels(), "e4m3")
    with pytest.raises(ValueError, match="expected"):
        E4m3Linear(rt, 8, 16).load(torch.zeros(8, 8))
    from roost_b200.engine.engine import RoostEngine
    with pytest.raises(ValueError, match="built with weights"):
        RoostEngine(build(tiny_model_dirs["A"], "stored"), weights="e4m3")


def test_a_part_without_the_form_refuses(tmp_path):
    from tests import zufusun_models as ZM
    cfg = ZM.config([(ZM.attention(), None)])
    with pytest.raises(ValueError, match="no form"):
        load_model(ZM.write_model(tmp_path, cfg, ZM.draw_tensors(cfg, 1)), torch.bfloat16, "cpu", FakeKernels(), "e4m3")


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_the_device_runs_what_the_plain_kernels_say(kernels, tiny_model_dirs, name, monkeypatch):
    """Sums in another order move a bfloat16 number to its neighbour now and then, and one bfloat16 step in sixteen moves a number of the 8 bits to
    its: below half of what the 8 bits themselves do to the logits."""
    ids = random_ids(70, 130, 5)
    model = build(tiny_model_dirs[name], "e4m3", "cuda", kernels)
    got = run_whole(StepExecutor(model, max_tokens=256), "r", ids)
    with monkeypatch.context() as m:      # the head's product on the CPU: whether torch.mm takes an output type is remembered from the device
        m.setattr(linear, "_MM_OUT_DTYPE", False)
        want = run_whole(StepExecutor(build(tiny_model_dirs[name], "e4m3"), max_tokens=128), "r", ids)
    err = rms_error(got, want)
    print(f"MEASURED {name}: {err:.4f}")
    assert err < E4M3_RMS / 2


@pytest.mark.gpu
def test_captured_steps_and_mixed_batches(kernels, tiny_model_dirs):
    """A step's rows do not feel one another, and a replayed step computes what the eager one does."""
    ids = {f"r{i}": random_ids(20 + 13 * i, 130, i) for i in range(4)}
    model = build(tiny_model_dirs["D"], "e4m3", "cuda", kernels)
    eager = run_mixed(StepExecutor(model, max_tokens=1024, use_graphs=False), ids, seed=1)
    graphs = run_mixed(StepExecutor(model, max_tokens=1024), ids, seed=1)
    again = run_mixed(StepExecutor(model, max_tokens=1024), ids, seed=1)
    alone = {rid: run_whole(StepExecutor(model, max_tokens=1024), rid, t) for rid, t in ids.items()}
    for rid in ids:
        assert torch.equal(graphs[rid], again[rid])
        assert rms_error(graphs[rid], eager[rid]) < E4M3_RMS / 2      # padded to captured sizes, so other forms of the product
        assert rms_error(graphs[rid], alone[rid]) < E4M3_RMS / 2


@pytest.mark.gpu
def test_the_engine_generates(kernels, tiny_model_dirs):
    from roost_b200 import GenerationOptions, RoostEngine
    options = GenerationOptions(max_output_tokens=12, ignore_eos=True)
    prompts = [random_ids(9, 130, 1), random_ids(30, 130, 2)]
    outs = [RoostEngine(tiny_model_dirs["D"], dtype="bfloat16", attention_blocks=64, weights="e4m3").generate(prompts, options) for _ in range(2)]
    assert [o.token_ids for o in outs[0]] == [o.token_ids for o in outs[1]] and all(len(o.token_ids) == 12 for o in outs[0])
