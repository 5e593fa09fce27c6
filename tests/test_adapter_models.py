"""Adapters through the engine: requests of several adapters and of none in the same steps, against models whose weights hold the adapter's product."""
import dataclasses
import json

import pytest
import torch

from roost_b200 import GenerationOptions, RoostEngine
from roost_b200.config.spec import RunEntry
from roost_b200.engine.executor import StepEntry, StepExecutor
from roost_b200.engine.model import Model, load_model
from roost_b200.engine.request import RequestError
from roost_b200.parts.adapters import AdapterError, AdapterSlots
from roost_b200.parts.base import Runtime
from roost_b200.weights.safetensors_io import SafetensorsFile, write_safetensors
from tests.fake_kernels import FakeKernels
from tests.helpers import BF16_RMS_BOUND, FP32_BOUND, random_ids, rms_error, run_whole, scaled_error

MODULES = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")


def write_adapter(folder, model_dir, rank, alpha, seed, modules=MODULES, rslora=False):
    """A random adapter for every layer's ``modules``; returns what it adds to each weight, in float64."""
    g = torch.Generator().manual_seed(seed)
    stored = SafetensorsFile(model_dir / "model.safetensors")
    tensors, added = {}, {}
    for name, entry in stored.entries.items():
        module = name.removesuffix(".weight")
        if not any(module.endswith(m) for m in modules):
            continue
        out, inner = entry.shape
        a, b = torch.randn(rank, inner, generator=g) * inner ** -0.5, torch.randn(out, rank, generator=g) * 0.1
        a, b = a.to(torch.bfloat16), b.to(torch.bfloat16)
        tensors[f"base_model.model.{module}.lora_A.weight"], tensors[f"base_model.model.{module}.lora_B.weight"] = a, b
        added[name] = (b.double() @ a.double()) * (alpha / (rank ** 0.5 if rslora else rank))
    folder.mkdir()
    write_safetensors(folder / "adapter_model.safetensors", tensors)
    (folder / "adapter_config.json").write_text(json.dumps({"r": rank, "lora_alpha": alpha, "use_rslora": rslora, "peft_type": "LORA", "bias": "none"}))
    return added


def merged(folder, model_dir, added):
    """The model with the adapter's product in its weights (float32)."""
    stored = SafetensorsFile(model_dir / "model.safetensors")
    tensors = {n: stored.tensor(n) for n in stored.entries}
    for n, d in added.items():
        tensors[n] = (tensors[n].double() + d).float()
    folder.mkdir()
    (folder / "config.json").write_text((model_dir / "config.json").read_text())
    write_safetensors(folder / "model.safetensors", tensors)
    return folder


@pytest.fixture(scope="module")
def adapters(tiny_model_dirs, tmp_path_factory):
    """Per model: two adapters' folders of different ranks, the second for some of the modules, and the merged models' folders."""
    root, out = tmp_path_factory.mktemp("adapters"), {}
    for name in ("A", "C", "D"):
        base = tiny_model_dirs[name]
        one = write_adapter(root / f"{name}-one", base, 4, 8.0, 1)
        two = write_adapter(root / f"{name}-two", base, 11, 11.0, 2, MODULES[:1] + MODULES[2:4] + MODULES[5:], rslora=True)
        out[name] = [(root / f"{name}-one", merged(root / f"{name}-m1", base, one)), (root / f"{name}-two", merged(root / f"{name}-m2", base, two))]
    return out


def build(model_dir, dtype, device, kernels, adapters=(3, 12), weights="stored"):
    return load_model(model_dir, dtype, device, kernels, weights, adapters)


def mixed_logits(model, folders, ids, **kw):
    """Four requests in common steps: an adapter, none, the other, the first again. {request: logits}"""
    for n, f in enumerate(folders):
        model.load_adapter(f"n{n}", f)
    ex = StepExecutor(model, max_tokens=1024, **kw)
    of = {"a": "n0", "c": "n1", "d": "n0"}
    outs = {r: [] for r in "abcd"}
    for r, n in of.items():
        ex.adapter_of[r] = model.rt.adapters.names[n]
    cuts = [(0, 9), (9, 10), (10, 11), (11, len(ids["a"]))]
    for lo, hi in cuts:
        logits = ex.step([StepEntry(r, ids[r][lo:hi], list(range(hi - lo))) for r in "abcd"])
        for i, r in enumerate("abcd"):
            outs[r].append(logits[i * (hi - lo):(i + 1) * (hi - lo)])
    return {r: torch.cat(v) for r, v in outs.items()}


def want_logits(model_dirs, ids, dtype, device, kernels):
    base, one, two = model_dirs
    of = {"a": one, "b": base, "c": two, "d": one}
    return {r: run_whole(StepExecutor(load_model(d, dtype, device, kernels), max_tokens=1024), r, ids[r]) for r, d in of.items()}


def step_ids():
    return {r: random_ids(24, 130, i) for i, r in enumerate("abcd")}


@pytest.mark.parametrize("name", ["A", "C"])
def test_mixed_requests_on_the_plain_kernels(tiny_model_dirs, adapters, name):
    ids, folders = step_ids(), adapters[name]
    got = mixed_logits(build(tiny_model_dirs[name], torch.float32, "cpu", FakeKernels()), [f for f, _ in folders], ids)
    want = want_logits([tiny_model_dirs[name]] + [m for _, m in folders], ids, torch.float32, "cpu", FakeKernels())
    for r in "abcd":
        assert scaled_error(got[r], want[r]) < FP32_BOUND, r
    assert scaled_error(want["a"], run_whole(StepExecutor(load_model(tiny_model_dirs[name], torch.float32, "cpu", FakeKernels()), max_tokens=64), "x", ids["a"])) > 1e-2


def test_slots_are_taken_replaced_and_freed(tiny_model_dirs, adapters, tmp_path):
    model = build(tiny_model_dirs["A"], torch.float32, "cpu", FakeKernels(), (2, 12))
    (one, _), (two, _) = adapters["A"]
    assert model.load_adapter("x", one) == 0 and model.load_adapter("y", two) == 1 and model.load_adapter("x", two) == 0
    a = model.blocks[0].mixer.qkv.adapters
    assert int(model.rt.adapters.ranks[0]) == 11 and not bool(a.a[0, 1].any()), "the module that the second adapter does not name adds nothing"
    with pytest.raises(AdapterError, match="slots"):
        model.load_adapter("z", one)
    model.rt.adapters.names.pop("x")
    assert model.load_adapter("z", one) == 0


def test_refusals(tiny_model_dirs, adapters, tmp_path):
    (one, _), (two, _) = adapters["A"]
    base = tiny_model_dirs["A"]
    with pytest.raises(AdapterError, match="without room"):
        load_model(base, torch.float32, "cpu", FakeKernels()).load_adapter("x", one)
    small = build(base, torch.float32, "cpu", FakeKernels(), (2, 8))
    with pytest.raises(AdapterError, match="rank 11"):
        small.load_adapter("x", two)
    with pytest.raises(AdapterError, match="cannot be read"):
        small.load_adapter("x", tmp_path)
    with pytest.raises(AdapterError):
        small.load_adapter("x", adapters["D"][0][0])      # another model's sizes
    with pytest.raises(ValueError):
        AdapterSlots(0, 4, torch.float32, "cpu", None)
    with pytest.raises(ValueError, match="beyond"):
        build(base, torch.float32, "cpu", FakeKernels(), (2, 200))

    spec = small.spec
    shared = dataclasses.replace(spec, schedule=[RunEntry(block=0), RunEntry(block=1, reads_cache_of=0)])
    Model(shared, Runtime(torch.float32, "cpu", FakeKernels()))
    with pytest.raises(ValueError, match="not served"):
        Model(shared, Runtime(torch.float32, "cpu", FakeKernels(), adapters=(2, 8)))

    def changed(name, config=None, rename=None, drop=None):
        f = tmp_path / name
        f.mkdir()
        c = json.loads((one / "adapter_config.json").read_text()) | (config or {})
        t = SafetensorsFile(one / "adapter_model.safetensors")
        tensors = {(rename or (lambda n: n))(n): t.tensor(n) for n in t.entries if not (drop and drop in n)}
        (f / "adapter_config.json").write_text(json.dumps(c))
        write_safetensors(f / "adapter_model.safetensors", tensors)
        return f

    for folder, what in ((changed("dora", {"use_dora": True}), "use_dora"), (changed("bias", {"bias": "all"}), "biases"), (changed("r", {"r": 5}), "expected rank"),
                         (changed("half", drop="layers.0.self_attn.q_proj.lora_A"), "one half"),
                         (changed("other", rename=lambda n: n.replace("q_proj", "w_proj")), "no projection"),
                         (changed("stray", rename=lambda n: n.replace("lora_A", "lora_X")), "no adapter's")):
        with pytest.raises(AdapterError, match=what):
            small.load_adapter("x", folder)
        assert "x" not in small.rt.adapters.names


def test_engine_requests_name_their_adapter(tiny_model_dirs, adapters):
    model = build(tiny_model_dirs["A"], torch.float32, "cpu", FakeKernels())
    with pytest.raises(ValueError, match="built with room"):
        RoostEngine(model, device="cpu", attention_blocks=64, adapter_slots=100)
    engine = RoostEngine(model, device="cpu", attention_blocks=64)
    (one, _), _ = adapters["A"]
    with pytest.raises(RequestError, match="not loaded"):
        engine.generate([[1, 2]], GenerationOptions(max_output_tokens=2, adapter="x"))
    engine.load_adapter("x", one)
    rid = engine.add_request([1, 2, 3], GenerationOptions(max_output_tokens=4, adapter="x").sampling())
    for call in (lambda: engine.load_adapter("x", one), lambda: engine.unload_adapter("x")):
        with pytest.raises(AdapterError, match="in use"):
            call()
    engine.cancel(rid)
    assert not engine.executor.adapter_of
    engine.generate([[1, 2, 3]], GenerationOptions(max_output_tokens=4, adapter="x"))
    assert not engine.executor.adapter_of
    engine.unload_adapter("x")
    with pytest.raises(AdapterError, match="not loaded"):
        engine.unload_adapter("x")


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name", ["A", "C", "D"])
def test_mixed_requests_on_the_device(kernels, tiny_model_dirs, adapters, name, graphs):
    ids, folders = step_ids(), adapters[name]
    got = mixed_logits(build(tiny_model_dirs[name], torch.float32, "cuda", kernels), [f for f, _ in folders], ids, use_graphs=graphs)
    want = want_logits([tiny_model_dirs[name]] + [m for _, m in folders], ids, torch.float32, "cuda", kernels)
    for r in "abcd":
        assert scaled_error(got[r], want[r]) < FP32_BOUND, r


@pytest.mark.gpu
@pytest.mark.parametrize("weights", ["stored", "e4m3"])
def test_mixed_requests_in_bfloat16(kernels, tiny_model_dirs, adapters, weights):
    """Each request beside others as alone. bfloat16: the same roundings, but for sums in another order where a step's size chooses another kernel."""
    ids, folders = step_ids(), [f for f, _ in adapters["D"]]
    model = build(tiny_model_dirs["D"], torch.bfloat16, "cuda", kernels, weights=weights)
    got = mixed_logits(model, folders, ids)
    plain = load_model(tiny_model_dirs["D"], torch.bfloat16, "cuda", kernels, weights)
    bound = BF16_RMS_BOUND if weights == "stored" else 0.09      # in 8 bits a bfloat16 step moves one number in sixteen by 2^-4 of itself
    assert rms_error(got["b"], run_whole(StepExecutor(plain, max_tokens=64), "b", ids["b"])) < bound
    for r, n in (("a", "n0"), ("c", "n1"), ("d", "n0")):
        ex = StepExecutor(model, max_tokens=64)
        ex.adapter_of[r] = model.rt.adapters.names[n]
        assert rms_error(got[r], run_whole(ex, r, ids[r])) < bound
        assert rms_error(got[r], run_whole(StepExecutor(plain, max_tokens=64), r, ids[r])) > 2 * bound, "the adapter counts"


@pytest.mark.gpu
def test_the_engine_mixes_adapters_in_its_steps(kernels, tiny_model_dirs, adapters):
    """float32, whose rows have the same bits in any batch: every request generates what it generates alone."""
    folders = [f for f, _ in adapters["D"]]
    prompts = [random_ids(5 + 7 * i, 130, i) for i in range(6)]
    names = ["x", None, "y", "x", None, "y"]

    def engine():
        e = RoostEngine(tiny_model_dirs["D"], dtype="float32", attention_blocks=128, adapter_slots=2, adapter_rank=12)
        e.load_adapter("x", folders[0]), e.load_adapter("y", folders[1])
        return e

    options = [GenerationOptions(max_output_tokens=10, ignore_eos=True, adapter=n) for n in names]
    together = engine().generate(prompts, options)
    one = engine()
    for p, o, t in zip(prompts, options, together):
        assert one.generate([p], o)[0].token_ids == t.token_ids
    assert together[0].token_ids != one.generate([prompts[0]], GenerationOptions(max_output_tokens=10, ignore_eos=True))[0].token_ids
