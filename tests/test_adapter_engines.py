"""Two engines over one model share its adapters."""
import gc

import pytest
import torch

from roost_b200 import GenerationOptions, RoostEngine
from roost_b200.engine.model import load_model
from roost_b200.parts.adapters import AdapterError
from tests.fake_kernels import FakeKernels
from tests.test_adapter_models import write_adapter


def test_an_adapter_that_another_engines_request_uses_is_neither_replaced_nor_freed(tiny_model_dirs, tmp_path):
    write_adapter(tmp_path / "one", tiny_model_dirs["A"], 4, 8.0, 1)
    model = load_model(tiny_model_dirs["A"], torch.float32, "cpu", FakeKernels(), adapters=(2, 8))
    first, second = (RoostEngine(model, device="cpu", attention_blocks=64) for _ in range(2))
    first.load_adapter("x", tmp_path / "one")
    options = GenerationOptions(max_output_tokens=4, adapter="x")
    rid = second.add_request([1, 2, 3], options.sampling())
    for engine in (first, second):
        for call in (lambda: engine.load_adapter("x", tmp_path / "one"), lambda: engine.unload_adapter("x")):
            with pytest.raises(AdapterError, match="in use"):
                call()
    second.cancel(rid)
    first.load_adapter("x", tmp_path / "one")
    second.add_request([1, 2, 3], options.sampling())
    del second, engine              # an engine that is gone holds nothing
    gc.collect()
    first.unload_adapter("x")
