"""Adapters whose configuration means something else than B A x beside the stored weights are refused."""
import json

import pytest
import torch

from roost_b200.parts.adapters import AdapterError, read_adapter
from roost_b200.weights.safetensors_io import write_safetensors


def folder_with(tmp_path, **config):
    write_safetensors(tmp_path / "adapter_model.safetensors", {"base_model.model.x.lora_A.weight": torch.ones(2, 4), "base_model.model.x.lora_B.weight": torch.ones(3, 2)})
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 2, "lora_alpha": 4, **config}))
    return tmp_path


@pytest.mark.parametrize("config,what", [({"peft_type": "ADALORA"}, "ADALORA"), ({"init_lora_weights": "pissa"}, "converted"), ({"init_lora_weights": "pissa_niter_16"}, "converted"),
                                         ({"init_lora_weights": "OLoRA"}, "converted"), ({"init_lora_weights": "loftq"}, "converted"), ({"layer_replication": [[0, 4], [2, 5]]}, "layer_replication"),
                                         ({"alora_invocation_tokens": [1, 2]}, "alora"), ({"use_qalora": True}, "use_qalora"), ({"lora_alpha": float("inf")}, "finite"),
                                         ({"lora_alpha": float("nan")}, "finite")])
def test_refused(tmp_path, config, what):
    with pytest.raises(AdapterError, match=what):
        read_adapter(folder_with(tmp_path, **config))


@pytest.mark.parametrize("config", [{}, {"peft_type": "LORA", "init_lora_weights": True}, {"init_lora_weights": "gaussian"}, {"init_lora_weights": "eva"}, {"layer_replication": None}])
def test_taken(tmp_path, config):
    modules, scale = read_adapter(folder_with(tmp_path, **config))
    assert list(modules) == ["x"] and scale == 2.0
