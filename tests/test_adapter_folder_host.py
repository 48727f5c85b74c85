"""What an adapter's folder must agree in."""

from __future__ import annotations

import json

import pytest
import torch

from kvforge_b200.parts.adapters import AdapterError, read_adapter
from kvforge_b200.weights.safetensors_io import write_safetensors


def test_tensors_of_another_rank_than_the_configurations(tmp_path):
    """The scale is ``lora_alpha`` over the rank: tensors of another rank would be added with a wrong one."""
    t = {"q.lora_A.weight": torch.randn(4, 8), "q.lora_B.weight": torch.randn(8, 4)}
    write_safetensors(tmp_path / "adapter_model.safetensors", t)
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 8, "lora_alpha": 16}))
    with pytest.raises(AdapterError, match="rank 4"):
        read_adapter(tmp_path)
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 16}))
    assert read_adapter(tmp_path)[1] == 4.0
