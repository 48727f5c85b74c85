"""Prompts of many rows with low-rank adapters through the engine."""

from __future__ import annotations

import pytest
import torch

from helpers import TINY, make_model_dir, random_tokens, rel_err
from plain_llama import PlainLlama
from test_gpu_beam_adapter_engine import engine_for, make_adapter, merged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("models")
    return {name: make_model_dir(tmp, name, store_dtype=torch.bfloat16) for name in TINY}


@pytest.mark.parametrize("graphs", [True, False])
def test_prompts_of_many_rows_in_bfloat16(folders, graphs):
    """Prompts of more rows than one kernel takes, with dependent launches, beside prompts without an adapter: logits of the base model within
    0.08 of its own in 32 bits (a bound that the engine's bfloat16 steps are held to elsewhere), with an adapter within twice that of the merged model's."""
    from kvforge_b200 import ops
    from kvforge_b200.engine.step import BatchItem

    name = "tiny-d"
    adapter, second = make_adapter(folders[name], 16, 4), make_adapter(folders[name], 5, 8)
    engine = engine_for(folders[name], name, dtype="bfloat16", max_num_batched_tokens=1536, max_model_len=512, num_blocks=512, cuda_graphs=graphs)
    assert engine.runner.pdl
    engine.load_adapter("it", *adapter)
    engine.load_adapter("second", *second)
    plains = {-1: PlainLlama(folders[name]), 0: merged(folders[name], adapter), 1: merged(folders[name], second)}
    vocab = TINY[name]["cfg"].vocab_size
    for turn in range(4 if graphs else 1):  # (a shape is captured at its second coming)
        prompts = [random_tokens(vocab, n, seed=turn * 10 + n) for n in (400, 350, 130)]
        slots = [0, -1, 1] if turn % 2 == 0 else [-1, 1, 0]
        assert sum(map(len, prompts)) >= ops.ADAPTER_MANY
        items = []
        for i, (p, slot) in enumerate(zip(prompts, slots)):
            engine.block_manager.allocate(f"s{i}", len(p) + 1)
            engine.core.state_slots.allocate(f"s{i}")
            items.append(BatchItem(f"s{i}", p, 0, "last", adapter=slot))
        logits = engine.runner.step(items).cpu()
        errors = {slot: rel_err(logits[i], plains[slot].logits(prompts[i])[-1]) for i, slot in enumerate(slots)}
        assert errors[-1] < 0.08 and max(errors[0], errors[1]) < 0.16, errors
        for i in range(3):
            engine.block_manager.free(f"s{i}")
            engine.core.state_slots.free(f"s{i}")
        engine.core.rt.check_error_flag()
