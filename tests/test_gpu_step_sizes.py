"""Configurations whose steps have fewer tokens than places for requests."""

from __future__ import annotations

import pytest
import torch

from helpers import TINY, make_model_dir
from plain_llama import PlainLlama
from test_gpu_beam_adapter_engine import engine_for, greedy, make_adapter, merged, prompts_for

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("models")
    return {name: make_model_dir(tmp, name, store_dtype=torch.bfloat16) for name in TINY}


@pytest.mark.parametrize("graphs", [True, False])
def test_beams_of_several_prompts_within_the_tokens_of_a_step(folders, graphs):
    """Twelve beams and room for six tokens a step: prompts wait for one another; more beams than tokens are refused."""
    from kvforge_b200 import BeamParams
    from kvforge_b200.engine.scheduler import RequestRejectedError

    name = "tiny-a"
    prompts = prompts_for(name, [9, 4, 14], seed=33)
    params = BeamParams(num_beams=4, max_tokens=6, num_return=4, ignore_eos=True)
    narrow = engine_for(folders[name], name, max_num_seqs=16, max_num_batched_tokens=6, cuda_graphs=graphs)
    wide = engine_for(folders[name], name, max_num_seqs=16, cuda_graphs=graphs)
    got, want = narrow.beam_search(prompts, params), wide.beam_search(prompts, params)
    assert [[h.token_ids for h in o.hypotheses] for o in got] == [[h.token_ids for h in o.hypotheses] for o in want]
    with pytest.raises(RequestRejectedError, match="max_num_batched_tokens"):
        narrow.beam_search(prompts, BeamParams(num_beams=8, max_tokens=6, ignore_eos=True))
    assert narrow.block_manager.num_free_blocks == narrow.block_manager.num_blocks


@pytest.mark.parametrize("graphs", [True, False])
def test_more_requests_than_a_step_has_tokens_for(folders, graphs):
    """18 decoding requests of 32 places and 20 tokens a step: a captured step has room for more rows than the budget of tokens."""
    name = "tiny-a"
    adapter = make_adapter(folders[name], 8, 21)
    engine = engine_for(folders[name], name, max_num_seqs=32, max_num_batched_tokens=20, cuda_graphs=graphs)
    engine.load_adapter("it", *adapter)
    prompts = prompts_for(name, [3 + i % 5 for i in range(18)], seed=90)
    chosen = ["it" if i % 2 else None for i in range(18)]
    outs = engine.generate(prompts, greedy(12), adapters=chosen)
    plains = {None: PlainLlama(folders[name]), "it": merged(folders[name], adapter)}
    for p, c, o in zip(prompts, chosen, outs):
        assert o.output_token_ids == plains[c].greedy(p, 12)
