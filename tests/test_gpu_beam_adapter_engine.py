"""Adapters and beams through the engine: requests with adapters of their own against models whose weights hold the adapter, beam search against a
search by full recomputation, both together, and the beams of models with recurrent states and windows against their own logits."""

from __future__ import annotations

import json
import math

import pytest
import torch

from helpers import TINY, make_model_dir, random_tokens, rel_err
from plain_llama import PlainLlama, read_safetensors

pytestmark = pytest.mark.gpu

PROJECTIONS = {
    "self_attn": ("q_proj", "k_proj", "v_proj", "o_proj"),
    "mlp": ("gate_proj", "up_proj", "down_proj"),
}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("models")
    return {name: make_model_dir(tmp, name, store_dtype=torch.bfloat16) for name in TINY}


def engine_for(folder, name, dtype="float32", num_blocks=256, adapters=True, **sched):
    from kvforge_b200 import AdapterConfig, CacheConfig, EngineConfig, InferenceEngine, SchedulerConfig

    sched = {"max_num_seqs": 8, "max_num_batched_tokens": 128, "max_model_len": 256, **sched}
    graphs = sched.pop("cuda_graphs", True)
    cfg = EngineConfig(
        cache=CacheConfig(block_size=TINY[name]["block_size"] if name in TINY else 16, num_blocks=num_blocks), scheduler=SchedulerConfig(**sched), dtype=dtype,
        cuda_graphs=graphs, adapters=AdapterConfig(max_adapters=4, max_rank=24) if adapters else None,
    )  # fmt: skip
    return InferenceEngine(cfg, model=folder)


def make_adapter(folder, rank, seed, targets=None):
    """(tensors, scale) of an adapter for every projection named in ``targets`` (all by default)."""
    g = torch.Generator().manual_seed(seed)
    weights = read_safetensors(folder / "model.safetensors")
    tensors = {}
    for name, w in weights.items():
        short = name[: -len(".weight")]
        if name.endswith(".weight") and any(short.endswith(f"{part}.{proj}") for part, projs in PROJECTIONS.items() for proj in projs):
            if targets is None or short.rsplit(".", 1)[1] in targets:
                tensors[f"base_model.model.{short}.lora_A.weight"] = torch.randn(rank, w.shape[1], generator=g).bfloat16().float() * 0.25
                tensors[f"base_model.model.{short}.lora_B.weight"] = torch.randn(w.shape[0], rank, generator=g).bfloat16().float() * 0.125
    return tensors, 0.5


def merged(folder, adapter):
    """The plain model with the adapter in its weights."""
    plain = PlainLlama(folder)
    tensors, scale = adapter
    for key in [k for k in tensors if k.endswith("lora_A.weight")]:
        short = key[len("base_model.model.") : -len(".lora_A.weight")]
        a, b = tensors[key], tensors[key.replace("lora_A", "lora_B")]
        own = short.removeprefix("model.") + ".weight"
        plain.w[own] = plain.w[own] + scale * (b @ a)
    return plain


def greedy(n):
    from kvforge_b200 import SamplingParams

    return SamplingParams(max_tokens=n, temperature=0.0, ignore_eos=True)


def prompts_for(name, lengths, seed=0):
    vocab = TINY[name]["cfg"].vocab_size
    return [random_tokens(vocab, n, seed=seed + i) for i, n in enumerate(lengths)]


# ------------------------------------------------------------------ adapters


@pytest.mark.parametrize("name", ["tiny-a", "tiny-b", "tiny-c", "tiny-d"])
@pytest.mark.parametrize("graphs", [True, False])
def test_requests_with_adapters_of_their_own(folders, name, graphs):
    """In 32 bits every request's tokens are those of the model with its adapter merged in, beside requests with others and none."""
    folder = folders[name]
    made = {"one": make_adapter(folder, 8, 1), "two": make_adapter(folder, 24, 2), "attention": make_adapter(folder, 3, 3, ("q_proj", "v_proj"))}
    engine = engine_for(folder, name, cuda_graphs=graphs)
    for key, (tensors, scale) in made.items():
        engine.load_adapter(key, tensors, scale)
    prompts = prompts_for(name, [2, 30, 7, 100, 1, 12, 9])
    chosen = ["one", None, "two", "attention", "one", "two", None]
    outs = engine.generate(prompts, greedy(10), adapters=chosen)
    plains = {None: PlainLlama(folder), **{k: merged(folder, a) for k, a in made.items()}}
    for p, c, o in zip(prompts, chosen, outs):
        assert o.output_token_ids == plains[c].greedy(p, 10)
    # without adapters the engine's tokens are the base model's, bit for bit those of an engine that keeps none
    plain_engine = engine_for(folder, name, adapters=False, cuda_graphs=graphs)
    assert [o.output_token_ids for o in engine.generate(prompts, greedy(10))] == [o.output_token_ids for o in plain_engine.generate(prompts, greedy(10))]


@pytest.mark.parametrize("name", ["tiny-a", "tiny-d", "tiny-e"])
def test_adapters_in_bfloat16(folders, name):
    """Logits of prompts and of single tokens: as far from the merged model's as the base model's are from its own (both round the
    same rows to bfloat16), within a factor of two."""
    from kvforge_b200.engine.step import BatchItem

    folder = folders[name]
    adapter = make_adapter(folder, 16, 4)
    engine = engine_for(folder, name, "bfloat16", cuda_graphs=False)
    engine.load_adapter("it", *adapter)
    plains = {-1: PlainLlama(folder), 0: merged(folder, adapter)}
    prompts = prompts_for(name, [3, 40, 17])
    errors = {}
    for slot in (-1, 0):
        items = []
        for i, p in enumerate(prompts):
            seq = f"{slot}.{i}"
            engine.block_manager.allocate(seq, len(p) + 1)
            engine.core.state_slots.allocate(seq)
            items.append(BatchItem(seq, p, 0, "all", adapter=slot))
        logits = engine.runner.step(items).cpu()
        want = torch.cat([plains[slot].logits(p) for p in prompts])
        single = engine.runner.step([BatchItem(it.seq_id, [5], len(p), "last", adapter=slot) for it, p in zip(items, prompts)]).cpu()
        want_single = torch.stack([plains[slot].logits([*p, 5])[-1] for p in prompts])
        errors[slot] = max(rel_err(logits, want), rel_err(single, want_single))
    assert errors[-1] < 0.08
    assert errors[0] <= 2 * errors[-1], errors
    engine.core.rt.check_error_flag()


def test_a_preempted_request_keeps_its_adapter(folders):
    name = "tiny-a"
    adapter = make_adapter(folders[name], 8, 5)
    engine = engine_for(folders[name], name, num_blocks=9)
    engine.load_adapter("it", *adapter)
    prompts = prompts_for(name, [30, 28, 25], seed=9)
    outs = engine.generate(prompts, greedy(30), adapters=["it", None, "it"])
    assert engine.stats()["scheduler"]["num_preemptions"] > 0
    plains = {None: PlainLlama(folders[name]), "it": merged(folders[name], adapter)}
    for p, c, o in zip(prompts, ["it", None, "it"], outs):
        assert o.output_token_ids == plains[c].greedy(p, 30)


def test_adapters_from_a_folder_come_and_go(folders, tmp_path):
    from kvforge_b200.parts.adapters import AdapterError
    from kvforge_b200.weights.safetensors_io import write_safetensors

    name = "tiny-b"
    folder = folders[name]
    tensors, _ = make_adapter(folder, 4, 6)
    write_safetensors(tmp_path / "adapter_model.safetensors", tensors)
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 2}))
    engine = engine_for(folder, name)
    engine.load_adapter("disk", tmp_path)
    prompt = prompts_for(name, [11])
    want = merged(folder, (tensors, 0.5)).greedy(prompt[0], 8)
    assert engine.generate(prompt, greedy(8), adapters="disk")[0].output_token_ids == want
    # its place goes to another, of a lower rank and fewer projections: nothing of the first is left
    other = make_adapter(folder, 2, 7, ("down_proj",))
    engine.unload_adapter("disk")
    engine.load_adapter("other", *other)
    assert engine.generate(prompt, greedy(8), adapters="other")[0].output_token_ids == merged(folder, other).greedy(prompt[0], 8)
    # refusals
    for bad in ("disk", "none"):
        with pytest.raises(AdapterError):
            engine.add_request(prompt[0], adapter=bad)
        with pytest.raises(AdapterError):
            engine.unload_adapter(bad)
    with pytest.raises(AdapterError):
        engine.load_adapter("other", *other)
    key = next(iter(tensors))
    for wrong in (
        {}, {"model.embed_tokens.lora_A.weight": torch.zeros(2, 8)}, {key: tensors[key]}, {**tensors, key: tensors[key][:, :-1]}, {**tensors, "x.weight": tensors[key]},
        make_adapter(folder, 25, 1)[0],
    ):  # fmt: skip
        with pytest.raises(AdapterError):
            engine.load_adapter("wrong", wrong, 1.0)
    engine.add_request(prompt[0], greedy(4), adapter="other")
    with pytest.raises(AdapterError, match="in use"):
        engine.unload_adapter("other")
    while engine.has_unfinished_requests():
        engine.step()
    engine.unload_adapter("other")
    for i in range(4):
        engine.load_adapter(f"n{i}", *other)
    with pytest.raises(AdapterError):
        engine.load_adapter("n4", *other)
    bare = engine_for(folder, name, adapters=False)
    with pytest.raises(AdapterError):
        bare.load_adapter("x", *other)
    with pytest.raises(AdapterError):
        bare.add_request(prompt[0], adapter="x")


# ------------------------------------------------------------------ beams


def plain_beams(plain, prompt, w, n, stops, penalty):
    """Beam search by full recomputation, in 64 bits behind the logits.  Returns (tokens, log probability) best first, and the smallest
    distance between neighbouring candidates that mattered."""
    beams, finished, gap = [([], 0.0)], [], math.inf
    k = min(64, w * (1 + max(1, len(stops))))
    for length in range(1, n + 1):
        every = []
        for b, (tokens, lp) in enumerate(beams):
            logp = torch.log_softmax(plain.logits(prompt + tokens)[-1].double(), 0) + lp
            every += [(float(v), b, t) for t, v in enumerate(logp)]
        every.sort(key=lambda c: (-c[0], c[1], c[2]))
        following = []
        for rank, (lp, b, t) in enumerate(every[:k]):
            tokens = [*beams[b][0], t]
            if t in stops:
                if rank < w:
                    finished.append((tokens, lp))
            elif len(following) < w:
                following.append((tokens, lp))
                last = rank
        # (what lies behind the last that goes on, and behind the first w, is not chosen from)
        last = max(last, w - 1) if following else k - 1
        gap = min([gap, *[a[0] - b[0] for a, b in zip(every[: last + 1], every[1 : last + 2])]])
        finished.sort(key=lambda h: -h[1] / len(h[0]) ** penalty)
        del finished[w:]
        beams = following
        if not beams:
            return finished, gap
        if len(finished) == w and beams[0][1] / length**penalty <= finished[-1][1] / len(finished[-1][0]) ** penalty:
            return finished, gap
    finished += beams
    finished.sort(key=lambda h: -h[1] / len(h[0]) ** penalty)
    return finished[:w], gap


@pytest.mark.parametrize("name,w,penalty", [("tiny-a", 4, 1.0), ("tiny-b", 3, 0.6), ("tiny-c", 1, 1.0), ("tiny-d", 2, 0.0)])
def test_beam_search_equals_a_search_by_recomputation(folders, name, w, penalty):
    from kvforge_b200 import BeamParams

    prompts = prompts_for(name, [5, 33, 16, 1, 18], seed=40)
    plain = PlainLlama(folders[name])
    vocab = TINY[name]["cfg"].vocab_size
    stops = list(range(0, vocab, 5))
    engine = engine_for(folders[name], name, max_num_seqs=3 * w)
    for stop in ([], stops):
        outs = engine.beam_search(prompts, BeamParams(num_beams=w, max_tokens=12, length_penalty=penalty, num_return=w, stop_token_ids=stop, ignore_eos=not stop))
        for p, o in zip(prompts, outs):
            want, gap = plain_beams(plain, p, w, 12, set(stop), penalty)
            assert gap > 1e-5, "the prompt's candidates lie too close to one another"
            assert o.prompt_token_ids == p
            assert [h.token_ids for h in o.hypotheses] == [t for t, _ in want]
            for h, (t, lp) in zip(o.hypotheses, want):
                assert abs(h.logprob - lp) < 1e-4 * max(1.0, abs(lp)) and abs(h.score - lp / len(t) ** penalty) < 1e-4 * max(1.0, abs(lp))
        engine.block_manager.check_invariants()
        assert engine.block_manager.num_free_blocks == engine.block_manager.num_blocks
        assert engine.core.state_slots.num_free == engine.core.state_slots.num_slots


def test_beams_of_requests_with_adapters(folders):
    """The two together: every prompt its adapter, beams against a search over the merged model; then sampling goes on as before."""
    from kvforge_b200 import BeamParams

    name = "tiny-a"
    folder = folders[name]
    made = {"one": make_adapter(folder, 8, 11), "two": make_adapter(folder, 20, 12)}
    engine = engine_for(folder, name, max_num_seqs=8, num_blocks=64)
    for key, a in made.items():
        engine.load_adapter(key, *a)
    plains = {None: PlainLlama(folder), **{k: merged(folder, a) for k, a in made.items()}}
    prompts, chosen = prompts_for(name, [20, 9, 31], seed=70), ["two", None, "one"]
    before = engine.generate(prompts, greedy(6), adapters=chosen)
    outs = engine.beam_search(prompts, BeamParams(num_beams=4, max_tokens=9, num_return=4, ignore_eos=True), adapters=chosen)
    for p, c, o in zip(prompts, chosen, outs):
        want, gap = plain_beams(plains[c], p, 4, 9, set(), 1.0)
        assert gap > 1e-5
        assert [h.token_ids for h in o.hypotheses] == [t for t, _ in want]
    after = engine.generate(prompts, greedy(6), adapters=chosen)
    assert [o.output_token_ids for o in before] == [o.output_token_ids for o in after] == [plains[c].greedy(p, 6) for p, c in zip(prompts, chosen)]


@pytest.mark.parametrize("preset", ["mopilorn-tiny", "setenex-tiny", "sonalix-tiny", "ritizen-tiny", "latuzen-tiny", "gukirax-tiny"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_beams_of_models_with_states_and_windows(tmp_path, preset, dtype):
    """Every hypothesis's log probability is that of its tokens fed one after another to a request of its own: pages and states
    followed their beams."""
    from kvforge_b200 import PRESETS, BeamParams, CacheConfig, EngineConfig, InferenceEngine, SchedulerConfig
    from kvforge_b200.engine.step import BatchItem

    cfg = EngineConfig(model=PRESETS[preset], cache=CacheConfig(block_size=16, num_blocks=128), scheduler=SchedulerConfig(max_num_seqs=8, max_num_batched_tokens=64, max_model_len=128), dtype=dtype)
    engine = InferenceEngine(cfg, init_std=0.15)
    vocab = engine.vocab_size
    prompts = [random_tokens(vocab, n, seed=n) for n in (5, 37, 16)]
    n = 24
    outs = engine.beam_search(prompts, BeamParams(num_beams=4, max_tokens=n, num_return=4, ignore_eos=True))
    assert all(len(o.hypotheses) == 4 and len({tuple(h.token_ids) for h in o.hypotheses}) == 4 for o in outs)
    # 32 bits: sums of the same rows in another order; bfloat16: rows that were rounded alike, beside other rows in the batch
    tol = 2e-3 if dtype == "float32" else 0.25
    for o in outs:
        for i, h in enumerate(o.hypotheses):
            seq = f"again-{i}"
            engine.block_manager.allocate(seq, len(o.prompt_token_ids))
            engine.core.state_slots.allocate(seq)
            logits = engine.runner.step([BatchItem(seq, o.prompt_token_ids, 0, "last")])
            total = 0.0
            for k, t in enumerate(h.token_ids):
                total += float(torch.log_softmax(logits[0].double(), 0)[t])
                if k + 1 < len(h.token_ids):
                    at = len(o.prompt_token_ids) + k
                    engine.block_manager.append_slots(seq, at + 1, at)
                    logits = engine.runner.step([BatchItem(seq, [t], at, "last")])
            engine.block_manager.free(seq)
            engine.core.state_slots.free(seq)
            assert abs(total - h.logprob) < tol, (o.prompt_token_ids, h, total)
    engine.block_manager.check_invariants()


def test_generate_with_an_unknown_adapter_leaves_nothing_behind(folders):
    engine = engine_for(folders["tiny-a"], "tiny-a")
    with pytest.raises(ValueError):
        engine.generate([[1, 2], [3]], greedy(2), adapters=[None, "none of them"])
    assert not engine.has_unfinished_requests()


def test_beam_search_of_prompts_cut_and_whole(folders):
    """How prompts come to their steps changes nothing, the cap on a portion without portions included."""
    from kvforge_b200 import BeamParams

    name = "tiny-a"
    prompts = prompts_for(name, [20, 18, 25, 3, 40], seed=5)
    outs = []
    for sched in (dict(), dict(max_prefill_chunk=8), dict(max_num_batched_tokens=48, enable_chunked_prefill=False, max_prefill_chunk=8)):
        engine = engine_for(folders[name], name, **sched)
        found = engine.beam_search(prompts, BeamParams(num_beams=2, max_tokens=4, num_return=2, ignore_eos=True))
        outs.append([[h.token_ids for h in o.hypotheses] for o in found])
    assert outs[0] == outs[1] == outs[2]


def test_beam_search_refusals_and_pressure(folders):
    from kvforge_b200 import BeamParams
    from kvforge_b200.engine.scheduler import RequestRejectedError

    name = "tiny-a"
    engine = engine_for(folders[name], name, num_blocks=12, max_num_seqs=8)
    prompts = prompts_for(name, [20, 18, 25, 3], seed=3)
    # room for one prompt's beams at a time: the others wait, and nothing changes in what comes out
    many = engine.beam_search(prompts, BeamParams(num_beams=3, max_tokens=20, num_return=3, ignore_eos=True))
    alone = [engine.beam_search([p], BeamParams(num_beams=3, max_tokens=20, num_return=3, ignore_eos=True))[0] for p in prompts]
    assert [[h.token_ids for h in o.hypotheses] for o in many] == [[h.token_ids for h in o.hypotheses] for o in alone]
    for bad, params in (([[]], BeamParams()), ([list(range(200)) * 2], BeamParams()), ([[1] * 100], BeamParams(num_beams=4, max_tokens=100)), ([[1, 2]], BeamParams(num_beams=9))):
        with pytest.raises((RequestRejectedError, ValueError)):
            engine.beam_search(bad, params)
    with pytest.raises(ValueError):
        engine.beam_search([[1, 10**6]])
    engine.add_request(prompts[0], greedy(3))
    with pytest.raises(RuntimeError, match="unfinished"):
        engine.beam_search([[1, 2]])
    while engine.has_unfinished_requests():
        engine.step()
    assert engine.block_manager.num_free_blocks == 12
    assert engine.beam_search([]) == []


def test_more_beams_than_continuations(folders, tmp_path):
    """A vocabulary of three tokens cannot fill eight beams at once: places stay empty until there are enough."""
    from kvforge_b200 import BeamParams, ModelConfig
    from kvforge_b200.models.folder import write_random_model

    cfg = ModelConfig(
        vocab_size=3, hidden_size=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=96, rms_norm_eps=1e-5, rope_theta=10000.0,
        tie_word_embeddings=False, max_position_embeddings=128,
    )  # fmt: skip
    write_random_model(tmp_path / "m", cfg, seed=3, store_dtype=torch.bfloat16, init_std=0.2, norm_std=0.1)
    engine = engine_for(tmp_path / "m", "tiny-a", max_num_seqs=16, max_model_len=64)
    out = engine.beam_search([[0, 1, 2, 1], [2]], BeamParams(num_beams=8, max_tokens=5, num_return=8, ignore_eos=True))
    plain = PlainLlama(tmp_path / "m")
    for prompt, o in zip(([0, 1, 2, 1], [2]), out):
        want, gap = plain_beams(plain, prompt, 8, 5, set(), 1.0)
        assert gap > 1e-5
        assert [h.token_ids for h in o.hypotheses] == [t for t, _ in want]


def test_command_line(folders, tmp_path):
    import os
    import subprocess
    import sys
    from pathlib import Path

    from kvforge_b200.weights.safetensors_io import write_safetensors

    folder = folders["tiny-a"]
    tensors, _ = make_adapter(folder, 4, 6)
    write_safetensors(tmp_path / "adapter_model.safetensors", tensors)
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 2}))
    root = Path(__file__).resolve().parent.parent
    cmd = [sys.executable, str(root / "bin" / "generate"), "--hf-model", str(folder), "--dtype", "float32", "--prompt-ids", "5,17,3", "--max-tokens", "6", "--ignore-eos",
           "--num-beams", "2", "--adapter", str(tmp_path), "--num-blocks", "64", "--max-model-len", "64"]  # fmt: skip
    res = subprocess.run(cmd, capture_output=True, text=True, env={**os.environ, "PYTHONPATH": str(root)}, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
    got = json.loads(res.stdout.strip().splitlines()[-1])
    want, _ = plain_beams(merged(folder, (tensors, 0.5)), [5, 17, 3], 2, 6, set(), 1.0)
    assert [h["output_token_ids"] for h in got["hypotheses"]] == [t for t, _ in want]
