"""The host side of beams and adapters: shared pages, slots that are not cleared, the rules of a choice, what adapters may be."""

from __future__ import annotations

import json
import random

import pytest
import torch

from kvforge_b200 import AdapterConfig, BeamParams
from kvforge_b200.cache.block_manager import RELEASED, BlockManager, GroupSpec, NoFreeBlocksError
from kvforge_b200.cache.state_slots import StateSlotPool
from kvforge_b200.engine.beam import BeamGroup, _Beam
from kvforge_b200.engine.request import FinishReason
from kvforge_b200.engine.step import BatchItem, _Layout
from kvforge_b200.parts.adapters import AdapterError, AdapterStore, read_adapter
from kvforge_b200.weights.safetensors_io import write_safetensors


def test_fork_shares_full_pages_and_copies_the_last():
    bm = BlockManager(16, 4)
    bm.allocate("a", 10)
    copies = bm.fork("a", "b", 10)
    a, b = bm.get_block_table("a"), bm.get_block_table("b")
    assert a[:2] == b[:2] and a[2] != b[2]
    assert copies == [(0, a[2], b[2], 2)]
    assert bm.num_free_blocks == 16 - 4
    bm.check_invariants()
    assert bm.stats().num_used_blocks == 4 and bm.stats().num_tokens == 4 + 4 + 2 + 2
    bm.append_slots("b", 13, 12)
    bm.free("a")
    bm.check_invariants()
    assert bm.num_free_blocks == 16 - 4  # two shared pages, b's third and fourth
    bm.free("b")
    bm.check_invariants()
    assert bm.num_free_blocks == 16


def test_fork_at_a_page_boundary_copies_nothing():
    bm = BlockManager(8, 4)
    bm.allocate("a", 8)
    assert bm.fork("a", "b", 8) == []
    assert bm.get_block_table("a") == bm.get_block_table("b") and bm.num_free_blocks == 6
    bm.append_slots("a", 9, 8)
    bm.append_slots("b", 9, 8)
    assert bm.get_block_table("a")[2] != bm.get_block_table("b")[2]
    bm.check_invariants()


def test_fork_refusals():
    bm = BlockManager(3, 4)
    bm.allocate("a", 10)
    with pytest.raises(NoFreeBlocksError):
        bm.fork("a", "b", 10)
    bm.check_invariants()
    assert not bm.has_seq("b")
    with pytest.raises(KeyError):
        bm.fork("x", "b", 1)
    with pytest.raises(ValueError):
        bm.fork("a", "b", 13)
    bm.fork("a", "b", 8)
    with pytest.raises(ValueError):
        bm.fork("a", "b", 8)


def test_fork_of_windows_shares_what_is_left():
    bm = BlockManager(12, 4, groups=[GroupSpec(), GroupSpec("window", 6)])
    bm.allocate("a", 4, 4)
    for n in range(5, 20):
        bm.append_slots("a", n, n - 1)
    copies = bm.fork("a", "b", 19)
    assert {c[0] for c in copies} == {0, 1} and all(c[3] == 3 for c in copies)
    assert bm.get_block_table("b", 1)[0] == RELEASED
    bm.check_invariants()
    # both walk on: a page that is shared comes back when the second of them has left it behind
    for n in range(20, 30):
        bm.append_slots("a", n, n - 1)
        bm.check_invariants()
        bm.append_slots("b", n, n - 1)
        bm.check_invariants()
    bm.free("a")
    bm.free("b")
    bm.check_invariants()
    assert bm.num_free_blocks == 12


def test_forks_at_random_lose_no_page():
    rng = random.Random(5)
    bm = BlockManager(200, 4, groups=[GroupSpec(), GroupSpec("window", 9, keep_first=3)])
    live = {}
    for i in range(600):
        if live and rng.random() < 0.35:
            seq = rng.choice(list(live))
            bm.free(seq)
            del live[seq]
        elif live and rng.random() < 0.6:
            seq = rng.choice(list(live))
            if len(live) < 12:
                bm.fork(seq, f"s{i}", live[seq])
                live[f"s{i}"] = live[seq]
            for s in (seq, *((f"s{i}",) if f"s{i}" in live else ())):
                if live[s] < 60:
                    bm.append_slots(s, live[s] + 1, live[s])
                    live[s] += 1
        elif len(live) < 12:
            live[f"s{i}"] = rng.randint(1, 20)
            bm.allocate(f"s{i}", live[f"s{i}"])
        bm.check_invariants()
    for seq in live:
        bm.free(seq)
    bm.check_invariants()
    assert bm.num_free_blocks == 200


def test_state_slots_that_are_not_cleared():
    pool = StateSlotPool(3)
    pool.allocate("a")
    pool.take_fresh()
    pool.allocate("b")
    pool.free("b")
    slot = pool.allocate("c", fresh=False)  # the slot that b left behind before any step
    assert slot not in pool.take_fresh()
    pool.check_invariants()


# ------------------------------------------------------------------ the rules of a choice


def group(w=2, **kw):
    g = BeamGroup([1, 2], BeamParams(num_beams=w, **kw), {9}, kw.get("max_tokens", 64))
    g.beams = [_Beam(str(i), [5 + i], -0.5 - i) for i in range(w)]
    return g


def test_choice_keeps_the_best_and_ends_hypotheses():
    g = group()
    # the first of four candidates is a stop token, the second and the fourth go on; the third stops beyond the first two
    assert g.choose([0, 1, 1, 0], [9, 4, 9, 7], [-1.0, -1.5, -1.6, -2.0]) == [(1, 4, -1.5), (0, 7, -2.0)]
    assert [(h.token_ids, h.finish_reason) for h in g.finished] == [([5, 9], FinishReason.STOP)]
    assert g.finished[0].score == -0.5 and not g.done


def test_choice_ends_when_no_beam_can_beat_what_is_finished():
    g = group()
    g.choose([0, 1, 0, 1], [9, 9, 3, 4], [-0.1, -0.2, -8.0, -9.0])
    assert g.done and [h.token_ids for h in g.finished] == [[5, 9], [6, 9]]


def test_choice_at_the_length_limit():
    g = group(max_tokens=2)
    assert g.choose([0, 0, 1, 1], [3, 4, 9, 5], [-1.0, -1.1, -1.2, -1.3]) == []
    assert g.done and [(h.token_ids, h.finish_reason) for h in g.finished] == [([5, 3], FinishReason.LENGTH), ([5, 4], FinishReason.LENGTH)]


def test_choice_without_candidates_and_with_few():
    g = group()
    assert g.choose([-1, -1], [-1, -1], [float("-inf")] * 2) == [] and g.done and g.finished == []
    g = group(w=3)
    assert g.choose([0, 2, -1, -1, -1, -1], [1, 2, -1, -1, -1, -1], [-1.0, -2.0] + [float("-inf")] * 4) == [(0, 1, -1.0), (2, 2, -2.0)]


def test_length_penalty():
    g = group(length_penalty=0.0)
    g.choose([0, 0, 1, 1], [9, 3, 4, 5], [-1.0, -3.0, -3.0, -4.0])
    assert g.finished[0].score == -1.0


def test_beam_parameter_refusals():
    for kw in (dict(num_beams=0), dict(num_beams=33), dict(max_tokens=0), dict(num_return=0), dict(num_beams=2, num_return=3), dict(length_penalty=float("inf")), dict(length_penalty=float("nan")), dict(length_penalty=1e4)):
        with pytest.raises(ValueError):
            BeamParams(**kw)


# ------------------------------------------------------------------ adapters


def test_adapter_config_refusals():
    for kw in (dict(max_adapters=0), dict(max_adapters=5000), dict(max_rank=0), dict(max_rank=129)):
        with pytest.raises(ValueError):
            AdapterConfig(**kw)


def test_read_adapter(tmp_path):
    with pytest.raises(AdapterError):
        read_adapter(tmp_path)
    t = {"base_model.model.model.layers.0.self_attn.q_proj.lora_A.weight": torch.randn(4, 8)}
    write_safetensors(tmp_path / "adapter_model.safetensors", t)
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 8}))
    tensors, scale = read_adapter(tmp_path)
    assert scale == 2.0 and torch.equal(tensors[next(iter(t))], t[next(iter(t))])
    for bad in ({"r": 0}, {"r": 4, "use_dora": True}, {"r": 4, "bias": "all"}, {"r": 4, "rank_pattern": {"q": 2}}):
        (tmp_path / "adapter_config.json").write_text(json.dumps(bad))
        with pytest.raises(AdapterError):
            read_adapter(tmp_path)
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 8, "use_rslora": True}))
    assert read_adapter(tmp_path)[1] == 4.0


def test_adapter_store_refusals():
    store = AdapterStore(2, 8, 16, torch.float32, torch.device("cpu"))
    store.declare(["q", "k"], [16, 8], 8)
    a, b = torch.randn(4, 8), torch.randn(16, 4)
    good = {"q.lora_A.weight": a, "q.lora_B.weight": b}
    for bad in (
        {}, {"q.lora_A.weight": a}, {**good, "q.bias": b}, {"v.lora_A.weight": a, "v.lora_B.weight": b}, {**good, "q.lora_A.weight": torch.tensor(1.0)},
        {**good, "q.lora_B.weight": torch.randn(4)}, {**good, "q.lora_B.weight": torch.randn(8, 4)}, {"q.lora_A.weight": torch.randn(9, 8), "q.lora_B.weight": torch.randn(16, 9)},
    ):  # fmt: skip
        with pytest.raises(AdapterError):
            store.load("x", bad, 1.0)
    with pytest.raises(AdapterError):
        store.load("x", good, float("nan"))
    assert not store.slots
    assert store.load("x", good, 2.0) == 0 and store.load("y", good, 1.0) == 1
    for name in ("x", "z"):
        with pytest.raises(AdapterError):
            store.load(name, good, 1.0)
    store.unload("x")
    with pytest.raises(AdapterError):
        store.unload("x")
    with pytest.raises(AdapterError):
        store.slot("x")
    assert store.load("z", good, 1.0) == 0 and store.slot("z") == 0 and store.slot(None) == -1


def test_a_steps_layout_carries_adapters_only_where_some_are_kept():
    without, with_ids = _Layout(8, 4, 2, 1, 4), _Layout(8, 4, 2, 1, 4, adapters=True)
    assert "adapter_ids" not in without.off and with_ids.total == without.total + 8
    assert BatchItem("a", [1], 0).adapter == -1
