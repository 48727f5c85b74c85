"""The operators of requests that share one base model, as they are measured.

* ``adapter``: low-rank adapters of many requests at once, added to what the shared projection made
  (``ops.group_by_adapter`` and ``ops.adapter_add``): row ``n`` of the result is
  ``base[n] + scale[s] * B[s] (A[s] x[n])`` with ``s = ids[n]``, and ``base[n]`` where that is -1.  A projection that
  stacks several matrices (queries, keys and values; gates and ups in alternating blocks of 8 rows) has a matrix ``A`` a section.
* ``select``: the best continuations of every prompt's beams (``ops.beam_select``): the ``k`` highest of
  ``score[beam] + log_softmax(logits[beam])[token]`` over a prompt's beams and the vocabulary, best first.
* ``pages`` and ``states``: what the choice moves (``ops.copy_pages``, ``ops.copy_states``): a beam's last, partly filled page
  in every layer, and its rows of the recurrent states, go to the beams that continue it.

Sizes are those of the presets (``kvforge_b200.PRESETS``): widths, heads, vocabulary, state sizes, 16 tokens a page.
"""

from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16  # tokens a page, the default of the engine's configuration
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
GATE_BLOCK = 8  # gates and ups alternate in blocks of so many columns

# projections of the presets: (input width, ends of the sections of the output, gates and ups alternate, 32-bit rows)
PROJECTIONS = {
    "1b-o": (2048, (2048,), False, True),
    "1b-gate-up": (2048, (8192, 16384), True, False),
    "1b-down": (8192, (2048,), False, True),
    "8b-qkv": (4096, (4096, 5120, 6144), False, False),
    "8b-o": (4096, (4096,), False, True),
    "8b-gate-up": (4096, (14336, 28672), True, False),
    "8b-down": (14336, (4096,), False, True),
    "tiny-qkv": (64, (64, 96, 128), False, False),
}
# caches of the presets: (layers that keep one, heads, key head, value head or 0 where values lie inside the keys)
CACHES = {
    "llama-3.2-1b": (16, 8, 64, 64),
    "llama-3.1-8b": (32, 8, 128, 128),
    "setenex-1b-window": (12, 8, 64, 64),
    "setenex-1b-latent": (4, 1, 576, 0),
}
# recurrent states of the presets: how many layers keep how many floats a request
STATES = {
    "sonalix-1b": ((4, 262144),),
    "latuzen-1b": ((4, 270352),),
    "ritizen-1b": ((4, 537344), (4, 262144)),
    "mopilorn-1b": ((8, 149504), (8, 280576)),
}


def listed() -> list[dict]:
    return [
        # one prompt in four beams, the smallest choice: latency is all of it
        dict(name="select-1x4", call="select", prompts=1, beams=4, vocab=128256, k=8, masked=0.0),
        # an odd vocabulary whose rows begin off 16 bytes, forbidden tokens, beams that are not alive yet
        dict(name="select-7x3-odd", call="select", prompts=7, beams=3, vocab=50021, k=6, masked=0.1),
        # a busy server's step: 64 prompts of eight beams over the vocabulary of the Llama shapes
        dict(name="select-64x8", call="select", prompts=64, beams=8, vocab=128256, k=16, masked=0.0),
        # the beams of eight prompts after a step: a dozen partly filled pages of a small model's cache
        dict(name="pages-1b-12", call="pages", cache="llama-3.2-1b", dtype="bfloat16", blocks=256, copies=12),
        # the forks of a busy server at the 8B shape
        dict(name="pages-8b-192", call="pages", cache="llama-3.1-8b", dtype="bfloat16", blocks=448, copies=192),
        # one beam of a small retention model forks: the smallest copy of states
        dict(name="states-sonalix-1", call="states", model="sonalix-1b", slots=8, copies=1),
        # a step of eight prompts in four beams of a delta-rule model: whole states of sixteen layers move
        dict(name="states-mopilorn-20", call="states", model="mopilorn-1b", slots=40, copies=20),
        # a decode step of eight requests, each with an adapter of its own: the smallest adapter call, three sections
        dict(name="adapter-decode-8", call="adapter", projection="8b-qkv", dtype="bfloat16", tokens=8, used=8, slots=16, rank=16, single=8),
        # a decode step of a busy server: 64 requests on 20 adapters (and the base), added to the 32-bit rows
        dict(name="adapter-decode-64-down", call="adapter", projection="1b-down", dtype="bfloat16", tokens=64, used=20, slots=32, rank=32, single=64),
        # a whole prompt of one request through the stacked projection of the 8B shape
        dict(name="adapter-prompt-2048", call="adapter", projection="8b-qkv", dtype="bfloat16", tokens=2048, used=1, slots=4, rank=16, single=0),
        # decoding requests beside two portions of prompts, through gates and ups of the 8B shape: the largest call
        dict(name="adapter-mixed-gate-up", call="adapter", projection="8b-gate-up", dtype="bfloat16", tokens=1057, used=24, slots=32, rank=64, single=33),
        # a ragged portion in true 32-bit, what exact replay and debugging run
        dict(name="adapter-float32", call="adapter", projection="1b-o", dtype="float32", tokens=515, used=3, slots=4, rank=16, single=2),
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    call = rng.choice(["select", "select", "pages", "states", "adapter", "adapter", "adapter"])
    if call == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        prompts = _log_uniform(rng, 1, 512 // beams)
        k = rng.choice([beams, 2 * beams, 2 * beams])
        return dict(call=call, prompts=prompts, beams=beams, vocab=_log_uniform(rng, 200, 128256), k=k, masked=rng.choice([0.0, 0.0, 0.2]))
    if call == "pages":
        blocks = _log_uniform(rng, 8, 448)
        return dict(call=call, cache=rng.choice(list(CACHES)), dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), blocks=blocks, copies=_log_uniform(rng, 1, max(1, blocks // 2 - 1)))
    if call == "states":
        slots = _log_uniform(rng, 2, 40)
        return dict(call=call, model=rng.choice(list(STATES)), slots=slots, copies=_log_uniform(rng, 1, slots // 2))
    projection = rng.choice(list(PROJECTIONS))
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    tokens = _log_uniform(rng, 1, 700 if dtype == "float32" or "gate-up" in projection else 2048)
    single = rng.choice([0, tokens, min(tokens, 32)])
    slots = _log_uniform(rng, 1, 32)
    used = rng.randint(1, slots)
    return dict(call=call, projection=projection, dtype=dtype, tokens=tokens, used=min(used, tokens), slots=slots, rank=rng.choice([4, 8, 16, 16, 24, 32, 64]), single=single)


# ------------------------------------------------------------------ inputs


def _generator(seed: int, salt: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + salt)


def _adapters_of(case: dict) -> list[int]:
    """Which of the adapters in use (0 .. used - 1; -1: the base alone) each row takes: ``single`` decoding requests turn by
    turn, every ninth without one, then portions of prompts of equal length."""
    used, n, single = case["used"], case["tokens"], case["single"]
    rows = [-1 if i % 9 == 8 else i % used for i in range(single)]
    portions = min(2, used)
    rows += [(i * portions // max(1, n - single)) % used for i in range(n - single)]
    return rows


def _padded(rank: int) -> int:
    return -(-rank // 16) * 16


def _prepare_adapter(case: dict, seed: int) -> dict:
    k, ends, alternating, wide = PROJECTIONS[case["projection"]]
    n, slots, rank, sections, width = case["tokens"], case["slots"], case["rank"], len(ends), ends[-1]
    dtype = TYPES[case["dtype"]]
    g = _generator(seed, 1)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    # adapters live in a bank of one size: ranks below it are filled with zeros (whole sixteens)
    a = torch.zeros((slots, sections, _padded(rank), k), dtype=dtype, device="cuda")
    b = torch.zeros((slots, width, _padded(rank)), dtype=dtype, device="cuda")
    a[:, :, :rank] = (normal(slots, sections, rank, k) * k**-0.5).to(dtype)
    b[:, :, :rank] = (normal(slots, width, rank) * 0.3 * rank**-0.5).to(dtype)
    order = random.Random(seed).sample(range(slots), case["used"])  # which slots are in use
    ids = [-1 if i < 0 else order[i] for i in _adapters_of(case)]
    # the plain form's rows, in blocks of one adapter each; row n stands for "none"
    size = 16 if n <= 256 else 64
    blocks, owners = [], []
    for s in sorted(set(ids) - {-1}):
        rows = [i for i, t in enumerate(ids) if t == s]
        for at in range(0, len(rows), size):
            part = rows[at : at + size]
            blocks.append(part + [n] * (size - len(part)))
            owners.append(s)
    if alternating:
        at = torch.arange(width, device="cuda") // GATE_BLOCK
        columns = [torch.nonzero(at % 2 == s)[:, 0] for s in range(2)]
    else:
        columns = [torch.arange(lo, hi, device="cuda") for lo, hi in zip((0, *ends[:-1]), ends)]
    base = normal(n, width)
    return {
        "x": normal(n, k).to(dtype), "a": a, "b": b, "scale": 2.0 / (1.0 + torch.arange(slots, device="cuda") % 3), "ends": ends,
        "alternating": alternating, "ids": torch.tensor(ids, dtype=torch.int32, device="cuda"), "base": base if wide else base.to(dtype),
        "blocks": torch.tensor(blocks or [[n] * size], device="cuda"), "owners": torch.tensor(owners or [0], device="cuda"),
        "columns": columns, "place": torch.argsort(torch.cat(columns)),
    }  # fmt: skip


def _prepare_select(case: dict, seed: int) -> dict:
    g = _generator(seed, 2)
    rows, v = case["prompts"] * case["beams"], case["vocab"]
    # the logits of a trained model: a broad body and a tail of a few likely tokens
    logits = 2.0 * torch.randn((rows, v), generator=g, device="cuda")
    logits -= torch.log(-torch.log(torch.rand((rows, v), generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)))
    scores = -25.0 * torch.rand((case["prompts"], case["beams"]), generator=g, device="cuda")
    if case["masked"]:
        logits.masked_fill_(torch.rand((rows, v), generator=g, device="cuda") < case["masked"], -math.inf)
        scores[::3, 1:] = -math.inf  # a prompt's first choice: one beam is alive
    return {"logits": logits, "scores": scores.reshape(-1), "prompts": case["prompts"], "k": case["k"]}


def _pairs(case: dict, seed: int, places: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Sources (a beam that is continued twice is one twice) and targets of the copies; no source is a target."""
    order = random.Random(seed).sample(range(places), places)
    targets, rest = order[: case["copies"]], order[case["copies"] :]
    sources = [rest[(i // 2) % len(rest)] for i in range(case["copies"])]
    return tuple(torch.tensor(t, dtype=torch.int32, device="cuda") for t in (sources, targets))


def prepare(case: dict, seed: int) -> dict:
    if case["call"] == "adapter":
        return {"call": "adapter", **_prepare_adapter(case, seed)}
    if case["call"] == "select":
        return {"call": "select", **_prepare_select(case, seed)}
    g = _generator(seed, 3)
    if case["call"] == "pages":
        layers, heads, d, dv = CACHES[case["cache"]]
        shape = (layers, case["blocks"], heads, PAGE)
        new = lambda width: torch.randn((*shape, width), generator=g, device="cuda", dtype=TYPES[case["dtype"]])  # noqa: E731
        src, dst = _pairs(case, seed, case["blocks"])
        # positions written of each page: 1 to 16, whatever the prompts' lengths are
        tokens = 1 + (torch.arange(case["copies"], device="cuda") * 5 % PAGE)
        return {"call": "pages", "k": new(d), "v": new(dv) if dv else None, "src": src, "dst": dst, "tokens": tokens.to(torch.int32)}
    src, dst = _pairs(case, seed, case["slots"])
    states = [torch.randn((case["slots"], width), generator=g, device="cuda") for count, width in STATES[case["model"]] for _ in range(count)]
    return {"call": "states", "states": states, "src": src, "dst": dst}


# ------------------------------------------------------------------ one pass


def _run_own(state: dict):
    from kvforge_b200 import ops

    if state["call"] == "adapter":
        if "bank" not in state:  # a program makes its bank, its groups and its rows once and keeps them
            state["bank"] = ops.AdapterBank(state["a"], state["b"], state["scale"], state["ends"], state["alternating"])
            state["groups"] = ops.AdapterGroups(state["x"].shape[0], state["a"].shape[0], state["x"].device)
            state["out"] = torch.empty_like(state["base"])
        ops.group_by_adapter(state["ids"], state["groups"])
        ops.adapter_add(state["x"], state["bank"], state["groups"], state["out"], base=state["base"])
        return state["out"]
    if state["call"] == "select":
        if "workspace" not in state:
            rows, v = state["logits"].shape
            shape = (state["prompts"], state["k"])
            state["workspace"] = ops.beam_workspace(rows, v, state["k"], state["logits"].device)
            state["parents"], state["tokens"] = (torch.empty(shape, dtype=torch.int32, device="cuda") for _ in range(2))
            state["best"] = torch.empty(shape, dtype=torch.float32, device="cuda")
        ops.beam_select(state["logits"], state["scores"], state["parents"], state["tokens"], state["best"], state["workspace"])
        return {"parents": state["parents"], "tokens": state["tokens"], "scores": state["best"]}
    if state["call"] == "pages":
        ops.copy_pages(state["k"], state["v"], state["src"], state["dst"], state["tokens"])
        return {"keys": state["k"], "values": state["v"]}
    if "table" not in state:
        state["table"] = ops.StateTable(state["states"])
    ops.copy_states(state["table"], state["src"], state["dst"])
    return state["states"]


def _plain_adapter(state: dict) -> torch.Tensor:
    x, a, b, owners = state["x"].float(), state["a"], state["b"], state["owners"]
    n, rank, width = x.shape[0], a.shape[2], b.shape[1]
    rows = torch.cat([x, x.new_zeros((1, x.shape[1]))])[state["blocks"]]
    inner = rows @ a[owners].flatten(1, 2).float().transpose(1, 2) * state["scale"][owners][:, None, None]
    outer = b[owners].float()
    parts = [inner[..., s * rank : (s + 1) * rank] @ outer[:, c].transpose(1, 2) for s, c in enumerate(state["columns"])]
    delta = torch.cat(parts, dim=-1)[..., state["place"]]
    out = torch.cat([state["base"].float(), x.new_zeros((1, width))])
    out.index_add_(0, state["blocks"].flatten(), delta.flatten(0, 1))
    return out[:n].to(state["base"].dtype)


def _plain_select(state: dict) -> dict:
    # 64 bits: the k-th candidate of a million lies next to others
    x, prompts, k = state["logits"].double(), state["prompts"], state["k"]
    v, scores = x.shape[1], state["scores"].double()[:, None]
    top = x.amax(dim=1, keepdim=True)
    total = top + torch.log(torch.exp(x - top).sum(dim=1, keepdim=True))
    every = scores + (x - total)
    every = torch.where(torch.isnan(every) | ~torch.isfinite(scores), -math.inf, every).view(prompts, -1)
    # the k highest, of equal ones those with the lowest place
    least = torch.topk(every, k, dim=1).values[:, -1:]
    above, equal = every > least, every == least
    taken = above | (equal & (torch.cumsum(equal, dim=1) <= k - above.sum(dim=1, keepdim=True)))
    place = torch.where(taken, torch.arange(every.shape[1], device=x.device), every.shape[1])
    place = torch.topk(place, k, dim=1, largest=False, sorted=True).values
    best, order = torch.sort(every.gather(1, place), dim=1, descending=True, stable=True)
    place = place.gather(1, order)
    none = best == -math.inf
    parents, tokens = (place // v).masked_fill(none, -1), (place % v).masked_fill(none, -1)
    return {"parents": parents.to(torch.int32), "tokens": tokens.to(torch.int32), "scores": best.float()}


def run(state: dict):
    if own:
        return _run_own(state)
    if state["call"] == "adapter":
        return _plain_adapter(state)
    if state["call"] == "select":
        return _plain_select(state)
    src, dst = state["src"].long(), state["dst"].long()
    if state["call"] == "states":
        return [t.index_copy_(0, dst, t[src]) for t in state["states"]]
    live = torch.arange(PAGE, device=src.device) < state["tokens"][:, None]
    live = live[None, :, None, :, None]
    caches = [t for t in (state["k"], state["v"]) if t is not None]
    moved = [t.index_copy_(1, dst, torch.where(live, t[:, src], t[:, dst])) for t in caches]
    return {"keys": moved[0], "values": moved[1] if len(moved) > 1 else None}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case: dict) -> dict:
    if case["call"] == "select":
        rows = case["prompts"] * case["beams"]
        return {"bytes": 4 * rows * case["vocab"] + 4 * rows + 12 * case["prompts"] * case["k"], "flops": 4 * rows * case["vocab"]}
    if case["call"] == "pages":
        layers, heads, d, dv = CACHES[case["cache"]]
        tokens = sum(1 + i * 5 % PAGE for i in range(case["copies"]))
        return {"bytes": 2 * tokens * layers * heads * (d + dv) * (4 if case["dtype"] == "float32" else 2) + 12 * case["copies"], "flops": 0}
    if case["call"] == "states":
        return {"bytes": 8 * case["copies"] * sum(count * width for count, width in STATES[case["model"]]) + 8 * case["copies"], "flops": 0}
    k, ends, _, wide = PROJECTIONS[case["projection"]]
    size = 4 if case["dtype"] == "float32" else 2
    width, rank = ends[-1], case["rank"]
    rows = [i for i in _adapters_of(case) if i >= 0]
    weights = len(set(rows)) * rank * (len(ends) * k + width) * size
    bytes_ = len(rows) * k * size + weights + 2 * case["tokens"] * width * (4 if wide else size) + 4 * case["tokens"]
    return {"bytes": bytes_, "flops": 2 * len(rows) * rank * (len(ends) * k + width)}


# ------------------------------------------------------------------ the same numbers in 64 bits


def exact(case: dict, seed: int):
    if case["call"] in ("pages", "states"):
        return None  # nothing is computed
    state = prepare(case, seed)
    if case["call"] == "select":
        return _exact_select(state)
    x, ids = state["x"].double(), state["ids"].tolist()
    k, ends, alternating, _ = PROJECTIONS[case["projection"]]
    out = state["base"].double()
    for s in set(ids) - {-1}:
        rows = torch.tensor([i for i, t in enumerate(ids) if t == s], device=x.device)
        h = torch.einsum("nk,grk->ngr", x[rows], state["a"][s].double()) * float(state["scale"][s])
        b = state["b"][s].double()
        for section in range(len(ends)):
            if alternating:
                columns = [c for c in range(ends[-1]) if c // GATE_BLOCK % 2 == section]
            else:
                columns = list(range(ends[section - 1] if section else 0, ends[section]))
            columns = torch.tensor(columns, device=x.device)
            out[rows[:, None], columns[None, :]] += torch.einsum("nr,cr->nc", h[:, section], b[columns])
    return out


def _exact_select(state: dict) -> dict:
    prompts, k = state["prompts"], state["k"]
    v = state["logits"].shape[1]
    beams = state["logits"].shape[0] // prompts
    parents, tokens, scores = [], [], []
    for p in range(prompts):
        rows = slice(p * beams, (p + 1) * beams)
        log_p = state["logits"][rows].double()
        log_p = log_p - torch.logsumexp(log_p, dim=1, keepdim=True)
        total = (log_p + state["scores"][rows].double()[:, None]).flatten()
        total = torch.nan_to_num(total, nan=-math.inf, neginf=-math.inf, posinf=math.inf)
        order = torch.sort(-total, stable=True).indices[:k]
        best = total[order]
        found = best > -math.inf
        parents.append(torch.where(found, order // v, -1))
        tokens.append(torch.where(found, order % v, -1))
        scores.append(best)
    return {"parents": torch.stack(parents).int(), "tokens": torch.stack(tokens).int(), "scores": torch.stack(scores)}
