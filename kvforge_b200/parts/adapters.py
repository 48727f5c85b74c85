"""Low-rank adapters beside a model's projections: what parts declare, where their tensors lie, how a folder fills them.

A part that lets requests bring adapters declares its stacked projections when it is bound (``AdapterStore.declare``) and
gets an ``ops.AdapterBank`` for each; in a step with adapters it adds them to what the shared product left
(``add``).  An adapter is a set of tensor pairs ``<projection>.lora_A.weight [r, in]`` and ``<projection>.lora_B.weight
[out, r]`` (projections by their checkpoint names without ``.weight``) and one scale; it adds ``scale * B (A x)`` to each projection
that it names.  All banks hold the same adapters in the same slots; a slot's rank in a bank is zero where the adapter leaves the projection
alone.
"""

from __future__ import annotations

import json
import math
from pathlib import Path

import torch

from .. import ops
from ..weights.safetensors_io import open_model_files

_PREFIXES = ("base_model.model.", "base_model.")


class AdapterError(ValueError):
    """An adapter that does not fit the model, or a name that means none."""


def read_adapter(source: str | Path) -> tuple[dict[str, torch.Tensor], float]:
    """(tensors by name, scale) of an adapter's folder: ``adapter_config.json`` (``r``, ``lora_alpha``, optional ``use_rslora``) and safetensors."""
    path = Path(source)
    try:
        cfg = json.loads((path / "adapter_config.json").read_text())
    except OSError as e:
        raise AdapterError(f"{path} has no adapter_config.json") from e
    r = int(cfg.get("r", 0))
    if r < 1:
        raise AdapterError(f"{path}: r must be positive")
    for key in ("use_dora", "modules_to_save", "rank_pattern", "alpha_pattern"):
        if cfg.get(key):
            raise AdapterError(f"{path}: {key} is not supported")
    if cfg.get("bias", "none") != "none":
        raise AdapterError(f"{path}: biases are not supported")
    scale = float(cfg.get("lora_alpha", r)) / (r**0.5 if cfg.get("use_rslora") else r)
    tensors: dict[str, torch.Tensor] = {}
    files = open_model_files(path)
    for f in files:
        tensors.update({name: f.tensor(name).clone() for name in f.keys()})
        f.close()
    # the scale is for rank r: of another rank they belong to another configuration
    for name, t in tensors.items():
        if name.endswith(".lora_A.weight") and t.dim() == 2 and t.shape[0] != r:
            raise AdapterError(f"{path}: {name} has rank {t.shape[0]}, the configuration says {r}")
    return tensors, scale


class _Declared:
    def __init__(self, names: list[str], widths: list[int], bank: "ops.AdapterBank") -> None:
        self.names, self.widths, self.bank = names, widths, bank


class AdapterStore:
    """``Runtime.adapters``: the banks of a model and the groups of its steps."""

    def __init__(self, max_adapters: int, max_rank: int, max_tokens: int, dtype: torch.dtype, device: torch.device) -> None:
        self.max_adapters, self.max_rank, self.max_tokens = int(max_adapters), int(max_rank), int(max_tokens)
        self.rank = -(-self.max_rank // 16) * 16
        self.dtype, self.device = dtype, device
        self._declared: list[_Declared] = []
        self._groups: ops.AdapterGroups | None = None
        self.slots: dict[str, int] = {}  # loaded adapters

    # ------------------------------------------------------------------ what parts declare
    def declare(self, names: list[str], widths: list[int], k: int, alternating: bool = False) -> "ops.AdapterBank | None":
        """A bank for the projections ``names`` (of ``widths`` rows, stacked in this order or alternating in blocks of 8), or ``None``
        where widths that are no multiples of 8 rule adapters out."""
        if k % 8 or any(w % 8 for w in widths) or len(widths) * self.rank > ops.ADAPTER_MAX_ROWS:
            return None
        s, n = self.max_adapters, sum(widths)
        ends = [sum(widths[: i + 1]) for i in range(len(widths))]
        zeros = lambda *shape, dtype=self.dtype: torch.zeros(shape, dtype=dtype, device=self.device)  # noqa: E731
        bank = ops.AdapterBank(
            zeros(s, len(widths), self.rank, k), zeros(s, n, self.rank), zeros(s, dtype=torch.float32), ends, alternating, zeros(s, dtype=torch.int32)
        )
        self._declared.append(_Declared(list(names), list(widths), bank))
        self._groups = None
        return bank

    def withdraw(self, bank: "ops.AdapterBank") -> None:
        self._declared = [d for d in self._declared if d.bank is not bank]
        self._groups = None

    @property
    def groups(self) -> "ops.AdapterGroups":
        if self._groups is None:
            rows = max((d.bank.sections * d.bank.rank for d in self._declared), default=self.rank)
            self._groups = ops.AdapterGroups(self.max_tokens, self.max_adapters, self.device, max_rows=rows)
        return self._groups

    # ------------------------------------------------------------------ what callers load
    def load(self, name: str, tensors: dict[str, torch.Tensor], scale: float) -> int:
        """Put an adapter into a free slot.  Every tensor must belong to a declared projection and fit it; nothing is written
        unless all do."""
        if name in self.slots:
            raise AdapterError(f"an adapter named {name!r} is already loaded")
        if len(self.slots) >= self.max_adapters:
            raise AdapterError(f"{self.max_adapters} adapters are loaded already")
        pairs: dict[str, dict[str, torch.Tensor]] = {}
        for full, t in tensors.items():
            short = next((full[len(p) :] for p in _PREFIXES if full.startswith(p)), full)
            for which in ("A", "B"):
                tail = f".lora_{which}.weight"
                if short.endswith(tail):
                    pairs.setdefault(short[: -len(tail)], {})[which] = t
                    break
            else:
                raise AdapterError(f"{full} is not a tensor of a low-rank adapter")
        places = {proj: (d, i) for d in self._declared for i, proj in enumerate(d.names)}
        if not pairs:
            raise AdapterError("the adapter has no tensors")
        if not math.isfinite(scale):
            raise AdapterError(f"the adapter's scale is {scale}")
        for proj, ab in pairs.items():
            if proj not in places:
                raise AdapterError(f"{proj} takes no adapters in this model")
            if set(ab) != {"A", "B"}:
                raise AdapterError(f"{proj} needs both lora_A and lora_B")
            d, i = places[proj]
            a, b = ab["A"], ab["B"]
            r = a.shape[0] if a.dim() else 0
            if a.dim() != 2 or b.dim() != 2 or tuple(a.shape) != (r, d.bank.k) or tuple(b.shape) != (d.widths[i], r) or r < 1:
                raise AdapterError(f"{proj}: lora_A {tuple(a.shape)} and lora_B {tuple(b.shape)} do not fit [{d.widths[i]}, {d.bank.k}]")
            if r > self.max_rank:
                raise AdapterError(f"{proj}: rank {r} is above max_rank = {self.max_rank}")
        slot = next(i for i in range(self.max_adapters) if i not in self.slots.values())
        for d in self._declared:
            self._fill(d, slot, pairs, scale)
        self.slots[name] = slot
        return slot

    def _fill(self, d: _Declared, slot: int, pairs: dict[str, dict[str, torch.Tensor]], scale: float) -> None:
        bank = d.bank
        bank.a[slot].zero_()
        bank.b[slot].zero_()
        bank.scales[slot] = scale
        rank = 0
        for i, proj in enumerate(d.names):
            ab = pairs.get(proj)
            if ab is None:
                continue
            r = ab["A"].shape[0]
            rank = max(rank, r)
            bank.a[slot, i, :r] = ab["A"].to(bank.a)
            b = ab["B"].to(bank.b)
            if bank.alternating:
                step = ops.ADAPTER_BLOCK
                bank.b[slot].view(-1, 2, step, bank.rank)[:, i, :, :r] = b.view(-1, step, r)
            else:
                end = bank.ends[i]
                bank.b[slot, end - d.widths[i] : end, :r] = b
        bank.ranks[slot] = rank

    def unload(self, name: str) -> None:
        if name not in self.slots:
            raise AdapterError(f"no adapter named {name!r} is loaded")
        del self.slots[name]

    def slot(self, name: str | None) -> int:
        if name is None:
            return -1
        if name not in self.slots:
            raise AdapterError(f"no adapter named {name!r} is loaded")
        return self.slots[name]


def add(ctx, bank: "ops.AdapterBank | None", x: torch.Tensor, out) -> None:
    """Add the step's adapters to the product of ``x`` (a tensor, or the slices of a split product: to the first)."""
    if bank is not None and ctx.adapters is not None:
        ops.adapter_add(x, bank, ctx.adapters, out.t[0] if isinstance(out, ops.Partials) else out)
