"""Low-rank adapters beside the layers' projections: y[t] += scale[s] B[s] (A[s] x[t]) for the tokens of requests that use the adapter in slot s.

A model that is built with slots keeps room for that many adapters beside every projection that takes them (``AdapterSlots.projection``). An adapter
is loaded into a slot while the model runs; a step's tokens are dealt out to their adapters by lists that the batch carries (``StepBatch.adapters``), so a
step may mix requests of any adapters and of none. Adapters are read as they are published: adapter_config.json (``r``, ``lora_alpha``) beside
adapter_model.safetensors with ``base_model.model.<module>.lora_A.weight`` [r, in] and ``lora_B.weight`` [out, r].
"""
from __future__ import annotations

import json
import math
import weakref
from dataclasses import dataclass
from pathlib import Path

import torch

OTHER_BASE = ("pissa", "olora", "corda", "loftq", "lora_ga")     # ways to begin an adapter that take something out of the base's weights
MAX_PARTS_RANK = 512     # parts times rank that a projection's adapters may have


class AdapterError(ValueError):
    pass


@dataclass
class ProjectionAdapters:
    """The adapters beside one projection, whose outputs are the parts ``widths`` one after the other."""
    slots: "AdapterSlots"
    a: torch.Tensor          # [slots, parts, rank, in]
    b: torch.Tensor          # [slots, out, rank]
    widths: tuple
    ranks: torch.Tensor      # [slots]: the adapters' ranks here; 0 where an adapter names no part of this projection, so that its tokens' rows are not touched

    def add_(self, y: torch.Tensor, x: torch.Tensor, plan) -> torch.Tensor:
        return self.slots.kernels.adapters_add_(y, x, self.a, self.b, self.slots.scale, plan, widths=self.widths, ranks=self.ranks)


class AdapterSlots:
    """Room for ``slots`` adapters of up to ``rank`` beside the projections of a model."""

    def __init__(self, slots: int, rank: int, dtype: torch.dtype, device, kernels):
        if slots <= 0 or rank <= 0:
            raise ValueError(f"adapters: {slots} slots and rank {rank} must be positive")
        self.count, self.rank = slots, -(-rank // 8) * 8     # rows of whole 16-byte pieces
        self.dtype, self.device, self.kernels = dtype, device, kernels
        self.scale = torch.zeros(slots, dtype=torch.float32, device=device)
        self.ranks = torch.zeros(slots, dtype=torch.int32, device=device)
        self.names: dict = {}        # adapter -> slot
        self.executors = weakref.WeakSet()     # whose requests use them (``StepExecutor.adapter_of``): several may run one model
        self.beside: list = []       # the projections that were given room since ``keep_only``

    def projection(self, out_features: int, in_features: int, widths: tuple | None = None) -> ProjectionAdapters:
        widths = (out_features,) if widths is None else tuple(widths)
        if sum(widths) != out_features:
            raise ValueError(f"adapters: parts {widths} are not the {out_features} outputs of the projection")
        if len(widths) * self.rank > MAX_PARTS_RANK:
            raise ValueError(f"adapters: rank {self.rank} beside a projection of {len(widths)} parts is beyond {MAX_PARTS_RANK // len(widths)}")
        zeros = lambda *shape, dtype=self.dtype: torch.zeros(shape, dtype=dtype, device=self.device)   # noqa: E731
        return ProjectionAdapters(self, zeros(self.count, len(widths), self.rank, in_features), zeros(self.count, out_features, self.rank), widths,
                                  zeros(self.count, dtype=torch.int32))

    def keep_only(self, pools: list) -> None:
        """Takes the room back from the projections whose ``ProjectionAdapters`` are not among ``pools``: no adapter can be loaded there."""
        kept = {id(p) for p in pools}
        for part in self.beside:
            if id(part.adapters) not in kept:
                part.adapters = None
        self.beside = []

    def in_use(self, name) -> bool:
        return name in self.names and any(self.names[name] in ex.adapter_of.values() for ex in self.executors)

    def free_slot(self) -> int:
        for s in range(self.count):
            if s not in self.names.values():
                return s
        raise AdapterError(f"all {self.count} adapter slots are taken ({', '.join(sorted(map(str, self.names)))})")


def read_adapter(folder) -> tuple[dict, float]:
    """(module -> (A, B), scale) of an adapter's folder."""
    from ..weights.safetensors_io import SafetensorsFile
    folder = Path(folder)
    try:
        config = json.loads((folder / "adapter_config.json").read_text())
        rank, alpha = int(config["r"]), float(config.get("lora_alpha", config["r"]))
    except (OSError, ValueError, KeyError, TypeError) as e:
        raise AdapterError(f"{folder}: adapter_config.json cannot be read ({e})") from None
    if str(config.get("peft_type", "LORA")).upper() != "LORA":
        raise AdapterError(f"{folder}: adapters of type {config['peft_type']!r} are not served")
    for key in ("use_dora", "modules_to_save", "rank_pattern", "alpha_pattern", "layer_replication", "alora_invocation_tokens", "use_qalora"):
        if config.get(key):
            raise AdapterError(f"{folder}: adapter_config.json asks for {key}, which is not served")
    if str(config.get("init_lora_weights", "")).lower().startswith(OTHER_BASE):
        raise AdapterError(f"{folder}: an adapter of init_lora_weights {config['init_lora_weights']!r} stands beside a base whose weights were changed with it; "
                           "save it converted to the stored base")
    if not math.isfinite(alpha):
        raise AdapterError(f"{folder}: lora_alpha {alpha} is not finite")
    if config.get("bias", "none") != "none":
        raise AdapterError(f"{folder}: adapters with biases are not served")
    if rank <= 0:
        raise AdapterError(f"{folder}: rank {rank} must be positive")
    file = SafetensorsFile(folder / "adapter_model.safetensors")
    halves: dict = {}
    for name in file.entries:
        stem, _, which = name.removesuffix(".weight").rpartition(".")
        if which not in ("lora_A", "lora_B"):
            raise AdapterError(f"{folder}: tensor '{name}' is no adapter's")
        halves.setdefault(stem.removeprefix("base_model.model."), {})[which] = file.tensor(name)
    for module, pair in halves.items():
        if len(pair) != 2:
            raise AdapterError(f"{folder}: '{module}' has one half of an adapter only")
        if pair["lora_A"].dim() != 2 or pair["lora_B"].dim() != 2 or pair["lora_A"].shape[0] != rank or pair["lora_B"].shape[1] != rank:
            raise AdapterError(f"{folder}: the adapter of '{module}' is {tuple(pair['lora_A'].shape)} and {tuple(pair['lora_B'].shape)}; expected rank {rank}")
    return {m: (p["lora_A"], p["lora_B"]) for m, p in halves.items()}, alpha / (math.sqrt(rank) if config.get("use_rslora") else rank)


def place_adapter(slots: AdapterSlots, projections: dict, name, modules: dict, scale: float) -> int:
    """Loads an adapter into a slot of its own (or the one it has) and returns the slot. ``projections``: module name -> (``ProjectionAdapters``, part).
    Everything is checked before anything is written."""
    ranks = {a.shape[0] for a, _ in modules.values()}
    if not modules or len(ranks) != 1:
        raise AdapterError(f"adapter {name!r}: its modules have ranks {sorted(ranks)}; expected one")
    rank = ranks.pop()
    if rank > slots.rank:
        raise AdapterError(f"adapter {name!r}: rank {rank} is beyond the {slots.rank} that the model has room for")
    unknown = sorted(set(modules) - set(projections))
    if unknown:
        raise AdapterError(f"adapter {name!r}: no projection takes an adapter for {', '.join(unknown[:4])}" + (" and others" if len(unknown) > 4 else ""))
    for module, (a, b) in modules.items():
        pool, part = projections[module]
        want = ((rank, pool.a.shape[3]), (pool.widths[part], rank))
        if (tuple(a.shape), tuple(b.shape)) != want:
            raise AdapterError(f"adapter {name!r}: '{module}' is {tuple(a.shape)} and {tuple(b.shape)}; expected {want[0]} and {want[1]}")
    slot = slots.names[name] if name in slots.names else slots.free_slot()
    for module, (pool, part) in projections.items():     # a projection the adapter does not name adds nothing
        lo = sum(pool.widths[:part])
        rows = slice(lo, lo + pool.widths[part])
        if module in modules:
            a, b = modules[module]
            pool.a[slot, part, :rank].copy_(a.to(device=slots.device, dtype=slots.dtype))
            pool.b[slot, rows, :rank].copy_(b.to(device=slots.device, dtype=slots.dtype))
        else:
            pool.a[slot, part].zero_()
            pool.b[slot, rows].zero_()
    named = {id(projections[module][0]) for module in modules}
    for pool, _ in projections.values():
        pool.ranks[slot] = rank if id(pool) in named else 0
    slots.scale[slot] = scale
    slots.ranks[slot] = rank
    slots.names[name] = slot
    return slot
