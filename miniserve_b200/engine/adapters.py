"""The low-rank adapters that an engine holds beside its model's projections, a slot each (``AdapterStore``).

An adapter comes as a folder with ``adapter_config.json`` (``r``, ``lora_alpha``) and safetensors, or as its tensors: for each adapted matrix ``<matrix>.lora_A.weight``
[r, inputs] and ``<matrix>.lora_B.weight`` [outputs, r], ``<matrix>.weight`` (or ``<matrix>``) being the model's tensor, with or without ``base_model.model.`` in front. It adds
alpha / r B A x to the matrix's product. Which matrices may have one is the parts' to say (``Part.adapted_products``); others are refused, all that is wrong in one error.
"""

from __future__ import annotations

import json
import math
from pathlib import Path
from typing import Mapping

import torch

from .. import ops

_PREFIX = "base_model.model."
_ENDS = {".lora_A.weight": 0, ".lora_B.weight": 1}


def _config(folder: Path) -> dict:
    """What ``adapter_config.json`` says, ``r`` a number."""
    try:
        cfg = json.loads((folder / "adapter_config.json").read_text())
    except FileNotFoundError:
        raise FileNotFoundError(f"no adapter_config.json in {folder}") from None
    try:
        cfg["r"] = int(cfg["r"])
    except (KeyError, TypeError, ValueError):
        raise ValueError(f"adapter_config.json in {folder} says no rank (r)") from None
    if cfg["r"] < 1:
        raise ValueError(f"adapter_config.json in {folder} says a rank of {cfg['r']}")
    return cfg


def rank_of(source: "str | Path | Mapping[str, torch.Tensor]") -> int:
    """The rank of an adapter, in a folder or as tensors by name."""
    if isinstance(source, (str, Path)):
        return _config(Path(source))["r"]
    return max((t.shape[0] for key, t in source.items() if key.endswith(".lora_A.weight") and t.dim()), default=1)


class AdapterStore:
    def __init__(self, model, slots: int, rank: int):
        """Room for ``slots`` adapters of a rank up to ``rank`` (made up to a multiple of 8) beside every projection of ``model`` that takes them."""
        if slots < 1 or not 1 <= rank <= ops.adapters.MAX_RANK:
            raise ValueError(f"max_adapters={slots} and max_adapter_rank={rank}: at least one adapter, a rank of 1 to {ops.adapters.MAX_RANK}")
        self.slots, self.rank = slots, rank
        self.names: dict[str, int] = {}
        # matrix -> (the LowRank of its product, its part there, the part's first row and the row behind)
        self.places: dict[str, tuple] = {}
        held = -(-rank // 8) * 8
        self.products: dict[tuple, ops.LowRank] = {}  # (part, product) -> its adapters

        def walk(part, prefix):
            decls = part.weights()
            for product, matrices in part.adapted_products().items():
                ends, at = [], 0
                for m in matrices:
                    at += decls[m].shape[0]
                    ends.append(at)
                inputs = decls[matrices[0]].shape[1]
                if inputs % 8:
                    continue  # (no kernel takes it; an adapter that names it is refused)
                low = self.products[part, product] = ops.LowRank.zeros(slots, inputs, tuple(ends), held, model.dtype, model.device)
                for p, m in enumerate(matrices):
                    self.places[prefix + m] = (low, p, ends[p - 1] if p else 0, ends[p])
            for sub, child in part.sub_parts().items():
                walk(child, prefix + sub)

        for prefix, layer in zip(model.prefixes, model.layers):
            walk(layer, prefix)
        if not self.places:
            raise ValueError(f"no projection of a {model.spec.architecture} model takes adapters")

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for low in self.products.values() for t in (low.a, low.b, low.scale))

    # ------------------------------------------------------------------ loading
    def load(self, name: str, source: "str | Path | Mapping[str, torch.Tensor]", alpha: float | None = None) -> int:
        """Put an adapter into a free slot; returns the slot. ``source``: a folder, or the tensors by name (then ``alpha`` says lora_alpha; left out, the rank:
        a factor of 1). Nothing is changed where anything is wrong with it."""
        if name in self.names:
            raise ValueError(f"there is an adapter {name!r} already")
        free = [s for s in range(self.slots) if s not in self.names.values()]
        if not free:
            raise ValueError(f"all {self.slots} adapters' places are taken ({', '.join(sorted(self.names))}): unload one, or ask for more (max_adapters)")
        factor = said = None
        if isinstance(source, (str, Path)):
            tensors, factor, said = self._read(Path(source))
            if alpha is not None:
                raise ValueError("alpha is what the adapter's folder says")
        else:
            tensors = dict(source)
        if factor is None and alpha is not None and not math.isfinite(alpha):
            raise ValueError(f"adapter {name!r} has a factor that is not finite")
        pairs = self._pairs(name, tensors, said)
        if factor is None:
            factor = 1.0 if alpha is None else float(alpha) / next(iter(pairs.values()))[0].shape[0]
        if not abs(factor) <= torch.finfo(torch.float32).max:
            raise ValueError(f"adapter {name!r} has a factor that is not finite in 32 bits: {factor}")
        slot = free[0]
        self._settle()  # (a step in flight may still read what the place held)
        for low in self.products.values():  # (beside all matrices: an earlier adapter's numbers, times a factor of 0, need not be 0)
            low.scale[slot] = 0.0
            low.a[slot].zero_()
            low.b[slot].zero_()
        for matrix, (a, b) in pairs.items():
            low, part, first, behind = self.places[matrix]
            r = a.shape[0]
            low.a[slot, part * low.rank:part * low.rank + r] = a.to(low.a.dtype)
            low.b[slot, first:behind, :r] = b.to(low.b.dtype)
            low.scale[slot] = factor
        self._settle()  # (steps may run on another stream)
        self.names[name] = slot
        return slot

    def _settle(self) -> None:
        device = next(iter(self.products.values())).a.device
        if device.type == "cuda":
            torch.cuda.synchronize(device)

    def unload(self, name: str) -> None:
        """Free the adapter's slot (no request that still runs may have it: the engine sees to that)."""
        self.slot(name)
        del self.names[name]

    def slot(self, name: str) -> int:
        try:
            return self.names[name]
        except KeyError:
            raise ValueError(f"no adapter named {name!r}; there are {sorted(self.names)}") from None

    def _read(self, folder: Path) -> tuple[dict, float, int]:
        """The tensors, the factor and the rank that the folder's configuration says."""
        from safetensors.torch import load_file

        cfg = _config(folder)
        odd = [k for k in ("use_dora", "rank_pattern", "alpha_pattern", "modules_to_save", "layer_replication", "fan_in_fan_out", "alora_invocation_tokens") if cfg.get(k)]
        if cfg.get("bias", "none") not in ("none", None):
            odd.append(f"bias={cfg['bias']}")
        if str(cfg.get("peft_type") or "LORA").upper() != "LORA":
            odd.append(f"peft_type={cfg['peft_type']}")
        if odd:
            raise ValueError(f"the adapter in {folder} has what there is nothing for here: {', '.join(odd)}")
        r = cfg["r"]
        files = sorted(folder.glob("*.safetensors"))
        if not files:
            raise FileNotFoundError(f"no .safetensors files in {folder}")
        tensors: dict = {}
        for f in files:
            more = load_file(str(f))
            twice = sorted(tensors.keys() & more.keys())
            if twice:
                raise ValueError(f"{f} holds tensors that another file of {folder} holds too: {', '.join(twice[:4])}")
            tensors.update(more)
        alpha = float(cfg.get("lora_alpha", r))
        return tensors, alpha / (math.sqrt(r) if cfg.get("use_rslora") else r), r

    def _pairs(self, name: str, tensors: Mapping[str, torch.Tensor], said: int | None = None) -> dict[str, tuple]:
        """(A, B) by the model's matrix, or one error about all that does not fit (``said``: the rank that they should have)."""
        halves: dict[str, list] = {}
        wrong: list[str] = []
        for key, t in tensors.items():
            at = key[len(_PREFIX):] if key.startswith(_PREFIX) else key
            end = next((e for e in _ENDS if at.endswith(e)), None)
            stem = at[:-len(end)] if end else None
            matrix = stem if stem in self.places else f"{stem}.weight"
            if matrix not in self.places:
                wrong.append(f"{key}: no projection here that takes an adapter")
                continue
            half = halves.setdefault(matrix, [None, None])
            if half[_ENDS[end]] is not None:
                wrong.append(f"{at}: given twice, with {_PREFIX} in front and without")
            half[_ENDS[end]] = t
        ranks = set()
        for matrix, (a, b) in halves.items():
            low, _, first, behind = self.places[matrix]
            if a is None or b is None:
                wrong.append(f"{matrix}: lora_{'A' if a is None else 'B'} is missing")
            elif a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or a.shape[1] != low.inputs or b.shape[0] != behind - first:
                wrong.append(f"{matrix}: A {tuple(a.shape)} and B {tuple(b.shape)} beside a matrix of {behind - first} x {low.inputs}")
            else:
                ranks.add(a.shape[0])
                if not all(bool(torch.isfinite(t.to(low.a.dtype)).all()) for t in (a, b)):
                    wrong.append(f"{matrix}: numbers that are not finite (other requests' tokens would meet them)")
                if not 1 <= a.shape[0] <= self.rank:
                    wrong.append(f"{matrix}: rank {a.shape[0]}, there is room for 1 to {self.rank} (max_adapter_rank)")
        if said is not None and ranks and ranks != {said}:
            wrong.append(f"tensors of rank {', '.join(map(str, sorted(ranks)))} beside a configuration that says {said} (the factor follows from it)")
        if len(ranks) > 1:
            wrong.append(f"ranks {sorted(ranks)}: all of an adapter's are one")
        if not halves and not wrong:
            wrong.append("it has no tensors")
        if wrong:
            more = f" ... and {len(wrong) - 12} more" if len(wrong) > 12 else ""
            raise ValueError(f"adapter {name!r} does not fit: {'; '.join(wrong[:12])}{more}")
        return {m: (a, b) for m, (a, b) in halves.items()}
