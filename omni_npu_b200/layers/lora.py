"""Low-rank adapters in the engine: named adapters in slots, applied beside the shared projections.

``AdapterManager`` gives every projection of a dense decoder a stack of slots (``ops.LoraStack``) and wraps its linear
method; a step whose requests use adapters carries a plan (``ops.lora_plan``) in its attention metadata, and a step without one
runs the projections as they are.  Adapters come in the PEFT layout: a directory with ``adapter_config.json`` and
``adapter_model.safetensors``.
"""
from __future__ import annotations

import itertools
import json
import math
import os
import re
from dataclasses import dataclass
from typing import Dict, Iterable, List, Optional, Tuple

import torch

from .. import ops
from ..attention.metadata import get_forward_context
from .linear import LinearBase, MergedColumnParallelLinear, QKVParallelLinear, RowParallelLinear


class LoraLinearMethod:
    """The projection's own method, followed by the adapters of the step's tokens."""

    def __init__(self, inner, stack: ops.LoraStack) -> None:
        self.inner, self.stack = inner, stack

    def process_weights_after_loading(self, layer) -> None:
        self.inner.process_weights_after_loading(layer)

    def apply(self, layer, x, bias, residual=None, swiglu: bool = False, out_dtype=None) -> torch.Tensor:
        md = get_forward_context().attn_metadata
        plan = md.extra.get("lora") if md is not None else None
        if plan is None:
            return self.inner.apply(layer, x, bias, residual=residual, swiglu=swiglu, out_dtype=out_dtype)
        y = self.inner.apply(layer, x, bias, residual=residual, out_dtype=out_dtype)
        if swiglu:
            return ops.lora_gated(y, x, self.stack, plan, act=layer.gated_act)
        return ops.lora_add(y, x, self.stack, plan, out=y)


_TENSOR = re.compile(r"^(?:base_model\.model\.)?(?P<module>.+)\.lora_(?P<which>[AB])(?:\.default)?\.weight$")


@dataclass
class Adapter:
    """A checked adapter whose factors are on the device, in no slot yet."""
    name: str
    scale: float
    factors: Dict[str, List[List[Optional[torch.Tensor]]]]       # of a projection: A of each slice, B of each slice


class AdapterManager:
    def __init__(self, model: torch.nn.Module, num_slots: int, max_rank: int, dtype: torch.dtype, device: torch.device) -> None:
        mapping = getattr(model, "stacked_params_mapping", None)
        if not getattr(model, "supports_adapters", False) or mapping is None:
            raise ValueError(f"{type(model).__name__} does not take low-rank adapters")
        if device.type == "cuda" and dtype != torch.bfloat16:
            raise ValueError("low-rank adapters on a GPU need a bf16 model")
        self.num_slots, self.max_rank = num_slots, max_rank
        self.slots: Dict[str, int] = {}
        self.keys: Dict[str, bytes] = {}             # told apart in the prefix cache, also from an earlier load of the name
        self._loads = itertools.count()
        self._lost = False                           # the stacks hold nothing that may be read
        self.layers: Dict[str, LinearBase] = {}
        self.stacks: Dict[str, ops.LoraStack] = {}
        # checkpoint module name -> (projection, its slice)
        self.parts: Dict[str, Tuple[str, int]] = {}
        stacked: Dict[str, List[Tuple[str, object]]] = {}
        for fused, part, shard in mapping:
            stacked.setdefault(fused, []).append((part, shard))
        for layer in model.modules():
            # (projections outside the decoder layers, such as those of a draft head, stay as they are)
            if not isinstance(layer, (QKVParallelLinear, MergedColumnParallelLinear, RowParallelLinear)) \
                    or not layer.prefix.startswith("model.layers."):
                continue
            name, interleaved = layer.prefix, False
            if isinstance(layer, QKVParallelLinear):
                k, slices = layer.in_features, [layer.q_size, layer.k_size, layer.v_size]
            elif isinstance(layer, MergedColumnParallelLinear):
                k, slices, interleaved = layer.in_features, layer.local_sizes, layer.swiglu_interleave
            else:
                k, slices = layer.in_local, [layer.out_features]
            self.layers[name] = layer
            self.stacks[name] = ops.LoraStack(num_slots, max_rank, k, slices, device=device, dtype=dtype,
                                              interleaved=interleaved)
            layer.quant_method = LoraLinearMethod(layer.quant_method, self.stacks[name])
            suffix = "." + name.rsplit(".", 1)[1]
            for part, shard in stacked.get(suffix, [(suffix, 0)]):
                self.parts[name[: -len(suffix)] + part] = (name, {"q": 0, "k": 1, "v": 2}.get(shard, shard))

    # ------------------------------------------------------------------ adapters
    def load(self, name: str, path: str) -> int:
        """Load a PEFT directory under ``name``; returns its slot."""
        return self.install(self.read(name, path))

    def load_tensors(self, name: str, config: dict, tensors: Iterable[Tuple[str, torch.Tensor]]) -> int:
        """Load an adapter from its configuration and (name, tensor) pairs."""
        return self.install(self.prepare(name, config, tensors))

    def read(self, name: str, path: str) -> Adapter:
        """The adapter of a PEFT directory.  Like ``prepare`` it changes nothing here, so steps may run meanwhile."""
        self._check_free(name)
        with open(os.path.join(path, "adapter_config.json")) as f:
            config = json.load(f)
        from safetensors import SafetensorError
        from ..models.utils import iter_safetensors
        try:
            return self.prepare(name, config, iter_safetensors(path))
        except SafetensorError as e:
            raise ValueError(f"adapter {name!r}: damaged file: {e}")

    def prepare(self, name: str, config: dict, tensors: Iterable[Tuple[str, torch.Tensor]]) -> Adapter:
        """Check an adapter and bring its factors to the device."""
        self._check_free(name)
        if not isinstance(config, dict):
            raise ValueError(f"adapter {name!r}: its configuration is not an object")
        for key, off in (("use_dora", False), ("bias", "none"), ("fan_in_fan_out", False), ("modules_to_save", None),
                         ("rank_pattern", {}), ("alpha_pattern", {}), ("peft_type", "LORA")):
            if config.get(key) and config[key] != off:
                raise ValueError(f"adapter {name!r}: {key} = {config[key]!r} is not supported")
        try:
            rank = int(config["r"])
            alpha = float(config.get("lora_alpha", rank))
        except (KeyError, TypeError, ValueError):
            raise ValueError(f"adapter {name!r}: r = {config.get('r')!r} and lora_alpha = {config.get('lora_alpha')!r} are not numbers")
        if not math.isfinite(alpha):
            raise ValueError(f"adapter {name!r}: lora_alpha = {alpha}")
        if not 1 <= rank <= self.max_rank:
            raise ValueError(f"adapter {name!r} has rank {rank}, the engine takes 1 to {self.max_rank}")
        scale = alpha / rank ** 0.5 if config.get("use_rslora") else alpha / rank
        found: Dict[str, List[List[Optional[torch.Tensor]]]] = {}
        for key, tensor in tensors:
            m = _TENSOR.match(key)
            part = self.parts.get(m["module"]) if m else None
            if part is None:
                raise ValueError(f"adapter {name!r}: {key} belongs to no projection that takes adapters")
            if tensor.dim() != 2 or tensor.shape["AB".index(m["which"])] != rank:
                # (the scale is the configuration's)
                raise ValueError(f"adapter {name!r}: {key} is {tuple(tensor.shape)}, its rank should be {rank}")
            proj, i = part
            stack = self.stacks[proj]
            n = len(stack.slices)
            found.setdefault(proj, [[None] * n, [None] * n])["AB".index(m["which"])][i] = tensor.to(stack.device, stack.dtype)
        if not found:
            raise ValueError(f"adapter {name!r} has no factors")
        return Adapter(name, scale, found)

    def install(self, adapter: Adapter) -> int:
        """Put an adapter into a free slot; returns it."""
        name = adapter.name
        self._check_free(name)
        if self._lost:
            for stack in self.stacks.values():
                stack.reset()
            self._lost = False
        slot = next(i for i in range(self.num_slots) if i not in self.slots.values())
        try:
            for proj, (a, b) in adapter.factors.items():
                self.stacks[proj].load(slot, a, b, adapter.scale)
        except Exception as e:
            self._clear(slot)
            raise ValueError(f"adapter {name!r}: {e}") if isinstance(e, ValueError) else e
        self.slots[name] = slot
        self.keys[name] = f"adapter {next(self._loads)} {name}".encode()
        return slot

    def _check_free(self, name: str) -> None:
        if not name or name in self.slots:
            raise ValueError(f"adapter {name!r} is already loaded" if name else "an adapter needs a name")
        if len(self.slots) == self.num_slots:
            raise ValueError(f"all {self.num_slots} adapter slots are taken")

    def unload(self, name: str) -> None:
        self._clear(self.slot(name))
        del self.slots[name], self.keys[name]

    def forget(self) -> None:
        """The stacks' memory is about to lose its contents: no adapter is loaded any more.  (No token names a slot before the
        next load, which empties them on the device first.)"""
        self.slots.clear()
        self.keys.clear()
        self._lost = True

    def slot(self, name: str) -> int:
        if name not in self.slots:
            raise ValueError(f"no adapter {name!r} is loaded (loaded: {sorted(self.slots)})")
        return self.slots[name]

    def _clear(self, slot: int) -> None:
        for stack in self.stacks.values():
            stack.clear(slot)

    # --------------------------------------------------------------------- steps
    def plan(self, slots: torch.Tensor) -> ops.LoraPlan:
        return ops.lora_plan(slots, self.num_slots)
