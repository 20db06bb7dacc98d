"""Low-rank adapters that requests bring to the model's projections.

A part names the projections that can have one (`Part.projections`).  For each the engine keeps a pool of `capacity` slots,
the same slot number in every projection being one adapter; a step's rows name their slot (`StepContext.row_adapter`), so
that one batch, and one captured graph, serves requests of any adapters.  An adapter adds ``scale (x A^T) B^T`` to
``x W^T``.  An engine without adapters keeps no pools, and a step none of whose rows has one takes the path without them.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Mapping, Optional, Tuple

import torch

from .. import kernels


class AdapterError(ValueError):
    pass


@dataclass(frozen=True)
class Projection:
    """A weight matrix of a part: the checkpoint tensors that it stacks, their widths, and its input's width."""
    names: Tuple[str, ...]
    widths: Tuple[int, ...]
    in_features: int


class ProjectionAdapters:
    """The pool of one projection: a [capacity, stacked tensors * rank, in], b [capacity, all widths, rank]; what lies beyond
    an adapter's own rank, and a tensor that it leaves alone, holds zeros."""

    def __init__(self, projection: Projection, capacity: int, rank: int, dtype: torch.dtype, device, scale: torch.Tensor):
        self.projection, self.rank, self.scale = projection, rank, scale
        n = len(projection.names)
        self.a = torch.zeros((capacity, n * rank, projection.in_features), dtype=dtype, device=device)
        self.b = torch.zeros((capacity, sum(projection.widths), rank), dtype=dtype, device=device)

    def linear(self, x: torch.Tensor, w: torch.Tensor, rows: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        kw = {} if out_dtype in (None, x.dtype) else {"out_dtype": out_dtype}
        return kernels.adapter_linear(x, w, self.a, self.b, self.scale, rows, self.projection.widths, **kw)

    def clear(self, slot: int) -> None:
        self.a[slot].zero_()
        self.b[slot].zero_()

    def put(self, slot: int, name: str, a: torch.Tensor, b: torch.Tensor) -> None:
        i = self.projection.names.index(name)
        first, width, r = sum(self.projection.widths[:i]), self.projection.widths[i], a.shape[0]
        self.a[slot, i * self.rank:i * self.rank + r].copy_(a)
        self.b[slot, first:first + width, :r].copy_(b)

    def nbytes(self) -> int:
        return (self.a.numel() + self.b.numel()) * self.a.element_size()


class AdapterBank:
    """All pools of a model, and which adapter holds which slot."""

    def __init__(self, model, capacity: int, rank: int, dtype: torch.dtype, device):
        self.capacity, self.rank = int(capacity), kernels.adapter_rank(rank)
        self.scale = torch.zeros((self.capacity,), dtype=torch.float32, device=device)
        self.all: List[ProjectionAdapters] = []
        self.pools: Dict[str, List[ProjectionAdapters]] = {}       # by tensor name (layers may share a tensor)
        self.slots: Dict[str, int] = {}                      # by adapter name
        self.held = [0] * self.capacity                      # holders of each slot beside the scheduler's requests
        for part in model.parts():
            pools = {what: ProjectionAdapters(p, self.capacity, self.rank, dtype, device, self.scale)
                     for what, p in part.projections().items()}
            part.adapters = pools
            for pool in pools.values():
                self.all.append(pool)
                for name in pool.projection.names:
                    self.pools.setdefault(name, []).append(pool)
        if not self.pools:
            raise AdapterError("no part of this model has a projection that takes adapters")

    def slot(self, name: Optional[str]) -> int:
        """The slot of a loaded adapter; -1 for None."""
        if name is None:
            return -1
        if name not in self.slots:
            raise AdapterError(f"no adapter {name!r}; loaded: {sorted(self.slots)}")
        return self.slots[name]

    def hold(self, slot: int) -> None:
        """An adapter is not dropped before whoever held its slot has released it: a slot's number says nothing of whose
        weights it has by then."""
        self.held[slot] += 1

    def release(self, slot: int) -> None:
        self.held[slot] -= 1

    def nbytes(self) -> int:
        return sum(p.nbytes() for p in self.all)

    def load(self, name: str, weights: Mapping[str, Tuple[torch.Tensor, torch.Tensor]], scale: float = 1.0) -> int:
        """Take an adapter into a free slot: for each adapted tensor of the checkpoint, by its name, A [r, in] and B
        [out, r].  All of it is checked before anything is written."""
        if name in self.slots:
            raise AdapterError(f"adapter {name!r} is loaded already")
        if not weights:
            raise AdapterError(f"adapter {name!r} adapts nothing")
        if not torch.isfinite(torch.tensor(float(scale), dtype=torch.float32)):
            raise AdapterError(f"adapter {name!r}: scale {scale} is not finite")
        unknown = sorted(n for n in weights if n not in self.pools)
        if unknown:
            raise AdapterError(f"adapter {name!r} adapts tensors that take no adapters: {unknown}; those that do: {sorted(self.pools)}")
        for n, (a, b) in weights.items():
            p = self.pools[n][0].projection
            width = p.widths[p.names.index(n)]
            if a.dim() != 2 or b.dim() != 2 or a.shape[1] != p.in_features or b.shape != (width, a.shape[0]):
                raise AdapterError(f"adapter {name!r}, {n}: A {tuple(a.shape)} and B {tuple(b.shape)} do not fit [{width}, {p.in_features}]")
            if not 1 <= a.shape[0] <= self.rank:
                raise AdapterError(f"adapter {name!r}, {n}: rank {a.shape[0]}; this engine takes up to {self.rank}")
            # rows of several requests share a product, in which another request's adapter is multiplied by zero
            dtype = self.pools[n][0].a.dtype
            if not (torch.isfinite(a.to(dtype)).all() and torch.isfinite(b.to(dtype)).all()):
                raise AdapterError(f"adapter {name!r}, {n}: not all weights are finite as {dtype}")
        taken = set(self.slots.values())
        free = [s for s in range(self.capacity) if s not in taken]
        if not free:
            raise AdapterError(f"all {self.capacity} adapter slots are taken: {sorted(self.slots)}")
        slot = free[0]
        for pool in self.all:
            pool.clear(slot)
        for n, (a, b) in weights.items():
            for pool in self.pools[n]:
                pool.put(slot, n, a, b)
        self.scale[slot] = float(scale)
        self.slots[name] = slot
        return slot

    def drop(self, name: str) -> None:
        """Give a slot back (its weights stay until another adapter takes it; no row names it any more)."""
        slot = self.slot(name)
        if self.held[slot]:
            raise AdapterError(f"adapter {name!r} is in use by {self.held[slot]} open session(s)")
        del self.slots[name]
