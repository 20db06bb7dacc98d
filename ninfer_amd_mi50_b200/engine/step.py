"""The step function: run a batch of (request, its next tokens) from the cache.

Reference: ``Model::forward_batch(tokens, positions, seq_ids)`` (src/models/model.h:74-77,
src/models/model.hip:994-1032) returns the logits of each group's last row and leaves
length bookkeeping to its callers (src/api/ninfer_c_api.cpp:190, 210, 239).  This step
takes whole entries, keeps the lengths in the cache manager, accepts portions of prompts
beside single decoded tokens cut anywhere, and returns logits at exactly the rows asked
for.  It runs only the tokens it is given; everything earlier comes from the cache.
"""

from __future__ import annotations

from typing import Dict, Hashable, List, Optional, Sequence, Tuple

import torch

from ..cache.manager import CacheManager
from ..cache.page_pool import OutOfPages
from ..parts.model import DecoderModel
from .batch import BatchError, StepEntry, TreeEntry, pack_step, tree_parents, tree_rows, validate_entries


class ModelRunner:
    def __init__(self, model: DecoderModel, cache: CacheManager, dtype: torch.dtype, device,
                 use_graph: bool = False):
        self.model, self.cache, self.dtype = model, cache, dtype
        self.device = torch.device(device)
        self.graphs = None
        self.adapters = None          # the bank of adapters, where the engine keeps one
        self.trees: Dict[Hashable, Tuple[int, List[int]]] = {}        # requests whose last step was a tree: tokens held before it, parents
        if use_graph and self.device.type == "cuda" and model.graph_safe:
            from .graphs import DecodeGraphs
            self.graphs = DecodeGraphs(self, cache.max_requests)
        self.steps_run = 0
        self.h2d_bytes = 0
        self.tokens_run = 0

    # ---- requests -------------------------------------------------------------------
    def open(self, req: Hashable) -> int:
        return self.cache.open(req)

    def close(self, req: Hashable) -> None:
        self.trees.pop(req, None)
        self.cache.close(req)

    def fork(self, req: Hashable, new: Hashable) -> int:
        """Admit `new` as a request that goes on from where `req` is (`CacheManager.fork`)."""
        return self.cache.fork(req, new)

    # ---- the step -------------------------------------------------------------------
    def reserve(self, entries: Sequence[StepEntry]) -> None:
        """Hold pages for every entry's new tokens, or no more of them than before: what a tree holds that may still be
        accepted stays."""
        done: List[Tuple[Hashable, int]] = []
        try:
            for e in entries:
                held = self.cache.reserved(e.req)
                self.cache.reserve(e.req, self.cache.length(e.req) + len(e.tokens))
                done.append((e.req, held))
        except OutOfPages:
            for req, held in done:
                self.cache.truncate(req, held)
            raise

    def _leave_trees(self, entries: Sequence[StepEntry]) -> None:
        """Forget trees that were not accepted and that the step is about to write over, with the pages that only they hold."""
        for e in entries:
            if self.trees.pop(e.req, None) is not None:
                self.cache.truncate(e.req, self.cache.length(e.req) + len(e.tokens))

    def step(self, entries: Sequence[StepEntry], device_tokens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """float32 logits [R, vocab] on the device, R = total wanted rows, in entry order.

        `device_tokens`: for a decode-only step replayed from a graph, the entries' token ids
        as an int32 tensor on the device, to be used instead of the (placeholder) ids in the
        entries; `can_take_device_tokens` says whether a step qualifies."""
        entries = list(entries)
        if not entries:
            return torch.empty((0, self.model.vocab_size), dtype=torch.float32, device=self.device)
        arrays = validate_entries(entries, self.cache, self.model.vocab_size)
        adapted = self._check_adapters(entries)
        self.reserve(entries)
        self._leave_trees(entries)
        try:
            if self.graphs is not None and self.graphs.eligible(entries):
                logits, moved = self._step_from_graph(entries, device_tokens)
            elif device_tokens is not None:
                raise ValueError("token ids on the device can only feed a step that is replayed from a graph")
            else:
                ctx = pack_step(entries, self.cache, self.dtype, self.device, arrays=arrays, adapted=adapted)
                logits, moved = self.run(ctx), ctx.scratch.get("h2d_bytes", 0)
        except Exception:
            for e in entries:
                self.cache.truncate(e.req)
            raise
        for e in entries:
            self.cache.commit(e.req, self.cache.length(e.req) + len(e.tokens))
        self.steps_run += 1
        self.h2d_bytes += moved
        self.tokens_run += sum(len(e.tokens) for e in entries)
        return logits

    def _check_adapters(self, entries: Sequence[StepEntry]) -> bool:
        """Whether some entry has an adapter; raises for one that is not there."""
        adapted = False
        for e in entries:
            if e.adapter != -1:
                if self.adapters is None or e.adapter not in self.adapters.slots.values():
                    raise BatchError(f"request {e.req!r}: no adapter in slot {e.adapter}")
                adapted = True
        return adapted

    # ---- trees of drafted tokens ------------------------------------------------------
    def tree_step(self, entries: Sequence[TreeEntry]) -> torch.Tensor:
        """Run every entry's tree -> float32 logits [nodes, vocab], row by row behind each node.

        Nothing is committed: `accept` says which path of the tree stands, and until then another step of the request
        starts where this one did.  For models whose mixers see all earlier tokens (`DecoderModel.tree_safe`)."""
        from .. import kernels
        entries = list(entries)
        if not self.model.tree_safe:
            raise BatchError("this model has layers that cannot run a tree of drafted tokens (states, windows or neighbouring tokens)")
        if not entries:
            return torch.empty((0, self.model.vocab_size), dtype=torch.float32, device=self.device)
        steps = [StepEntry(e.req, e.tokens, range(len(e.tokens)), e.adapter) for e in entries]
        arrays = validate_entries(steps, self.cache, self.model.vocab_size)
        parents = [tree_parents(e, kernels.MAX_TREE_NODES) for e in entries]
        adapted = self._check_adapters(steps)
        self.reserve(steps)
        self._leave_trees(steps)
        lengths = [self.cache.length(e.req) for e in entries]
        try:
            ctx = pack_step(steps, self.cache, self.dtype, self.device, arrays=arrays, adapted=adapted)
            ctx.tree = tree_rows(lengths, parents, self.device)
            logits = self.run(ctx)
        except Exception:
            for e in entries:
                self.cache.truncate(e.req)
            raise
        for e, held, p in zip(entries, lengths, parents):
            self.trees[e.req] = (held, p)
        self.steps_run += 1
        self.h2d_bytes += ctx.scratch.get("h2d_bytes", 0) + 4 * (ctx.tree.positions.numel() + ctx.tree.mask.numel())
        self.tokens_run += sum(len(e.tokens) for e in entries)
        return logits

    def accept(self, paths: Dict[Hashable, Sequence[int]]) -> None:
        """Commit, for each request, the root of its last tree and the nodes of `paths[req]` behind it, from the root's child
        down (none: the root alone).  Their cache entries move up to where they would be had they been run in a line."""
        from .. import kernels
        for req, path in paths.items():
            if req not in self.trees or self.trees[req][0] != self.cache.length(req):
                raise BatchError(f"request {req!r}: its last step was not a tree")
            parents, at = self.trees[req][1], 0
            for node in path:
                if not 0 < int(node) < len(parents) or parents[int(node)] != at:
                    raise BatchError(f"request {req!r}: {list(path)} is not a path down its tree")
                at = int(node)
        moving = [req for req, path in paths.items() if any(int(p) != j + 1 for j, p in enumerate(path))]
        if moving:
            most = max(len(paths[r]) for r in moving)
            rows = [[self.cache.length(r), len(paths[r])] + [int(p) for p in paths[r]] + [-1] * (most - len(paths[r])) for r in moving]
            small = torch.tensor(rows, dtype=torch.int32)
            lengths, accepted, path = (t.contiguous().to(self.device) for t in (small[:, 0], small[:, 1], small[:, 2:]))
            for g in self.cache.groups:
                width = max(len(self.cache.block_table(g.index, r)) for r in moving)
                table = torch.from_numpy(self.cache.block_rows(g.index, [self.cache.slot(r) for r in moving], width)).to(self.device)
                kernels.compact_cache(g.pages, table, lengths, path, accepted)
        for req, path in paths.items():
            del self.trees[req]
            self.cache.commit(req, self.cache.length(req) + 1 + len(path))
            self.cache.truncate(req)           # (pages that only nodes left behind had use for)

    def can_take_device_tokens(self, n_entries: int) -> bool:
        """Whether a step of `n_entries` single tokens would be replayed from a graph."""
        return self.graphs is not None and 0 < n_entries <= self.graphs.max_rows

    def _step_from_graph(self, entries: Sequence[StepEntry], device_tokens: Optional[torch.Tensor] = None):
        """A decode-only step: replay the captured graph for this many rows."""
        g = self.graphs.get(entries)
        logits = g.run(entries, device_tokens)
        n = len(entries)
        if all(len(e.want) == 1 for e in entries):
            return logits[:n], g.h2d_bytes
        rows = [i for i, e in enumerate(entries) for _ in e.want]
        if not rows:
            return logits[:0], g.h2d_bytes
        return logits.index_select(0, torch.tensor(rows, device=self.device)), g.h2d_bytes

    def run(self, ctx) -> torch.Tensor:
        cache = self.cache
        return self.model.forward(
            ctx,
            lambda slot, append: cache.view(slot, ctx.block_tables, append),
            cache.state_of)
