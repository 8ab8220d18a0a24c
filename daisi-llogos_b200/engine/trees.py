"""Steps over trees of drafted tokens, and caches that keys are taken out of: what the step function does around the operators
``attn_tree``, ``tree_accept``, ``key_weights``, ``keep_keys`` and ``CacheRows.move``.

The reference verifies one chain of drafted tokens by a batched forward pass and rolls its cache back to the accepted length
(Inference/SpeculativeDecoder.cs, Inference/ForwardPass.cs:718-760); it cannot take keys out of the middle of its cache.

A tree step writes the keys and values of all nodes behind the cached ones, node i's at place ``length + i``, while a node's position (its
rotation, its window) is ``depth`` behind the last cached token's.  Accepting a path moves its rows to the front of the tree's in all
layers; lengths advance by the path, and nothing was committed before.  Tree steps of sizes that come again are recorded as CUDA graphs.
"""
from __future__ import annotations

import weakref
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..cache.slots import CacheError
from ..parts.base import Mixer
from .context import StepContext, Workspace

RECORDED_SIZES = 8       # tree sizes whose buffers and graph are kept; the ones used longest ago make room
RECORDED_BYTES = 1 << 30      # and what their buffers may take together: logits of 512 nodes over 128,256 ids alone are 263 MB


class _Pending:
    """A tree step that has not been accepted: nothing of it is committed."""

    def __init__(self, slots, counts, len_before, tokens, meta, logits):
        self.slots, self.counts, self.len_before, self.tokens, self.meta, self.logits = slots, counts, len_before, tokens, meta, logits


class _Recorded:
    """Static buffers (and later the CUDA graph) of tree steps of one batch of tree sizes."""

    def __init__(self, ints: int, device: torch.device):
        self.meta = torch.zeros(ints, dtype=torch.int32, device=device)
        self.workspace = Workspace(device)
        self.graph = None
        self.logits: Optional[torch.Tensor] = None
        self.kernels = 0


def ancestor_bits(parents: Sequence[int]) -> List[int]:
    """Per node the bits of its ancestors and itself."""
    bits: List[int] = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return bits


class TreeSteps:
    """The engine's tree steps and evictions."""

    def __init__(self, engine):
        # (not a reference: an engine in a cycle is freed whenever the collector runs, and graphs that are freed while another is recorded
        # end that recording)
        self._engine = weakref.ref(engine)
        self.pending: Optional[_Pending] = None
        self._seen: Dict[tuple, int] = {}
        self._recorded: Dict[tuple, _Recorded] = {}
        self._large = set()              # sizes whose buffers alone are more than RECORDED_BYTES
        self._accept: Dict[int, Tuple[torch.Tensor, ...]] = {}

    @property
    def engine(self):
        return self._engine()

    # ---- which models take them ------------------------------------------------------------
    def refused(self, shorten: bool = False) -> Optional[str]:
        """Why the model cannot take a drafted tree (``shorten``: why keys cannot be taken out of its cache); ``None``: it can."""
        model, cache = self.engine.model, self.engine.cache
        if cache.state:
            return "it keeps a fixed-size state per sequence"
        if not cache.kv_groups:
            return "it keeps no keys and values"
        for block in model.blocks:
            for part in block.parts.values():
                if isinstance(part, Mixer) or part.cache_need() is not None:
                    # (a part that keeps a cache and is no Mixer says nothing: it takes none)
                    why = getattr(part, "placed_steps_refused", lambda part=part: Mixer.placed_steps_refused(part))()
                    if why is not None:
                        return why
        if shorten:
            if any(g.window > 0 for g in cache.kv_groups):
                return "a window slides over its keys"
            if any(e.cache_of is not None for e in model.spec.schedule):
                return "a layer reads another layer's keys"
        return None

    # ---- a tree step -----------------------------------------------------------------------
    def drop(self) -> None:
        """Forgets a tree step that was not accepted: its nodes' pages go back."""
        if self.pending is not None:
            p, self.pending = self.pending, None
            for slot, lb, c in zip(p.slots, p.len_before, p.counts):
                self.engine.cache.settle(slot, lb, lb + c)

    def uncommitted(self) -> List[Tuple[int, int]]:
        """Per slot of a tree step that was not accepted the tokens that its pages hold, the nodes included."""
        p = self.pending
        return [] if p is None else [(slot, lb + c) for slot, lb, c in zip(p.slots, p.len_before, p.counts)]

    def _check(self, entries):
        from .engine import StepError
        e = self.engine
        why = self.refused()
        if why is not None:
            raise StepError(f"step_tree: this model takes no drafted trees: {why}")
        if e.weigh_keys:
            raise StepError("step_tree: an engine that weighs its keys takes no drafted trees (nodes that are not accepted would count)")
        if len(entries) == 0:
            raise StepError("a step needs at least one sequence")
        most = getattr(e.ops, "TREE_MAX_NODES", 64)
        slots, toks, parents = [], [], []
        for i, (slot, t, par) in enumerate(entries):
            t = np.asarray(t, dtype=np.int64).reshape(-1)
            par = [int(x) for x in par]
            if not 0 < t.size <= most:
                raise StepError(f"entry {i} (slot {slot}): a tree has 1 to {most} nodes, got {t.size}")
            if len(par) != t.size:
                raise StepError(f"entry {i} (slot {slot}): {t.size} tokens and {len(par)} parents")
            if par[0] != -1 or any(not 0 <= p < j for j, p in enumerate(par) if j):
                raise StepError(f"entry {i} (slot {slot}): the first node's parent is -1, every other node's one before it, got {par}")
            if t.min() < 0 or t.max() >= e.vocab:
                bad = int(t[(t < 0) | (t >= e.vocab)][0])
                raise StepError(f"entry {i} (slot {slot}): token id {bad} is outside the vocabulary [0, {e.vocab})")
            slots.append(int(slot))
            toks.append(t)
            parents.append(par)
        return slots, toks, parents

    def step(self, entries) -> torch.Tensor:
        from .engine import StepError
        e = self.engine
        slots, toks, parents = self._check(entries)
        counts = [int(t.size) for t in toks]
        growth = list(zip(slots, counts))
        try:
            e.cache.check_room(growth, self.uncommitted())
        except CacheError as err:
            raise StepError(str(err)) from None
        len_before = [e.cache.length(s) for s in slots]
        bits = [ancestor_bits(p) for p in parents]
        depth = [[b.bit_count() - 1 for b in tree] for tree in bits]
        limit = e.model.position_limit()
        longest = max(lb + max(d) + 1 for lb, d in zip(len_before, depth))
        if limit is not None and longest > limit:
            raise StepError(f"a sequence would reach {longest} tokens, the position tables hold {limit}")
        self.drop()
        updates = e.cache.grow(growth)
        try:
            meta, logits = self._launch(slots, toks, parents, counts, len_before, bits, depth, updates)
        except BaseException:
            e.cache.ungrow(growth, updates)          # (pages whose entries may not have reached the table)
            raise
        self.pending = _Pending(slots, counts, len_before, [t.tolist() for t in toks], self._views(meta, sum(counts), len(slots)), logits)
        return logits

    def _launch(self, slots, toks, parents, counts, len_before, bits, depth, updates):
        """Uploads a checked step and runs it: its integers on the device and its logits."""
        from .engine import length_bucket
        e = self.engine
        n, b = sum(counts), len(slots)
        cu = np.zeros(b + 1, dtype=np.int32)
        np.cumsum(counts, out=cu[1:])
        words = np.array([x for tree in bits for x in tree], dtype=np.uint64)
        places = np.concatenate([np.arange(lb, lb + c, dtype=np.int32) for lb, c in zip(len_before, counts)])
        positions = np.concatenate([lb + np.asarray(d, dtype=np.int32) for lb, d in zip(len_before, depth)])
        # the words first: they lie on 8 bytes
        host = [words.view(np.int32), np.concatenate(toks).astype(np.int32), positions, np.repeat(np.arange(b, dtype=np.int32), counts), places,
                np.concatenate([np.asarray(p, dtype=np.int32) for p in parents]), np.arange(n, dtype=np.int32),
                np.asarray(slots, dtype=np.int32), cu, np.asarray(len_before, dtype=np.int32)]
        fixed = sum(h.size for h in host)
        plan = e._apply_updates(updates, host)
        block = np.concatenate(host)
        bound = min(e.cache.max_seq_len, length_bucket(max(lb + c for lb, c in zip(len_before, counts))))
        key = (tuple(counts), bound)
        rec = self._state(key, fixed) if e.use_graphs else None
        meta = e._ensure_meta(block.size)
        e._staging.upload(block, meta)
        for g, off, k in plan:
            e.ops.scatter_i32(g.page_table, meta[off:off + k], meta[off + k:off + 2 * k])
        if rec is not None:
            rec.meta.copy_(meta[:fixed], non_blocking=True)
            meta = rec.meta
        logits = self._run(rec, meta, n, b, counts, bound)
        if rec is not None:
            self._make_room(key, rec)
        return meta, logits

    @staticmethod
    def _views(meta: torch.Tensor, n: int, b: int) -> Dict[str, torch.Tensor]:
        out, o = {"ancestors": meta[:2 * n].view(torch.int64)}, 2 * n
        for name, k in (("tokens", n), ("positions", n), ("seq_of_token", n), ("places", n), ("parents", n), ("rows", n), ("slots", b),
                        ("cu", b + 1), ("len_before", b)):
            out[name] = meta[o:o + k]
            o += k
        return out

    def _state(self, key, ints: int) -> Optional[_Recorded]:
        """Buffers of their own for sizes that have come before."""
        rec = self._recorded.pop(key, None)
        if rec is None:
            if key in self._large:
                return None
            if len(self._seen) > 256:
                self._seen.clear()
            self._seen[key] = self._seen.get(key, 0) + 1
            if self._seen[key] < 2:
                return None
            while len(self._recorded) >= RECORDED_SIZES:
                del self._recorded[next(iter(self._recorded))]
            rec = _Recorded(ints, self.engine.device)
        self._recorded[key] = rec
        return rec

    def _make_room(self, key, rec: _Recorded) -> None:
        """The sizes used longest ago go until the buffers of the rest are no more than they may be."""
        if rec.workspace.bytes() > RECORDED_BYTES:
            if len(self._large) > 256:
                self._large.clear()
            self._large.add(key)
            del self._recorded[key]
            return
        while sum(r.workspace.bytes() for r in self._recorded.values()) > RECORDED_BYTES:
            del self._recorded[next(iter(self._recorded))]

    def _run(self, rec: Optional[_Recorded], meta, n, b, counts, bound) -> torch.Tensor:
        e = self.engine
        if rec is not None and rec.graph is not None:
            rec.graph.replay()
            e.graph_kernels += rec.kernels
            return rec.logits
        m = self._views(meta, n, b)

        def forward():
            ctx = StepContext(n_tokens=n, n_seqs=b, decode=False, counts=counts, max_count=max(counts), token_ids=m["tokens"],
                              positions=m["positions"], seq_of_token=m["seq_of_token"], slots=m["slots"], cu_tokens=m["cu"],
                              len_before=m["len_before"], dtype=e.dtype, device=e.device, ops=e.ops,
                              workspace=e._workspace if rec is None else rec.workspace, max_len_after=bound, cache_positions=m["places"],
                              tree_ancestors=m["ancestors"])
            return e.model.forward(ctx, e.cache, m["rows"])

        if rec is None or rec.logits is None:
            logits = forward()                       # (of sizes that come again: their buffers exist from here on)
            if rec is not None:
                rec.logits = logits
            return logits
        graph = torch.cuda.CUDAGraph()
        rec.workspace.frozen = True
        before = getattr(e.ops, "launches", lambda: 0)()
        with torch.cuda.graph(graph):
            rec.logits = forward()
        rec.kernels = getattr(e.ops, "launches", lambda: 0)() - before
        rec.graph = graph
        graph.replay()
        e.graph_kernels += rec.kernels
        return rec.logits

    # ---- accepting -------------------------------------------------------------------------
    def accept(self, picked: Optional[torch.Tensor] = None) -> List[Tuple[List[int], int]]:
        from .engine import StepError
        e, p = self.engine, self.pending
        if p is None:
            raise StepError("accept_tree: no tree step was made, or another step, truncate or close came behind it")
        n, b = sum(p.counts), len(p.slots)
        if picked is not None and (picked.dtype != torch.int32 or tuple(picked.shape) != (n,) or picked.device != p.logits.device):
            raise StepError(f"accept_tree: picked tokens are int32 [{n}] on the engine's device")
        bufs = self._accept.get(b)
        if bufs is None:
            # path, count and next of one tensor, so that one copy brings them to the host
            whole = torch.empty(b * 66, dtype=torch.int32, device=e.device)
            bufs = self._accept[b] = (whole, whole[:64 * b].view(b, 64), whole[64 * b:65 * b], whole[65 * b:])
        whole, path, count, nxt = bufs
        m = p.meta
        if picked is None:
            need = e.ops.tree_accept_scratch(n, b)
            scratch = e._workspace.get("tree.accept", (need,), torch.int64, zero=True)
            e.ops.tree_accept(m["tokens"], m["parents"], m["cu"], path, count, nxt, logits=p.logits, scratch=scratch)
        else:
            e.ops.tree_accept(m["tokens"], m["parents"], m["cu"], path, count, nxt, picked=picked.contiguous())
        for g, rows in [(g, g.rows(e.ops)) for g in e.cache.kv_groups]:      # (made before the first row moves)
            rows.move(g.page_table, g.ring_pages, m["slots"], m["len_before"], path.view(1, b, 1, 64), count)
        got = whole.cpu().numpy()
        self.pending = None
        out = []
        for i, (slot, lb, c) in enumerate(zip(p.slots, p.len_before, p.counts)):
            k = int(got[64 * b + i])
            e.cache.settle(slot, lb + k, lb + c)
            out.append((got[64 * i:64 * i + k].tolist(), int(got[65 * b + i])))
        return out

    # ---- eviction --------------------------------------------------------------------------
    def evict(self, entries, first: int, recent: int) -> None:
        from .engine import StepError
        e = self.engine
        if not e.weigh_keys:
            raise StepError("evict: needs an engine that weighs its keys (weigh_keys)")
        if first < 0 or recent < 0:
            raise StepError(f"evict: first {first} and recent {recent} must not be negative")
        seen = set()
        for slot, keep in entries:
            try:
                length = e.cache.length(slot)
            except CacheError as err:
                raise StepError(str(err)) from None
            if slot in seen:
                raise StepError(f"evict: slot {slot} appears twice")
            seen.add(slot)
            if not max(1, first + recent) <= keep <= length:
                raise StepError(f"evict: slot {slot} holds {length} keys, cannot keep {keep} with the first {first} and the newest {recent}")
        work = [(int(s), int(k), e.cache.length(s)) for s, k in entries if k < e.cache.length(s)]
        if not work:
            return
        b, most, longest = len(work), max(k for _, k, _ in work), max(n for _, _, n in work)
        block = np.asarray([[s for s, _, _ in work], [k for _, k, _ in work], [n for _, _, n in work], [0] * b], dtype=np.int32).reshape(-1)
        meta = e._ensure_meta(block.size)
        e._staging.upload(block, meta)
        slots, keep, lengths, base = (meta[i * b:(i + 1) * b] for i in range(4))
        moves = []
        for g in e.cache.kv_groups:                       # (all that can fail for want of memory is done before the first row moves)
            chosen = torch.empty((len(g.units), b, g.need.num_kv_heads, most), dtype=torch.int32, device=e.device)
            e.ops.keep_keys(g.weights, slots, lengths, keep, chosen, first=first, recent=recent, max_len=longest)
            moves.append((g, g.rows(e.ops), chosen))
        for g, rows, chosen in moves:
            rows.move(g.page_table, g.ring_pages, slots, base, chosen, keep)
        for slot, k, n in work:
            e.cache.shorten(slot, k)
            e._taken[slot] = e._taken.get(slot, 0) + n - k
            e._kept[slot] = k
