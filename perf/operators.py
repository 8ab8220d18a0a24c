"""What is timed of the operators around drafted trees of tokens and a cache that keeps the keys which were looked at most.

A case is a dict of plain values.  ``op`` says what one pass is:

* ``attend``: attention of every sequence's tree of drafted tokens (its first node is the last token that is certain) over the
  paged cache: a node sees the cached keys and, of the tree, its ancestors and itself (``ops.attn_tree``).
* ``accept``: which path of every tree the model's logits confirm, and the token behind it (``ops.tree_accept``).
* ``weigh``: what the step's last queries gave each cached key, added up per key/value head (``ops.key_weights``).
* ``choose``: which keys of every layer, sequence and head stay: the first, the newest, and those of most weight (``ops.keep_keys``).
* ``move``: the rows of a paged cache that stay, brought together at its front in all layers (``ops.CacheRows.move``): a
  confirmed path's few nodes, or the thousands of keys that an eviction leaves.

Lengths are spread between ``low`` and ``high``, and the trees' sizes between ``nodes_low`` and ``nodes``, by the case's own
numbers; values, trees and choices come from the seed.  Pages lie in the pool in no order.
"""
import importlib
import math
import random

import torch

own = False
PAGE = 64
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
# (query heads, key/value heads, head size) of the dense models that the library's numbers are quoted on, and of small ones
HEADS = {"8b": (32, 8, 128), "14b": (40, 8, 128), "1b": (32, 8, 64), "odd": (6, 3, 32), "wide": (9, 3, 48), "one": (5, 1, 80)}


def listed():
    return [
        # a chat with a small model that drafts seven tokens a step: latency is what its user waits for
        {"name": "attend_1b_one", "op": "attend", "dtype": "bfloat16", "heads": "1b", "batch": 1, "low": 611, "high": 611,
         "nodes_low": 8, "nodes": 8, "window": 0},
        # a server's batch at the context that the library's numbers are quoted on, trees of unequal sizes
        {"name": "attend_8b_eight", "op": "attend", "dtype": "bfloat16", "heads": "8b", "batch": 8, "low": 7900, "high": 8190,
         "nodes_low": 13, "nodes": 32, "window": 0},
        # full trees over ragged long contexts of a model with groups of five heads
        {"name": "attend_14b_full", "op": "attend", "dtype": "bfloat16", "heads": "14b", "batch": 16, "low": 256, "high": 8192,
         "nodes_low": 64, "nodes": 64, "window": 0},
        # the 32-bit path that answers are checked against
        {"name": "attend_1b_float32", "op": "attend", "dtype": "float32", "heads": "1b", "batch": 3, "low": 301, "high": 1999,
         "nodes_low": 5, "nodes": 16, "window": 0},
        # the logits of one chat's tree
        {"name": "accept_one", "op": "accept", "vocab": 128256, "batch": 1, "nodes_low": 16, "nodes": 16, "greedy": True},
        # the logits of a server's trees
        {"name": "accept_batch", "op": "accept", "vocab": 151936, "batch": 32, "nodes_low": 9, "nodes": 32, "greedy": True},
        # a decode step of eight long sequences whose keys are weighed as they go
        {"name": "weigh_decode", "op": "weigh", "dtype": "bfloat16", "heads": "8b", "batch": 8, "low": 7900, "high": 8190,
         "new_low": 1, "new": 1, "last": 1},
        # a prompt step: what the last 32 tokens of long prompts looked at
        {"name": "weigh_prompt", "op": "weigh", "dtype": "bfloat16", "heads": "8b", "batch": 4, "low": 0, "high": 700,
         "new_low": 1000, "new": 8000, "last": 32},
        # one chat's cache of a small model, cut to a quarter
        {"name": "choose_one", "op": "choose", "heads": "1b", "layers": 16, "batch": 1, "low": 2011, "high": 2011, "share": 0.25,
         "first": 4, "recent": 32},
        # a batch of long sequences, all layers of a model of 8B parameters
        {"name": "choose_batch", "op": "choose", "heads": "8b", "layers": 32, "batch": 8, "low": 5000, "high": 8190, "share": 0.25,
         "first": 4, "recent": 128},
        # confirmed paths of a batch's trees
        {"name": "move_paths", "op": "move", "dtype": "bfloat16", "heads": "8b", "layers": 16, "batch": 8, "low": 500, "high": 2000,
         "nodes_low": 13, "nodes": 32, "share": 0.0},
        # an eviction: a quarter of long sequences' keys stay, others in each head
        {"name": "move_evicted", "op": "move", "dtype": "bfloat16", "heads": "8b", "layers": 8, "batch": 8, "low": 5000, "high": 8190,
         "nodes_low": 0, "nodes": 0, "share": 0.25},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("attend", "attend", "attend", "accept", "weigh", "weigh", "choose", "move", "move"))
    if op == "accept":
        batch = _log(rng, 1, 48)
        nodes = rng.randint(1, min(64, 1000 // batch))
        return {"op": op, "vocab": rng.choice((32000, 128256, 151936, 152064, 1003)), "batch": batch,
                "nodes_low": rng.randint(1, nodes), "nodes": nodes, "greedy": rng.random() < 0.8}
    if op == "choose":
        high = _log(rng, 30, 12000)
        layers, batch = _log(rng, 1, 32), _log(rng, 1, max(1, min(16, 60000 // high)))
        first = rng.randint(0, 8)
        return {"op": op, "heads": rng.choice(sorted(HEADS)), "layers": layers, "batch": batch, "low": _log(rng, max(20, high // 8), high),
                "high": high, "share": rng.choice((0.1, 0.25, 0.5, 0.9, 1.0)), "first": first, "recent": rng.randint(0, 10)}
    dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
    case = {"op": op, "dtype": dtype, "heads": rng.choice(sorted(HEADS))}
    batch = _log(rng, 1, 24)
    high = _log(rng, 5, min(16000, 80000 // batch) // (4 if dtype == "float32" else 1))
    low = rng.randint(0, high) if op == "weigh" else _log(rng, max(1, high // 16), high)
    case.update(batch=batch, low=0 if op == "attend" and rng.random() < 0.1 else low, high=high)
    if op == "attend":
        nodes = rng.randint(1, 64 if dtype == "bfloat16" else 24)
        case.update(nodes_low=rng.randint(1, nodes), nodes=nodes, window=rng.choice((0, 0, 0, 70, 1000)))
    elif op == "weigh":
        new = rng.choice((1, 1, _log(rng, 2, 400)))
        case.update(new_low=rng.randint(1, new), new=new, last=1 if new == 1 else rng.randint(1, 32))
    else:
        layers = rng.randint(1, 8)
        paths = rng.random() < 0.5
        nodes = rng.randint(1, 64) if paths else 0
        case.update(layers=layers, nodes_low=rng.randint(1, nodes) if paths else 0, nodes=nodes,
                    share=0.0 if paths else rng.choice((0.1, 0.3, 0.6, 1.0)))
    return case


def _spread(case, low, high, salt):
    r = random.Random(1000003 * case["batch"] + 1009 * low + high + salt)
    return [r.randint(low, high) for _ in range(case["batch"])]


def _lengths(case):
    return _spread(case, case["low"], case["high"], 0)


def _nodes(case):
    return _spread(case, case["nodes_low"], case["nodes"], 1)


def _brings(case):
    return _spread(case, case["new_low"], case["new"], 2)


def _keeps(case):
    """How many keys of each sequence stay."""
    least = case.get("first", 0) + case.get("recent", 0)
    return [max(min(least, n), 1, int(n * case["share"])) for n in _lengths(case)]


# ---- what a program has in hand -------------------------------------------------------------------

class State:
    pass


def prepare(case, seed):
    st, op = State(), case["op"]
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    r = random.Random(seed)
    batch = case["batch"]
    st.case = case

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return torch.randn(*shape, device=dev, generator=g, dtype=dtype).mul_(scale)

    def trees(sizes):
        """Parents of every tree's nodes (a node hangs on one of the few before it) and each node's ancestors as bits."""
        parents, bits = [], []
        for n in sizes:
            above = [-1] + [r.randint(max(0, i - 6), i - 1) for i in range(1, n)]
            mine = []
            for i, p in enumerate(above):
                mine.append((mine[p] if p >= 0 else 0) | 1 << i)
            parents.append(above)
            bits += mine
        return parents, torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64, device=dev)

    def starts(sizes):
        return ints([sum(sizes[:i]) for i in range(len(sizes) + 1)])

    if op == "accept":
        st.sizes = _nodes(case)
        parents, st.ancestors = trees(st.sizes)
        n, v = sum(st.sizes), case["vocab"]
        st.tokens = torch.randint(0, v, (n,), device=dev, generator=g, dtype=torch.int32)
        st.parents, st.cu = ints([p for t in parents for p in t]), starts(st.sizes)
        st.logits = normal(n, v, scale=2.0)
        # a good draft: most nodes' most likely next token is among their children
        st.picked = torch.randint(0, v, (n,), device=dev, generator=g, dtype=torch.int32)
        at, likely = [], []
        for b, above in enumerate(parents):
            base = sum(st.sizes[:b])
            for i in range(len(above)):
                children = [j for j, p in enumerate(above) if p == i]
                if children and r.random() < 0.8:
                    at.append(base + i)
                    likely.append(base + r.choice(children))
        if at:
            rows, toks = torch.tensor(at, device=dev), st.tokens[torch.tensor(likely, device=dev)].long()
            st.logits[rows, toks] = 14.0
            st.picked[rows] = toks.int()
        st.path = torch.empty(batch, PAGE, dtype=torch.int32, device=dev)
        st.count = torch.empty(batch, dtype=torch.int32, device=dev)
        st.next = torch.empty(batch, dtype=torch.int32, device=dev)
        if own:
            st.ops = importlib.import_module("daisi-llogos_b200.kernels.ops")
            st.scratch = torch.zeros(st.ops.tree_accept_scratch(n, batch), dtype=torch.int64, device=dev)
        return st
    nh, nkv, hd = HEADS[case["heads"]]
    lens = _lengths(case)
    st.lens = lens
    n_slots = batch + 2
    st.slots = ints(r.sample(range(n_slots), batch))
    if op in ("weigh", "choose"):
        width = max(lens) + (case["new"] if op == "weigh" else 0)
        st.weights = normal(case.get("layers", 1), n_slots, nkv, width).square_().mul_(4.0 / width)      # a few steps' shares
    if op == "choose":
        keeps = _keeps(case)
        st.lengths, st.keep = ints(lens), ints(keeps)
        st.chosen = torch.full((case["layers"], batch, nkv, max(keeps)), -1, dtype=torch.int32, device=dev)
        if own:
            st.ops = importlib.import_module("daisi-llogos_b200.kernels.ops")
        return st

    # the paged cache: a pool of pages, each sequence's in no order, one page beyond that no sequence has
    dtype = DTYPES[case["dtype"]]
    window = case.get("window", 0)
    more = case["new"] if op == "weigh" else case["nodes"]
    pages = (max(lens) + more + PAGE - 1) // PAGE
    st.ring = min(pages, (window + PAGE - 1) // PAGE + 1) if window else pages
    n_pages = batch * st.ring + 1
    order = list(range(n_pages - 1))
    r.shuffle(order)
    table = [[n_pages - 1] * st.ring for _ in range(n_slots)]
    for i, s in enumerate(st.slots.tolist()):
        table[s] = order[i * st.ring:(i + 1) * st.ring]
    st.table = ints(table)
    layers = case.get("layers", 1)
    st.k = normal(layers, n_pages, nkv, PAGE, hd, dtype=dtype)
    st.v = normal(layers, n_pages, nkv, PAGE, hd, dtype=dtype) if op != "weigh" else None
    st.before = ints(lens)
    st.scale = hd ** -0.5
    if op == "attend":
        st.sizes = _nodes(case)
        st.ancestors = trees(st.sizes)[1]
        st.max_len = max(a + b for a, b in zip(lens, st.sizes))
    elif op == "weigh":
        st.sizes = _brings(case)
        st.max_len = max(a + b for a, b in zip(lens, st.sizes))
    if op in ("attend", "weigh"):
        n = sum(st.sizes)
        st.cu = starts(st.sizes)
        st.q = normal(n, nh, hd, scale=2.0).to(dtype)           # scores that spread: a few keys stand out
    if op == "attend":
        st.out = torch.empty(n, nh * hd, dtype=dtype, device=dev)
    if op == "move":
        if case["nodes"]:
            # confirmed paths: nodes in ascending order, the first always among them, the same in all layers and heads
            st.base = ints(lens)
            paths = [[0] + sorted(r.sample(range(1, n), r.randint(0, min(5, n - 1)))) if n > 1 else [0] for n in _nodes(case)]
            width = max(len(p) for p in paths)
            st.source = ints([p + [0] * (width - len(p)) for p in paths]).view(1, batch, 1, width)
            st.count = ints([len(p) for p in paths])
        else:
            st.base = ints([0] * batch)
            keeps = _keeps(case)
            st.count = ints(keeps)
            width = max(keeps)
            order = torch.rand(layers, batch, nkv, max(lens), device=dev, generator=g)
            order.masked_fill_(torch.arange(max(lens), device=dev) >= st.before.view(1, -1, 1, 1), 2.0)
            picked = order.argsort(-1)[..., :width]
            picked.masked_fill_(torch.arange(width, device=dev) >= st.count.view(1, -1, 1, 1), 1 << 30)
            st.source = picked.sort(-1).values.int().contiguous()
    if own:
        ops = st.ops = importlib.import_module("daisi-llogos_b200.kernels.ops")
        if op == "attend":
            st.plan = ops.attn_tree_plan(dtype, batch, case["nodes"], nh, nkv, hd, st.max_len)
        elif op == "weigh":
            st.plan = ops.key_weights_plan(dtype, batch, case["last"], nh, nkv, hd, st.max_len)
        else:
            st.rows = ops.CacheRows(list(st.k), list(st.v))
        if op in ("attend", "weigh"):
            st.scratch = torch.empty(max(1, st.plan.scratch_floats), device=dev)
            st.counters = torch.zeros(max(1, st.plan.n_counters), dtype=torch.int32, device=dev)
    return st


# ---- a pass ---------------------------------------------------------------------------------------

def run(st):
    case, op = st.case, st.case["op"]
    if own:
        ops = st.ops
        if op == "attend":
            ops.attn_tree(st.q, st.k[0], st.v[0], st.table, st.ring, st.slots, st.cu, st.before, st.ancestors, st.out, st.scratch,
                          scale=st.scale, window=case["window"], plan=st.plan, counters=st.counters)
            return st.out
        if op == "accept":
            source = {"logits": st.logits, "scratch": st.scratch} if case["greedy"] else {"picked": st.picked}
            ops.tree_accept(st.tokens, st.parents, st.cu, st.path, st.count, st.next, **source)
            return {"path": st.path, "count": st.count, "next": st.next}
        if op == "weigh":
            ops.key_weights(st.q, st.k[0], st.table, st.slots, st.cu, st.before, st.weights[0], st.scratch, scale=st.scale,
                            last=case["last"], plan=st.plan, counters=st.counters)
            return st.weights
        if op == "choose":
            ops.keep_keys(st.weights, st.slots, st.lengths, st.keep, st.chosen, first=case["first"], recent=case["recent"])
            return st.chosen
        st.rows.move(st.table, st.ring, st.slots, st.base, st.source, st.count)
        return {"k": st.k, "v": st.v}
    return {"attend": plain_attend, "accept": plain_accept, "weigh": plain_weigh, "choose": plain_choose, "move": plain_move}[op](st)


def _pages(pool, st):
    """A layer's rows of every sequence in the order of their positions: float32 [batch, kv heads, positions, head size]."""
    count = (st.max_len + PAGE - 1) // PAGE
    at = st.table[st.slots.long()][:, torch.arange(count, device=pool.device) % st.ring].long()
    rows = pool[at].float().transpose(1, 2)
    return rows.reshape(rows.shape[0], rows.shape[1], count * PAGE, -1)


def plain_attend(st):
    n, nh, hd = st.q.shape
    dev, batch, most = st.q.device, len(st.sizes), max(st.sizes)
    k, v = _pages(st.k[0], st), _pages(st.v[0], st)
    nkv = k.shape[1]
    cu, before = st.cu.long(), st.before.long()
    node = torch.arange(most, device=dev)
    here = node < (cu[1:] - cu[:-1])[:, None]                                # [batch, most]
    at = torch.where(here, cu[:-1, None] + node, 0)
    q = st.q.float()[at].view(batch, most, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q, k.unsqueeze(2).transpose(-1, -2)) * st.scale          # [batch, nkv, group, most, positions]
    pos = torch.arange(k.shape[2], device=dev)
    place = pos - before[:, None]                                            # [batch, positions]
    bits = (st.ancestors[at][:, :, None] >> torch.arange(PAGE, device=dev)) & 1
    depth = bits.sum(-1) - 1
    own_node = torch.gather(bits, 2, place.clamp(0, PAGE - 1)[:, None].expand(-1, most, -1)) == 1
    sees = torch.where(place[:, None] < 0, True, own_node & (place[:, None] < PAGE))
    if st.case["window"]:
        # a node stands as many places behind the cached keys as it has ancestors
        deep = torch.gather(depth, 1, place.clamp(0, most - 1))
        stands = torch.where(place < 0, place, deep)
        sees &= depth[:, :, None] - stands[:, None] < st.case["window"]
    sees = sees[:, None, None]
    s = s.masked_fill(~sees, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v.unsqueeze(2)) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch * most, nh * v.shape[-1])
    seq = torch.searchsorted(cu[1:], torch.arange(n, device=dev), right=True)
    return o[seq * most + torch.arange(n, device=dev) - cu[seq]].to(st.q.dtype)


def plain_accept(st):
    dev, batch, most = st.tokens.device, len(st.sizes), max(st.sizes)
    best = st.logits.argmax(-1) if st.case["greedy"] else st.picked.long()
    if st.case["greedy"]:
        top = st.logits.gather(1, best[:, None])
        best = (st.logits == top).int().argmax(-1)                           # of equal ones the first
    cu = st.cu.long()
    node = torch.arange(most, device=dev)
    here = node < (cu[1:] - cu[:-1])[:, None]
    at = torch.where(here, cu[:-1, None] + node, 0)
    tokens, parents, best = st.tokens.long()[at], st.parents.long()[at], best[at]
    # a node is taken where its token is what its parent's logits say, and no node before it with the same parent has that token
    twin = (parents[:, :, None] == parents[:, None]) & (tokens[:, :, None] == tokens[:, None]) & (node[None, :] < node[:, None])
    taken = (torch.gather(best, 1, parents.clamp(0)) == tokens) & ~twin.any(-1)
    taken[:, 0] = True
    bits = (st.ancestors[at][:, :, None] >> node) & 1                        # [batch, node, ancestor]
    on = here & ((bits == 0) | taken[:, None]).all(-1)
    count = on.sum(-1)
    order = torch.where(on, node, PAGE).sort(-1).values
    path = torch.full((batch, PAGE), -1, dtype=torch.int32, device=dev)
    path[:, :most] = torch.where(order < PAGE, order, -1).int()
    last = torch.gather(order, 1, count[:, None] - 1)
    return {"path": path, "count": count.int(), "next": torch.gather(best, 1, last)[:, 0].int()}


def plain_weigh(st):
    n, nh, hd = st.q.shape
    dev, batch, last = st.q.device, len(st.sizes), st.case["last"]
    k = _pages(st.k[0], st)
    nkv = k.shape[1]
    cu, before = st.cu.long(), st.before.long()
    brings = cu[1:] - cu[:-1]
    back = torch.arange(last, device=dev)                                    # queries counted from the newest
    here = back < brings[:, None]
    at = torch.where(here, cu[1:, None] - 1 - back, 0)
    q = st.q.float()[at].view(batch, last, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q, k.unsqueeze(2).transpose(-1, -2)) * st.scale
    pos = torch.arange(k.shape[2], device=dev)
    after = before + brings
    sees = (pos[None, None] <= (after[:, None] - 1 - back)[:, :, None]) & here[:, :, None]
    s = s.masked_fill(~sees[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    new = (e / torch.where(total > 0, total, 1.0)).sum((2, 3))                # [batch, nkv, positions]
    width = min(k.shape[2], st.weights.shape[-1])
    new, pos = new[..., :width], pos[:width]
    held = st.weights[0, st.slots.long(), :, :width]
    kept = torch.where(pos < before[:, None, None], held, 0.0) + new
    st.weights[0, st.slots.long(), :, :width] = torch.where(pos < after[:, None, None], kept, held)
    return st.weights


def plain_choose(st):
    most = max(st.lens)
    w = st.weights[:, st.slots.long()][..., :most]
    pos = torch.arange(most, device=w.device)
    length, keep = st.lengths.view(1, -1, 1, 1), st.keep.view(1, -1, 1, 1)
    stays = (pos < st.case["first"]) | (pos >= length - st.case["recent"])
    w = w.masked_fill(stays, math.inf).masked_fill(pos >= length, -math.inf)
    order = w.sort(dim=-1, descending=True, stable=True).indices[..., :st.chosen.shape[-1]]
    order = order.masked_fill(torch.arange(order.shape[-1], device=w.device) >= keep, 1 << 30).sort(-1).values
    st.chosen.copy_(torch.where(order < 1 << 30, order, st.chosen))
    return st.chosen


def plain_move(st):
    layers, n_pages, nkv, _, hd = st.k.shape
    dev, batch, width = st.k.device, st.slots.numel(), st.source.shape[-1]
    table = st.table[st.slots.long()].long()
    head = torch.arange(nkv, device=dev).view(1, 1, -1, 1)
    layer = torch.arange(layers, device=dev).view(-1, 1, 1, 1)

    def row(pos):
        """Where the row of a position lies in the pool of all layers: [layers, batch, heads, width]."""
        page = torch.gather(table, 1, (pos // PAGE % st.ring).transpose(0, 1).reshape(batch, -1)).view(batch, *pos.shape[:1], *pos.shape[2:])
        return ((layer * n_pages + page.transpose(0, 1)) * nkv + head) * PAGE + pos % PAGE

    j = torch.arange(width, device=dev).view(1, 1, 1, -1)
    real = j < st.count.view(1, -1, 1, 1)
    base = st.base.long().view(1, -1, 1, 1)
    spare = ((layer + 1) * n_pages * nkv - 1) * PAGE                          # a row of the page that no sequence has
    source = torch.where(real, row(base + torch.where(real, st.source.long(), 0)), spare)
    target = torch.where(real, row((base + torch.where(real, j, 0)).expand(*st.source.shape[:3], -1)), spare)
    for pool in (st.k, st.v):
        rows = pool.view(-1, hd)
        rows[target.reshape(-1)] = rows[source.reshape(-1)]
    return {"k": st.k, "v": st.v}


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "accept":
        n = sum(_nodes(case))
        return {"bytes": 4.0 * n * (2 + (case["vocab"] if case["greedy"] else 1)) + 4.0 * case["batch"] * (PAGE + 2),
                "flops": float(n * case["vocab"]) if case["greedy"] else 0.0}
    nh, nkv, hd = HEADS[case["heads"]]
    lens = _lengths(case)
    if op == "choose":
        pairs = case["layers"] * nkv
        return {"bytes": 4.0 * pairs * (sum(lens) + sum(_keeps(case))), "flops": float(pairs * sum(lens))}
    e = 2.0 if case["dtype"] == "bfloat16" else 4.0
    if op == "attend":
        sizes, w = _nodes(case), case["window"]
        seen = [min(n, w) if w else n for n in lens]
        keys = sum(a + b for a, b in zip(seen, sizes))
        pairs = sum(a * b + b for a, b in zip(seen, sizes))
        return {"bytes": e * (2 * keys * nkv * hd + 2 * sum(sizes) * nh * hd) + 8.0 * sum(sizes), "flops": 4.0 * nh * hd * pairs}
    if op == "weigh":
        brings = _brings(case)
        queries = [min(b, case["last"]) for b in brings]
        keys = sum(lens) + sum(brings)
        pairs = sum(a * (n + b) for a, n, b in zip(queries, lens, brings))
        return {"bytes": e * (keys * nkv * hd + sum(queries) * nh * hd) + 4.0 * nkv * (sum(lens) + keys), "flops": 2.0 * nh * hd * pairs}
    # paths: at most five nodes behind the first; of an eviction every row that stays
    rows = sum(min(n, 3) for n in _nodes(case)) if case["nodes"] else sum(_keeps(case))
    return {"bytes": 2.0 * 2 * e * case["layers"] * rows * nkv * hd, "flops": 0.0}


# ---- the same in float64 --------------------------------------------------------------------------

def exact(case, seed):
    op = case["op"]
    if op in ("accept", "choose"):
        return None                                              # whole numbers
    st, F64 = prepare(case, seed), torch.float64

    def keys(pool, b, count, head):
        """Rows of the first ``count`` positions of sequence b (of a ring: those that it still has)."""
        pos = torch.arange(count, device=pool.device)
        return pool[st.table[int(st.slots[b])][pos // PAGE % st.ring].long(), head, pos % PAGE]

    if op == "move":
        k, v = st.k.clone(), st.v.clone()
        for b, count in enumerate(st.count.tolist()):
            table, base = st.table[int(st.slots[b])].long(), int(st.base[b])
            to = torch.arange(count, device=k.device) + base
            for layer in range(k.shape[0]):
                for head in range(k.shape[2]):
                    src = st.source[min(layer, st.source.shape[0] - 1), b, min(head, st.source.shape[2] - 1), :count].long() + base
                    for old, new in ((st.k, k), (st.v, v)):
                        new[layer, table[to // PAGE % st.ring], head, to % PAGE] = old[layer, table[src // PAGE % st.ring], head, src % PAGE]
        return {"k": k, "v": v}
    nh, nkv, hd = HEADS[case["heads"]]
    group = nh // nkv
    if op == "attend":
        out = torch.zeros(sum(st.sizes), nh, hd, dtype=F64, device=st.q.device)
    else:
        out = st.weights.to(F64)
    for b, count in enumerate(st.sizes):
        lo, before = int(st.cu[b]), st.lens[b]
        total = before + count
        pos = torch.arange(total, device=st.q.device)
        if op == "attend":
            bits = [int(x) & ((1 << 64) - 1) for x in st.ancestors[lo:lo + count]]
            where = torch.tensor([before + bin(x).count("1") - 1 for x in bits], device=st.q.device)
            place = torch.cat([pos[:before], where])
            sees = torch.ones(count, total, dtype=torch.bool, device=st.q.device)
            sees[:, before:] = torch.tensor([[bool(x >> j & 1) for j in range(count)] for x in bits], device=st.q.device)
            if case["window"]:
                sees &= place[None] > where[:, None] - case["window"]
            rows = range(lo, lo + count)
        else:
            rows = range(max(lo, lo + count - case["last"]), lo + count)
            sees = pos[None] <= torch.tensor([before + i - lo for i in rows], device=st.q.device)[:, None]
        for head in range(nkv):
            k = keys(st.k[0], b, total, head).to(F64)
            q = st.q[rows.start:rows.stop, head * group:(head + 1) * group].to(F64)          # [rows, group, hd]
            s = torch.einsum("rgd,jd->rgj", q, k) / math.sqrt(hd)
            p = torch.softmax(s.masked_fill(~sees[:, None], -math.inf), -1)
            if op == "attend":
                out[rows.start:rows.stop, head * group:(head + 1) * group] = torch.einsum("rgj,jd->rgd", p, keys(st.v[0], b, total, head).to(F64))
            else:
                w = out[0, int(st.slots[b]), head]
                w[before:total] = 0.0
                w[:total] += p.sum((0, 1))
    return out.view(sum(st.sizes), -1) if op == "attend" else out
