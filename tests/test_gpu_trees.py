"""Drafted trees over the paged cache, and caches cut by accumulated weight: each operator against the plain float64 forms of ``tree_plain``, at
the sizes, masks and contents where it can go wrong.  ``slack`` there says what rounding allows."""
import importlib
import random

import pytest
import torch

import tree_plain as T

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("daisi-llogos_b200.kernels.ops")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def normal(*shape, seed, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


def tree(r, n, chain=False):
    return [-1][:n] + [i - 1 if chain else r.randint(max(0, i - 5), i - 1) for i in range(1, n)]


class Case:
    """A batch of trees over paged keys, on the host and on the GPU."""

    def __init__(self, dtype, nh, nkv, hd, before, nodes, *, vd=0, window=0, seed=0, extra=0, chain=False, bits=None, spoil=None):
        r = random.Random(seed)
        vd = vd or hd
        self.dtype, self.window, self.before, self.nodes = dtype, window, before, nodes
        b = len(before)
        self.bits = bits or [T.tree_bits(tree(r, n, chain)) for n in nodes]
        self.k = [normal(lb + n, nkv, hd, seed=seed + 10 * i + 1).to(dtype) for i, (lb, n) in enumerate(zip(before, nodes))]
        self.v = [normal(lb + n, nkv, vd, seed=seed + 10 * i + 2).to(dtype) for i, (lb, n) in enumerate(zip(before, nodes))]
        if spoil:
            spoil(self)
        n = sum(nodes)
        self.q = normal(n + extra, nh, hd, seed=seed + 3, scale=2.0).to(dtype)
        self.scale = hd ** -0.5
        self.max_len = max(lb + m for lb, m in zip(before, nodes))
        pages = max(1, -(-self.max_len // 64))
        self.ring = min(pages, -(-window // 64) + 1) if window else pages
        self.slots = r.sample(range(b + 3), b)
        (kp, vp), table = T.pages_of(list(zip(self.k, self.v)), nkv, (hd, vd), dtype, self.ring, b + 3, self.slots, seed, device=DEV)
        self.cu = [sum(nodes[:i]) for i in range(b + 1)]
        self.args = [self.q.to(DEV), kp, vp, table, self.ring, ints(self.slots), ints(self.cu), ints(before),
                     torch.tensor(T.signed([x for t in self.bits for x in t]) + [-1] * extra, dtype=torch.int64, device=DEV)]
        self.shape = (nh, nkv, hd, vd)

    def call(self, ops, max_nodes=None, max_len=None):
        nh, nkv, hd, vd = self.shape
        plan = ops.attn_tree_plan(self.dtype, len(self.before), max_nodes or max(1, max(self.nodes)), nh, nkv, hd, max_len or self.max_len, vd)
        out = torch.full((self.q.shape[0], nh * vd), 7.0, dtype=self.dtype, device=DEV)
        scratch = torch.full((max(1, plan.scratch_floats),), float("nan"), device=DEV)
        counters = torch.zeros(max(1, plan.n_counters), dtype=torch.int32, device=DEV)

        def go():
            ops.attn_tree(*self.args, out, scratch, scale=self.scale, window=self.window, plan=plan, counters=counters)
        go()
        assert not counters.any()
        return out, go

    def want(self):
        outs, slacks = [], []
        for i, n in enumerate(self.nodes):
            q = self.q[self.cu[i]:self.cu[i] + n]
            o, s = T.attend(q, self.k[i], self.v[i], T.sees(self.before[i], n, self.bits[i], self.window), self.scale, self.dtype)
            outs.append(o)
            slacks.append(s)
        nh, _, _, vd = self.shape
        return torch.cat(outs).reshape(-1, nh * vd), torch.cat(slacks).reshape(-1, nh * vd)

    def check(self, ops, **kw):
        out, _ = self.call(ops, **kw)
        want, slack = self.want()
        n = sum(self.nodes)
        got = out[:n].cpu().double()
        assert torch.isfinite(got).all()
        off = (got - want).abs() - slack
        assert float(off.max()) <= 1e-7, (float(off.max()), int(off.argmax()))
        assert (out[n:] == 7.0).all()                            # rows behind the last tree are left as they were
        return out


HEADS = [(F32, 4, 2, 16, 0), (F32, 6, 3, 32, 0), (F32, 5, 1, 48, 0), (F32, 3, 3, 20, 0), (F32, 8, 2, 64, 0), (F32, 4, 1, 128, 64),
         (F32, 2, 1, 384, 0), (F32, 4, 2, 30, 7), (BF16, 8, 2, 64, 0), (BF16, 8, 1, 128, 0), (BF16, 5, 1, 128, 0), (BF16, 6, 3, 80, 0),
         (BF16, 4, 4, 96, 0), (BF16, 16, 1, 64, 0), (BF16, 4, 2, 64, 128), (BF16, 4, 2, 20, 0), (BF16, 2, 1, 192, 0), (BF16, 9, 3, 48, 0),
         (BF16, 12, 4, 24, 40), (BF16, 7, 1, 8, 0)]


@pytest.mark.parametrize("dtype,nh,nkv,hd,vd", HEADS, ids=lambda x: str(x).replace("torch.", ""))
def test_trees_of_every_head_layout(ops, dtype, nh, nkv, hd, vd):
    Case(dtype, nh, nkv, hd, [70, 0, 129, 64], [5, 3, 17, 1], vd=vd, seed=nh + hd).check(ops)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("before,nodes", [
    ([0], [1]), ([0], [64]), ([1], [1]), ([63], [1]), ([63], [2]), ([64], [1]), ([65], [63]), ([127], [64]), ([128], [64]), ([1000], [33]),
    ([0, 500, 64, 3], [64, 1, 40, 7]), ([2500], [8]), ([31, 32, 33], [16, 16, 16]), ([300] * 9, [2, 4, 8, 16, 32, 64, 1, 3, 5])],
    ids=lambda x: "_".join(map(str, x)))
def test_trees_of_every_length(ops, dtype, hd, before, nodes):
    Case(dtype, 8, 2, hd, before, nodes, seed=hd + sum(nodes)).check(ops)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 5, 63, 64, 65, 128, 200])
def test_a_window_goes_by_the_nodes_depth(ops, dtype, window):
    """Rings have gone round: pages hold the newest keys alone, the older ones are not there."""
    Case(dtype, 6, 3, 64, [300, 10, 64, 511], [20, 12, 64, 33], window=window, seed=window).check(ops)
    Case(dtype, 4, 2, 64, [130, 257], [30, 9], window=window, seed=window, chain=True).check(ops)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_nodes_that_see_nothing_or_few(ops, dtype):
    """No cached keys and no bits: zeros.  A node may also see others than a tree would give it, itself not among them."""
    bits = [[0, 1, 0b110, 0], [0b1000, 0, 0b1, 0b1011]]
    c = Case(dtype, 4, 2, 64, [0, 0], [4, 4], bits=bits, seed=3)
    out = c.check(ops)
    assert not out[0].any() and not out[3].any() and not out[5].any()
    Case(dtype, 4, 2, 64, [70, 0], [4, 4], bits=bits, seed=4).check(ops)


@pytest.mark.parametrize("dtype,hd", [(F32, 64), (BF16, 64), (BF16, 128), (BF16, 48), (BF16, 20)], ids=["f32", "bf16", "bf16_128", "bf16_48", "bf16_20"])
def test_what_a_node_does_not_see_has_no_part(ops, dtype, hd):
    """A node's key and value are NaN or infinite; only the node itself sees it, and only its rows may show it."""
    r = random.Random(5)
    for bad in (float("nan"), float("inf"), float("-inf")):
        parents = [-1, 0, 0, 1, 2, 2, 4]
        bits = T.tree_bits(parents)

        def spoil(c):
            c.k[0][90 + 5, :, r.randrange(hd)] = bad
            c.v[0][90 + 5, :, 3] = bad
            c.v[0][90 + 3] = bad                                 # the whole value
        c = Case(dtype, 8, 2, hd, [90], [7], bits=[bits], seed=9, spoil=spoil)
        out, _ = c.call(ops)
        want, slack = c.want()
        clean = [0, 1, 2, 4, 6]
        got = out.cpu().double()
        assert torch.isfinite(got[clean]).all()
        assert ((got - want).abs()[clean] <= slack[clean] + 1e-7).all()
        assert not torch.isfinite(got[3]).any()


def test_an_infinite_value_that_a_window_hides(ops):
    """At a window's edge the rows of a tile differ in what they see; a cached value that the deepest nodes do not see is infinite."""
    for dtype in (F32, BF16):
        def spoil(c):
            c.v[0][100 - 10 + 4] = float("inf")                  # depth 4 and more do not see it
        c = Case(dtype, 4, 2, 64, [100], [8], window=10, chain=True, seed=2, spoil=spoil)
        out, _ = c.call(ops)
        want, slack = c.want()
        got = out.cpu().double()
        fine = torch.isfinite(want).all(1)
        assert fine.tolist() == [False] * 4 + [True] * 4
        assert ((got - want).abs()[4:] <= slack[4:] + 1e-7).all() and not torch.isfinite(got[:4]).any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_batches_with_an_empty_tree_and_rows_behind(ops, dtype):
    Case(dtype, 8, 2, 64, [40, 100, 70], [6, 0, 9], seed=1, extra=5).check(ops)
    Case(dtype, 8, 2, 64, [0, 100], [0, 9], seed=2, extra=1).check(ops)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_a_plan_for_more_gives_the_same(ops, dtype):
    """A plan for longer sequences and larger trees only cuts the keys elsewhere."""
    c = Case(dtype, 8, 2, 128, [700, 90], [11, 30], seed=6)
    pages = torch.cat([c.args[3], c.args[3][:, :1].expand(-1, 60)], 1).contiguous()
    c.args[3], c.args[4] = pages, pages.shape[1]
    c.check(ops, max_nodes=64, max_len=pages.shape[1] * 64)


@pytest.mark.parametrize("dtype,hd", [(F32, 64), (BF16, 64), (BF16, 128)], ids=["f32", "bf16_64", "bf16_128"])
def test_the_same_bits_twice_in_a_graph_and_on_another_stream(ops, dtype, hd):
    c = Case(dtype, 8, 2, hd, [900, 33, 257], [40, 1, 12], seed=8)
    out, go = c.call(ops)
    first = out.clone()
    out.fill_(0)
    go()
    assert torch.equal(first, out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out.fill_(0)
        go()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    other = Case(dtype, 8, 2, hd, [500, 100, 256], [3, 33, 17], seed=11)
    for a, x in zip(c.args, other.args):                          # other lengths, trees, keys in the recorded buffers
        if isinstance(a, torch.Tensor) and a.shape == x.shape:
            a.copy_(x)
    c.args[0][:53].copy_(other.args[0])
    c.args[8][:53].copy_(other.args[8])
    for i in (1, 2):
        assert c.args[i].shape[0] >= other.args[i].shape[0]
        c.args[i][:other.args[i].shape[0]].copy_(other.args[i])
    c.args[3][:, :other.args[3].shape[1]].copy_(other.args[3])
    for _ in range(2):
        out.fill_(7)
        graph.replay()
        want, slack = other.want()
        got = out[:53].cpu().double()
        assert ((got - want).abs() <= slack + 1e-7).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("before,nodes", [([0], [17]), ([0, 1, 2, 3], [20, 17, 64, 33]), ([40] * 40, [20] * 40), ([64, 700, 0, 9], [64, 33, 1, 2]),
                                          ([5000], [64]), ([3000, 20], [40, 64])], ids=lambda x: "_".join(map(str, x[:4])))
@pytest.mark.parametrize("nh,nkv", [(8, 2), (10, 2), (3, 3), (16, 1)])
def test_many_rows(ops, hd, before, nodes, nh, nkv, monkeypatch):
    """Row blocks of 128: one and several, whole and with a few rows, runs of one key tile and of many; on both matrix paths."""
    c = Case(BF16, nh, nkv, hd, before, nodes, seed=hd + nh)
    c.check(ops)
    monkeypatch.setattr(ops, "USE_TC_TREE", False)
    c.check(ops)


@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("before,nodes", [([0, 63, 64, 300], [5, 9, 16, 12]), ([1000, 2], [9, 5])], ids=str)
def test_a_few_rows_on_both_matrix_paths(ops, hd, before, nodes, window, monkeypatch):
    c = Case(BF16, 8, 2, hd, before, nodes, window=window, seed=hd)
    for rows in ({}, {64: 0, 128: 0}):
        monkeypatch.setattr(ops, "TREE_MMA_ROWS", rows)
        c.check(ops)


@pytest.mark.parametrize("tc", [True, False], ids=["tc", "mma"])
@pytest.mark.parametrize("hd", [64, 128])
def test_what_many_rows_do_not_see_has_no_part(ops, hd, tc, monkeypatch):
    """Values that are not finite, in a tree of many rows: at its first tile, at a later one, with rows that rise in between."""
    monkeypatch.setattr(ops, "USE_TC_TREE", tc)
    for before in (0, 30, 64, 200, 1000):
        parents = [-1, 0, 0, 1, 2, 2, 4] + [6 + i for i in range(20)]
        bits = T.tree_bits(parents)

        def spoil(c):
            c.v[0][before + 5] = float("nan")
            c.v[0][before + 3, :, 1] = float("inf")
            c.k[0][before + 3] *= 8
        c = Case(BF16, 16, 2, hd, [before], [27], bits=[bits], seed=9, spoil=spoil)
        out, _ = c.call(ops)
        want, slack = c.want()
        got = out.cpu().double().view(27, 16, hd)
        clean = torch.tensor([i for i in range(27) if not bits[i] >> 5 & 1 and not bits[i] >> 3 & 1])
        assert torch.isfinite(got[clean]).all() and len(clean) > 20
        assert ((got - want.view(27, 16, hd)).abs()[clean] <= slack.view(27, 16, hd)[clean] + 1e-7).all()
        assert torch.isnan(got[5]).all() and not torch.isfinite(got[3, :, 1]).any() and torch.isfinite(got[3, :, 2:]).all()


@pytest.mark.parametrize("dtype,nh,hd", [(F32, 8, 64), (BF16, 8, 64), (BF16, 8, 20), (BF16, 32, 128)], ids=["f32", "mma", "simt", "tc"])
def test_queries_that_are_no_numbers_show(ops, dtype, nh, hd):
    c = Case(dtype, nh, 2, hd, [500, 70], [9, 3], seed=4)
    c.args[0][2] = float("nan")
    c.args[0][10, 1] = float("nan")
    out, _ = c.call(ops)
    out = out.view(12, nh, hd)
    assert torch.isnan(out[2]).all() and torch.isnan(out[10, 1]).all()
    out[2] = out[10, 1] = 0.0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("hd,vd", [(64, 64), (128, 128), (80, 48), (8, 128)])
def test_bfloat16_trees_on_the_cuda_cores(ops, hd, vd, monkeypatch):
    monkeypatch.setattr(ops, "USE_MMA_TREE", False)
    monkeypatch.setattr(ops, "USE_TC_TREE", False)
    Case(BF16, 8, 2, hd, [70, 0, 600, 64], [5, 3, 64, 1], vd=vd, seed=hd).check(ops)


def test_no_wait_has_run_out(ops):
    """Behind the tests above: none of their launches gave a wait up."""
    assert ops.attn_tree_status() == 0


def test_pages_far_behind(ops):
    """Pools of more than 2^32 bytes and 2^31 elements: the last pages are the sequence's."""
    nkv, hd, n_pages = 8, 128, 34000
    c = Case(BF16, 16, nkv, hd, [200], [9], seed=12)
    used = c.args[1].shape[0]
    for i in (1, 2):
        big = torch.empty(n_pages, nkv, 64, hd, dtype=BF16, device=DEV)
        big[n_pages - used:].copy_(c.args[i])
        c.args[i] = big
    c.args[3] = c.args[3] + (n_pages - used)
    assert big.numel() > 2 ** 31
    c.check(ops)


# ---- the confirmed path ---------------------------------------------------------------------------

def draft(r, n, vocab):
    parents = tree(r, n)
    return parents, [r.randrange(vocab) for _ in range(n)]


def run_accept(ops, trees, logits=None, picked=None, extra=0, scratch=None):
    b = len(trees)
    cu = [sum(len(t[0]) for t in trees[:i]) for i in range(b + 1)]
    n = cu[-1] + extra
    tokens, parents = ints([x for t in trees for x in t[1]] + [0] * extra), ints([x for t in trees for x in t[0]] + [-1] * extra)
    path = torch.full((b, 64), 99, dtype=torch.int32, device=DEV)
    count, nxt = torch.full((b,), 99, dtype=torch.int32, device=DEV), torch.full((b,), 99, dtype=torch.int32, device=DEV)
    if logits is not None:
        scratch = torch.zeros(ops.tree_accept_scratch(n, b), dtype=torch.int64, device=DEV) if scratch is None else scratch
        for _ in range(2):                                         # the scratch is left as it was found
            ops.tree_accept(tokens, parents, ints(cu), path, count, nxt, logits=logits, scratch=scratch)
        assert not scratch.any()
    else:
        ops.tree_accept(tokens, parents, ints(cu), path, count, nxt, picked=picked)
    return path.tolist(), count.tolist(), nxt.tolist(), cu


def check_accept(trees, cu, best, path, count, nxt):
    longest = 0
    for b, (parents, tokens) in enumerate(trees):
        want, last = T.walk(tokens, parents, best[cu[b]:cu[b + 1]])
        assert (count[b], nxt[b]) == (len(want), last)
        assert path[b] == want + [-1] * (64 - len(want))
        longest = max(longest, len(want))
    return longest


@pytest.mark.parametrize("vocab", [7, 1003, 32000, 128256])
@pytest.mark.parametrize("sizes", [[1], [64], [16], [5, 0, 64, 1, 33, 32, 31], [0, 3]], ids=lambda s: "_".join(map(str, s)))
def test_the_path_that_logits_confirm(ops, vocab, sizes):
    r = random.Random(vocab + sum(sizes))
    trees = [draft(r, n, vocab) if n else ([], []) for n in sizes]
    n = sum(sizes)
    logits = normal(n + 2, vocab, seed=vocab, scale=2.0)
    base = 0
    for parents, tokens in trees:
        for i in range(len(parents)):
            children = [j for j, p in enumerate(parents) if p == i]
            if children and r.random() < 0.9:
                logits[base + i, tokens[r.choice(children)]] = 20.0
        base += len(parents)
    best = logits.argmax(-1).tolist()
    path, count, nxt, cu = run_accept(ops, trees, logits=logits.to(DEV), extra=2)
    longest = check_accept(trees, cu, best, path, count, nxt)
    assert longest > 1 or max(sizes) < 4
    picked = ints(best)
    check_accept(trees, cu, best, *run_accept(ops, trees, picked=picked, extra=2)[:3])


def test_equal_logits_go_to_the_lowest_token_and_equal_children_to_the_first(ops):
    vocab = 50000
    for places in ([0, 49999], [40000, 41], [1, 2, 3], [8191, 8192], [20000, 20001]):
        logits = torch.full((3, vocab), -1.5)
        logits[:, places] = 3.0
        low = min(places)
        trees = [([-1, 0, 0], [5, low, low])]
        path, count, nxt, _ = run_accept(ops, trees, logits=logits.to(DEV))
        assert path[0][:3] == [0, 1, -1] and count == [2] and nxt == [low]
    zeros = torch.zeros(1, 20000)
    zeros[0, ::2] = -0.0                                            # minus zero is zero
    assert run_accept(ops, [([-1], [5])], logits=zeros.to(DEV))[2] == [0]


def test_logits_that_are_no_numbers(ops):
    nan, inf = float("nan"), float("inf")
    logits = torch.full((4, 30011), -inf)
    logits[1] = nan
    logits[2, 7] = nan
    logits[2, 29000] = -4.0
    logits[3, 9] = inf
    logits[3, 3] = nan
    trees = [([-1], [1])] * 4
    assert run_accept(ops, trees, logits=logits.to(DEV))[2] == [0, 0, 29000, 9]


def test_a_chain_of_64_is_confirmed_whole_and_a_view_of_logits_is_taken(ops):
    vocab = 1000
    tokens = [(7 * i) % vocab for i in range(64)]
    wide = torch.zeros(65, vocab + 1, device=DEV)
    logits = wide.view(-1)[1:1 + 64 * vocab].view(64, vocab)          # does not start on 16 bytes
    for i in range(64):
        logits[i, tokens[i + 1] if i < 63 else 321] = 1.0
    path, count, nxt, _ = run_accept(ops, [([-1] + list(range(63)), tokens)], logits=logits)
    assert path[0] == list(range(64)) and count == [64] and nxt == [321]


# ---- what queries give each key -------------------------------------------------------------------

@pytest.mark.parametrize("dtype,nh,nkv,hd", [(F32, 4, 2, 16), (F32, 5, 1, 48), (F32, 6, 3, 30), (F32, 2, 1, 384), (BF16, 8, 2, 64), (BF16, 8, 1, 128),
                                             (BF16, 5, 1, 128), (BF16, 6, 3, 80), (BF16, 12, 4, 20), (BF16, 3, 3, 48), (BF16, 20, 1, 64)],
                         ids=lambda x: str(x).replace("torch.", ""))
@pytest.mark.parametrize("before,brings,last", [([0], [1], 1), ([63, 64, 65, 700], [1, 1, 1, 1], 1), ([0, 130], [90, 3], 32), ([5, 0, 64], [1, 200, 64], 8),
                                                ([100, 20], [0, 4], 4)],
                         ids=["first", "decode", "prompt", "mixed", "empty"])
def test_weights_of_keys(ops, dtype, nh, nkv, hd, before, brings, last):
    r = random.Random(hd)
    b, extra = len(before), 2
    totals = [x + y for x, y in zip(before, brings)]
    width, pages = max(totals) + 5, -(-max(totals) // 64)
    slots = r.sample(range(b + 2), b)
    k = [normal(t, nkv, hd, seed=7 + i).to(dtype) for i, t in enumerate(totals)]
    (kp,), table = T.pages_of([[x] for x in k], nkv, (hd,), dtype, pages, b + 2, slots, hd, device=DEV)
    cu = [sum(brings[:i]) for i in range(b + 1)]
    q = normal(cu[-1] + extra, nh, hd, seed=hd, scale=2.0).to(dtype)
    held = normal(b + 2, nkv, width, seed=1).abs() * 0.02
    for i, s in enumerate(slots):
        held[s, :, before[i]:] = float("nan")                          # what lies behind the cached keys is not added to
    weights = held.to(DEV)
    plan = ops.key_weights_plan(dtype, b, last, nh, nkv, hd, max(totals))
    scratch = torch.full((plan.scratch_floats,), float("nan"), device=DEV)
    counters = torch.zeros(plan.n_counters, dtype=torch.int32, device=DEV)

    def go():
        ops.key_weights(q.to(DEV), kp, table, ints(slots), ints(cu), ints(before), weights, scratch, scale=hd ** -0.5, last=last, plan=plan,
                        counters=counters)
    go()
    assert not counters.any()
    got = weights.cpu()
    for i, s in enumerate(slots):
        if brings[i] == 0:
            assert torch.equal(got[s].nan_to_num(9.0), held[s].nan_to_num(9.0))
            continue
        want, slack = T.key_weights(q[cu[i]:cu[i + 1]], k[i], before[i], last, hd ** -0.5, held[s])
        t = totals[i]
        assert ((got[s, :, :t].double() - want[:, :t]).abs() <= slack[:, :t] + 1e-9).all()
        assert torch.isnan(got[s, :, t:]).all()
    for s in set(range(b + 2)) - set(slots):
        assert torch.equal(got[s], held[s])
    once = weights.clone()
    weights.copy_(held)
    go()
    assert torch.equal(once.nan_to_num(9.0), weights.nan_to_num(9.0))    # sums run in one order


@pytest.mark.parametrize("hd", [64, 128, 40])
def test_bfloat16_weights_on_the_cuda_cores(ops, hd, monkeypatch):
    monkeypatch.setattr(ops, "USE_MMA_WEIGHTS", False)
    test_weights_of_keys(ops, BF16, 8, 2, hd, [5, 0, 64], [1, 200, 64], 8)


@pytest.mark.parametrize("keep", [True, False], ids=["kept", "twice"])
@pytest.mark.parametrize("dtype,nh,nkv,hd,last", [(F32, 8, 2, 64, 40), (F32, 5, 1, 80, 20), (F32, 3, 3, 200, 9), (BF16, 8, 2, 20, 33), (F32, 8, 1, 128, 1)], ids=str)
def test_weights_of_many_queries_on_the_cuda_cores(ops, dtype, nh, nkv, hd, last, keep, monkeypatch):
    """Scores kept between the passes, and worked out twice; several row blocks, row ends worked out in several goes."""
    monkeypatch.setattr(ops, "USE_MMA_WEIGHTS", False)
    monkeypatch.setattr(ops, "KEY_SCORE_FLOATS", 1 << 24 if keep else 0)
    test_weights_of_keys(ops, dtype, nh, nkv, hd, [300, 0, 127], [1, 230, 41], last)


@pytest.mark.parametrize("hd", [64, 128])
def test_weights_of_many_queries_on_mma_sync(ops, hd, monkeypatch):
    monkeypatch.setattr(ops, "USE_TC_WEIGHTS", False)
    test_weights_of_keys(ops, BF16, 8, 2, hd, [5, 0, 64], [1, 200, 64], 20)


@pytest.mark.parametrize("nh,nkv,hd,last", [(8, 2, 128, 64), (5, 1, 64, 40), (40, 8, 128, 9), (33, 1, 64, 1), (128, 1, 128, 2)], ids=str)
def test_weights_of_many_queries(ops, nh, nkv, hd, last):
    """More rows than one row block of 128, splits of several pairs of pages that end in a page, in one key and in a whole pair."""
    test_weights_of_keys(ops, BF16, nh, nkv, hd, [700, 0, 1023, 320], [1, 1153, 1, 64], last)


@pytest.mark.parametrize("dtype,hd,last,keep", [(BF16, 64, 30, True), (BF16, 128, 6, True), (BF16, 80, 30, True), (F32, 64, 30, True), (F32, 64, 30, False),
                                                (BF16, 20, 4, True)], ids=str)
def test_a_query_that_is_no_number_shows_in_the_keys_it_sees(ops, dtype, hd, last, keep, monkeypatch):
    """The rows of one head of one query hold NaN, the pages NaN behind the sequence: its keys' entries show it, later keys' and other heads' do not."""
    monkeypatch.setattr(ops, "KEY_SCORE_FLOATS", 1 << 24 if keep else 0)
    nh, nkv, before, count = 4, 2, 100, 40
    total, bad = before + count, count - 3
    k = normal(total, nkv, hd, seed=3).to(dtype)
    (kp,), table = T.pages_of([[k]], nkv, (hd,), dtype, 4, 2, [1], hd, device=DEV)
    q = normal(count, nh, hd, seed=5).to(dtype)
    q[bad, 1] = float("nan")
    plan = ops.key_weights_plan(dtype, 1, last, nh, nkv, hd, total)
    weights = torch.zeros(2, nkv, 200, device=DEV)
    ops.key_weights(q.to(DEV), kp, table, ints([1]), ints([0, count]), ints([before]), weights, torch.empty(plan.scratch_floats, device=DEV),
                    scale=hd ** -0.5, last=last, plan=plan, counters=torch.zeros(plan.n_counters, dtype=torch.int32, device=DEV))
    got = weights[1].cpu()
    assert torch.isnan(got[0, :before + bad + 1]).all()
    clean = q.clone()
    clean[bad, 1] = 0
    want, slack = T.key_weights(clean, k, before, last, hd ** -0.5, torch.zeros(nkv, 200))
    late = slice(before + bad + 1, total)
    assert ((got[0, late].double() - want[0, late]).abs() <= slack[0, late] + 1e-9).all()
    assert ((got[1].double() - want[1]).abs() <= slack[1] + 1e-9).all()


def test_weights_of_long_sequences_in_a_graph(ops):
    """Thousands of keys: many blocks' sums are joined; every query's shares add up to one."""
    nh, nkv, hd, before = 8, 2, 128, [3900, 100]
    pages = 64
    kp = torch.randn(2 * pages + 1, nkv, 64, hd, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(BF16)
    table = torch.arange(2 * pages, dtype=torch.int32, device=DEV).view(2, pages)
    for last, brings in ((1, [1, 1]), (32, [100, 40])):
        q = normal(sum(brings), nh, hd, seed=4, scale=2.0).to(BF16).to(DEV)
        plan = ops.key_weights_plan(BF16, 2, last, nh, nkv, hd, 4096)
        scratch, counters = torch.empty(plan.scratch_floats, device=DEV), torch.zeros(plan.n_counters, dtype=torch.int32, device=DEV)
        weights = torch.zeros(2, nkv, 4096, device=DEV)
        args = [q, kp, table, ints([1, 0]), ints([0, brings[0], sum(brings)]), ints(before)]
        ops.key_weights(*args, weights, scratch, scale=hd ** -0.5, last=last, plan=plan, counters=counters)
        rows = nh // nkv * last
        # a share is off by at most 2 e, e below (hd + 3) 2^-23 * 32 + L 2^-23 for these scores
        assert ((weights.double().sum(-1) - rows).abs() <= rows * 2 * (131 * 32 + 4096) * 2.0 ** -23).all()
        graph = torch.cuda.CUDAGraph()
        again = torch.zeros_like(weights)
        with torch.cuda.graph(graph):
            ops.key_weights(*args, again, scratch, scale=hd ** -0.5, last=last, plan=plan, counters=counters)
        graph.replay()
        assert torch.equal(again, weights)
        for i, (slot, lb) in enumerate(((1, before[0]), (0, before[1]))):
            k = kp[table[slot].long()].transpose(0, 1).reshape(nkv, -1, hd).transpose(0, 1)[:lb + brings[i]]
            c0 = sum(brings[:i])
            want, slack = T.key_weights(q[c0:c0 + brings[i]].cpu(), k.cpu(), lb, last, hd ** -0.5, torch.zeros(nkv, 4096))
            assert ((weights[slot].cpu().double() - want).abs() <= slack + 1e-9).all()


# ---- which keys stay ------------------------------------------------------------------------------

@pytest.mark.parametrize("lengths,keeps,first,recent,bound", [
    ([1], [1], 0, 0, None), ([5, 64], [5, 1], 0, 0, None), ([700, 33, 512], [100, 20, 511], 4, 16, None), ([2048, 2000], [17, 1999], 0, 3, None),
    ([9000, 100], [2000, 99], 4, 64, None), ([9000, 100], [2000, 99], 4, 64, 9000), ([300], [20], 15, 10, None), ([300], [20], 30, 0, None),
    ([17000], [3333], 4, 100, None), ([40], [40], 100, 100, None), ([513, 511], [300, 300], 0, 0, 513)],
    ids=lambda x: "_".join(map(str, x)) if isinstance(x, list) else str(x))
def test_keys_of_most_weight(ops, lengths, keeps, first, recent, bound):
    r = random.Random(sum(lengths))
    b, layers, nkv = len(lengths), 2, 3
    width, most = max(lengths) + (7 if bound is None else 12000), max(keeps) + 2
    w = normal(layers, b + 2, nkv, width, seed=2).abs()
    w[0] = (w[0] * 3).round() / 3                                   # many equal ones
    w[1, :, 0] = -w[1, :, 0]
    w[1, :, 1, ::3] = 0.0
    w[1, :, 1, 1::9] = -0.0
    slots = r.sample(range(b + 2), b)
    chosen = torch.full((layers, b, nkv, most), -7, dtype=torch.int32, device=DEV)
    ops.keep_keys(w.to(DEV), ints(slots), ints(lengths), ints(keeps), chosen, first=first, recent=recent, max_len=bound)
    got = chosen.tolist()
    for layer in range(layers):
        for i, s in enumerate(slots):
            for h in range(nkv):
                want = T.keep(w[layer, s, h], lengths[i], keeps[i], first, recent)
                assert got[layer][i][h] == want + [-7] * (most - len(want)), (layer, i, h)


def test_weights_that_are_no_numbers_stay_last(ops):
    nan, inf = float("nan"), float("inf")
    w = torch.tensor([nan, 1.0, -inf, nan, inf, 0.5, -2.0, nan]).view(1, 1, 1, 8)
    for keep in range(1, 9):
        chosen = torch.full((1, 1, 1, 8), -7, dtype=torch.int32, device=DEV)
        ops.keep_keys(w.to(DEV), ints([0]), ints([8]), ints([keep]), chosen, first=0, recent=0)
        order = [4, 1, 5, 6, 2, 0, 3, 7]
        assert chosen[0, 0, 0].tolist() == sorted(order[:keep]) + [-7] * (8 - keep)


# ---- rows to new places ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,nkv,hd,vd", [(F32, 2, 16, 16), (BF16, 3, 64, 64), (BF16, 8, 128, 128), (BF16, 1, 80, 48), (F32, 2, 6, 10), (BF16, 2, 7, 3), (F32, 1, 384, 0)],
                         ids=lambda x: str(x).replace("torch.", ""))
@pytest.mark.parametrize("per_layer,per_head", [(True, True), (False, False), (True, False), (False, True)])
def test_rows_that_stay_come_together(ops, dtype, nkv, hd, vd, per_layer, per_head):
    r = random.Random(hd + nkv)
    layers, lengths, base = 3, [700, 64, 130, 5], [0, 3, 60, 4]
    b, pages, n_slots = len(lengths), 12, 6
    slots = r.sample(range(n_slots), b)
    n_pages = b * pages + 1
    table = torch.full((n_slots, pages), n_pages - 1, dtype=torch.int32)
    order = r.sample(range(n_pages - 1), b * pages)
    for i, s in enumerate(slots):
        table[s] = torch.tensor(order[i * pages:(i + 1) * pages])
    pools = [[normal(n_pages, nkv, 64, d, seed=layer * 2 + j).to(dtype) for layer in range(layers)] for j, d in enumerate((hd, vd)) if d]
    weights = normal(layers, n_slots, nkv, 750, seed=9)
    counts = [r.randint(0, n - s) for n, s in zip(lengths, base)]
    counts[0] = 600
    width = max(counts)
    source = torch.zeros(layers if per_layer else 1, b, nkv if per_head else 1, width, dtype=torch.int32)
    for layer in range(source.shape[0]):
        for i in range(b):
            for h in range(source.shape[2]):
                pick = sorted(r.sample(range(lengths[i] - base[i]), counts[i]))
                source[layer, i, h, :counts[i]] = torch.tensor(pick, dtype=torch.int32)
    dev = [[p.to(DEV) for p in ps] for ps in pools]
    w = weights.to(DEV)
    rows = ops.CacheRows(dev[0], dev[1] if vd else None, weights=w)
    rows.move(table.to(DEV), pages, ints(slots), ints(base), source.to(DEV), ints(counts))
    for j, ps in enumerate(pools):
        for layer in range(layers):
            want = ps[layer].clone()
            for i, s in enumerate(slots):
                for h in range(nkv):
                    for n in range(counts[i]):
                        src = base[i] + int(source[layer if per_layer else 0, i, h if per_head else 0, n])
                        dst = base[i] + n
                        want[table[s, dst // 64], h, dst % 64] = ps[layer][table[s, src // 64], h, src % 64]
            assert torch.equal(dev[j][layer].cpu(), want), (j, layer)
    want = weights.clone()
    for layer in range(layers):
        for i, s in enumerate(slots):
            for h in range(nkv):
                for n in range(counts[i]):
                    want[layer, s, h, base[i] + n] = weights[layer, s, h, base[i] + int(source[layer if per_layer else 0, i, h if per_head else 0, n])]
    assert torch.equal(w.cpu(), want)


def test_rows_move_within_a_ring_and_in_a_graph(ops):
    ring, base = 3, 185                                             # positions 185 .. 230 lie over the ring's end
    pool = normal(4, 2, 64, 64, seed=3).to(BF16)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    source = torch.tensor([0, 3, 4, 9, 40], dtype=torch.int32).view(1, 1, 1, 5)
    dev, values = pool.to(DEV), pool.neg().to(DEV)
    rows = ops.CacheRows([dev], [values])
    args = (table.to(DEV), ring, ints([0]), ints([base]), source.to(DEV), ints([5]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows.move(*args)
    assert torch.equal(dev.cpu(), pool)                              # recorded, not run
    graph.replay()
    want = pool.clone()
    for j, s in enumerate(source.view(-1).tolist()):
        src, dst = base + s, base + j
        want[table[0, dst // 64 % ring], :, dst % 64] = pool[table[0, src // 64 % ring], :, src % 64]
    assert torch.equal(dev.cpu(), want) and torch.equal(values.cpu(), want.neg())


def test_no_wait_for_keys_has_run_out(ops):
    """Behind the tests above."""
    assert ops.key_weights_status() == 0 and ops.attn_tree_status() == 0
