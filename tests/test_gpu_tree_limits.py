"""Drafted trees and weighed keys on the GPU at the ends of what plans take: layers that differ, scores that outgrow a workspace, lists of work that
outgrow a launch's counts, many sequences."""
import importlib

import pytest
import torch

import tree_models as M

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("daisi-llogos_b200.kernels.ops")


@pytest.mark.parametrize("dtype,tol", [(F32, 2e-5), (BF16, 4e-2)], ids=["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[64, 32], [32, 64]], ids=str)
def test_layers_of_two_value_sizes_are_weighed(llogos, ops, dtype, tol, sizes):
    """An engine that weighs its keys gives the logits of one that does not: before an eviction both look at the same keys.  (How close: as in
    ``test_gpu_tree_engine.py``, relative to the largest logit.)"""
    model = M.two_value_sizes(M.CFG, sizes, dtype=dtype, device="cuda:0", ops=ops)
    plain = llogos.engine.Engine(model, max_tokens=64 * 8)
    weighed = llogos.engine.Engine(model, max_tokens=64 * 8, weigh_keys=4)
    steps = [[[5] * 70, [3, 9, 1]]] + [[[7 + i], [11 + i]] for i in range(4)]
    got = []
    for eng in (plain, weighed):
        slots = [eng.open(), eng.open()]
        got.append([eng.step(list(zip(slots, toks))).cpu().double() for toks in steps])
    for a, b in zip(*got):
        assert float((a - b).abs().max()) <= tol * float(a.abs().max())
    weighed.evict([(0, 40)], first=2, recent=8)
    assert torch.isfinite(weighed.step([(0, [5]), (1, [6])])).all()


def shared_pages(n_seqs, nkv, hd, before, width):
    """A few pages that all sequences read, and a table as wide as the longest sequence that a plan allows for."""
    g = torch.Generator().manual_seed(hd + n_seqs)
    k, v = (torch.randn(5, nkv, 64, hd, generator=g).to(BF16) for _ in range(2))
    table = torch.zeros(n_seqs, width, dtype=torch.int32)
    table[:, :2] = torch.tensor([[i % 5, (i * 3 + 1) % 5] for i in range(n_seqs)], dtype=torch.int32)
    return k, v, table, [before[i % len(before)] for i in range(n_seqs)]


@pytest.mark.parametrize("kind,n_seqs,nkv,group,hd,max_len", [("tc", 256, 8, 8, 128, 131072), ("mma", 1024, 32, 2, 64, 1 << 20), ("simt", 1024, 32, 8, 64, 1 << 20)])
def test_plans_for_long_sequences_of_many_fall_through_to_a_kernel_that_takes_them(ops, kind, n_seqs, nkv, group, hd, max_len):
    """Sequences that may be long and are not, as an engine's bound for one long chat in a batch makes them: the plan is for what may be."""
    import tree_plain as T
    nh = nkv * group
    k, v, table, before = shared_pages(n_seqs, nkv, hd, [5, 100, 64, 0], max_len // 64)
    q = torch.randn(n_seqs, nh, hd, generator=torch.Generator().manual_seed(3)).to(BF16)
    plan = ops.attn_tree_plan(BF16, n_seqs, 64, nh, nkv, hd, max_len)
    assert plan.kind == kind

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda:0")
    out = torch.full((n_seqs, nh * hd), 7.0, dtype=BF16, device="cuda:0")
    ops.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), max_len // 64, ints(list(range(n_seqs))), ints(list(range(n_seqs + 1))), ints(before),
                  torch.ones(n_seqs, dtype=torch.int64, device="cuda:0"), out, torch.empty(max(1, plan.scratch_floats), device="cuda:0"), scale=hd ** -0.5,
                  plan=plan, counters=torch.zeros(max(1, plan.n_counters), dtype=torch.int32, device="cuda:0"))
    got = out.cpu().double().view(n_seqs, nh, hd)
    assert torch.isfinite(got).all() and not (got == 7.0).all(-1).any()
    for i in (0, 1, 2, 3, 129, n_seqs // 2 + 1, n_seqs - 2, n_seqs - 1):
        pages = table[i, :2].long()
        rows = [x[pages].transpose(0, 1).reshape(nkv, 128, hd).transpose(0, 1)[:before[i] + 1] for x in (k, v)]
        want, slack = T.attend(q[i:i + 1], *rows, [list(range(before[i] + 1))], hd ** -0.5, BF16)
        assert ((got[i] - want[0]).abs() <= slack[0] + 1e-7).all()
    assert ops.attn_tree_status() == 0


@pytest.mark.parametrize("n_seqs", [130, 200, 500, 1024])
@pytest.mark.parametrize("rows", [{}, {64: 0}], ids=["mma", "tc"])
def test_batches_of_many_sequences(ops, n_seqs, rows, monkeypatch):
    """More sequences than a block stages or has threads: each works out the list's sums over several of them."""
    import test_gpu_trees as G
    monkeypatch.setattr(ops, "TREE_MMA_ROWS", rows or {64: 1 << 30})
    before = [(i * 37) % 150 for i in range(n_seqs)]
    nodes = [(i * 5) % 4 for i in range(n_seqs)]
    G.Case(BF16, 4, 2, 64, before, nodes, seed=n_seqs).check(ops)


FEW = [(8, 2, 64, 4), (8, 2, 128, 1), (8, 1, 128, 2), (5, 1, 80, 3), (12, 4, 24, 5)]
MORE = [(8, 2, 64, 8), (8, 2, 128, 5), (5, 1, 80, 6), (12, 4, 24, 10), (4, 4, 64, 17)]


@pytest.mark.parametrize("nh,nkv,hd,last,kept", [(*h, kept) for kept in (0, 3, 1) for h in FEW] + [(*h, kept) for kept in (0, 1) for h in MORE], ids=str)
def test_weights_of_few_rows_with_a_bound_on_the_scores(ops, nh, nkv, hd, last, kept, monkeypatch):
    """Up to 32 rows on mma.sync where the batch's scores are more than may be kept: worked out twice, or a few sequences at a time."""
    import test_gpu_trees as G
    before, brings = [300, 0, 127, 64, 1, 500, 9], [1, 230, 41, 1, 0, 3, 20]
    max_len = max(x + y for x, y in zip(before, brings))
    rows = nh // nkv * last
    monkeypatch.setattr(ops, "KEY_SCORE_FLOATS", kept * nkv * rows * (-(-max_len // 256) * 256))
    plan = ops.key_weights_plan(BF16, len(before), last, nh, nkv, hd, max_len)
    assert plan.kind == "mma" and (bool(plan.scores), plan.together) == ((True, {3: 3, 1: 1}[kept]) if kept and rows <= ops.KEY_GOES_ROWS else (False, 7))
    G.test_weights_of_keys(ops, BF16, nh, nkv, hd, before, brings, last)
    assert ops.key_weights_status() == 0


@pytest.mark.parametrize("kept", [0, 2], ids=["twice", "some"])
def test_weights_with_a_bound_on_the_scores_in_a_graph(ops, kept, monkeypatch):
    """Recorded and replayed over other keys: the goes of a call follow one another on its scratch."""
    nh, nkv, hd, last, b = 8, 2, 64, 4, 5
    monkeypatch.setattr(ops, "KEY_SCORE_FLOATS", kept * nkv * 16 * 1024)
    plan = ops.key_weights_plan(BF16, b, last, nh, nkv, hd, 1000)
    assert bool(plan.scores) == (kept > 0)
    g = torch.Generator("cuda:0").manual_seed(1)
    kp = torch.randn(b * 16, nkv, 64, hd, device="cuda:0", generator=g).to(BF16)
    q = torch.randn(b * last, nh, hd, device="cuda:0", generator=g).to(BF16)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda:0")
    args = [q, kp, torch.arange(b * 16, dtype=torch.int32, device="cuda:0").view(b, 16), ints([4, 2, 0, 1, 3]), ints([last * i for i in range(b + 1)]),
            ints([900, 20, 0, 64, 700])]
    scratch, counters = torch.empty(plan.scratch_floats, device="cuda:0"), torch.zeros(1, dtype=torch.int32, device="cuda:0")
    weights = [torch.zeros(b, nkv, 1000, device="cuda:0") for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    kw = dict(scale=hd ** -0.5, last=last, plan=plan, counters=counters)
    ops.key_weights(*args, weights[0], scratch, **kw)
    with torch.cuda.graph(graph):
        ops.key_weights(*args, weights[1], scratch, **kw)
    graph.replay()
    assert torch.equal(*weights)
    kp.copy_(torch.randn(kp.shape, device="cuda:0", generator=g))
    for w in weights:
        w.zero_()
    graph.replay()
    ops.key_weights(*args, weights[0], scratch, **kw)
    assert torch.equal(*weights)
    rows = nh // nkv * last
    assert ((weights[0].double().sum(-1) - rows).abs() <= rows * 2 * (67 * 32 + 1000) * 2.0 ** -23).all()      # (as in the test of long sequences)


@pytest.mark.parametrize("dtype,nh,hd", [(F32, 4, 64), (BF16, 4, 64), (BF16, 4, 20), (BF16, 16, 64), (BF16, 32, 128)], ids=["f32", "mma", "simt", "tc64", "tc128"])
@pytest.mark.parametrize("window", [40, 64, 100, 200])
def test_a_nodes_depth_is_its_bits_however_few_nodes_there_are(ops, dtype, nh, hd, window):
    """Words with more bits than the tree has nodes: they are no nodes' and show nothing, and they count for the depth that a window goes by."""
    import test_gpu_trees as G
    bits = [[1, 3 | ((1 << 50) - 1) << 5, 5, (1 << 64) - 1, 9, (1 << 40) - 1], [1, 3 | 1 << 60, (1 << 63) - 1, 2, 1 << 63]]
    G.Case(dtype, nh, 2, hd, [330, 205], [6, 5], bits=bits, window=window, seed=window).check(ops)
    G.Case(dtype, nh, 2, hd, [70, 0], [6, 5], bits=bits, window=window, seed=window + 1).check(ops)


@pytest.mark.parametrize("dtype,nh,hd", [(F32, 4, 64), (BF16, 4, 64), (BF16, 4, 20), (BF16, 16, 64), (BF16, 32, 128)], ids=["f32", "mma", "simt", "tc64", "tc128"])
def test_a_window_ends_between_a_node_and_one_without_bits(ops, dtype, nh, hd):
    """A node that sees nothing, itself included, stands one place before the tree's first: a node whose depth is the window less one is a window behind it."""
    import test_gpu_trees as G
    for window in (1, 2, 3, 5, 8):
        bits = [[0, 0b10, 0b11, 0b111, 0b1111, 0b11111, 0b111111, 0b1111111, 0b11111111, 0b1], [1, 0, 0b111, 0b1111, 2]]
        G.Case(dtype, nh, 2, hd, [200, 0], [10, 5], bits=bits, window=window, seed=window).check(ops)


def test_calls_on_two_streams_at_once_give_what_they_give_alone(ops):
    """Every kernel beside every other, each with a scratch of its own; no block of one waits for another's."""
    import test_gpu_trees as G

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda:0")
    jobs = []
    for dtype, nh, hd, nodes in ((BF16, 16, 128, 64), (BF16, 8, 64, 4), (F32, 8, 64, 9), (BF16, 8, 64, 40)):
        c = G.Case(dtype, nh, 2, hd, [900, 33, 257], [nodes, 1, nodes // 2], seed=nodes)
        out, go = c.call(ops)
        jobs.append((go, out, out.clone()))
    for dtype, hd, last in ((BF16, 128, 40), (BF16, 64, 4), (F32, 64, 3)):
        nh, nkv, before, brings = 8, 2, [900, 60], [50, 45]
        kp = torch.randn(32, nkv, 64, hd, device="cuda:0", generator=torch.Generator("cuda:0").manual_seed(last)).to(dtype)
        q = torch.randn(95, nh, hd, device="cuda:0", generator=torch.Generator("cuda:0").manual_seed(hd)).to(dtype)
        plan = ops.key_weights_plan(dtype, 2, last, nh, nkv, hd, 1000)
        scratch, counters, weights = torch.empty(plan.scratch_floats, device="cuda:0"), ints([0]), torch.zeros(2, nkv, 1000, device="cuda:0")
        args = (q, kp, torch.arange(32, dtype=torch.int32, device="cuda:0").view(2, 16), ints([1, 0]), ints([0, 50, 95]), ints(before), weights, scratch)

        def go(args=args, hd=hd, last=last, plan=plan, counters=counters, weights=weights):
            weights.zero_()
            ops.key_weights(*args, scale=hd ** -0.5, last=last, plan=plan, counters=counters)
        go()
        jobs.append((go, weights, weights.clone()))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(len(jobs)):
        for j in range(len(jobs)):
            if i == j:
                continue
            for _ in range(3):
                for stream, (go, _, _) in zip(streams, (jobs[i], jobs[j])):
                    with torch.cuda.stream(stream):
                        go()
            torch.cuda.synchronize()
            assert torch.equal(jobs[i][1], jobs[i][2]) and torch.equal(jobs[j][1], jobs[j][2]), (i, j)
    assert ops.attn_tree_status() == 0 and ops.key_weights_status() == 0
