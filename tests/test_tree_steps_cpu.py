"""Steps over drafted trees and weighed keys: what a step's host logic keeps, gives back and forgets, on CPU tensors with stand-ins for the kernels."""
import pytest
import torch

import tree_models as M
import tree_ops


def engine_for(llogos, model, **kw):
    kw.setdefault("max_tokens", 64 * 14)
    return llogos.engine.Engine(model, use_graphs=False, **kw)


def test_layers_of_two_value_sizes_have_a_decode_plan_each(llogos, monkeypatch):
    """The sizes that a plan is asked for by are the same for both layers; the values' size comes with the attention's form."""
    class Plan:
        scratch_floats, n_counters = 1, 0

        def __init__(self, vd):
            self.vd = vd

    def plan(dtype, n_seqs, n_heads, n_kv_heads, head_dim, max_len, form=tree_ops.PLAIN_ATTENTION):
        return Plan(form.vd(head_dim))

    attend, seen = tree_ops.attn_decode, []

    def decode(*args, plan, form=tree_ops.PLAIN_ATTENTION, **kw):
        seen.append((plan.vd, form.vd(args[0].shape[2])))
        attend(*args, plan=plan, form=form, **kw)

    monkeypatch.setattr(tree_ops, "attn_decode_plan", plan)
    monkeypatch.setattr(tree_ops, "attn_decode", decode)
    model = M.two_value_sizes(M.CFG, [64, 32], dtype=torch.float32, device="cpu", ops=tree_ops)
    eng = engine_for(llogos, model, weigh_keys=2)
    slot = eng.open()
    eng.step([(slot, [1, 2, 3])])
    eng.step([(slot, [4])])
    assert seen == [(64, 64), (32, 32)]


class Failure(Exception):
    pass


def table_is_the_hosts(eng):
    """Every page that a sequence has stands in the table that the kernels read."""
    for g in eng.cache.kv_groups:
        for slot, pages in g.pages_of.items():
            assert g.page_table[slot, :len(pages)].tolist() == pages
    eng.cache.audit()


@pytest.mark.parametrize("name", ["llama", "qwen3"])
@pytest.mark.parametrize("where", ["upload", "meta", "scatter", "forward"])
@pytest.mark.parametrize("kind", ["tree", "prompt", "decode", "assume"])
def test_a_step_that_fails_leaves_no_page_without_its_entry(llogos, model_dirs, monkeypatch, name, where, kind):
    """Pages that a step took and whose entries never reached the table went to the next step, which wrote through what stood there before: another
    sequence's page.  In rings too, whose pages a step of more tokens than they hold takes all at once."""
    if kind == "assume" and where == "forward":
        pytest.skip("nothing runs")
    model = llogos.weights.load_model(model_dirs[name], dtype=torch.float32, device="cpu", ops=tree_ops)
    eng = engine_for(llogos, model)
    other, slot = eng.open(), eng.open()
    eng.step([(other, [3] * 100), (slot, [1] * 64)], [[], []])
    free = [g.pool.free_count for g in eng.cache.kv_groups]
    act = {"tree": lambda: eng.step_tree([(slot, [1, 2, 3], [-1, 0, 0])]), "prompt": lambda: eng.step([(slot, [4] * 130)]),
           "decode": lambda: eng.step([(slot, [4])]), "assume": lambda: eng.assume(slot, 200)}[kind]

    def fails(*args, **kw):
        raise Failure

    with monkeypatch.context() as m:
        target = {"upload": (eng._staging, "upload"), "meta": (eng, "_ensure_meta"), "scatter": (tree_ops, "scatter_i32"),
                  "forward": (model, "forward")}[where]
        m.setattr(*target, fails)
        with pytest.raises(Failure):
            act()
    assert [g.pool.free_count for g in eng.cache.kv_groups] == free and eng.length(slot) == 64
    table_is_the_hosts(eng)
    act()
    table_is_the_hosts(eng)


@pytest.mark.parametrize("name", ["llama", "qwen3"])
def test_a_refused_call_forgets_no_tree(llogos, model_dirs, name):
    """Another step, truncate and close forget a tree that was not accepted; one that is refused changes nothing."""
    E = llogos.engine.StepError
    model = llogos.weights.load_model(model_dirs[name], dtype=torch.float32, device="cpu", ops=tree_ops)
    eng = engine_for(llogos, model, max_tokens=64 * 4, max_seq_len=64 * 4, n_slots=3)
    slot, other = eng.open(), eng.open()
    eng.step([(slot, [1] * 60), (other, [2] * 60)], [[], []])
    eng.step_tree([(slot, [1, 2, 3], [-1, 0, 1])])
    for call, error in ((lambda: eng.truncate(other, 61), E), (lambda: eng.truncate(2, 1), E),
                        (lambda: eng.close(2), RuntimeError), (lambda: eng.close(7), RuntimeError), (lambda: eng.step([(2, [1])]), E),
                        (lambda: eng.step([(slot, [1] * 300)]), E), (lambda: eng.step([(other, [1] * 190)]), E), (lambda: eng.assume(2, 5), E),
                        (lambda: eng.step_tree([(2, [1], [-1])]), E), (lambda: eng.step_tree([(slot, [1], [0])]), E),
                        (lambda: eng.step_tree([(slot, [1], [-1]), (slot, [1], [-1])]), E)):
        with pytest.raises(error):
            call()
        assert eng.trees.pending is not None and eng.length(slot) == 60
    best = torch.tensor([2, 3, 9], dtype=torch.int32)
    assert eng.accept_tree(best) == [([0, 1, 2], 9)] and eng.length(slot) == 63
    eng.cache.audit()


def test_a_forgotten_trees_pages_count_as_free(llogos, model_dirs):
    """The pages of a tree that a step will forget are there for that step: for its own sequence and for another."""
    model = llogos.weights.load_model(model_dirs["llama"], dtype=torch.float32, device="cpu", ops=tree_ops)
    for own in (True, False):
        eng = engine_for(llogos, model, max_tokens=64 * 3, max_seq_len=64 * 3, n_slots=2)
        slot, other = eng.open(), eng.open()
        eng.step([(slot, [1] * 60), (other, [2] * 60)], [[], []])
        eng.step_tree([(slot, [1] * 20, [-1] + [0] * 19)])
        assert eng.cache.free_pages() == 0
        eng.step([(slot if own else other, [1] * 20)])
        assert (eng.length(slot), eng.length(other)) == ((80, 60) if own else (60, 80))
        table_is_the_hosts(eng)


def test_a_truncation_to_a_negative_length_is_refused(llogos, model_dirs):
    model = llogos.weights.load_model(model_dirs["llama"], dtype=torch.float32, device="cpu", ops=tree_ops)
    eng = engine_for(llogos, model, weigh_keys=1)
    slot = eng.open()
    eng.step([(slot, [1] * 10)], [[]])
    for says in ("cannot truncate 10 tokens", "6 keys were left by an eviction"):
        with pytest.raises(llogos.engine.StepError, match=says):
            eng.truncate(slot, -1)
        eng.evict([(slot, 6)], first=1, recent=1) if eng.length(slot) == 10 else None
    assert eng.length(slot) == 6


def test_what_tree_steps_are_recorded_in_is_bounded_in_bytes(llogos, model_dirs, monkeypatch):
    """Sizes that come again have buffers of their own (their logits among them): the ones used longest ago make room, and sizes that are too
    large by themselves have none."""
    import importlib
    trees = importlib.import_module("daisi-llogos_b200.engine.trees")
    model = llogos.weights.load_model(model_dirs["llama"], dtype=torch.float32, device="cpu", ops=tree_ops)

    def twice(eng, slot, n):
        for _ in range(2):                                 # (the third of a size would be recorded on a GPU)
            eng.step_tree([(slot, [1] * n, [-1] + [0] * (n - 1))])
        return eng.trees._recorded

    def made(limit):
        monkeypatch.setattr(trees, "RECORDED_BYTES", limit)
        eng = engine_for(llogos, model)
        eng.use_graphs = True
        slot = eng.open()
        eng.step([(slot, [1, 2, 3])], [[]])
        return eng, slot

    eng, slot = made(1 << 40)
    for n in (4, 8, 9):
        kept = twice(eng, slot, n)
    size = {key[0][0]: rec.workspace.bytes() for key, rec in kept.items()}
    assert sorted(size) == [4, 8, 9] and size[4] >= 4 * 4 * 256        # logits of four nodes over 256 ids
    eng, slot = made(size[8] + size[9] + 1000)
    for n in (4, 8, 9):
        kept = twice(eng, slot, n)
        assert sum(r.workspace.bytes() for r in kept.values()) <= trees.RECORDED_BYTES
    assert [key[0] for key in kept] == [(8,), (9,)]
    eng, slot = made(size[8] - 1)
    assert [key[0] for key in twice(eng, slot, 4)] == [(4,)]
    for _ in range(2):
        assert [key[0] for key in twice(eng, slot, 8)] == [(4,)]       # too large by itself, and nobody makes room for it
    assert eng.accept_tree(torch.zeros(8, dtype=torch.int32)) == [([0], 0)]


MIXERS = {"value_blend": dict(changes=[dict(value_blend="g")] * 2), "value_dim": dict(changes=[dict(value_dim=32), dict(value_dim=24)]),
          "out_gate": dict(changes=[dict(out_gate=True)] * 2), "out_bias": dict(changes=[dict(out_bias=True), {}]),
          "window": dict(changes=[dict(window=20), {}]), "borrowed": dict(changes=[{}, dict(own_kv=False)], cache_of=((1, 0),)),
          "borrowed_window": dict(changes=[dict(window=20), dict(window=20, own_kv=False)], cache_of=((1, 0),))}


@pytest.mark.parametrize("name", list(MIXERS))
def test_a_chain_of_drafted_tokens_has_the_logits_of_a_prompts_step(llogos, name):
    """For every form of the attention that takes tree steps, twice as long as a page: a chain is what a step brings, and what is accepted of it is what
    the next step looks at."""
    model = M.with_mixers(M.CFG, **MIXERS[name], dtype=torch.float32, device="cpu", ops=tree_ops)
    eng = engine_for(llogos, model)
    toks = [(7 * i + i * i) % 256 for i in range(200)]
    trees, steps = eng.open(), eng.open()
    for slot in (trees, steps):
        eng.step([(slot, toks[:60])], [[]])
    at = 60
    for n in (9, 64, 30):
        part = toks[at:at + n]
        want = eng.step([(steps, part)], [list(range(n))]).clone()
        got = eng.step_tree([(trees, part, list(range(-1, n - 1)))]).clone()
        assert float((got - want).abs().max()) <= 2e-4 * float(want.abs().max())
        assert eng.accept_tree(torch.tensor(part[1:] + [5], dtype=torch.int32)) == [(list(range(n)), 5)]
        at += n
    want, got = (eng.step([(slot, [11])]).clone() for slot in (steps, trees))
    assert float((got - want).abs().max()) <= 2e-4 * float(want.abs().max())


@pytest.mark.parametrize("name", ["value_blend", "value_dim", "out_gate", "out_bias"])
def test_weighed_keys_leave_every_forms_logits(llogos, name):
    """An engine that weighs its keys, before an eviction, and one that does not."""
    model = M.with_mixers(M.CFG, **MIXERS[name], dtype=torch.float32, device="cpu", ops=tree_ops)
    engines = [engine_for(llogos, model), engine_for(llogos, model, weigh_keys=3)]
    slots = [e.open() for e in engines]
    for part in ([3] * 70, [5], [9, 8, 7], [2]):
        want, got = (e.step([(s, part)]).clone() for e, s in zip(engines, slots))
        assert float((got - want).abs().max()) <= 2e-4 * float(want.abs().max())


def test_a_view_of_keys_is_made_with_the_arguments_it_had(llogos):
    """What a mixer's own tests make by position: what is shared between the entries of a step is the ninth."""
    shared = {}
    view = llogos.cache.store.KvView(None, None, None, 1, 0, 3, True, False, shared)
    assert view.shared is shared and view.weights is None


def two_groups(llogos, **kw):
    """An engine whose layers keep their keys in two groups (values of two sizes)."""
    model = M.with_mixers(M.CFG, [dict(value_dim=32), dict(value_dim=24)], dtype=torch.float32, device="cpu", ops=tree_ops)
    eng = engine_for(llogos, model, **kw)
    assert len(eng.cache.kv_groups) == 2
    return eng


def fails_second(monkeypatch, target, name):
    """The second call of ``target.name`` fails, once."""
    real, calls = getattr(target, name), []

    def act(*args, **kw):
        calls.append(1)
        if len(calls) == 2:
            raise Failure
        return real(*args, **kw)
    monkeypatch.setattr(target, name, act)


@pytest.mark.parametrize("where", ["keep_keys", "CacheRows"])
def test_an_eviction_that_fails_has_moved_nothing(llogos, monkeypatch, where):
    """One group's keys at their new places and another's not would be an answer from keys that are not the tokens'."""
    eng = two_groups(llogos, weigh_keys=2)
    slot = eng.open()
    eng.step([(slot, [(5 * i) % 256 for i in range(90)])], [[]])
    before = [[t.clone() for t in (*g.k.values(), *g.v.values(), g.weights)] for g in eng.cache.kv_groups]
    with monkeypatch.context() as m:
        fails_second(m, tree_ops, where)
        with pytest.raises(Failure):
            eng.evict([(slot, 40)], first=2, recent=8)
    for g, old in zip(eng.cache.kv_groups, before):
        assert all(torch.equal(a, b) for a, b in zip((*g.k.values(), *g.v.values(), g.weights), old))
    assert eng.length(slot) == eng.position(slot) == 90
    eng.evict([(slot, 40)], first=2, recent=8)
    assert (eng.length(slot), eng.position(slot)) == (40, 90)


def test_an_acceptance_that_fails_can_be_made_again(llogos, monkeypatch):
    eng, other = two_groups(llogos), two_groups(llogos)
    parts = [3] * 70, ([1, 2, 3, 4], [-1, 0, 0, 2]), torch.tensor([3, 9, 4, 7], dtype=torch.int32)
    logits = []
    for e in (eng, other):
        slot = e.open()
        e.step([(slot, parts[0])], [[]])
        e.step_tree([(slot, *parts[1])])
        if e is eng:
            with monkeypatch.context() as m:
                fails_second(m, tree_ops, "CacheRows")
                with pytest.raises(Failure):
                    e.accept_tree(parts[2])
        assert e.accept_tree(parts[2]) == [([0, 2, 3], 7)]
        logits.append(e.step([(slot, [7])]).clone())
    assert torch.equal(*logits)
