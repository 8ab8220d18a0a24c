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
