"""Drafted trees and evictions through the engine's host logic, on CPU tensors with stand-ins for the kernels."""
import pytest
import torch

import tree_engine as E
import tree_ops
from conftest import TINY, TINY_LLAMA, read_weights


@pytest.fixture(scope="module")
def setup(llogos, model_dirs):
    return {name: (llogos.weights.load_model(model_dirs[name], dtype=torch.float32, device="cpu", ops=tree_ops),
                   read_weights(llogos, model_dirs[name]), model_dirs[name]) for name in TINY}


def engine_for(llogos, model, **kw):
    kw.setdefault("max_tokens", 64 * 14)
    return llogos.engine.Engine(model, use_graphs=False, **kw)


@pytest.mark.parametrize("name", list(TINY))
def test_trees_agree_with_plain(llogos, setup, name):
    model, w, key = setup[name]
    E.check_trees(engine_for(llogos, model), key, w, TINY[name], torch.float32, [70, 30], [9, 14], 2, 3)


def test_greedy_with_drafts_is_greedy(llogos, setup):
    model, w, _ = setup["llama"]
    E.check_greedy(engine_for(llogos, model), TINY["llama"], torch.float32, [[5, 6, 7], [9] * 20], 9, 4)


def test_trees_that_nobody_accepts(llogos, setup):
    for name in ("llama", "qwen3"):
        model, w, key = setup[name]
        E.check_forgotten(engine_for(llogos, model), llogos, key, w, TINY[name], torch.float32, 5)


def test_refusals(llogos, setup):
    model, _, _ = setup["llama"]
    E.check_refusals(engine_for(llogos, model), llogos, TINY["llama"])
    eng = engine_for(llogos, model, max_tokens=64 * 2)
    slot = eng.open()
    eng.step([(slot, [1] * 120)], [[]])
    with pytest.raises(llogos.engine.StepError, match="longest sequence"):
        eng.step_tree([(slot, [1] * 9, [-1] + [0] * 8)])
    assert eng.length(slot) == 120
    eng.step_tree([(slot, [1] * 8, [-1] + [0] * 7)])
    assert eng.accept_tree(torch.tensor([3] * 8, dtype=torch.int32)) == [([0], 3)] and eng.length(slot) == 121


def test_evictions_agree_with_plain(llogos, setup):
    model, w, _ = setup["llama"]
    E.check_evictions(lambda **kw: engine_for(llogos, model, **kw), w, TINY["llama"], torch.float32, 2e-4, 6, rounds=2)


def test_models_that_take_neither(llogos, setup):
    """Windows keep their trees but no evictions; a mixer that says nothing takes neither."""
    with pytest.raises(ValueError, match="slides"):
        engine_for(llogos, setup["qwen3"][0], weigh_keys=4)
    with pytest.raises(ValueError, match="must not be negative"):
        engine_for(llogos, setup["llama"][0], weigh_keys=-1)
    model = setup["llama"][0]
    mixer = model.blocks[0].parts["mixer"]
    assert llogos.parts.base.Mixer.placed_steps_refused(mixer) is not None
    mixer.sink_kind = "learned"
    try:
        eng = engine_for(llogos, model)
        slot = eng.open()
        with pytest.raises(llogos.engine.StepError, match="sinks"):
            eng.step_tree([(slot, [1], [-1])])
        with pytest.raises(ValueError, match="sinks"):
            engine_for(llogos, model, weigh_keys=4)
    finally:
        mixer.sink_kind = None


def test_positions_run_out_before_the_cache(llogos):
    """After evictions a short cache outlives its length, up to the model's positions."""
    cfg = dict(TINY_LLAMA, max_position_embeddings=96)
    model = llogos.weights.random_model(cfg, 3, dtype=torch.float32, device="cpu", ops=tree_ops)
    eng = engine_for(llogos, model, max_tokens=64, weigh_keys=1)
    slot = eng.open()
    eng.step([(slot, [1] * 60)], [[]])
    eng.evict([(slot, 20)], first=1, recent=4)
    eng.step([(slot, [1] * 36)], [[]])
    assert (eng.length(slot), eng.position(slot)) == (56, 96)
    with pytest.raises(llogos.engine.StepError, match="97"):
        eng.step([(slot, [1])])


def test_an_engine_is_freed_with_its_last_reference(llogos, setup):
    """Not when a collector next runs, which may be while a graph is recorded: graphs freed then end the recording."""
    import gc
    import weakref
    eng = engine_for(llogos, setup["llama"][0])
    slot = eng.open()
    eng.step_tree([(slot, [1, 2], [-1, 0])])
    eng.accept_tree()
    there = weakref.ref(eng)
    gc.disable()
    try:
        del eng
        assert there() is None
    finally:
        gc.enable()
