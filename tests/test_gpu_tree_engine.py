"""Drafted trees and evictions through the engine on the GPU, float32 and bfloat16, launched one by one and as recorded graphs.

How close logits have to be is said in ``compare.py``.  A key's weight is a sum of softmax shares: in float32 a share is off by the scores' error, 2
(hd + 3) 2^-23 times the largest sum of magnitudes (below 50 for these models: 1.2e-4 at hd 64), and the activations' 2e-5.  In bfloat16 q and k
are rounded (half a step, 2^-8 of a value, in every summand of a score): scores of up to ten are off by up to 2 * 2^-8 * 10 in the worst case
and a root of the summands' number less in all others, so 0.08 of the largest weight bounds shares that are off by 0.02 each way and the
activations' 4e-2."""
import pytest
import torch

import tree_engine as E
from conftest import TINY, read_weights

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


@pytest.fixture(scope="module")
def setup(llogos, model_dirs):
    cache = {}

    def get(name, dtype):
        if (name, dtype) not in cache:
            cache[name, dtype] = llogos.weights.load_model(model_dirs[name], dtype=dtype, device="cuda:0")
        return cache[name, dtype], read_weights(llogos, model_dirs[name]), model_dirs[name]
    return get


def engine_for(llogos, model, graphs=True, **kw):
    kw.setdefault("max_tokens", 64 * 16)
    return llogos.engine.Engine(model, use_graphs=graphs, **kw)


@pytest.mark.parametrize("graphs", [True, False], ids=["graph", "eager"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("name", list(TINY))
def test_trees_agree_with_plain(llogos, setup, name, dtype, graphs):
    model, w, key = setup(name, dtype)
    eng = engine_for(llogos, model, graphs)
    E.check_trees(eng, key, w, TINY[name], dtype, [70, 1, 129], [9, 1, 20], 5, 3)
    E.check_trees(eng, key, w, TINY[name], dtype, [62], [64], 3, 4)
    assert eng.trees._recorded == {} if not graphs else any(r.graph is not None for r in eng.trees._recorded.values())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("name", list(TINY))
def test_greedy_with_drafts_is_greedy(llogos, setup, name, dtype):
    """(The two runs add sums in other orders: prompts are such that no two logits are as near as that.)"""
    model, w, key = setup(name, dtype)
    E.check_greedy(engine_for(llogos, model), TINY[name], dtype, [[5, 6, 7], [9, 8] * 20, [11] * 63], 12, 4)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_trees_that_nobody_accepts(llogos, setup, dtype):
    for name in ("llama", "qwen3", "wide"):
        model, w, key = setup(name, dtype)
        E.check_forgotten(engine_for(llogos, model), llogos, key, w, TINY[name], dtype, 5)


def test_refusals(llogos, setup):
    model, _, _ = setup("llama", torch.float32)
    E.check_refusals(engine_for(llogos, model), llogos, TINY["llama"])


@pytest.mark.parametrize("graphs", [True, False], ids=["graph", "eager"])
@pytest.mark.parametrize("name,dtype,tol,weights_tol", [("llama", torch.float32, 2e-5, 1.5e-4), ("deep", torch.float32, 2e-5, 1.5e-4),
                                                        ("llama", torch.bfloat16, 4e-2, 8e-2), ("deep", torch.bfloat16, 4e-2, 8e-2)],
                         ids=["llama_f32", "deep_f32", "llama_bf16", "deep_bf16"])
def test_evictions_agree_with_plain(llogos, setup, name, dtype, tol, weights_tol, graphs):
    model, w, _ = setup(name, dtype)
    E.check_evictions(lambda **kw: engine_for(llogos, model, graphs, **kw), w, TINY[name], dtype, tol, 6, weights_tol=weights_tol)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_sampler_picks_for_every_node(llogos, model_dirs, dtype):
    """The public model: a sampler's draws for all nodes of a tree step say the path."""
    import importlib
    import tree_plain as T
    api = importlib.import_module("daisi-llogos_b200.api")
    m = api.LlogosModel.load(model_dirs["llama"], dtype=dtype, max_context=256, max_batch=2)
    slots = [m.open(), m.open()]
    m.step([(slots[0], [1, 2, 3]), (slots[1], [4] * 70)], [[], []])
    params = importlib.import_module("daisi-llogos_b200.sampling.params").GenerationParams(temperature=0.9, seed=3)
    trees = [([7, 8, 9, 8], [-1, 0, 0, 1]), ([5, 6], [-1, 0])]
    logits = m.step_tree([(s, t, p) for s, (t, p) in zip(slots, trees)])
    picked = m.sampler.sample_device(logits, params, seed=3, step=0, seq_ids=list(range(6)))
    got = m.accept_tree(picked[:6])
    best = picked[:6].tolist()
    assert got[0] == T.walk(*trees[0], best[:4]) and got[1] == T.walk(*trees[1], best[4:])
    assert [m.engine.length(s) for s in slots] == [3 + len(got[0][0]), 70 + len(got[1][0])]
