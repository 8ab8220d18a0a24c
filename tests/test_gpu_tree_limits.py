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
