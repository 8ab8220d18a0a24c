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
