"""What plans of drafted trees and weighed keys go by at the ends of their ranges: rules on the host, asked without a GPU."""
import importlib
import random

import pytest

ops = importlib.import_module("daisi-llogos_b200.kernels.ops")
LIMIT = 2 ** 31


def up(x, y):
    return -(-x // y)


def tc_list(n_seqs, group, nodes, nkv, max_len):
    """The weight of the tcgen05 kernel's list if every sequence is as long as it may be: 5 a tile of a row block and 8 a row block at most."""
    tile = 128 // group
    return n_seqs * nkv * up(nodes, tile if nodes <= tile else 2 * tile) * (5 * up(max_len, 64) + 8)


def mma_list(n_seqs, rows, nkv, max_len):
    return n_seqs * nkv * up(rows, 16 if rows <= 16 else 32 if rows <= 32 else 64) * up(max_len, 64)


def test_kernels_take_the_trees_whose_lists_fit_their_counts():
    """Each by its own list's length: 256 sequences of up to 131,072 positions, 64 nodes, 8 key/value heads of 8 query heads are 43 million units, no
    reason to refuse them; where the list is too long the next kernel's turn comes."""
    tc = ops._lib("attention_tree_tc").llg_attn_tree_tc_supported
    mma = ops._lib("attention_tree_mma").llg_attn_tree_mma_supported
    assert tc(128, 128, 256, 8, 64, 8, 131072) and mma(128, 128, 256, 512, 8, 131072)
    rng, seen = random.Random(1), {(a, b): 0 for a in (0, 1) for b in (0, 1)}
    for _ in range(20000):
        n_seqs, group, nodes, nkv, max_len = (int(2 ** rng.uniform(low, high)) for low, high in ((0, 10), (0, 7), (0, 6), (0, 7), (0, 30)))
        a, b = tc(64, 64, n_seqs, group, nodes, nkv, max_len), mma(64, 64, n_seqs, nodes * group, nkv, max_len)
        for taken, units in ((a, tc_list(n_seqs, group, nodes, nkv, max_len)), (b, mma_list(n_seqs, nodes * group, nkv, max_len))):
            assert not taken or units + 2 ** 20 < LIMIT
            assert taken or units * 1.01 + 2 ** 21 > LIMIT      # (the room that is left: a million, rounded down to a head's)
        seen[a, b] += 1
    assert min(seen[1, 1], seen[0, 0]) > 100
    assert not tc(64, 64, 1025, 4, 8, 8, 100) and not mma(64, 64, 1025, 32, 8, 100)
    assert not tc(64, 64, 1024, 2, 64, 32, 1 << 20) and mma(64, 64, 1024, 128, 32, 1 << 20)
    assert not tc(64, 64, 1024, 8, 64, 32, 1 << 20) and not mma(64, 64, 1024, 512, 32, 1 << 20)


def test_no_plan_keeps_more_scores_than_a_workspace_should(monkeypatch):
    """What keys are weighed in is bounded whatever the batch and its longest sequence are, on every kernel: 64 MB of scores."""
    import torch
    monkeypatch.setattr(ops, "sm_count", lambda: 148)
    rng = random.Random(2)
    kinds = set()
    for i in range(3000):
        n_seqs, nkv, group, last, max_len = (int(2 ** rng.uniform(low, high)) for low, high in ((0, 8.1), (0, 5.1), (0, 3.1), (0, 5.1), (0, 17.1)))
        if i == 0:
            n_seqs, nkv, group, last, max_len = 32, 8, 4, 8, 131072
        dtype, hd = rng.choice(((torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 80), (torch.bfloat16, 20), (torch.float32, 64)))
        plan = ops.key_weights_plan(dtype, n_seqs, last, nkv * group, nkv, hd, max_len)
        assert plan.scores <= 1 << 24, (plan.kind, plan.scores)
        assert plan.scratch_floats >= plan.scores + 2 * plan.together * nkv * group * last * plan.splits and plan.splits * plan.split_keys >= max_len
        assert plan.together == n_seqs or group * last <= ops.KEY_GOES_ROWS
        if plan.scores:
            assert plan.scores == plan.together * nkv * group * last * plan.splits * plan.split_keys and plan.together <= n_seqs
        else:
            assert plan.together == n_seqs
        kinds.add((plan.kind, bool(plan.scores), plan.together < n_seqs))
    assert kinds == {("mma", True, False), ("mma", True, True), ("mma", False, False), ("simt", True, False), ("simt", False, False), ("tc", False, False)}


@pytest.mark.parametrize("source", ["attention_tree.cu", "attention_tree_mma.cu", "attention_tree_tc.cu"])
def test_only_sizes_slots_and_pages_are_read_before_the_wait(source):
    """Ahead of its wait for the kernel before it an attention of trees reads what its entry point says: not the words of what nodes see, which a
    caller's own kernel may just be writing."""
    import os
    import re
    with open(os.path.join(os.path.dirname(ops.__file__), "..", "csrc", source)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    ahead = text[text.index("__global__"):text.index("  pdl_wait();")]
    assert set(re.findall(r"\ba\.(cu_tokens|len_before|slots|page_table|ancestors|q|k_pages|v_pages|out|part|counters)\s*\[", ahead)) <= {
        "cu_tokens", "len_before", "slots", "page_table"}
