"""Logits that are no numbers beside logits of minus infinity: the confirmed path's tokens on the GPU."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [30011, 30012, 5])
def test_a_logit_that_is_no_number_is_never_chosen_before_minus_infinity(vocab):
    """Of minus infinities the lowest id, wherever the ids lie that are NaN: ahead of it, in whole slices of the row, in a thread's first places.  A
    row of NaN alone gives token 0."""
    ops = importlib.import_module("daisi-llogos_b200.kernels.ops")
    nan, inf = float("nan"), float("inf")
    low = [i for i in (0, 1, 2, 3, 4, 5, 255, 256, 1024, 4095, 4096, 8191, 12288, 20001, vocab - 1) if i < vocab] + [None]
    logits = torch.full((len(low), vocab), nan)
    for row, at in zip(logits, low):
        if at is not None:
            row[at::7] = -inf
    b = len(low)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda:0")
    path, count, nxt = (torch.full(s, 99, dtype=torch.int32, device="cuda:0") for s in ((b, 64), (b,), (b,)))
    scratch = torch.zeros(ops.tree_accept_scratch(b, b), dtype=torch.int64, device="cuda:0")
    for _ in range(2):
        ops.tree_accept(ints([1] * b), ints([-1] * b), ints(list(range(b + 1))), path, count, nxt, logits=logits.cuda(), scratch=scratch)
        assert nxt.tolist() == [0 if at is None else at for at in low] and count.tolist() == [1] * b and not scratch.any()
