"""What the operators around drafted trees and shortened caches refuse, and their argument blocks, without a GPU: every refusal comes before a
library is asked for."""
import ctypes
import importlib
import os

import pytest
import torch

import test_prototypes as P
import test_warp_whole as W
import tree_plain as T

ops = importlib.import_module("daisi-llogos_b200.kernels.ops")
F32, BF16, I32, I64 = torch.float32, torch.bfloat16, torch.int32, torch.int64


def test_the_argument_blocks_are_those_of_the_header():
    text = P._text(os.path.join(P.CSRC, "cache_args.h"))
    for name in ("TreeArgs", "KeyWeightArgs", "MoveArgs"):
        block = getattr(ops, "_" + name)
        assert [(f, ctypes.sizeof(t)) for f, t in block._fields_] == [
            (f, s) if f != "row_bytes" else (f, 8) for f, s in _fields(text, name)], name


def _fields(text, name):
    """As ``test_prototypes`` reads a structure, with array counts that are plain numbers."""
    return P._c_struct(text.replace("void* const* pools", "void* pools"), name, {})


@pytest.mark.parametrize("source,least", [("attention_tree_tc.cu", 8), ("key_weights_tc.cu", 3)])
def test_the_warp_is_whole_where_tensor_memory_wants_it(source, least):
    with open(os.path.join(P.CSRC, source)) as f:
        found = W.lines_that_want_the_warp(f.read())
    assert len(found) >= least, found
    assert not [x for x in found if not x[2]]


def tree_call(**change):
    nh, nkv, hd, b, n = 4, 2, 16, 2, 5
    plan = change.pop("plan", ops.TreePlan("simt", (F32, b, nh, nkv, hd, hd), 2, 4, 130, 100, 4))
    given = dict(q=torch.zeros(n, nh, hd), k_pages=torch.zeros(6, nkv, 64, hd), v_pages=torch.zeros(6, nkv, 64, hd),
                 page_table=torch.zeros(3, 3, dtype=I32), ring_pages=3, slots=torch.zeros(b, dtype=I32), cu_tokens=torch.zeros(b + 1, dtype=I32),
                 len_before=torch.zeros(b, dtype=I32), ancestors=torch.zeros(n, dtype=I64), out=torch.zeros(n, nh * hd), scratch=torch.zeros(100))
    kw = dict(scale=0.25, window=0, counters=torch.zeros(4, dtype=I32))
    for key, value in change.items():
        (given if key in given else kw)[key] = value
    ops.attn_tree(*given.values(), plan=plan, **kw)


@pytest.mark.parametrize("change,says", [
    (dict(), "not on the GPU"),
    (dict(q=torch.zeros(5, 4, 16, dtype=BF16)), "the plan is for"),
    (dict(q=torch.zeros(5, 6, 16)), "the plan is for"),
    (dict(v_pages=torch.zeros(5, 2, 64, 16)), "v_pages has shape"),
    (dict(k_pages=torch.zeros(6, 2, 32, 16)), "k_pages has shape"),
    (dict(k_pages=torch.zeros(6, 2, 64, 16, dtype=BF16)), "k_pages is"),
    (dict(cu_tokens=torch.zeros(2, dtype=I32)), "cu_tokens has shape"),
    (dict(len_before=torch.zeros(2, dtype=I64)), "len_before is"),
    (dict(ancestors=torch.zeros(5, dtype=I32)), "ancestors is"),
    (dict(ancestors=torch.zeros(4, dtype=I64)), "ancestors has shape"),
    (dict(out=torch.zeros(5, 32)), "out has shape"),
    (dict(out=torch.zeros(5, 64, dtype=BF16)), "out is"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
    (dict(window=-1), "window -1"),
    (dict(ring_pages=4), "4 ring pages"),
    (dict(ring_pages=2), "do not hold 130 positions"),
    (dict(ring_pages=1, window=60), "does not hold a window"),
    (dict(scratch=torch.zeros(99)), "scratch of 99"),
    (dict(scratch=torch.zeros(100, dtype=BF16)), "scratch of 100"),
    (dict(counters=torch.zeros(3, dtype=I32)), "3 counters"),
    (dict(page_table=torch.zeros(3, 3, dtype=I64)), "page_table is"),
    (dict(slots=torch.zeros(2, device="meta", dtype=I32)), "tensors on cpu and on meta"),
])
def test_attention_of_trees_refuses(change, says):
    with pytest.raises(ops.KernelError, match=says):
        tree_call(**change)


@pytest.mark.parametrize("args,says", [
    ((torch.float16, 1, 4, 4, 2, 16, 100), "float32 or bfloat16"), ((F32, 1, 65, 4, 2, 16, 100), "65 nodes"), ((F32, 1, 0, 4, 2, 16, 100), "0 nodes"),
    ((F32, 1, 4, 5, 2, 16, 100), "no multiple"), ((F32, 1, 4, 4, 2, 385, 400), "385"), ((F32, 0, 4, 4, 2, 16, 100), "needs sequences"),
    ((F32, 1, 4, 4, 2, 16, 0), "needs sequences")])
def test_plans_of_trees_refuse(args, says):
    with pytest.raises(ops.KernelError, match=says):
        ops.attn_tree_plan(*args)


@pytest.mark.parametrize("change,says", [
    (dict(), "not on the GPU"), (dict(logits=None), "either logits or picked"), (dict(picked=torch.zeros(5, dtype=I32)), "either logits or picked"),
    (dict(tokens=torch.zeros(5, dtype=I64)), "tokens is"), (dict(parents=torch.zeros(4, dtype=I32)), "parents has shape"),
    (dict(cu_tokens=torch.zeros(2, dtype=I32)), "cu_tokens has shape"), (dict(path=torch.zeros(2, 63, dtype=I32)), "path has shape"),
    (dict(next_token=torch.zeros(1, dtype=I32)), "next_token has shape"), (dict(logits=torch.zeros(5, 9, dtype=BF16)), "logits is"),
    (dict(logits=torch.zeros(4, 9)), "logits has shape"), (dict(logits=torch.zeros(45)), "logits of shape"), (dict(scratch=None), "zeroed int64"),
    (dict(scratch=torch.zeros(6, dtype=I64)), "zeroed int64"), (dict(logits=None, picked=torch.zeros(4, dtype=I32)), "picked has shape"),
    (dict(tokens=torch.zeros(0, dtype=I32), parents=torch.zeros(0, dtype=I32)), "none with a node")])
def test_the_confirmed_path_refuses(change, says):
    given = dict(tokens=torch.zeros(5, dtype=I32), parents=torch.zeros(5, dtype=I32), cu_tokens=torch.zeros(3, dtype=I32),
                 path=torch.zeros(2, 64, dtype=I32), n_path=torch.zeros(2, dtype=I32), next_token=torch.zeros(2, dtype=I32),
                 logits=torch.zeros(5, 9), picked=None, scratch=torch.zeros(7, dtype=I64))
    given.update(change)
    with pytest.raises(ops.KernelError, match=says):
        ops.tree_accept(**given)


@pytest.mark.parametrize("change,says", [
    (dict(), "not on the GPU"), (dict(last=2), "the plan is for"), (dict(q=torch.zeros(5, 4, 8)), "the plan is for"),
    (dict(k_pages=torch.zeros(6, 2, 64, 8)), "k_pages has shape"), (dict(weights=torch.zeros(2, 130)), "weights of shape"),
    (dict(weights=torch.zeros(2, 2, 130)), "weights has shape"), (dict(weights=torch.zeros(3, 2, 129)), "129 weights a row"),
    (dict(weights=torch.zeros(3, 2, 130, dtype=BF16)), "weights is"), (dict(page_table=torch.zeros(3, 2, dtype=I32)), "2 pages"),
    (dict(scale=-1.0), "scale must be positive"), (dict(scratch=torch.zeros(59)), "scratch of 59"), (dict(counters=torch.zeros(4)), "4 counters")])
def test_weights_of_keys_refuse(change, says):
    plan = ops.KeyWeightPlan("simt", (F32, 2, 4, 2, 16), 1, 130, 1, 192, 40, 20)
    given = dict(q=torch.zeros(5, 4, 16), k_pages=torch.zeros(6, 2, 64, 16), page_table=torch.zeros(3, 3, dtype=I32), slots=torch.zeros(2, dtype=I32),
                 cu_tokens=torch.zeros(3, dtype=I32), len_before=torch.zeros(2, dtype=I32), weights=torch.zeros(3, 2, 130), scratch=torch.zeros(60),
                 scale=0.25, last=1, plan=plan, counters=torch.zeros(4, dtype=I32))
    given.update(change)
    with pytest.raises(ops.KernelError, match=says):
        ops.key_weights(**given)


@pytest.mark.parametrize("args,says", [((F32, 0, 1, 4, 2, 16, 10), "needs sequences"), ((F32, 1, 0, 4, 2, 16, 10), "needs sequences"),
                                       ((F32, 1, 1, 4, 3, 16, 10), "no multiple"), ((F32, 1, 1, 4, 2, 400, 10), "400"), ((I32, 1, 1, 4, 2, 16, 10), "float32 or")])
def test_plans_of_weights_refuse(args, says):
    with pytest.raises(ops.KernelError, match=says):
        ops.key_weights_plan(*args)


@pytest.mark.parametrize("change,says", [
    (dict(), "not on the GPU"), (dict(weights=torch.zeros(3, 2, 50)), "weights are"), (dict(weights=torch.zeros(1, 3, 2, 50, dtype=BF16)), "weights is"),
    (dict(keep=torch.zeros(1, dtype=I32)), "keep has shape"), (dict(lengths=torch.zeros(2, dtype=I64)), "lengths is"),
    (dict(chosen=torch.zeros(1, 2, 3, 8, dtype=I32)), "chosen has shape"), (dict(first=-1), "must not be negative"), (dict(max_len=51), "lengths up to 51"),
    (dict(max_len=0), "lengths up to 0")])
def test_the_choice_of_keys_refuses(change, says):
    given = dict(weights=torch.zeros(1, 3, 2, 50), slots=torch.zeros(2, dtype=I32), lengths=torch.zeros(2, dtype=I32), keep=torch.zeros(2, dtype=I32),
                 chosen=torch.zeros(1, 2, 2, 8, dtype=I32), first=0, recent=0)
    given.update(change)
    with pytest.raises(ops.KernelError, match=says):
        ops.keep_keys(**given)


@pytest.mark.parametrize("args,says", [
    (([], []), "0 layers"), (([torch.zeros(3, 2, 64, 8)], []), "value pages of 0"), (([torch.zeros(3, 2, 32, 8)],), "pages of shape"),
    (([torch.zeros(3, 2, 64, 8, dtype=I32)],), "float32 or bfloat16"), (([torch.zeros(3, 2, 64, 8), torch.zeros(4, 2, 64, 8)],), "key pages has shape"),
    (([torch.zeros(3, 2, 64, 8)], [torch.zeros(3, 2, 64, 8, dtype=BF16)]), "value pages is"),
    (([torch.zeros(3, 2, 64, 8)], None, torch.zeros(2, 5, 2, 9)), "weights of shape"), (([torch.zeros(3, 2, 64, 8)],), "not on the GPU")])
def test_cache_rows_refuse(args, says):
    with pytest.raises(ops.KernelError, match=says):
        ops.CacheRows(*args)


@pytest.mark.parametrize("change,says", [
    (dict(count=torch.zeros(3, dtype=I32)), "count has shape"), (dict(source=torch.zeros(2, 2, 1, 4, dtype=I32)), "sources of shape"),
    (dict(source=torch.zeros(1, 2, 3, 4, dtype=I32)), "sources of shape"), (dict(source=torch.zeros(1, 2, 1, 4, dtype=I64)), "source is"),
    (dict(ring_pages=0), "0 ring pages"), (dict(ring_pages=4), "4 ring pages"), (dict(base=torch.zeros(2)), "base is")])
def test_moves_refuse(change, says):
    rows = object.__new__(ops.CacheRows)
    rows.k, rows.v, rows.nkv, rows.weights, rows.args = [torch.zeros(3, 2, 64, 8)], None, 2, None, ops._MoveArgs()
    rows.pools = torch.zeros(1, dtype=I64)
    given = dict(page_table=torch.zeros(3, 3, dtype=I32), ring_pages=3, slots=torch.zeros(2, dtype=I32), base=torch.zeros(2, dtype=I32),
                 source=torch.zeros(1, 2, 1, 4, dtype=I32), count=torch.zeros(2, dtype=I32))
    given.update(change)
    with pytest.raises(ops.KernelError, match=says):
        rows.move(**given)


def test_the_plain_forms_agree_with_a_softmax():
    """The oracle's masks against a dense product: a chain of drafted tokens is a causal step, a window counts positions."""
    g = torch.Generator().manual_seed(1)
    before, n, nh, nkv, hd = 7, 5, 4, 2, 8
    q = torch.randn(n, nh, hd, generator=g, dtype=torch.float64)
    k, v = (torch.randn(before + n, nkv, hd, generator=g, dtype=torch.float64) for _ in range(2))
    for window in (0, 3):
        bits = T.tree_bits([-1, 0, 1, 2, 3])
        out, _ = T.attend(q, k, v, T.sees(before, n, bits, window), 0.5, F32)
        i, j = torch.arange(n)[:, None] + before, torch.arange(before + n)[None]
        see = (j <= i) & ((j > i - window) if window else True)
        s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(2, 1)) * 0.5
        p = torch.softmax(s.masked_fill(~see, -float("inf")), -1)
        assert torch.allclose(out, torch.einsum("hij,jhd->ihd", p, v.repeat_interleave(2, 1)))
    assert T.walk([9, 1, 1, 4], [-1, 0, 0, 2], [1, 4, 4, 6]) == ([0, 1], 4)
    assert T.walk([9, 2, 1, 4], [-1, 0, 0, 2], [1, 0, 4, 6]) == ([0, 2, 3], 6)
    assert T.keep(torch.tensor([1.0, 5.0, 2.0, 5.0, 0.0]), 5, 3, 1, 1) == [0, 1, 4]


def test_the_look_over_of_a_calls_tensors_takes_nothing_that_is_not_as_said():
    """In native code; what is right on a GPU is in the operators' own tests."""
    build = importlib.import_module("daisi-llogos_b200.csrc.build")
    look = ctypes.PyDLL(build.compile_library("tensor_args")).llg_tensor_addresses
    look.argtypes = [ctypes.py_object, ctypes.c_int, ctypes.c_void_p]
    out = (ctypes.c_ulonglong * 4)(*[7] * 4)
    t = torch.zeros(3, 4)
    for specs in ([("t", t, None, F32)], (t,), (("t", t, None),), (("t", 5, None, F32),), (("t", t, None, "float32"),), (("t", t, ("x", 4), F32),),
                  (("t", t, None, F32),), (("t", t, (3, 4), BF16),), (("t", t.to_sparse(), None, F32),), (("t", t.to("meta"), None, F32),)):
        assert look(specs, 0, out) == 1
    assert list(out) == [7] * 4 and look((), 0, out) == 0
