"""What an engine has to do with drafted trees and shortened caches, against the plain model: run on CPU tensors with stand-ins for the kernels
(``test_trees_cpu_engine.py``) and on the GPU (``test_gpu_tree_engine.py``)."""
import random

import pytest
import torch

import tree_plain as T
from compare import reference


def random_tree(r, n, vocab):
    parents = [-1] + [r.randint(max(0, i - 4), i - 1) for i in range(1, n)]
    return [r.randrange(vocab) for _ in range(n)], parents


def path_to(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


def check_trees(eng, key, weights, cfg, dtype, lengths, sizes, rounds, seed):
    """Rounds of: a tree for every sequence, every node's logits against the plain model on its own path, a path of the test's choice accepted, one
    more token decoded; and at the end the whole sequences once more without trees."""
    r = random.Random(seed)
    vocab = cfg["vocab_size"]
    seqs = [[r.randrange(vocab) for _ in range(n)] for n in lengths]
    slots = [eng.open() for _ in seqs]
    eng.step([(s, t) for s, t in zip(slots, seqs)], [[]] * len(seqs))
    for rnd in range(rounds):
        trees = [random_tree(r, n, vocab) for n in (sizes if rnd % 4 != 3 else sizes[::-1])]
        logits = eng.step_tree([(s, t, p) for s, (t, p) in zip(slots, trees)])
        assert logits.shape == (sum(len(t) for t, _ in trees), vocab)
        assert [eng.length(s) for s in slots] == [len(t) for t in seqs]
        best, base, ends = [], 0, []
        for b, (tokens, parents) in enumerate(trees):
            n = len(tokens)
            ends.append(r.randrange(n))
            for i in sorted(set(r.sample(range(n), min(n, 5)) + [ends[-1], n - 1])):
                way = path_to(parents, i)
                ref = reference(key, weights, cfg, seqs[b] + [tokens[j] for j in way])
                ref.check(logits[base + i], [len(seqs[b]) + len(way) - 1], dtype, ("round", rnd, "tree", b, "node", i))
            # what follows each node, so that the way to the chosen end is confirmed; another child of equal token is not meant
            way = path_to(parents, ends[-1])
            follow = [vocab - 1 - rnd] * n
            for a, c in zip(way, way[1:]):
                follow[a] = tokens[c]
            best += follow
            base += n
        got = eng.accept_tree(torch.tensor(best, dtype=torch.int32, device=eng.device))
        base = 0
        for b, (tokens, parents) in enumerate(trees):
            want, nxt = T.walk(tokens, parents, best[base:base + len(tokens)])
            assert got[b] == (want, nxt)
            seqs[b] += [tokens[j] for j in want]
            base += len(tokens)
        assert [eng.length(s) for s in slots] == [len(t) for t in seqs]
        eng.cache.audit()
        more = [r.randrange(vocab) for _ in seqs]
        logits = eng.step([(s, [t]) for s, t in zip(slots, more)])
        for b, t in enumerate(more):
            seqs[b].append(t)
            reference(key, weights, cfg, seqs[b]).check(logits[b], [len(seqs[b]) - 1], dtype, ("round", rnd, "decoded", b))
    for s in slots:
        eng.close(s)
    eng.cache.audit()


def check_greedy(eng, cfg, dtype, prompts, steps, seed):
    """Greedy generation with drafts, right and wrong ones, gives the tokens of greedy generation without."""
    r = random.Random(seed)
    vocab = cfg["vocab_size"]
    plain = []
    for p in prompts:
        slot = eng.open()
        logits, out = eng.step([(slot, p)]), []
        for _ in range(steps):
            out.append(int(logits[0].argmax()))
            logits = eng.step([(slot, [out[-1]])])
        plain.append(out)
        eng.close(slot)
    slots = [eng.open() for _ in prompts]
    made = [[int(x.argmax())] for x in eng.step(list(zip(slots, prompts)))]
    used = 0
    while min(len(m) for m in made) < steps:
        trees = []
        for b, m in enumerate(made):
            # the last certain token, a right draft of up to three tokens, a wrong one beside each
            ahead = plain[b][len(m):len(m) + 3]
            tokens, parents, at = [m[-1]], [-1], 0
            for t in ahead:
                tokens += [(t + 1 + r.randrange(vocab - 1)) % vocab, t]
                parents += [at, at]
                at = len(tokens) - 1
            trees.append((tokens, parents))
        eng.step_tree([(s, t, p) for s, (t, p) in zip(slots, trees)])
        for b, (way, nxt) in enumerate(eng.accept_tree()):
            made[b] += [trees[b][0][j] for j in way[1:]] + [nxt]
        used += 1
    assert used < steps                                    # fewer steps than tokens
    for m, p in zip(made, plain):
        assert m[:steps] == p
    for s in slots:
        eng.close(s)
    eng.cache.audit()


def check_forgotten(eng, llogos, key, weights, cfg, dtype, seed):
    """A tree that nobody accepts leaves no trace: other steps, truncation and the end of a sequence."""
    r = random.Random(seed)
    vocab = cfg["vocab_size"]
    seq = [r.randrange(vocab) for _ in range(62)]
    slot, other = eng.open(), eng.open()
    eng.step([(slot, seq)], [[]])
    free = eng.cache.free_pages()
    tree = random_tree(r, 9, vocab)
    eng.step_tree([(slot, *tree)])
    eng.step_tree([(slot, *random_tree(r, 20, vocab))])     # another tree in its place
    logits = eng.step([(other, seq[:5])])
    reference(key, weights, cfg, seq[:5]).check(logits[0], [4], dtype)
    with pytest.raises(llogos.engine.StepError, match="no tree step"):
        eng.accept_tree()
    eng.close(other)
    assert eng.cache.free_pages() == free
    eng.step_tree([(slot, *tree)])
    eng.truncate(slot, 60)
    logits = eng.step([(slot, seq[60:])], [[0, 1]])
    reference(key, weights, cfg, seq).check(logits, [60, 61], dtype)
    eng.step_tree([(slot, *tree)])
    eng.close(slot)
    eng.cache.audit()


def check_refusals(eng, llogos, cfg):
    E = llogos.engine.StepError
    slot, vocab = eng.open(), cfg["vocab_size"]
    eng.step([(slot, [1, 2, 3])], [[]])
    for entries, says in (([], "at least one"), ([(slot, [], [])], "1 to 64 nodes"), ([(slot, [1] * 65, [-1] * 65)], "1 to 64 nodes"),
                          ([(slot, [1, 2], [-1])], "2 tokens and 1 parents"), ([(slot, [1, 2], [0, 0])], "first node's parent"),
                          ([(slot, [1, 2], [-1, 1])], "first node's parent"), ([(slot, [1, 2], [-1, -1])], "first node's parent"),
                          ([(slot, [1, vocab], [-1, 0])], "outside the vocabulary"), ([(slot, [1, -1], [-1, 0])], "outside the vocabulary"),
                          ([(slot, [1], [-1]), (slot, [1], [-1])], "twice"), ([(slot + 1, [1], [-1])], "not in use")):
        with pytest.raises(E, match=says):
            eng.step_tree(entries)
    assert eng.length(slot) == 3
    with pytest.raises(E, match="no tree step"):
        eng.accept_tree()
    eng.step_tree([(slot, [1, 2], [-1, 0])])
    with pytest.raises(E, match="picked tokens"):
        eng.accept_tree(torch.zeros(2, dtype=torch.int64, device=eng.device))
    with pytest.raises(E, match="weighs its keys"):
        eng.evict([(slot, 2)])
    eng.close(slot)


def check_evictions(make, weights, cfg, dtype, tol, seed, rounds=3, weights_tol=None):
    """Prompts, decoding, eviction and more of both, the logits and the weights against the plain model that holds the same keys."""
    r = random.Random(seed)
    vocab, last = cfg["vocab_size"], 6
    eng = make(weigh_keys=last)
    models, slots = [], []
    for n in (70, 131, 9):
        slots.append(eng.open())
        models.append(T.KeptModel(weights, cfg))
    prompts = [[r.randrange(vocab) for _ in range(n)] for n in (70, 131, 9)]
    logits = eng.step(list(zip(slots, prompts)))

    def compare(got, want, what):
        for b, (x, y) in enumerate(zip(got, want)):
            off = float((x.detach().cpu().double() - y).abs().max()) / float(y.abs().max())
            assert off <= tol, (what, b, off, tol)

    compare(logits, [m.step(p, last)[-1] for m, p in zip(models, prompts)], "prompt")
    for rnd in range(rounds):
        for _ in range(4):
            toks = [r.randrange(vocab) for _ in slots]
            logits = eng.step([(s, [t]) for s, t in zip(slots, toks)])
            compare(logits, [m.step([t], 1)[0] for m, t in zip(models, toks)], ("decode", rnd))
        g = eng.cache.kv_groups[0]
        for s, m in zip(slots, models):
            n = eng.length(s)
            got = g.weights[:, s, :, :n].cpu().double()
            want = torch.tensor(m.given, dtype=torch.float64)
            assert float((got - want).abs().max()) <= (weights_tol or tol) * float(want.abs().max()), ("weights", rnd)
        # the engine's own weights say what stays: two keys of nearly equal weight may go either way
        cut = [(s, max(8, eng.length(s) * 2 // 3)) for s in slots[:2]]
        stays = [[[T.keep(g.weights[i, s, h].cpu(), eng.length(s), keep, 2, 5) for h in range(models[0].nkv)] for i in range(models[0].layers)]
                 for s, keep in cut]
        position = [eng.position(s) for s in slots]
        eng.evict(cut, first=2, recent=5)
        for m, st in zip(models, stays):
            m.keep(st)
        assert [eng.length(s) for s in slots[:2]] == [k for _, k in cut] and [eng.position(s) for s in slots] == position
        eng.cache.audit()
        more = [[r.randrange(vocab) for _ in range(n)] for n in (3, 20, 1)]        # the next turns, after keys are gone
        logits = eng.step(list(zip(slots, more)))
        compare(logits, [m.step(t, last)[-1] for m, t in zip(models, more)], ("turn", rnd))
    held = eng.length(slots[0])
    eng.truncate(slots[0], held - 2)                               # tokens behind the eviction can be forgotten ...
    assert eng.position(slots[0]) == position[0] + 1
    with pytest.raises(ValueError, match="left by an eviction"):   # ... the ones that it left cannot
        eng.truncate(slots[0], cut[0][1] - 1)
    for entries, says in (([(slots[0], held)], "cannot keep"), ([(slots[0], 6)], "cannot keep"), ([(slots[0], 20), (slots[0], 20)], "twice"),
                          ([(99, 20)], "not in use")):
        with pytest.raises(ValueError, match=says):
            eng.evict(entries, first=2, recent=5)
    with pytest.raises(ValueError, match="weighs its keys"):
        eng.step_tree([(slots[0], [1], [-1])])
    for s in slots:
        eng.close(s)
    eng.cache.audit()
    slot = eng.open()                                              # a new sequence in a slot that was shortened begins anew
    assert eng.position(slot) == 0
    m = T.KeptModel(weights, cfg)
    compare(eng.step([(slot, prompts[2])]), [m.step(prompts[2], last)[-1]], "a new sequence")
    eng.close(slot)
