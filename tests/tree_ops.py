"""Stand-ins on CPU tensors for the kernels, those around drafted trees and shortened caches included (``cpu_ops`` has the others)."""
import torch

import tree_plain as T
from cpu_ops import *  # noqa: F401,F403
from cpu_ops import _gather, _rows_of

TREE_MAX_NODES = 64


class _Plan:
    scratch_floats, n_counters = 1, 0


def attn_tree_plan(dtype, n_seqs, max_nodes, n_heads, n_kv_heads, head_dim, max_len, value_dim=0):
    return _Plan()


def attn_tree(q, k_pages, v_pages, page_table, ring_pages, slots, cu_tokens, len_before, ancestors, out, scratch, *, scale, window=0, plan, counters):
    n, nh, hd = q.shape
    group = nh // k_pages.shape[1]
    o = out.view(n, nh, -1)
    for b in range(slots.numel()):
        t0, t1, lb = int(cu_tokens[b]), int(cu_tokens[b + 1]), int(len_before[b])
        bits = [int(x) & (1 << 64) - 1 for x in ancestors[t0:t1]]
        for i, seen in enumerate(T.sees(lb, t1 - t0, bits, window)):
            for h in range(nh):
                ks, vs = _gather(k_pages, v_pages, page_table, ring_pages, int(slots[b]), seen, h // group)
                p = torch.softmax(torch.stack(ks).float() @ q[t0 + i, h].float() * scale, 0)
                o[t0 + i, h] = (p @ torch.stack(vs).float()).to(out.dtype)


def tree_accept_scratch(n_tokens, n_seqs):
    return n_tokens + n_seqs


def tree_accept(tokens, parents, cu_tokens, path, n_path, next_token, *, logits=None, picked=None, scratch=None):
    best = picked.tolist() if picked is not None else logits.argmax(-1).tolist()
    path.fill_(-1)
    for b in range(n_path.numel()):
        t0, t1 = int(cu_tokens[b]), int(cu_tokens[b + 1])
        way, nxt = T.walk(tokens[t0:t1].tolist(), parents[t0:t1].tolist(), best[t0:t1])
        path[b, :len(way)] = torch.tensor(way, dtype=torch.int32)
        n_path[b], next_token[b] = len(way), nxt


def key_weights_plan(dtype, n_seqs, last, n_heads, n_kv_heads, head_dim, max_len):
    return _Plan()


def key_weights(q, k_pages, page_table, slots, cu_tokens, len_before, weights, scratch, *, scale, last, plan, counters):
    nkv, ring = k_pages.shape[1], page_table.shape[1]
    for b in range(slots.numel()):
        t0, t1, lb, slot = int(cu_tokens[b]), int(cu_tokens[b + 1]), int(len_before[b]), int(slots[b])
        total = lb + t1 - t0
        k = torch.stack([torch.stack([k_pages[_rows_of(page_table, ring, slot, p, h, nkv)] for h in range(nkv)]) for p in range(total)])
        new, _ = T.key_weights(q[t0:t1], k, lb, last, scale, weights[slot])
        weights[slot, :, :total] = new[:, :total].float()


def keep_keys(weights, slots, lengths, keep, chosen, *, first, recent, max_len=None):
    for layer in range(weights.shape[0]):
        for b, s in enumerate(slots.tolist()):
            for h in range(weights.shape[2]):
                stays = T.keep(weights[layer, s, h], int(lengths[b]), int(keep[b]), first, recent)
                chosen[layer, b, h, :len(stays)] = torch.tensor(stays, dtype=torch.int32)


class CacheRows:
    def __init__(self, k_pages, v_pages=None, weights=None):
        self.pools, self.weights = list(zip(k_pages, v_pages)) if v_pages is not None else [(k,) for k in k_pages], weights

    def move(self, page_table, ring_pages, slots, base, source, count):
        nkv = self.pools[0][0].shape[1]
        for layer, pools in enumerate(self.pools):
            for b, s in enumerate(slots.tolist()):
                for h in range(nkv):
                    src = source[min(layer, source.shape[0] - 1), b, min(h, source.shape[2] - 1), :int(count[b])].tolist()
                    at = int(base[b])
                    for pool in pools:
                        rows = [pool[_rows_of(page_table, ring_pages, s, at + j, h, nkv)].clone() for j in src]
                        for j, row in enumerate(rows):
                            pool[_rows_of(page_table, ring_pages, s, at + j, h, nkv)] = row
                    if self.weights is not None:
                        w = self.weights[layer, s, h]
                        w[at:at + len(src)] = w[[at + j for j in src]].clone()
