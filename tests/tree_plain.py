"""Plain float64 forms of the operators around drafted trees and shortened caches, with what each element may be off by.

Every form walks sequences, heads and rows one by one over a dense copy of the sequence's keys; nothing is shared with the library.  ``slack`` is
what rounding allows an implementation that multiplies in the storage type, adds in float32 and rounds softmax weights and result to the storage
type, worked out from the data:

* a score is a sum of ``hd`` products whose partial sums are at most ``A = scale sum |q_d k_d|``; each float32 addition is off by at most
  2^-23 of that (half a step, or a whole one where a matrix unit cuts off): ``e = (hd + 3) 2^-23 A``, which the exponential turns into a factor
  of ``1 +- e`` on the weight; a maximum and an exponential of a few units in the last place add ``8 2^-23``.
* the weights' and the outputs' sums have ``L`` terms: ``L 2^-23`` of the sum of magnitudes; the quotient twice that.
* bfloat16: a weight is rounded once (half a step, 2^-8 of it) and so is the result.
"""
import math

import torch

F64 = torch.float64
PAGE = 64
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def pages_of(seqs, nkv, dims, dtype, ring, n_slots, slots, seed, fill=float("nan"), spare=2, device="cpu"):
    """Pools ``[pages, nkv, 64, d]`` for each of ``dims`` and the page table, every row that holds nothing filled with ``fill``.

    ``seqs``: per sequence a list of dense tensors ``[positions, nkv, d]``, one per pool; a ring keeps the newest ``ring`` pages."""
    g = torch.Generator().manual_seed(seed)
    n_pages = len(seqs) * ring + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    table = torch.full((n_slots, ring), order[-1], dtype=torch.int32)
    pools = [torch.full((n_pages, nkv, PAGE, d), fill, dtype=dtype) for d in dims]
    for i, dense in enumerate(seqs):
        mine = order[i * ring:(i + 1) * ring]
        table[slots[i]] = torch.tensor(mine, dtype=torch.int32)
        for pool, rows in zip(pools, dense):
            for p in range(rows.shape[0]):                       # newer positions of a ring overwrite older ones
                pool[mine[p // PAGE % ring], :, p % PAGE] = rows[p].to(dtype)
    return [p.to(device) for p in pools], table.to(device)


def tree_bits(parents):
    """Each node's ancestors and itself as bits of an unsigned 64-bit number."""
    bits = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return bits


def signed(bits):
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def sees(before, nodes, bits, window):
    """Per node the positions (cached ones, then nodes) that it sees."""
    depth = [bin(b).count("1") - 1 for b in bits]
    out = []
    for i in range(nodes):
        at = before + depth[i]
        row = [p for p in range(before) if not window or p > at - window]
        row += [before + j for j in range(nodes) if bits[i] >> j & 1 and (not window or depth[i] - depth[j] < window)]
        out.append(row)
    return out


def attend(q, k, v, seen, scale, dtype):
    """q [rows, nh, hd], k and v [positions, nkv, d], ``seen`` per row a list of positions: (out, slack) [rows, nh, vd]."""
    rows, nh, hd = q.shape
    group = nh // k.shape[1]
    out = torch.zeros(rows, nh, v.shape[2], dtype=F64)
    slack = torch.zeros_like(out)
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    for i in range(rows):
        if not seen[i]:
            continue
        at = torch.tensor(seen[i])
        for h in range(nh):
            kk, vv = k[at, h // group], v[at, h // group]
            s = kk @ q[i, h] * scale
            p = torch.softmax(s, 0)
            e = ((hd + 3) * (kk.abs() @ q[i, h].abs()).max() * scale + 8) * 2.0 ** -23
            out[i, h] = p @ vv
            big = p @ vv.abs()
            slack[i, h] = big * (2 * e + 3 * len(at) * 2.0 ** -23) + STEP[dtype] * out[i, h].abs() + (STEP[dtype] * big if dtype == torch.bfloat16 else 0)
    return out, slack


def key_weights(q, k, before, last, scale, held):
    """q [count, nh, hd] of one sequence's step, k [positions, nkv, hd], held [nkv, width]: (weights, slack) [nkv, width]."""
    count, nh, hd = q.shape
    nkv, total = k.shape[1], k.shape[0]
    group = nh // nkv
    new = held.to(F64).clone()
    new[:, before:total] = 0.0
    slack = torch.zeros_like(new)
    q, k = q.to(F64), k.to(F64)
    for i in range(max(0, count - last), count):
        end = before + i + 1
        for h in range(nh):
            kk = k[:end, h // group]
            p = torch.softmax(kk @ q[i, h] * scale, 0)
            e = ((hd + 3) * (kk.abs() @ q[i, h].abs()).max() * scale + 8 + end) * 2.0 ** -23
            new[h // group, :end] += p
            slack[h // group, :end] += p * 2 * e
    slack[:, :total] += new[:, :total].abs() * (min(count, last) * group + 2) * 2.0 ** -23
    return new, slack


def keep(weights, length, count, first, recent):
    """The positions of one head that stay, ascending."""
    w = weights.tolist()
    order = sorted(range(length), key=lambda p: (not (p < first or p >= length - recent), math.isnan(w[p]), 0.0 if math.isnan(w[p]) else -w[p], p)
                   if not (p < first or p >= length - recent) else (False, False, 0.0, p))
    return sorted(order[:min(count, length)])


def walk(tokens, parents, best):
    """The confirmed path and the token behind it."""
    if not tokens:
        return [], -1
    path = [0]
    while True:
        nxt = [j for j in range(path[-1] + 1, len(tokens)) if parents[j] == path[-1] and tokens[j] == best[path[-1]]]
        if not nxt:
            return path, best[path[-1]]
        path.append(nxt[0])


class KeptModel:
    """The dense decoder token by token in float64, with a list of keys and values per layer and key/value head that keys can be taken out of,
    and what queries gave each key so far.  The formulas are ``plain_model``'s."""

    def __init__(self, weights, cfg):
        import plain_model as P
        self.P, self.w, self.cfg = P, weights, cfg
        self.nh, self.nkv = cfg["num_attention_heads"], cfg["num_key_value_heads"]
        self.hd = cfg.get("head_dim") or cfg["hidden_size"] // self.nh
        self.layers = cfg["num_hidden_layers"]
        arch = cfg["architectures"][0]
        self.qk_norm = arch == "Qwen3ForCausalLM"
        self.bias = cfg.get("attention_bias", arch == "Qwen2ForCausalLM")
        self.freq = P.rope_inverse_frequencies(int(self.hd * cfg.get("partial_rotary_factor", 1.0)), cfg["rope_theta"], cfg.get("rope_scaling"))
        assert not any(P.layer_windows(cfg))
        self.k = [[[] for _ in range(self.nkv)] for _ in range(self.layers)]
        self.v = [[[] for _ in range(self.nkv)] for _ in range(self.layers)]
        self.given = [[[] for _ in range(self.nkv)] for _ in range(self.layers)]
        self.position = 0

    def step(self, tokens, last):
        """Logits of the step's tokens; its last ``last`` queries count."""
        return torch.stack([self._token(t, i >= len(tokens) - last) for i, t in enumerate(tokens)])

    def _token(self, token, counts):
        P, cfg, w = self.P, self.cfg, self.w
        eps = cfg["rms_norm_eps"]
        h = P.embedding(w["model.embed_tokens.weight"], [token])
        for i in range(self.layers):
            p = f"model.layers.{i}."
            x = P.rms_norm(h, w[p + "input_layernorm.weight"], eps)
            a = p + "self_attn."
            q, k, v = (P.linear(x, w[a + f"{n}_proj.weight"]).view(1, -1, self.hd) for n in "qkv")
            if self.qk_norm:
                q, k = P.per_head_rms_norm(q, w[a + "q_norm.weight"], eps), P.per_head_rms_norm(k, w[a + "k_norm.weight"], eps)
            if self.bias:
                q, k, v = (t + w[a + f"{n}_proj.bias"].to(F64).view(-1, self.hd) for t, n in ((q, "q"), (k, "k"), (v, "v")))
            q, k = (P.rope_rotate(t, [self.position], self.freq, "half") for t in (q, k))
            o = torch.empty(self.nh, self.hd, dtype=F64)
            for kvh in range(self.nkv):
                self.k[i][kvh].append(k[0, kvh])
                self.v[i][kvh].append(v[0, kvh])
                self.given[i][kvh].append(0.0)
                keys, values = torch.stack(self.k[i][kvh]), torch.stack(self.v[i][kvh])
                for g in range(self.nh // self.nkv):
                    head = kvh * (self.nh // self.nkv) + g
                    share = torch.softmax(keys @ q[0, head] / math.sqrt(self.hd), 0)
                    o[head] = share @ values
                    if counts:
                        self.given[i][kvh] = [x + y for x, y in zip(self.given[i][kvh], share.tolist())]
            h = h + P.linear(o.view(1, -1), w[a + "o_proj.weight"])
            x = P.rms_norm(h, w[p + "post_attention_layernorm.weight"], eps)
            m = p + "mlp."
            h = h + P.swiglu(x, w[m + "gate_proj.weight"], w[m + "up_proj.weight"], w[m + "down_proj.weight"])
        self.position += 1
        x = P.rms_norm(h, w["model.norm.weight"], eps)
        return P.linear(x, w["model.embed_tokens.weight"] if cfg.get("tie_word_embeddings") else w["lm_head.weight"])[0]

    def keep(self, stays):
        """``stays[layer][head]``: the places of the keys that stay."""
        for lists in (self.k, self.v, self.given):
            for i in range(self.layers):
                for h in range(self.nkv):
                    lists[i][h] = [lists[i][h][j] for j in stays[i][h]]
