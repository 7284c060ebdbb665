"""The operators of drafted tokens from their definitions, in 64 bits and one number after the other, on the host."""
import math

import torch

PAGE = 64
UNITS = 2 ** 40


def attention(q, k, v, n, words, scale):
    """q [n, heads, d], a sequence's keys and values [keys, kv, d] (its last n the step's own), ``words`` its tokens' ancestors or None -> (out fp64 [n, heads, d], and of
    every row the weighted sum of the values' magnitudes [n, heads, d] and the largest sum of |q k| scale of a key that it sees [n, heads])."""
    keys, kv = k.shape[:2]
    heads, d = q.shape[1:]
    out, size, terms = torch.zeros(n, heads, d, dtype=torch.float64), torch.zeros(n, heads, d, dtype=torch.float64), torch.zeros(n, heads, dtype=torch.float64)
    for t in range(n):
        seen = [j for j in range(keys) if j < keys - n or (j - (keys - n) <= t if words is None else words[t] >> (j - (keys - n)) & 1)]
        if not seen:
            continue
        for h in range(heads):
            kk, vv = k[seen, h * kv // heads].double(), v[seen, h * kv // heads].double()
            x = q[t, h].double()
            p = torch.softmax((kk @ x) * scale, 0)
            out[t, h], size[t, h] = p @ vv, p @ vv.abs()
            terms[t, h] = (kk.abs() @ x.abs()).max() * scale
    return out, size, terms


def ancestors(parents):
    """Words and depths of one sequence's tokens."""
    words, depth = [], []
    for i, p in enumerate(parents):
        there = 0 <= p < i
        words.append((words[p] if there else 0) | 1 << i)
        depth.append(depth[p] + 1 if there else 0)
    return words, depth


def signed(word):
    return word - (1 << 64) if word >> 63 else word


def kept(z, temperature, top_k, top_p, min_p):
    """Units of every token that the filters keep (list of whole numbers), and log-probabilities (fp64)."""
    z = z.float()
    vocab = z.numel()
    if not bool((z > -math.inf).any()) or temperature <= 0:
        best = int(torch.where(z.isnan(), torch.full_like(z, -math.inf), z).argmax())
        if not bool((z > -math.inf).any()):
            best = 0
        units = [0] * vocab
        units[best] = UNITS
        lp = torch.full((vocab,), -math.inf, dtype=torch.float64)
        lp[best] = 0.0 if bool((z > -math.inf).any()) else -math.inf
        return units, lp
    top = z[~z.isnan()].max()
    below = torch.where(z == math.inf, torch.zeros_like(z), torch.full_like(z, -math.inf)) if top == math.inf else (z - top) / torch.tensor(temperature)
    w = torch.where(below.isnan(), torch.zeros_like(below), torch.exp(below))
    units = [int(x * UNITS) for x in w.double().tolist()]
    order = sorted(range(vocab), key=lambda i: (-float(w[i]), i))
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        need = float(torch.tensor(top_p)) * float(sum(units[i] for i in order))
        run = 0
        for n, i in enumerate(order):
            run += units[i]
            if float(run) >= need:
                order = order[:n + 1]
                break
    if min_p > 0:
        order = [i for i in order if w[i] >= torch.tensor(min_p)] or order[:1]
    mine = set(order)
    units = [x if i in mine else 0 for i, x in enumerate(units)]
    return units, below.double() - math.log(sum(units) / UNITS)


def drawn(units, u):
    total = sum(units)
    target = min(int(float(u) * float(total)), total - 1)
    run = 0
    for i, x in enumerate(units):
        run += x
        if run > target:
            return i
    return 0


def verify(z, ids, uniform, settings, parents=None, probs=None, accept=None):
    """One sequence: rows z [n, vocab], its tokens, numbers and (temperature, top_k, top_p, min_p) -> (tokens, path, log-probabilities)."""
    tokens, path, logs, at = [], [0], [], 0
    n = len(ids)
    while True:
        units, lp = kept(z[at], *settings)
        total = sum(units)
        if probs is not None and at + 1 < n:
            q = [int(min(max(x, 0.0), 1.0) * float(total)) if x == x else 0 for x in probs[at].double().tolist()]
            x = ids[at + 1]
            if 0 <= x < len(units) and float(accept[at]) * float(q[x]) < float(units[x]):
                tokens.append(x)
                logs.append(float(lp[x]))
                at += 1
                path.append(at)
                continue
            rest = [max(0, a - b) for a, b in zip(units, q)]
            x = drawn(rest if sum(rest) else units, uniform[at])
            return tokens + [x], path, logs + [float(lp[x])]
        x = drawn(units, uniform[at])
        tokens.append(x)
        logs.append(float(lp[x]))
        if probs is not None:
            return tokens, path, logs
        up = parents if parents is not None else range(-1, n - 1)
        child = next((j for j in range(at + 1, n) if up[j] == at and ids[j] == x), None)
        if child is None:
            return tokens, path, logs
        at = child
        path.append(at)
