"""The 4-bit cache, copying of pages and filtered sampling by their definitions, in 64 bits where a number is computed.

Shares no code with the package; the tests compare the kernels with it."""
import math

import torch


def quantised(x: torch.Tensor):
    """Rows x [..., d] -> (values they are stored as, fp32 [..., d]; scales fp32 [..., 2]).  Half a row from lo to hi: s = bf16((hi - lo) / 15),
    m = bf16(lo + 8 s), c = clamp(round((x - m) / s) + 8, 0, 15), value m + s (c - 8).  Every step is rounded to 32 bits once."""
    h = x.float().unflatten(-1, (2, -1))
    lo, hi = h.amin(-1), h.amax(-1)
    s = ((hi - lo) / 15.0).bfloat16().float()
    m = (lo + 8.0 * s).bfloat16().float()
    inverse = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    c = (torch.round((h - m[..., None]) * inverse[..., None]) + 8.0).clamp(0, 15)
    v = m[..., None] + s[..., None] * (c - 8.0)
    return v.flatten(-2), s


def rotated(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, magnitude: float) -> torch.Tensor:
    """x [tokens, heads, d]: pairs (c, c + d/2) turned by position * inv_freq[c], in 64 bits."""
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin = angle.cos()[:, None] * magnitude, angle.sin()[:, None] * magnitude
    a, b = x.double().chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def attention(q, k, v, first: int, scale: float, window: int) -> torch.Tensor:
    """q [tokens, heads, d] at positions first, first + 1, ... against k, v [keys, kv, d], in 64 bits -> [tokens, heads, d]; a query
    that sees no key gives zeros.  Keys that a query does not see have no part in it, whatever they hold."""
    n, heads, d = q.shape
    out = torch.zeros(n, heads, d, dtype=torch.float64)
    group = heads // k.shape[1]
    for i in range(n):
        p = first + i
        lo, hi = (max(0, p - window + 1) if window else 0), min(p + 1, k.shape[0])
        if hi <= lo:
            continue
        for h in range(heads):
            s = k[lo:hi, h // group].double() @ q[i, h].double() * scale
            out[i, h] = torch.softmax(s, 0) @ v[lo:hi, h // group].double()
    return out


UNIT = 2.0 ** 40


def sampled(z: torch.Tensor, u: float, t: float, k: int, p: float, ratio: float):
    """(token, log-probability) of one row of logits, by the definition: weights are whole multiples of 2^-40 of the largest."""
    z = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z.float())
    top = float(z.max())
    if top == -math.inf:
        return 0, -math.inf
    if not t > 0:
        return int((z == top).nonzero()[0]), 0.0
    x = torch.where(z == top, torch.zeros_like(z), (z - top) / torch.tensor(t))
    w = torch.exp(x)
    weight = [int(float(a) * UNIT) for a in w]
    order = sorted(range(len(weight)), key=lambda i: (-float(w[i]), i))
    if p <= 0 or ratio > 1:
        k = 1
    kept = order[:k] if k > 0 else order
    if p < 1 and p > 0:
        need, run, n = float(torch.tensor(p)) * float(sum(weight[i] for i in kept)), 0, 0
        while float(run) < need:
            run += weight[kept[n]]
            n += 1
        kept = kept[:max(1, n)]
    if ratio > 0:
        kept = [i for i in kept if float(w[i]) >= float(torch.tensor(ratio))] or kept[:1]
    kept = sorted(kept)
    total = sum(weight[i] for i in kept)
    target = min(int(float(torch.tensor(u)) * float(total)), total - 1)
    run = 0
    for i in kept:
        run += weight[i]
        if run > target:
            return i, float(x[i].double()) - math.log(total / UNIT)
    raise AssertionError("the running sum ends at the total")
