"""Operators of a cache held in 4 bits, of its pages, and of drawing tokens: the measured cases and their plain forms.

``run`` computes an operator either by elementary torch operations in 32 bits (``own`` False) or by the calls of
``cpmcu_b200`` that a user makes (``own`` True).  ``exact`` computes the same from the definitions in 64 bits.

A page of the 4-bit cache holds 64 tokens of one key-value head as one record of 64 * d + 1024 bytes: key codes, value codes,
key parameters, value parameters.  Every half row of d/2 channels has a bf16 scale s and a bf16 middle m, and a
code c (0..15) stands for m + s * (c - 8).  Where a code lies in the record is said at ``_places``.
"""
import functools
import math
import random

import torch

own = False

PAGE = 64
DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

# heads, key-value heads and head size of the two benchmark configurations, and of smaller ones
LAYERS_8B = {"heads": 32, "kv": 2, "d": 128}
LAYERS_HALF_B = {"heads": 16, "kv": 2, "d": 64}


def listed():
    return [
        # one decode step of a full batch of conversations: 64 new tokens are rotated, put into 4 bits and stored
        dict(name="store_step", op="store", seqs=64, tokens=1, history=4000, type="bf16", **LAYERS_HALF_B),
        # a full chunk of a prompt
        dict(name="store_prompt", op="store", seqs=1, tokens=2048, history=1000, type="bf16", **LAYERS_8B),
        # one conversation, one token: what a single user waits for
        dict(name="attend_one", op="attend", seqs=1, shortest=1000, longest=1000, queries=1, window=0, type="bf16", **LAYERS_8B),
        # a full batch of conversations of very unequal length
        dict(name="attend_batch", op="attend", seqs=64, shortest=1, longest=8192, queries=1, window=0, type="bf16", **LAYERS_HALF_B),
        # one document that is far longer than everything else
        dict(name="attend_long", op="attend", seqs=1, shortest=131071, longest=131071, queries=1, window=0, type="bf16", **LAYERS_8B),
        # a full chunk of a prompt behind a history
        dict(name="attend_prompt", op="attend", seqs=1, shortest=6149, longest=6149, queries=2048, window=0, type="bf16", **LAYERS_8B),
        # the 32-bit path, which replays and comparisons use
        dict(name="attend_fp32", op="attend", seqs=5, shortest=300, longest=2500, queries=1, window=0, type="fp32", **LAYERS_HALF_B),
        # seven further answers to one prompt: its last, partial page is copied for each in all layers
        dict(name="fork_pages", op="pages", lanes=24, kv=2, d=64, pages=64, moved=7, fork=True, type="bf16"),
        # what many ended conversations left is closed up: the last pages move into the holes
        dict(name="compact_pages", op="pages", lanes=32, kv=2, d=128, pages=600, moved=250, fork=False, type="bf16"),
        # one conversation's next token
        dict(name="sample_one", op="sample", rows=1, vocab=73448, top_k=50, top_p=0.9, min_p=0.0, temperature=0.8, mixed=False),
        # the next token of every conversation of a full batch, each with settings of its own
        dict(name="sample_batch", op="sample", rows=64, vocab=73448, top_k=200, top_p=0.95, min_p=0.02, temperature=1.0, mixed=True),
        # many rows of a smaller vocabulary by mass alone
        dict(name="sample_rows", op="sample", rows=512, vocab=32000, top_k=0, top_p=0.8, min_p=0.0, temperature=1.3, mixed=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "attend", "pages", "sample", "sample"])
    if op == "store":
        tokens = rng.choice([1, _log_int(rng, 2, 2048)])
        d = rng.choice([32, 64, 96, 128])
        return dict(op=op, seqs=_log_int(rng, 1, 64) if tokens == 1 else _log_int(rng, 1, max(1, min(16, 2048 // tokens))), tokens=tokens,
                    history=_log_int(rng, 1, 8000) - 1, type="bf16", heads=2 * rng.choice([1, 2, 3, 4, 8, 16]), kv=2, d=d)
    if op == "attend":
        queries = rng.choice([1, 1, _log_int(rng, 2, 2048)])
        kv, group, d = rng.choice([1, 2, 4]), rng.choice([1, 2, 3, 5, 8, 16]), rng.choice([32, 64, 64, 96, 128, 128])
        seqs = _log_int(rng, 1, 64) if queries == 1 else _log_int(rng, 1, max(1, min(4, 2048 // queries)))
        most = max(queries + 1, min(131071, 4_000_000 // (seqs * kv * d) if queries == 1 else 12_000_000 // (queries * seqs * kv)))
        longest = max(queries, _log_int(rng, 1, most))
        if queries > 1:
            while group > 1 and queries * longest * seqs * kv * group * d > 2048 * 6149 * 32 * 128:
                group -= 1
        return dict(op=op, seqs=seqs, shortest=max(queries, min(longest, _log_int(rng, 1, max(1, longest)))), longest=longest, queries=queries,
                    window=rng.choice([0, 0, _log_int(rng, 1, max(2, longest))]), type=rng.choice(["bf16", "bf16", "bf16", "fp32"]),
                    heads=kv * group, kv=kv, d=d)
    if op == "pages":
        pages = _log_int(rng, 16, 600)
        fork = rng.random() < 0.5
        return dict(op=op, lanes=_log_int(rng, 1, 32), kv=rng.choice([1, 2]), d=rng.choice([32, 64, 96, 128]), pages=pages,
                    moved=_log_int(rng, 1, max(1, pages // 3)), fork=fork, type=rng.choice(["bf16", "bf16", "fp32"]))
    return dict(op=op, rows=_log_int(rng, 1, 64), vocab=_log_int(rng, 300, 73448), top_k=rng.choice([0, 1, _log_int(rng, 2, 3000)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]), min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]),
                temperature=round(rng.uniform(0.3, 2.0), 3), mixed=rng.random() < 0.5)


def _lengths(case):
    """Keys and new tokens of each sequence, from the case alone."""
    n, lo, hi, q = case["seqs"], case["shortest"], case["longest"], case["queries"]
    kv = [hi if i == 0 else lo + (hi - lo) * ((i * 37 + 11) % 101) // 100 for i in range(n)]
    new = [q if i == 0 else max(1, q - (i * 7) % max(1, q // 3)) for i in range(n)]
    return kv, [min(a, b) for a, b in zip(new, kv)]


def _visible(case):
    """(query-key pairs that are seen, keys that some query sees) over all sequences."""
    pairs = keys = 0
    w = case["window"]
    for L, q in zip(*_lengths(case)):
        first = L - q
        if not w:
            pairs += q * first + q * (q + 1) // 2
            keys += L
        else:
            pairs += sum(min(w, p + 1) for p in range(first, L))
            keys += min(L, q + w - 1)
    return pairs, keys


def work(case):
    op = case["op"]
    if op == "pages":
        each = case["lanes"] * case["kv"] * PAGE * case["d"] * (2 if case["type"] == "bf16" else 4) * 2
        sources = 1 if case["fork"] else case["moved"]
        return {"bytes": each * (sources + case["moved"]) + 8 * case["moved"], "flops": 0}
    if op == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 28), "flops": 4 * case["rows"] * case["vocab"]}
    size, d, kv, heads = (2 if case["type"] == "bf16" else 4), case["d"], case["kv"], case["heads"]
    if op == "store":
        n = case["seqs"] * case["tokens"]
        # the projections read, the turned queries written, codes and parameters written, the values they stand for read back
        return {"bytes": n * ((heads + 2 * kv) * d * size + heads * d * size + kv * (d + 16) * 2 + 2 * kv * d * size), "flops": 8 * n * (heads + 2 * kv) * d}
    pairs, keys = _visible(case)
    n = sum(_lengths(case)[1])
    return {"bytes": keys * kv * (d + 16) + 2 * n * heads * d * size, "flops": 4 * pairs * heads * d}


# ---------------------------------------------------------------------------
# the 4-bit page by elementary operations
# ---------------------------------------------------------------------------

def _places(d, values, device):
    """Nibble number within the record of every code of a page: int64 [64 tokens, d].

    A page is cut into slices of 16 tokens of 8 * d bytes.  In a slice words of 32 bits follow one another by (pair of blocks of 16
    channels) and by 32 lanes.  Keys: lane = (token % 8) * 4 + (channel % 16) / 4, a word holds eight channels of one token.
    Values: lane = ((channel % 16) / 2) * 4 + (token % 8) / 2, a word holds four channels of two neighbouring tokens."""
    t = torch.arange(PAGE, device=device)[:, None]
    c = torch.arange(d, device=device)[None, :]
    block, r = c // 16, t % 16
    pair, odd = block // 2, block % 2
    if values:
        lane = (c % 16) // 2 * 4 + (r % 8) // 2
        nibble = (r % 2) * 4 + odd * 2 + c % 2
    else:
        lane = (r % 8) * 4 + (c % 16) // 4
        nibble = 2 * odd + (c % 4) // 2 + 4 * (c % 2)
    run = 2 if d % 64 == 0 else 1                     # pairs of blocks that lie together, so that a lane reads 16 or 8 bytes
    byte = (t // 16) * (8 * d) + (pair // run) * (256 * run) + lane * (8 * run) + (pair % run) * 8 + (r // 8) * 4
    return (byte + (32 * d if values else 0)) * 2 + nibble


def _to_codes(x):
    """x fp32 [..., d] -> codes uint8 [..., d], scale and middle bf16 [..., 2]."""
    h = x.unflatten(-1, (2, -1))
    lo, hi = h.amin(-1), h.amax(-1)
    scale = ((hi - lo) / 15.0).bfloat16()
    s = scale.float()
    middle = (lo + 8.0 * s).bfloat16()
    inverse = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    c = torch.round((h - middle.float()[..., None]) * inverse[..., None]) + 8.0
    return c.clamp(0, 15).to(torch.uint8).flatten(-2), scale, middle


def _nibbles(records):
    return torch.stack((records & 15, records >> 4), dim=-1).flatten(-2)


def _bytes(nibbles):
    pairs = nibbles.unflatten(-1, (-1, 2))
    return pairs[..., 0] | (pairs[..., 1] << 4)


def _parameters(records, d):
    """(scale, middle) fp32 [..., 2 (keys, values), 64, 2] of records [..., bytes]."""
    p = records[..., 64 * d:].contiguous().view(torch.bfloat16).float().unflatten(-1, (2, PAGE, 2, 2))
    return p[..., 0], p[..., 1]


def _values(records, d):
    """What records [..., 64 * d + 1024] stand for: keys and values fp32 [..., 64, d]."""
    nib = _nibbles(records[..., :64 * d])
    scale, middle = _parameters(records, d)
    k = nib[..., _places(d, False, records.device)].float()
    v = nib[..., _places(d, True, records.device)].float()
    each = lambda c, i: (middle[..., i, :, :, None] + scale[..., i, :, :, None] * (c.unflatten(-1, (2, -1)) - 8.0)).flatten(-2)  # noqa: E731
    return each(k, 0), each(v, 1)


def _records(k, v, d):
    """Records uint8 [..., 64 * d + 1024] of keys and values fp32 [..., 64, d]."""
    kc, ks, km = _to_codes(k)
    vc, vs, vm = _to_codes(v)
    nib = torch.zeros(*k.shape[:-2], 128 * d, dtype=torch.uint8, device=k.device)
    nib[..., _places(d, False, k.device)] = kc
    nib[..., _places(d, True, k.device)] = vc
    par = torch.stack((torch.stack((ks, km), -1), torch.stack((vs, vm), -1)), dim=-4)      # [..., 2, 64, 2, 2]
    return torch.cat((_bytes(nib), par.flatten(-4).contiguous().view(torch.uint8)), -1)


# ---------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------

def _inv_freq(d):
    return (1.0 / 10000.0 ** (torch.arange(0, d, 2, dtype=torch.float32) / d)).to(DEVICE)


def _tables(g, pages_per_seq):
    """Page table int32 [slots, pages], the sequences' slots int32, and the number of pages; pages lie in no order."""
    n, most = len(pages_per_seq), max(1, max(pages_per_seq))
    total = sum(pages_per_seq) + 1
    order = torch.randperm(total, generator=g, device=DEVICE).to(torch.int32)
    slots = torch.randperm(n, generator=g, device=DEVICE).to(torch.int32)
    table = torch.zeros(n, most, dtype=torch.int32, device=DEVICE)
    counts = torch.tensor(pages_per_seq, device=DEVICE)
    at = torch.cumsum(counts, 0) - counts
    col = torch.arange(most, device=DEVICE)[None, :]
    rows = torch.where(col < counts[:, None], order[(at[:, None] + col).clamp(max=total - 1)], torch.zeros_like(table))
    table[slots.long()] = rows
    return table, slots, total, order[-1:]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    op = case["op"]
    if op == "pages":
        shape = (case["lanes"], case["pages"], case["kv"])
        dtype = TYPES[case["type"]]
        k = torch.empty(*shape, PAGE, case["d"], dtype=dtype, device=DEVICE).normal_(generator=g)
        v = torch.empty(*shape, case["d"], PAGE, dtype=dtype, device=DEVICE).normal_(generator=g)
        order = torch.randperm(case["pages"], generator=g, device=DEVICE).to(torch.int32)
        m = case["moved"]
        src, dst = order[:m].clone(), order[m:2 * m].clone()
        if case["fork"]:
            src = src[:1].repeat(m)
        return {"case": case, "k": k, "v": v, "src": src, "dst": dst}
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # many unlikely tokens and a few likely ones, as a model's logits have them
        logits = normal(rows, vocab) * 1.7
        few = min(vocab, 60)
        places = torch.randint(0, vocab, (rows, few), generator=g, device=DEVICE)
        logits.scatter_add_(1, places, normal(rows, few).abs() * 3.0 + 4.0)
        f = lambda v: torch.full((rows,), float(v), device=DEVICE)  # noqa: E731
        temperature, top_p, min_p = f(case["temperature"]), f(case["top_p"]), f(case["min_p"])
        top_k = torch.full((rows,), case["top_k"], dtype=torch.int32, device=DEVICE)
        if case["mixed"]:                          # every conversation has settings of its own, some of them greedy, some without limits
            i = torch.arange(rows, device=DEVICE)
            temperature = torch.where(i % 5 == 4, torch.zeros_like(temperature), temperature * (0.5 + (i % 7) / 7.0))
            top_k = torch.where(i % 3 == 1, torch.zeros_like(top_k), top_k)
            top_p = torch.where(i % 4 == 2, torch.ones_like(top_p), top_p)
            min_p = torch.where(i % 2 == 1, torch.zeros_like(min_p), min_p)
        return {"case": case, "logits": logits, "uniform": torch.rand(rows, generator=g, device=DEVICE), "temperature": temperature,
                "top_k": top_k, "top_p": top_p, "min_p": min_p}
    heads, kv, d, dtype = case["heads"], case["kv"], case["d"], TYPES[case["type"]]
    size = 64 * d + 1024
    # some key channels are far larger than the others in every token
    loud = 1.0 + 4.0 * (torch.rand(kv, 1, d, generator=g, device=DEVICE) > 0.95).float()
    if op == "store":
        n, seqs = case["tokens"], case["seqs"]
        first = [max(0, case["history"] - 13 * i) for i in range(seqs)]
        table, slots, total, spare = _tables(g, [(f + n + PAGE - 1) // PAGE for f in first])
        qkv = normal(seqs * n, heads + 2 * kv, d)
        qkv[:, heads:heads + kv] *= loud[:, 0]
        return {"case": case, "qkv": qkv.flatten(1).to(dtype), "positions": (i32(first)[:, None] + torch.arange(n, device=DEVICE, dtype=torch.int32)).flatten(),
                "token_seq": torch.arange(seqs, device=DEVICE, dtype=torch.int32).repeat_interleave(n), "slots": slots, "table": table,
                "inv_freq": _inv_freq(d), "spare": spare.long(), "first": i32(first),
                "records": torch.randint(0, 256, (total, kv, size), generator=g, device=DEVICE, dtype=torch.uint8)}
    lengths, new = _lengths(case)
    table, slots, total, _ = _tables(g, [(n + PAGE - 1) // PAGE for n in lengths])
    records = torch.empty(total, kv, size, dtype=torch.uint8, device=DEVICE)
    for at in range(0, total, 256):                                 # in pieces, for the memory
        n = min(256, total - at)
        records[at:at + n] = _records(normal(n, kv, PAGE, d) * loud, normal(n, kv, PAGE, d) + 0.3, d)
    # what the pages hold behind a sequence's last token is what earlier sequences left there, with parameters that are no numbers among it
    last = i32([(n - 1) // PAGE for n in lengths])
    page = table[slots.long(), last.long()].long()
    par = records[page][..., 64 * d:].contiguous().view(torch.bfloat16).unflatten(-1, (2, PAGE, 4))
    behind = torch.arange(PAGE, device=DEVICE)[None, :] > (i32(lengths) - 1)[:, None] % PAGE
    par = torch.where(behind[:, None, None, :, None], torch.full_like(par, float("nan")), par)
    records[page] = torch.cat((records[page][..., :64 * d], par.flatten(-3).contiguous().view(torch.uint8)), -1)
    q = normal(sum(new), heads, d) * 0.8
    cu = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
    tiles = [(i, r) for i, n in enumerate(new) for r in range(0, n, PAGE)]
    return {"case": case, "q": q.to(dtype), "records": records, "table": table, "slots": slots, "kv_len": i32(lengths), "cu_q": cu,
            "tiles": (i32([t[0] for t in tiles]), i32([t[1] for t in tiles]), len(tiles)), "scale": 1.0 / math.sqrt(d)}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _ops(dtype):
    from cpmcu_b200.ops.ops import Ops
    return Ops(dtype, DEVICE)


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        return {"store": _store_own, "attend": _attend_own, "pages": _pages_own, "sample": _sample_own}[op](s, case)
    return {"store": _store, "attend": _attend, "pages": _pages, "sample": _sample}[op](s, case)


def _store_own(s, case):
    ops = _ops(s["qkv"].dtype)
    kv, d = case["kv"], case["d"]
    q = ops.rope_store_kv4(s["qkv"], case["heads"], kv, d, s["positions"], s["token_seq"], s["slots"], s["table"], s["records"],
                           s["inv_freq"], 1.0, d)
    k, v = ops.kv4_values(s["records"], s["positions"], s["token_seq"], s["slots"], s["table"], kv, d)
    return q, k, v


def _store(s, case):
    heads, kv, d = case["heads"], case["kv"], case["d"]
    dtype = s["qkv"].dtype
    x = s["qkv"].float().unflatten(1, (heads + 2 * kv, d))
    angle = s["positions"].float()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[:, :heads + kv, :d // 2], x[:, :heads + kv, d // 2:]
    turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    k, v = turned[:, heads:], x[:, heads + kv:]
    kc, ks, km = _to_codes(k)
    vc, vs, vm = _to_codes(v)
    # the pages that the new tokens lie in, as far as the sequence with the most of them needs (the others' rest goes to a spare page)
    first_page = s["first"] // PAGE
    n_pages = (case["tokens"] + 2 * PAGE - 2) // PAGE
    n_pages = min(n_pages, s["table"].shape[1])
    col = first_page[:, None] + torch.arange(n_pages, device=x.device)
    ends = (s["first"] + case["tokens"] - 1) // PAGE
    page = torch.where(col <= ends[:, None], s["table"][s["slots"].long()].gather(1, col.clamp(max=s["table"].shape[1] - 1).long()).long(), s["spare"])
    records = s["records"][page]                                                        # [seqs, pages, kv, bytes]
    nib = _nibbles(records[..., :64 * d]).transpose(1, 2).flatten(2)                      # [seqs, kv, pages * 128 d]
    par = records[..., 64 * d:].contiguous().view(torch.bfloat16).unflatten(-1, (2, PAGE, 4)).clone()
    seq = s["token_seq"].long()
    mine = (s["positions"].long() // PAGE) - first_page.long()[seq]
    inside = s["positions"].long() % PAGE
    head = torch.arange(kv, device=x.device)
    for values, codes in ((False, kc), (True, vc)):
        at = mine[:, None] * (128 * d) + _places(d, values, x.device)[inside]             # [tokens, d]
        nib[seq[:, None, None], head[None, :, None], at[:, None, :]] = codes
    for i, (scale, middle) in enumerate(((ks, km), (vs, vm))):
        par[seq[:, None], mine[:, None], head[None, :], i, inside[:, None]] = torch.stack((scale, middle), -1).flatten(-2)
    nib = nib.unflatten(2, (n_pages, 128 * d)).transpose(1, 2)
    records = torch.cat((_bytes(nib), par.flatten(-3).contiguous().view(torch.uint8)), -1)
    s["records"][page] = records
    k, v = _values(records, d)
    take = lambda t: t[seq, mine, :, inside].to(dtype)  # noqa: E731
    return turned[:, :heads].to(dtype), take(k), take(v)


def _attend_own(s, case):
    ops = _ops(s["q"].dtype)
    prompt = dict(cu_q=s["cu_q"], tiles=s["tiles"]) if case["queries"] > 1 else {}
    return ops.kv4_attention(s["q"], s["records"], s["kv_len"], s["slots"], s["table"], case["kv"], s["scale"], window=case["window"], **prompt)


def _attend(s, case):
    heads, kv, d, most = case["heads"], case["kv"], case["d"], case["queries"]
    q, cu, kv_len = s["q"], s["cu_q"].long(), s["kv_len"].long()
    k, v = _values(s["records"][s["table"][s["slots"].long()].long()], d)                 # [seqs, pages, kv, 64, d]
    k, v = (t.transpose(1, 2).flatten(2, 3) for t in (k, v))                              # [seqs, kv, keys, d]
    n_q = cu[1:] - cu[:-1]
    i = torch.arange(most, device=q.device)
    x = q.float()[(cu[:-1, None] + i).clamp(max=q.shape[0] - 1)].unflatten(2, (kv, -1))   # [seqs, most, kv, group, d]
    x = x.permute(0, 2, 3, 1, 4).flatten(2, 3)
    j = torch.arange(k.shape[2], device=q.device)
    there = j < kv_len[:, None]
    k, v = (torch.where(there[:, None, :, None], t, torch.zeros_like(t)) for t in (k, v))
    own_place = (kv_len - n_q)[:, None] + i
    seen = (j <= own_place[..., None]) & there[:, None]
    if case["window"]:
        seen = seen & (j > own_place[..., None] - case["window"])
    score = (x @ k.transpose(-1, -2)) * s["scale"]                                        # [seqs, kv, group * most, keys]
    score = score.unflatten(2, (-1, most)).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v).unflatten(2, (-1, most)) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 3, 1, 2, 4).flatten(2)                                           # [seqs, most, heads * d]
    return out[i < n_q[:, None]].to(q.dtype) if most > 1 else out[:, 0].to(q.dtype)


def _pages_own(s, case):
    _ops(torch.bfloat16).copy_pages([s["k"], s["v"]], s["src"], s["dst"])
    return s["k"], s["v"]


def _pages(s, case):
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return s["k"], s["v"]


def _sample_own(s, case):
    return _ops(torch.bfloat16).sample_filtered(s["logits"], s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


# A token's weight exp((z - max) / T) is held as a whole number of units of 2^-40, so that sums have no order.
UNIT = float(2 ** 40)


def _sample(s, case):
    z = s["logits"]
    vocab = z.shape[1]
    greedy = s["temperature"] <= 0
    top = z.amax(1, keepdim=True)
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"])[:, None]
    w = torch.exp((z - top) / t)
    weight = (w.double() * UNIT).long()
    order = torch.argsort(w, dim=1, descending=True, stable=True)
    mass = weight.gather(1, order).cumsum(1)
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab).long().clamp(max=vocab)
    within = mass.gather(1, k[:, None] - 1)
    need = s["top_p"].clamp(max=1.0).double()[:, None] * within.double()
    by_mass = torch.where(s["top_p"] < 1, 1 + (mass.double() < need).sum(1), vocab)
    by_ratio = torch.where(s["min_p"] > 0, (w >= s["min_p"][:, None]).sum(1), vocab)
    kept = torch.minimum(torch.minimum(k, by_mass), by_ratio).clamp(min=1)
    kept = torch.where(greedy, torch.ones_like(kept), kept)
    keep = torch.zeros_like(z, dtype=torch.bool).scatter(1, order, torch.arange(vocab, device=z.device) < kept[:, None])
    c = torch.where(keep, weight, 0).cumsum(1)
    total = c[:, -1:]
    target = torch.minimum((s["uniform"].double()[:, None] * total.double()).long(), total - 1)
    token = (c <= target).sum(1)
    chosen = (z.gather(1, token[:, None]) - top) / t
    logprob = chosen[:, 0] - torch.log((total[:, 0].double() / UNIT).float())
    return token.int(), torch.where(greedy, torch.zeros_like(logprob), logprob)


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _store_exact, "attend": _attend_exact, "pages": _pages_exact, "sample": _sample_exact}[case["op"]](s, case)


def _pages_exact(s, case):
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        for t in (s["k"], s["v"]):
            t[:, b] = t[:, a]
    return s["k"], s["v"]


def _half_rows(x):
    """The values that a row's 4-bit form stands for, in 64 bits."""
    out = torch.empty_like(x)
    half = x.shape[-1] // 2
    for i in range(2):
        part = x[..., i * half:(i + 1) * half]
        low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        s = ((high - low) / 15).bfloat16().double()
        m = (low + 8 * s).bfloat16().double()
        code = torch.where(s > 0, torch.round((part - m) / s), torch.zeros_like(part)).clamp(-8, 7)
        out[..., i * half:(i + 1) * half] = m + s * code
    return out


def _store_exact(s, case):
    heads, kv, d = case["heads"], case["kv"], case["d"]
    x = s["qkv"].double().view(-1, heads + 2 * kv, d)
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=x.device), s["positions"].double()[:, None] * s["inv_freq"].double())[:, None]
    z = torch.complex(x[:, :heads + kv, :d // 2].contiguous(), x[:, :heads + kv, d // 2:].contiguous()) * turn
    turned = torch.cat((z.real, z.imag), -1)
    return turned[:, :heads], _half_rows(turned[:, heads:]), _half_rows(x[:, heads + kv:])


@functools.lru_cache(maxsize=None)
def _where_codes(d, values):
    """Byte and shift of every code of a page, one by one from the description of the layout."""
    byte, shift = [], []
    together = 2 if d % 64 == 0 else 1
    for token in range(PAGE):
        for channel in range(d):
            row, block, e = token % 16, channel // 16, channel % 16
            if values:
                lane, nib = (e // 2) * 4 + (row % 8) // 2, 4 * (row % 2) + 2 * (block % 2) + e % 2
            else:
                lane, nib = (row % 8) * 4 + e // 4, 2 * (block % 2) + (e % 4) // 2 + 4 * (e % 2)
            at = (token // 16) * 8 * d + (block // 2 // together) * 256 * together + lane * 8 * together + (block // 2 % together) * 8 + (row // 8) * 4
            byte.append((32 * d if values else 0) + at + nib // 2)
            shift.append(4 * (nib % 2))
    return torch.tensor(byte, device=DEVICE), torch.tensor(shift, device=DEVICE, dtype=torch.uint8)


def _rows_exact(records, head, d, values):
    """Keys or values of one head of a sequence's records [pages, kv, bytes], fp64 [pages * 64, d]."""
    r = records[:, head]
    byte, shift = _where_codes(d, values)
    code = ((r[:, byte] >> shift) & 15).double().view(-1, 2, d // 2)
    at = 64 * d + (512 if values else 0)
    par = r[:, at:at + 512].contiguous().view(torch.bfloat16).double().view(-1, 2, 2)
    return (par[..., 1:] + par[..., :1] * (code - 8)).view(-1, d)


def _attend_exact(s, case):
    heads, kv, d = case["heads"], case["kv"], case["d"]
    out = torch.zeros(s["q"].shape[0], heads, d, dtype=torch.float64, device=DEVICE)
    cu, lengths, slots = s["cu_q"].tolist(), s["kv_len"].tolist(), s["slots"].tolist()
    for i, n in enumerate(lengths):
        records = s["records"][s["table"][slots[i], :(n + PAGE - 1) // PAGE].long()]
        rows = torch.arange(cu[i], cu[i + 1], device=DEVICE)
        place = rows - cu[i + 1] + n
        j = torch.arange(n, device=DEVICE)
        hidden = j[None] > place[:, None]
        if case["window"]:
            hidden = hidden | (j[None] <= place[:, None] - case["window"])
        for h in range(kv):
            k, v = (_rows_exact(records, h, d, values)[:n] for values in (False, True))
            for e in range(h * (heads // kv), (h + 1) * (heads // kv)):
                score = s["q"][rows, e].double() @ k.T * s["scale"]
                out[rows, e] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v
    return out.flatten(1)


def _sample_exact(s, case):
    z = s["logits"].double()
    found = torch.zeros(z.shape[0], dtype=torch.float64, device=DEVICE)
    for i in range(z.shape[0]):
        t, k, p, low = (float(s[n][i]) for n in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            continue
        prob = torch.softmax(z[i] / t, 0)
        ranked, order = torch.sort(prob, descending=True, stable=True)
        n = int(k) if k > 0 else z.shape[1]
        ranked, order = ranked[:n], order[:n]
        if p < 1:
            n = int((ranked.cumsum(0) < p * ranked.sum()).sum()) + 1
            ranked, order = ranked[:n], order[:n]
        if low > 0:
            n = max(1, int((ranked >= low * ranked[0]).sum()))
            ranked, order = ranked[:n], order[:n]
        by_index, back = torch.sort(order)
        c = ranked[back].cumsum(0)
        at = int((c <= float(s["uniform"][i]) * c[-1]).sum().clamp(max=len(c) - 1))
        found[i] = torch.log(prob[by_index[at]] / ranked.sum())
    return None, found
