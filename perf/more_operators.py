"""Operators of drafted tokens: the measured cases and their plain forms.

A sequence whose cache holds some tokens brings a few more at once: its last token (the root) and tokens that were drafted to follow it, one
behind the other (a chain) or as a tree.  ``step_tables`` makes the step's description from the requests' lengths, ``draft_attention`` lets every token see the
tokens before the step and of the step's its ancestors, ``verify_drafts`` accepts a path of drafted tokens and draws one more, and ``keep_drafts`` moves the
accepted ones' keys and values to where the sequence goes on.

``run`` computes an operator either by elementary torch operations (``own`` False) or by the calls of ``cpmcu_b200`` that a user makes (``own``
True).  ``exact`` computes the same from the definitions, in 64 bits.
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

# heads, key-value heads and head size of the two benchmark configurations
LAYERS_8B = {"heads": 32, "kv": 2, "d": 128}
LAYERS_HALF_B = {"heads": 16, "kv": 2, "d": 64}


def listed():
    return [
        # one conversation, four tokens drafted in a row: what a single user waits for
        dict(name="attend_one", op="attend", seqs=1, shortest=1000, longest=1000, tokens=5, tree=False, type="bf16", **LAYERS_8B),
        # a full batch of conversations of very unequal length, each with a few drafted tokens
        dict(name="attend_batch", op="attend", seqs=64, shortest=6, longest=8192, tokens=5, tree=False, type="bf16", **LAYERS_HALF_B),
        # some conversations with a small tree each
        dict(name="attend_trees", op="attend", seqs=16, shortest=500, longest=6000, tokens=16, tree=True, type="bf16", **LAYERS_8B),
        # one document that is far longer than everything else, and the largest tree
        dict(name="attend_long", op="attend", seqs=1, shortest=131071, longest=131071, tokens=64, tree=True, type="bf16", **LAYERS_8B),
        # the 32-bit path, which replays and comparisons use
        dict(name="attend_fp32", op="attend", seqs=3, shortest=300, longest=2500, tokens=7, tree=True, type="fp32", **LAYERS_HALF_B),
        # one conversation's drafted tokens against a small model's probabilities
        dict(name="verify_one", op="verify", seqs=1, tokens=5, vocab=73448, tree=False, probs=True, top_k=50, top_p=0.9, min_p=0.0, temperature=0.8, mixed=False),
        # a full batch of them, each conversation with settings of its own
        dict(name="verify_batch", op="verify", seqs=64, tokens=5, vocab=73448, tree=False, probs=True, top_k=200, top_p=0.95, min_p=0.02, temperature=1.0, mixed=True),
        # trees of looked-up continuations, which have no probabilities
        dict(name="verify_trees", op="verify", seqs=32, tokens=16, vocab=32000, tree=True, probs=False, top_k=0, top_p=0.8, min_p=0.0, temperature=0.7, mixed=True),
        # one conversation accepted four tokens of a tree: they move together in all layers
        dict(name="keep_one", op="keep", lanes=32, kv=2, d=128, seqs=1, tokens=64, accepted=5, history=4000, type="bf16"),
        # a full batch's accepted tokens
        dict(name="keep_batch", op="keep", lanes=24, kv=2, d=64, seqs=64, tokens=16, accepted=6, history=1000, type="bf16"),
        # the description of one batch's step, whose pages are there
        dict(name="tables_step", op="tables", seqs=64, tokens=5, history=4000, tree=False, pages=False),
        # the description of a large batch of trees, pages handed out on the way
        dict(name="tables_trees", op="tables", seqs=512, tokens=64, history=2000, tree=True, pages=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "verify", "verify", "keep", "tables"])
    if op == "attend":
        kv, group, d = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 5, 8, 16]), rng.choice([32, 64, 64, 96, 128, 128])
        seqs, tokens = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        type_ = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        most = min(131071, 8_000_000 // (seqs * kv * d) * (4 if d < 64 else 1), 128_000_000 // (seqs * kv * group * tokens) // (8 if type_ == "fp32" else 1))
        longest = max(tokens, _log_int(rng, 1, max(2, most)))
        return dict(op=op, seqs=seqs, shortest=max(tokens, min(longest, _log_int(rng, 1, max(2, longest)))), longest=longest, tokens=tokens,
                    tree=rng.random() < 0.6, type=type_, heads=kv * group, kv=kv, d=d)
    if op == "verify":
        vocab = _log_int(rng, 300, 73448)
        tokens = _log_int(rng, 2, 32)
        probs = rng.random() < 0.6
        return dict(op=op, seqs=_log_int(rng, 1, max(2, min(64, 12_000_000 // (vocab * tokens)))), tokens=tokens, vocab=vocab, tree=not probs and rng.random() < 0.7,
                    probs=probs, top_k=rng.choice([0, 1, _log_int(rng, 2, 2000)]), top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                    min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]), temperature=round(rng.uniform(0.3, 2.0), 3), mixed=rng.random() < 0.5)
    if op == "keep":
        tokens = _log_int(rng, 2, 64)
        return dict(op=op, lanes=_log_int(rng, 1, 32), kv=rng.choice([1, 2, 4]), d=rng.choice([32, 64, 96, 128]), seqs=_log_int(rng, 1, 64), tokens=tokens,
                    accepted=rng.randint(1, tokens), history=_log_int(rng, 1, 2000) - 1, type=rng.choice(["bf16", "bf16", "fp32"]))
    return dict(op=op, seqs=_log_int(rng, 1, 512), tokens=_log_int(rng, 1, 64), history=_log_int(rng, 1, 8000) - 1, tree=rng.random() < 0.6,
                pages=rng.random() < 0.6)


def _new(case):
    """Tokens that each sequence brings, from the case alone."""
    n = case["tokens"]
    return [n if i == 0 else max(1, n - (i * 7) % max(1, n // 2)) for i in range(case["seqs"])]


def _lengths(case):
    """Keys of each sequence, the step's tokens among them."""
    lo, hi = case["shortest"], case["longest"]
    return [hi if i == 0 else lo + (hi - lo) * ((i * 37 + 11) % 101) // 100 for i in range(case["seqs"])]


def work(case):
    op, new = case["op"], _new(case)
    if op == "attend":
        size, d, kv, heads = (2 if case["type"] == "bf16" else 4), case["d"], case["kv"], case["heads"]
        lengths = _lengths(case)
        return {"bytes": 2 * sum(lengths) * kv * d * size + 2 * sum(new) * heads * d * size,
                "flops": 4 * heads * d * sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, lengths))}
    if op == "verify":
        rows = sum(new)
        return {"bytes": 4 * case["vocab"] * (rows + (rows - len(new) if case["probs"] else 0)), "flops": 4 * rows * case["vocab"]}
    if op == "keep":
        moved = sum(min(case["accepted"], n) - 1 for n in new)
        return {"bytes": 4 * max(1, moved) * case["lanes"] * case["kv"] * case["d"] * (2 if case["type"] == "bf16" else 4), "flops": 0}
    return {"bytes": 20 * len(new) + sum(new) * (24 + (12 if case["tree"] else 0)), "flops": 0}


# ---------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------

def _parents(g, new, tree):
    """Parents of the packed tokens (int32; a sequence's first has none), one of the six tokens before it in a tree."""
    cu, seq, i = _packed(new)
    back = torch.randint(1, 7, (len(seq),), generator=g, device=DEVICE) if tree else torch.ones(len(seq), dtype=torch.int64, device=DEVICE)
    return torch.where(i == 0, -1, (i - back).clamp(min=0)).int()


def _packed(new):
    """Offsets [seqs + 1], and for every token its sequence and its place among its sequence's new ones (int64)."""
    n = torch.tensor(new, device=DEVICE)
    cu = torch.cat((torch.zeros(1, dtype=torch.int64, device=DEVICE), n.cumsum(0)))
    seq = torch.arange(len(new), device=DEVICE).repeat_interleave(n)
    return cu, seq, torch.arange(sum(new), device=DEVICE) - cu[seq]


def _tables(g, pages_per_seq, spare=0):
    """Page table int32 [slots, pages], the sequences' slots int32, the number of pages, and ``spare`` further pages; pages lie in no order."""
    n, most = len(pages_per_seq), max(1, max(pages_per_seq))
    total = sum(pages_per_seq) + spare + 1
    order = torch.randperm(total, generator=g, device=DEVICE).to(torch.int32)
    slots = torch.randperm(n, generator=g, device=DEVICE).to(torch.int32)
    table = torch.zeros(n, most, dtype=torch.int32, device=DEVICE)
    counts = torch.tensor(pages_per_seq, device=DEVICE)
    at = torch.cumsum(counts, 0) - counts
    col = torch.arange(most, device=DEVICE)[None, :]
    table[slots.long()] = torch.where(col < counts[:, None], order[(at[:, None] + col).clamp(max=total - 1)], torch.zeros_like(table))
    return table, slots, total, order[total - 1 - spare:total - 1]


def _pages(tokens):
    return (tokens + PAGE - 1) // PAGE


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    op, new = case["op"], _new(case)
    cu, seq, inside = _packed(new)
    if op == "tables":
        held = [max(0, case["history"] - 13 * i % (case["history"] + 1)) for i in range(case["seqs"])]
        want = [_pages(h + n) - _pages(h) for h, n in zip(held, new)]
        table, slots, _, spare = _tables(g, [_pages(h + (0 if case["pages"] else n)) for h, n in zip(held, new)], sum(want) + 7)
        if case["pages"]:                               # room for the step's
            table = torch.cat((table, torch.zeros(len(new), 1 + _pages(case["tokens"]), dtype=torch.int32, device=DEVICE)), 1)
        return {"case": case, "lengths": i32(held), "new": i32(new), "slots": slots, "table": table, "n": sum(new),
                "parents": _parents(g, new, True) if case["tree"] else None, "free": spare.clone() if case["pages"] else None}
    if op == "keep":
        lanes, kv, d, dtype = case["lanes"], case["kv"], case["d"], TYPES[case["type"]]
        held = [max(0, case["history"] - 13 * i % (case["history"] + 1)) for i in range(case["seqs"])]
        # only the pages that the step's tokens lie in are made, the others' numbers go to one page
        first = [h // PAGE for h in held]
        mine = [_pages(h + n) - f for h, n, f in zip(held, new, first)]
        table, slots, total, spare = _tables(g, mine, 1)
        wide = spare.repeat(case["seqs"] * max(f + m for f, m in zip(first, mine))).view(case["seqs"], -1).clone()
        col = torch.arange(table.shape[1], device=DEVICE)
        row = slots.long()
        at = torch.tensor(first, device=DEVICE)[:, None] + col
        there = col < torch.tensor(mine, device=DEVICE)[:, None]
        wide[row[:, None].expand_as(at)[there], at[there]] = table[row][there]
        k = torch.empty(lanes, total, kv, PAGE, d, dtype=dtype, device=DEVICE).normal_(generator=g)
        v = torch.empty(lanes, total, kv, d, PAGE, dtype=dtype, device=DEVICE).normal_(generator=g)
        # an accepted path: the root, and tokens that lie further and further back
        most = max(new)
        places = torch.rand(len(new), most, generator=g, device=DEVICE)
        places = torch.where(torch.arange(most, device=DEVICE) < i32(new)[:, None], places, 2.0)
        places[:, 0] = -1.0
        count = i32([min(case["accepted"], n) for n in new])
        chosen = places.argsort(1)
        path = torch.where(torch.arange(most, device=DEVICE) < count[:, None], chosen, most).sort(1).values
        path = torch.where(path < most, path, -1).int()
        return {"case": case, "k": k, "v": v, "lengths": i32(held), "path": path, "count": count, "slots": slots, "table": wide}
    if op == "verify":
        rows, vocab = sum(new), case["vocab"]
        # many unlikely tokens and a few likely ones, as a model's logits have them
        logits = normal(rows, vocab) * 1.7
        few = min(vocab, 60)
        places = torch.randint(0, vocab, (rows, few), generator=g, device=DEVICE)
        logits.scatter_add_(1, places, normal(rows, few).abs() * 3.0 + 4.0)
        f = lambda v: torch.full((len(new),), float(v), device=DEVICE)  # noqa: E731
        temperature, top_p, min_p = f(case["temperature"]), f(case["top_p"]), f(case["min_p"])
        top_k = torch.full((len(new),), case["top_k"], dtype=torch.int32, device=DEVICE)
        if case["mixed"]:                          # every conversation has settings of its own, some of them greedy, some without limits
            i = torch.arange(len(new), device=DEVICE)
            temperature = torch.where(i % 5 == 4, torch.zeros_like(temperature), temperature * (0.5 + (i % 7) / 7.0))
            top_k = torch.where(i % 3 == 1, torch.zeros_like(top_k), top_k)
            top_p = torch.where(i % 4 == 2, torch.ones_like(top_p), top_p)
            min_p = torch.where(i % 2 == 1, torch.zeros_like(min_p), min_p)
        uniform, accept = torch.rand(rows, generator=g, device=DEVICE), torch.rand(rows, generator=g, device=DEVICE)
        parents = _parents(g, new, True) if case["tree"] else None
        # what was drafted: by a smaller model, whose logits are near the large one's, or looked up, which is right more often than not
        near = torch.softmax((logits + 0.7 * normal(rows, vocab)) / 0.9, 1)
        drawn = torch.multinomial(near, 1, generator=g)[:, 0]
        right = torch.where(torch.rand(rows, generator=g, device=DEVICE) < 0.5, logits.argmax(1), drawn)
        before = (cu[seq] + parents.clamp(min=0)) if case["tree"] else (torch.arange(rows, device=DEVICE) - 1).clamp(min=0)
        ids = (drawn if case["probs"] else right)[before].int()
        return {"case": case, "logits": logits, "ids": ids, "cu": cu.int(), "seq": seq.int(), "uniform": uniform, "accept": accept if case["probs"] else None,
                "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "parents": parents, "probs": near if case["probs"] else None}
    heads, kv, d, dtype = case["heads"], case["kv"], case["d"], TYPES[case["type"]]
    lengths = _lengths(case)
    table, slots, total, _ = _tables(g, [_pages(n) for n in lengths])
    # some key channels are far larger than the others in every token
    loud = 1.0 + 3.0 * (torch.rand(kv, 1, d, generator=g, device=DEVICE) > 0.95).float()
    k = torch.empty(total, kv, PAGE, d, dtype=dtype, device=DEVICE)
    v = torch.empty(total, kv, d, PAGE, dtype=dtype, device=DEVICE)
    for at in range(0, total, 512):                                 # in pieces, for the memory
        n = min(512, total - at)
        k[at:at + n] = (normal(n, kv, PAGE, d) * loud).to(dtype)
        v[at:at + n] = (normal(n, kv, d, PAGE) + 0.3).to(dtype)
    # what the pages hold behind a sequence's last token is what earlier sequences left there, numbers that are none among it
    last = table[slots.long(), i32([(n - 1) // PAGE for n in lengths]).long()].long()
    behind = torch.arange(PAGE, device=DEVICE)[None, :] > (i32(lengths) - 1)[:, None] % PAGE
    k[last] = torch.where(behind[:, None, :, None], torch.full_like(k[last], float("nan")), k[last])
    v[last] = torch.where(behind[:, None, None, :], torch.full_like(v[last], float("nan")), v[last])
    ancestors = None
    if case["tree"]:
        ancestors = _bits(_reach(_parents(g, new, True), cu, case["tokens"]))[seq, inside]
    return {"case": case, "q": (normal(sum(new), heads, d) * 0.8).to(dtype), "k": k, "v": v, "table": table, "slots": slots, "kv_len": i32(lengths),
            "cu": cu.int(), "ancestors": ancestors, "scale": 1.0 / math.sqrt(d)}


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
        return {"attend": _attend_own, "verify": _verify_own, "keep": _keep_own, "tables": _tables_own}[op](s, case)
    return {"attend": _attend, "verify": _verify, "keep": _keep, "tables": _tables_plain}[op](s, case)


def _attend_own(s, case):
    return _ops(s["q"].dtype).draft_attention(s["q"], s["k"], s["v"], s["kv_len"], s["cu"], s["slots"], s["table"], case["kv"], s["scale"], case["tokens"],
                                              ancestors=s["ancestors"])


def _attend(s, case):
    heads, kv, most = case["heads"], case["kv"], case["tokens"]
    q, cu, kv_len = s["q"], s["cu"].long(), s["kv_len"].long()
    pages = s["table"][s["slots"].long()].long()
    k = s["k"][pages].transpose(1, 2).flatten(2, 3).float()                               # [seqs, kv, keys, d]
    v = s["v"][pages].permute(0, 2, 1, 4, 3).flatten(2, 3).float()
    n_q = cu[1:] - cu[:-1]
    i = torch.arange(most, device=q.device)
    at = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
    x = q.float()[at].unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)         # [seqs, kv, group * most, d]
    j = torch.arange(k.shape[2], device=q.device)
    there = j < kv_len[:, None]
    k, v = (torch.where(there[:, None, :, None], t, torch.zeros_like(t)) for t in (k, v))
    own_place = j - (kv_len - n_q)[:, None]                                               # of a key among the step's tokens
    if s["ancestors"] is None:
        seen = own_place[:, None] <= i[:, None]
    else:
        seen = (own_place[:, None] < 0) | ((s["ancestors"][at][..., None] >> own_place.clamp(0, 63)[:, None]) & 1).bool()
    seen = seen & there[:, None]
    score = (x @ k.transpose(-1, -2)) * s["scale"]
    score = score.unflatten(2, (-1, most)).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v).unflatten(2, (-1, most)) / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(0, 3, 1, 2, 4).flatten(2)[i < n_q[:, None]].to(q.dtype)


def _verify_own(s, case):
    return _ops(torch.bfloat16).verify_drafts(s["logits"], s["ids"], s["cu"], s["seq"], case["tokens"], s["uniform"], s["temperature"], s["top_k"], s["top_p"],
                                              s["min_p"], parents=s["parents"], draft_probs=s["probs"], accept=s["accept"])


# A token's weight exp((z - max) / T) is held as a whole number of units of 2^-40, so that sums have no order.
UNIT = float(2 ** 40)


def _kept(s):
    """The weights of the tokens that temperature, top-k, top-p and min-p leave (int64 units, 0 elsewhere), (z - max) / T, and which rows are greedy."""
    z, seq = s["logits"], s["seq"].long()
    vocab = z.shape[1]
    temperature, top_p, min_p, k = s["temperature"][seq], s["top_p"][seq], s["min_p"][seq], s["top_k"][seq]
    greedy = temperature <= 0
    top = z.amax(1, keepdim=True)
    below = (z - top) / torch.where(greedy, torch.ones_like(temperature), temperature)[:, None]
    w = torch.exp(below)
    weight = (w.double() * UNIT).long()
    order = torch.argsort(w, dim=1, descending=True, stable=True)
    mass = weight.gather(1, order).cumsum(1)
    k = torch.where(k > 0, k, vocab).long().clamp(max=vocab)
    within = mass.gather(1, k[:, None] - 1)
    need = top_p.clamp(max=1.0).double()[:, None] * within.double()
    by_mass = torch.where(top_p < 1, 1 + (mass.double() < need).sum(1), vocab)
    by_ratio = torch.where(min_p > 0, (w >= min_p[:, None]).sum(1), vocab)
    kept = torch.minimum(torch.minimum(k, by_mass), by_ratio).clamp(min=1)
    keep = torch.zeros_like(z, dtype=torch.bool).scatter(1, order, torch.arange(vocab, device=z.device) < kept[:, None])
    largest = torch.zeros_like(keep).scatter(1, z.argmax(1, keepdim=True), True)
    return torch.where(torch.where(greedy[:, None], largest, keep), weight, 0), below, greedy


def _drawn(units, uniform):
    """Where the number falls in the masses in index order."""
    c = units.cumsum(1)
    total = c[:, -1:]
    return (c <= torch.minimum((uniform.double()[:, None] * total.double()).long(), total - 1)).sum(1)


def _verify(s, case):
    ids, cu, seq, most = s["ids"].long(), s["cu"].long(), s["seq"].long(), case["tokens"]
    rows = ids.shape[0]
    units, below, greedy = _kept(s)
    total = units.sum(1, keepdim=True)
    i = torch.arange(most, device=ids.device)
    n = (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None] + i).clamp(max=rows - 1)
    inside = i < n
    if s["probs"] is not None:
        refused = (s["probs"].clamp(0, 1).double() * total.double()).long()                 # what the drafter's probability takes of a token's units
        x = ids.roll(-1)[:, None]
        ok = s["accept"].double() * refused.gather(1, x)[:, 0].double() < units.gather(1, x)[:, 0].double()
        ok = ok[at] & (i + 1 < n)
        accepted = torch.cat((torch.ones_like(ok[:, :1]), ok.long().cumprod(1).bool()), 1)[:, :most] & inside
        count = accepted.sum(1)
        stop = cu[:-1] + count - 1
        rest = (units[stop] - refused[stop]).clamp(min=0)
        rest = torch.where((count[:, None] < n) & (rest.sum(1, keepdim=True) > 0), rest, units[stop])
        following = _drawn(rest, s["uniform"][stop])
        path = torch.where(accepted, i, -1)
    else:
        drawn = _drawn(units, s["uniform"])
        parents = s["parents"] if s["parents"] is not None else (torch.arange(rows, device=ids.device) - cu[seq] - 1).int()
        parent = torch.where(inside, parents.long()[at], -1)
        token = ids[at]
        hit = (parent >= 0) & (token == drawn[at].gather(1, parent.clamp(min=0)))           # a child that has its parent's token
        same = (parent[:, :, None] == parent[:, None, :]) & hit[:, :, None] & hit[:, None, :] & (i[None, :] < i[:, None])
        live = (hit & ~same.any(2)) | (i == 0)
        seen = _reach(parents, cu, most)
        accepted = ~(seen & ~live[:, None, :]).any(2) & inside
        count = accepted.sum(1)
        path = torch.where(accepted, i, most).sort(1).values
        path = torch.where(path < most, path, -1)
        stop = cu[:-1] + path.gather(1, count[:, None] - 1)[:, 0]
        following = drawn[stop]
    there = i < count[:, None]
    row = torch.where(there, cu[:-1, None] + path.clamp(min=0), 0)
    behind = torch.where(i + 1 < count[:, None], cu[:-1, None] + path.roll(-1, 1).clamp(min=0), 0)
    token = torch.where(i + 1 < count[:, None], ids[behind], following[:, None])
    logprob = below[row, token] - torch.log((total[row, 0].double() / UNIT).float())
    logprob = torch.where(there & ~greedy[row], logprob, torch.zeros_like(logprob))
    return torch.where(there, token, -1).int(), count.int(), path.int(), logprob


def _reach(parents, cu, most):
    """Which of its sequence's new tokens (``most`` at most) a token descends from, itself among them: bool [seqs, most, most]."""
    t = torch.arange(parents.shape[0], device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    i = t - cu[seq]
    step = torch.eye(most, dtype=torch.float64, device=parents.device).repeat(cu.shape[0] - 1, 1, 1)
    up = parents.long().clamp(min=0)
    step[seq, i, up] = torch.where(parents >= 0, torch.ones_like(step[seq, i, up]), step[seq, i, up])
    return torch.linalg.matrix_power(step, 64) > 0


def _bits(reach):
    """The same as words of 64 bits (int64 [seqs, most])."""
    return (reach.long() << torch.arange(reach.shape[1], device=reach.device)).sum(2)


def _keep_own(s, case):
    _ops(TYPES[case["type"]]).keep_drafts([(s["k"], s["v"])], s["lengths"], s["path"], s["count"], s["slots"], s["table"])
    return s["k"], s["v"]


def _keep(s, case):
    table, path = s["table"][s["slots"].long()].long(), s["path"].long()
    i = torch.arange(path.shape[1], device=path.device)
    which, to = torch.nonzero((i < s["count"][:, None]) & (path != i), as_tuple=True)
    held = s["lengths"].long()[which]
    a, b = held + path[which, to], held + to
    page_a, page_b = table[which, a // PAGE], table[which, b // PAGE]
    k, v = s["k"][:, page_a, :, a % PAGE], s["v"][:, page_a, :, :, a % PAGE]
    s["k"][:, page_b, :, b % PAGE] = k
    s["v"][:, page_b, :, :, b % PAGE] = v
    return s["k"], s["v"]


def _tables_own(s, case):
    t = _ops(torch.bfloat16).step_tables(s["lengths"], s["new"], s["slots"], s["table"], s["n"], parents=s["parents"], free=s["free"])
    return t.cu_q, t.kv_len, t.token_seq, t.positions, t.places, t.slot_map, t.ancestors, t.taken, s["table"]


def _tables_plain(s, case):
    held, new = s["lengths"].long(), s["new"].long()
    cu = torch.cat((torch.zeros_like(new[:1]), new.cumsum(0)))
    t = torch.arange(s["n"], device=new.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    i = t - cu[seq]
    place = held[seq] + i
    position, ancestors, taken = place, None, None
    if s["parents"] is not None:
        reach = _reach(s["parents"], cu, case["tokens"])
        position = held[seq] + reach.sum(2)[seq, i] - 1
        ancestors = _bits(reach)[seq, i]
    row = s["slots"].long()
    fits = torch.ones_like(new, dtype=torch.bool)
    have = (held + PAGE - 1) // PAGE
    if s["free"] is not None:
        want = (held + new + PAGE - 1) // PAGE - have
        upto = want.cumsum(0)
        taken = upto[-1:].int()
        fits = upto <= s["free"].numel()
        col = torch.arange(s["table"].shape[1], device=new.device)
        inside = (col >= have[:, None]) & (col < (have + want)[:, None]) & fits[:, None]
        at = ((upto - want - have)[:, None] + col).clamp(0, max(0, s["free"].numel() - 1))
        s["table"][row] = torch.where(inside, s["free"][at], s["table"][row])
    page = s["table"][row[seq], (place // PAGE).clamp(max=s["table"].shape[1] - 1)].long()
    there = (place // PAGE < s["table"].shape[1]) & (fits[seq] | (place // PAGE < have[seq]))
    slot_map = torch.where(there, page * PAGE + place % PAGE, -1)
    return cu.int(), (held + new).int(), seq.int(), position.int(), place.int(), slot_map, ancestors, taken, s["table"]


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _attend_exact, "verify": _verify_exact, "keep": _keep_exact, "tables": _tables_exact}[case["op"]](s, case)


def _attend_exact(s, case):
    heads, kv, d = case["heads"], case["kv"], case["d"]
    out = torch.zeros(s["q"].shape[0], heads, d, dtype=torch.float64, device=DEVICE)
    cu, lengths, slots = s["cu"].tolist(), s["kv_len"].tolist(), s["slots"].tolist()
    words = None if s["ancestors"] is None else s["ancestors"].tolist()
    for i, n in enumerate(lengths):
        pages = s["table"][slots[i], :_pages(n)].long()
        new = cu[i + 1] - cu[i]
        hidden = torch.zeros(new, n, dtype=torch.bool)
        for t in range(new):
            for j in range(new):
                hidden[t, n - new + j] = j > t if words is None else not words[cu[i] + t] >> j & 1
        hidden = hidden.to(DEVICE)
        for h in range(kv):
            k = s["k"][pages, h].double().reshape(-1, d)[:n]
            v = s["v"][pages, h].double().permute(0, 2, 1).reshape(-1, d)[:n]
            for e in range(h * (heads // kv), (h + 1) * (heads // kv)):
                score = s["q"][cu[i]:cu[i + 1], e].double() @ k.T * s["scale"]
                out[cu[i]:cu[i + 1], e] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v
    return out.flatten(1)


def _verify_exact(s, case):
    cu, most = s["cu"].tolist(), case["tokens"]
    found = torch.zeros(len(cu) - 1, most, dtype=torch.float64)
    ids = s["ids"].tolist()
    for b in range(len(cu) - 1):
        t, k, p, low = (float(s[n][b]) for n in ("temperature", "top_k", "top_p", "min_p"))
        at, done = cu[b], 0
        while True:
            z = s["logits"][at].double()
            if t <= 0:
                prob = torch.zeros_like(z)
                prob[int(z.argmax())] = 1.0
            else:
                prob = torch.softmax(z / t, 0)
                ranked, order = torch.sort(prob, descending=True, stable=True)
                n = int(k) if k > 0 else len(z)
                ranked, order = ranked[:n], order[:n]
                if p < 1:
                    n = int((ranked.cumsum(0) < p * ranked.sum()).sum()) + 1
                    ranked, order = ranked[:n], order[:n]
                if low > 0:
                    n = max(1, int((ranked >= low * ranked[0]).sum()))
                    ranked, order = ranked[:n], order[:n]
                prob = torch.zeros_like(z)
                prob[order] = ranked / ranked.sum()
            following = None
            number = float(s["uniform"][at])
            if s["probs"] is not None and at + 1 < cu[b + 1]:
                x, q = ids[at + 1], s["probs"][at].double()
                if float(s["accept"][at]) * float(q[x]) < float(prob[x]):
                    following = at + 1
                else:
                    rest = (prob - q).clamp(min=0)
                    prob_of = rest if float(rest.sum()) > 0 else prob
            else:
                prob_of = prob
            if following is None:
                c = prob_of.cumsum(0)
                x = int((c <= number * c[-1]).sum().clamp(max=len(c) - 1))
                if s["probs"] is None:
                    children = [j for j in range(at + 1, cu[b + 1])
                                if ids[j] == x and (int(s["parents"][j]) if s["parents"] is not None else j - cu[b] - 1) == at - cu[b]]
                    following = children[0] if children else None
            if t > 0:
                found[b, done] = torch.log(prob[x])
            done += 1
            if following is None:
                break
            at = following
    return None, None, None, found.to(DEVICE)


def _keep_exact(s, case):
    held, count, slots, path, table = (s[n].tolist() for n in ("lengths", "count", "slots", "path", "table"))
    for b, n in enumerate(count):
        for j in range(n):                      # a token lies where it goes to or further back
            x, y = held[b] + path[b][j], held[b] + j
            a, c = table[slots[b]][x // PAGE], table[slots[b]][y // PAGE]
            s["k"][:, c, :, y % PAGE] = s["k"][:, a, :, x % PAGE].clone()
            s["v"][:, c, :, :, y % PAGE] = s["v"][:, a, :, :, x % PAGE].clone()
    return s["k"], s["v"]


def _tables_exact(s, case):
    held, new, slots, table = (s[n].tolist() for n in ("lengths", "new", "slots", "table"))
    parents = None if s["parents"] is None else s["parents"].tolist()
    free = None if s["free"] is None else s["free"].tolist()
    cu, seq, position, place, slot_map, words, taken = [0], [], [], [], [], [], 0
    for b, (h, n) in enumerate(zip(held, new)):
        fits = True
        if free is not None:
            columns = range(_pages(h), _pages(h + n))
            fits = taken + len(columns) <= len(free)
            for c in columns:
                if fits and c < len(table[0]):
                    table[slots[b]][c] = free[taken + c - _pages(h)]
            taken += len(columns)
        depth, word = [], []
        for i in range(n):
            up = -1 if parents is None else parents[cu[b] + i]
            depth.append(i if parents is None else depth[up] + 1 if up >= 0 else 0)
            word.append((word[up] if up >= 0 else 0) | 1 << i)
            seq.append(b)
            place.append(h + i)
            position.append(h + depth[i])
            c = (h + i) // PAGE
            slot_map.append(table[slots[b]][c] * PAGE + (h + i) % PAGE if c < len(table[0]) and (fits or c < _pages(h)) else -1)
        words += [w - (1 << 64) if w >> 63 else w for w in word]
        cu.append(cu[-1] + n)
    i32, i64 = dict(dtype=torch.int32, device=DEVICE), dict(dtype=torch.int64, device=DEVICE)
    return (torch.tensor(cu, **i32), torch.tensor([h + n for h, n in zip(held, new)], **i32), torch.tensor(seq, **i32), torch.tensor(position, **i32),
            torch.tensor(place, **i32), torch.tensor(slot_map, **i64), None if parents is None else torch.tensor(words, **i64),
            None if free is None else torch.tensor([taken], **i32), torch.tensor(table, **i32))


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(n)) for n in range(6)]:
        print(c, work(c))
