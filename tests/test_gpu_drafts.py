"""Operators of drafted tokens against their definitions (tests/plain/drafts_plain.py)."""
import math

import pytest
import torch

from tests.plain import drafts_plain as plain

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
PAGE = 64


def _ops(dtype):
    from cpmcu_b200.ops.ops import Ops
    return Ops(DT[dtype], "cuda:0")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def _tables(lengths, seed, spare=3):
    """Page table [slots, pages], slots and the number of pages; pages and slots in no order."""
    g = torch.Generator().manual_seed(seed)
    pages = [(n + PAGE - 1) // PAGE for n in lengths]
    total = sum(pages) + spare
    order = torch.randperm(total, generator=g).tolist()
    slots = torch.randperm(len(lengths) + 2, generator=g)[:len(lengths)].tolist()
    table = torch.zeros(len(lengths) + 2, max(pages + [1]) + 1, dtype=torch.int32)
    for s, n in zip(slots, pages):
        table[s, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table, slots, total


def _trees(new, seed, wide=6):
    g = torch.Generator().manual_seed(seed)
    return [[-1] + [max(0, i - 1 - int(torch.randint(0, wide, (1,), generator=g))) for i in range(1, n)] for n in new]


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _attention_case(dtype, d, heads, kv, lengths, new, words, seed, q_scale=1.0, poison=float("nan")):
    """A cache that holds the sequences' keys and values in pages in no order, ``poison`` wherever there is none; returns what ``draft_attention`` takes, and rows of keys and
    values."""
    g = torch.Generator().manual_seed(seed)
    table, slots, total = _tables(lengths, seed)
    k = torch.full((total, kv, PAGE, d), poison, dtype=DT[dtype])
    v = torch.full((total, kv, d, PAGE), poison, dtype=DT[dtype])
    rows = []
    for s, n in zip(slots, lengths):
        kk = torch.randn(n, kv, d, generator=g).to(DT[dtype])
        vv = (torch.randn(n, kv, d, generator=g) + 0.2).to(DT[dtype])
        for t in range(0, n, PAGE):
            page, m = int(table[s, t // PAGE]), min(PAGE, n - t)
            k[page, :, :m] = kk[t:t + m].transpose(0, 1)
            v[page, :, :, :m] = vv[t:t + m].permute(1, 2, 0)
        rows.append((kk, vv))
    q = (torch.randn(sum(new), heads, d, generator=g) * q_scale).to(DT[dtype])
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    anc = None if words is None else torch.tensor([plain.signed(w) for ws in words for w in ws], dtype=torch.int64).cuda()
    args = dict(q=q.cuda(), k_cache=k.cuda(), v_cache=v.cuda(), kv_len=_i32(lengths), cu_q=_i32(cu), slots=_i32(slots), page_table=table.cuda(), n_kv=kv,
                scale=1.0 / math.sqrt(d), most=max(new + [1]), ancestors=anc)
    return args, rows, cu


def _check_attention(dtype, args, rows, cu, words, weight_bits, got):
    """Half a step of the output's type, half a step of the weights' (``weight_bits``) on the values' magnitudes, and fp32 throughout else: scores of d terms, an exponential, and
    a sum over the keys."""
    q = args["q"].cpu()
    heads, d = q.shape[1:]
    half = torch.finfo(DT[dtype]).eps / 2
    got = got.cpu().double().view(-1, heads, d)
    for s, (kk, vv) in enumerate(rows):
        a, b = cu[s], cu[s + 1]
        out, size, terms = plain.attention(q[a:b], kk, vv, b - a, None if words is None else words[s], args["scale"])
        inner = 2 * (d + 8) * terms * 2.0 ** -24 + (2 * kk.shape[0] ** 0.5 + 16) * 2.0 ** -23
        tol = half * out.abs() + (2.0 ** -weight_bits * 2 + inner[..., None]) * size * 1.01 + 1e-30
        off = (got[a:b] - out).abs()
        assert bool((off <= tol).all()), f"sequence {s}: {float((off / tol).max()):.2f} of the tolerance"


def _weight_bits(ops, dtype, d, heads, kv):
    return 9 if ops.draft_attention_on_tensor_cores(d, heads, kv) else 24          # bf16 weights: a half step is 2^-9 of the power of two above, 2^-8 of the least


@pytest.mark.parametrize("form", ["tcgen05", "plain"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,heads,kv", [(32, 4, 1), (64, 16, 2), (96, 6, 2), (128, 32, 2), (64, 5, 5), (128, 10, 2), (64, 6, 2), (128, 21, 1)])
@pytest.mark.parametrize("tree", [False, True])
def test_attention(form, dtype, d, heads, kv, tree):
    ops = _ops(dtype)
    ops.use_tcgen05_draft = form == "tcgen05"
    if form == "tcgen05" and dtype == "float32":
        pytest.skip("a form of bf16")
    new = [1, 7, 3, 64, 16, 2]
    lengths = [1, 7, 64, 130, 300, 65]
    words = [plain.ancestors(p)[0] for p in _trees(new, 5)] if tree else None
    args, rows, cu = _attention_case(dtype, d, heads, kv, lengths, new, words, seed=d + heads)
    got = ops.draft_attention(**args)
    _check_attention(dtype, args, rows, cu, words, _weight_bits(ops, dtype, d, heads, kv), got)
    assert torch.equal(got, ops.draft_attention(**args))


@pytest.mark.parametrize("form", ["tcgen05", "plain"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("lengths,new", [([5000], [5]), ([2000], [64]), ([1], [1]), ([3000, 1, 64, 1500], [1, 1, 1, 1]), ([70] * 40, [3] * 40), ([40 * i + 9 for i in range(60)], [9] * 60)])
def test_attention_of_lengths(form, dtype, lengths, new):
    """Few and many sequences, keys shared out or not."""
    if form == "tcgen05" and dtype == "float32":
        pytest.skip("a form of bf16")
    ops = _ops(dtype)
    ops.use_tcgen05_draft = form == "tcgen05"
    words = [plain.ancestors(p)[0] for p in _trees(new, 6)]
    args, rows, cu = _attention_case(dtype, 64, 4, 2, lengths, new, words, seed=3)
    _check_attention(dtype, args, rows, cu, words, _weight_bits(ops, dtype, 64, 4, 2), ops.draft_attention(**args))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [4, 20, 48, 160, 256])
def test_attention_of_other_head_sizes(dtype, d):
    ops = _ops(dtype)
    new, lengths = [3, 5], [90, 5]
    if dtype == "bfloat16" and d % 8:
        lengths = [90, 64]
    args, rows, cu = _attention_case(dtype, d, 6, 2, lengths, new, None, seed=d)
    _check_attention(dtype, args, rows, cu, None, 24, ops.draft_attention(**args))


@pytest.mark.parametrize("form", ["tcgen05", "plain"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_of_rows_that_see_nothing_and_of_no_sequence(form, dtype):
    ops = _ops(dtype)
    ops.use_tcgen05_draft = form == "tcgen05"
    new, lengths = [3, 0, 2], [3, 100, 80]
    words = [[1, 0, 0b101], [], [0, 0b11]]                 # one row without any key, one that sees the history alone
    args, rows, cu = _attention_case(dtype, 64, 4, 2, lengths, new, words, seed=1)
    args["q"] = torch.cat((args["q"], torch.ones(2, 4, 64, dtype=DT[dtype]).cuda()))
    args["ancestors"] = torch.cat((args["ancestors"], torch.ones(2, dtype=torch.int64).cuda()))
    marked = torch.full((7, 256), 7.0, dtype=DT[dtype]).cuda()
    ops.empty, make = (lambda *shape, **kw: marked if shape == (7, 256) else make(*shape, **kw)), ops.empty
    got = ops.draft_attention(**args)
    assert got is marked and bool((got[5:] == 7).all()) and bool((got[1] == 0).all())
    _check_attention(dtype, args, rows, cu, words, _weight_bits(ops, dtype, 64, 4, 2), got[:5])


@pytest.mark.parametrize("form", ["tcgen05", "plain"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("history", [40, 61, 500])
def test_attention_keeps_numbers_that_are_none_to_the_rows_that_see_them(form, dtype, bad, history):
    """A key or a value of a tree's branch that is no number reaches its descendants alone, in its own channel; what lies behind the keys reaches nobody."""
    ops = _ops(dtype)
    ops.use_tcgen05_draft = form == "tcgen05"
    new, lengths = [8], [history + 8]
    parents = [-1, 0, 0, 1, 2, 3, 4, 4]
    words = [plain.ancestors(parents)[0]]
    args, rows, cu = _attention_case(dtype, 64, 4, 2, lengths, new, words, seed=2, poison=bad)
    clean = ops.draft_attention(**args).clone()
    _check_attention(dtype, args, rows, cu, words, _weight_bits(ops, dtype, 64, 4, 2), clean)
    place = history + 2                                      # the third token: an ancestor of itself, 4, 6 and 7
    page = int(args["page_table"][int(args["slots"][0]), place // PAGE])
    for what, where in (("v_cache", (page, 1, 13, place % PAGE)), ("k_cache", (page, 0, place % PAGE, 5))):
        t = args[what].clone()
        t[where] = bad
        got = ops.draft_attention(**{**args, what: t}).view(8, 4, 64)
        want = clean.view(8, 4, 64).clone()
        seeing = [2, 4, 6, 7]
        if what == "v_cache":                                # of the second key-value head: query heads 2 and 3
            want[seeing, 2:, 13] = bad
            assert torch.equal(torch.isfinite(got), torch.isfinite(want)) and torch.equal(got.isnan(), want.isnan())
            assert torch.equal(got[torch.isfinite(want)], want[torch.isfinite(want)])
        else:
            others = [i for i in range(8) if i not in seeing]
            assert torch.equal(got[others], clean.view(8, 4, 64)[others]) and torch.equal(got[:, 2:], clean.view(8, 4, 64)[:, 2:])
            if math.isnan(bad):
                assert bool(got[seeing, :2].isnan().all())


@pytest.mark.parametrize("form", ["tcgen05", "plain"])
def test_attention_does_not_depend_on_neighbours(form):
    """A row's result is within its tolerance whatever else is in the batch; the same launch gives the same bits."""
    ops = _ops("bfloat16")
    ops.use_tcgen05_draft = form == "tcgen05"
    new, lengths = [4] * 30, [37 * i + 4 for i in range(30)]
    args, rows, cu = _attention_case("bfloat16", 128, 8, 1, lengths, new, None, seed=9)
    got = ops.draft_attention(**args)
    for i in (0, 11, 29):
        one = {**args, "q": args["q"][cu[i]:cu[i + 1]].contiguous(), "kv_len": args["kv_len"][i:i + 1].contiguous(), "slots": args["slots"][i:i + 1].contiguous(), "cu_q": _i32([0, 4])}
        alone = ops.draft_attention(**one)
        _check_attention("bfloat16", one, rows[i:i + 1], [0, 4], None, _weight_bits(ops, "bfloat16", 128, 8, 1), alone)
    assert torch.equal(got, ops.draft_attention(**args))


@pytest.mark.parametrize("form", ["tcgen05", "plain"])
def test_attention_captured_and_on_another_stream(form):
    ops = _ops("bfloat16")
    ops.use_tcgen05_draft = form == "tcgen05"
    new, lengths = [5, 9], [500, 90]
    args, rows, cu = _attention_case("bfloat16", 64, 16, 2, lengths, new, None, seed=4)
    want = ops.draft_attention(**args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.draft_attention(**args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.draft_attention(**args)
    for n in (300, 77):                                      # other lengths in the same recording
        args["kv_len"].copy_(_i32([n, 80]))
        graph.replay()
        assert torch.equal(got, ops.draft_attention(**args))


@pytest.mark.parametrize("form", ["tcgen05", "plain"])
@pytest.mark.parametrize("d,heads,kv", [(64, 4, 2), (128, 20, 1)])
def test_attention_of_more_sequences_than_a_launch_takes(form, d, heads, kv):
    """1,100 short sequences: several launches, and units that have no place of their own for their parts."""
    ops = _ops("bfloat16")
    ops.use_tcgen05_draft = form == "tcgen05"
    new = [1 + i % 3 for i in range(1100)]
    lengths = [n + (i * 7) % 130 for i, n in enumerate(new)]
    lengths[700] = 900
    args, rows, cu = _attention_case("bfloat16", d, heads, kv, lengths, new, None, seed=12)
    got = ops.draft_attention(**args)
    for some in (slice(0, 40), slice(500, 530), slice(690, 710), slice(1080, 1100)):
        _check_attention("bfloat16", args, rows[some], cu[some] + [cu[some.stop]], None, _weight_bits(ops, "bfloat16", d, heads, kv), got)


def test_offsets_beyond_32_bits():
    """Keys and values that lie behind 2^32 bytes: attention in both forms, and the moving of accepted tokens."""
    ops = _ops("bfloat16")
    d, kv, new, lengths = 128, 2, [5], [130]
    args, rows, cu = _attention_case("bfloat16", d, 8, kv, lengths, new, None, seed=6)
    pages = 2 ** 32 // (kv * PAGE * d * 2) + 40
    k = torch.empty(pages, kv, PAGE, d, dtype=torch.bfloat16, device="cuda")
    v = torch.empty(pages, kv, d, PAGE, dtype=torch.bfloat16, device="cuda")
    n = args["k_cache"].shape[0]
    k[-n:], v[-n:] = args["k_cache"], args["v_cache"]
    args.update(k_cache=k, v_cache=v, page_table=args["page_table"] + (pages - n))
    for form in (True, False):
        ops.use_tcgen05_draft = form
        _check_attention("bfloat16", args, rows, cu, None, _weight_bits(ops, "bfloat16", d, 8, kv), ops.draft_attention(**args))
    ops.keep_drafts([(k[None], v[None])], _i32([125]), _i32([[0, 3]]), _i32([2]), args["slots"], args["page_table"])
    table = args["page_table"][int(args["slots"][0])]
    a, b = int(table[1]), int(table[2])
    assert torch.equal(k[a, :, 126 - 64], k[b, :, 0]) and torch.equal(v[a, :, :, 126 - 64], v[b, :, :, 0])


def test_another_current_device_is_refused(monkeypatch):
    """Tensors of one device while another is the current one."""
    from cpmcu_b200.ops import ops as module

    ops = _ops("bfloat16")
    args, _, _ = _attention_case("bfloat16", 64, 4, 2, [70], [3], None, seed=1)
    more, _ = _verify_case([3], 50, 2, False)
    table = _i32([[0, 1]])
    k = torch.zeros(1, 2, 1, PAGE, 8).bfloat16().cuda()
    monkeypatch.setattr(module, "_current_device", lambda: 1)
    for call in (lambda: ops.draft_attention(**args), lambda: ops.verify_drafts(**more), lambda: ops.step_tables(_i32([3]), _i32([1]), _i32([0]), table, 1),
                 lambda: ops.keep_drafts([(k, None)], _i32([0]), _i32([[0, 1]]), _i32([2]), _i32([0]), table)):
        with pytest.raises(ValueError, match="current device"):
            call()


def test_refusals_of_attention():
    ops = _ops("bfloat16")
    args, _, _ = _attention_case("bfloat16", 64, 4, 2, [70, 3], [3, 2], None, seed=1)
    q = args["q"]
    off = torch.zeros(q.numel() + 1, dtype=q.dtype).cuda()[1:].view(q.shape)
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q[..., :32]), dict(n_kv=3), dict(n_kv=0), dict(most=0), dict(most=65), dict(kv_len=_i32([1])), dict(slots=_i32([0])),
                dict(cu_q=_i32([0, 5])), dict(ancestors=torch.zeros(4, dtype=torch.int64).cuda()), dict(ancestors=_i32([1] * 5)), dict(k_cache=args["k_cache"].float()),
                dict(k_cache=args["k_cache"][..., :32].contiguous()), dict(v_cache=args["v_cache"][:2]), dict(page_table=args["page_table"][0]), dict(kv_len=args["kv_len"].long()),
                dict(q=q.cpu()), dict(q=off)):
        with pytest.raises(ValueError):
            ops.draft_attention(**{**args, **bad})
    none = ops.draft_attention(**{**args, "q": q[:0], "kv_len": args["kv_len"][:0], "slots": args["slots"][:0], "cu_q": _i32([0])})
    assert none.shape == (0, 256)


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------

def _rows(n, vocab, g, spread=3.0):
    z = torch.randn(n, vocab, generator=g) * spread
    return z


def _settings(n, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda: torch.rand(n, generator=g)  # noqa: E731
    t = torch.where(r() < 0.2, torch.zeros(n), 0.3 + 1.5 * r())
    k = torch.where(r() < 0.4, torch.zeros(n), (vocab * r() ** 3).ceil()).int()
    p = torch.where(r() < 0.4, torch.ones(n), r())
    m = torch.where(r() < 0.5, torch.zeros(n), 0.2 * r())
    return t, k, p, m


def _check_verify(got, z, ids, cu, u, settings, parents=None, probs=None, accept=None):
    tokens, count, path, logs = (x.cpu() for x in got)
    most = tokens.shape[1]
    for s in range(len(cu) - 1):
        a, b = cu[s], cu[s + 1]
        mine = tuple(float(x[s]) if x.dtype == torch.float32 else int(x[s]) for x in settings)
        w_tokens, w_path, w_logs = plain.verify(z[a:b], ids[a:b], u[a:b], mine, None if parents is None else parents[s], None if probs is None else probs[a:b],
                                                None if accept is None else accept[a:b])
        n = len(w_tokens)
        assert int(count[s]) == n, f"sequence {s}"
        assert tokens[s].tolist() == w_tokens + [-1] * (most - n), f"sequence {s}"
        assert path[s].tolist() == w_path + [-1] * (most - n)
        want = torch.tensor(w_logs, dtype=torch.float64)
        # (z - max) / T rounded twice, a logarithm, and their difference
        size = 2.0 ** -23 * (want.abs() + math.log(z.shape[1]) + 2)
        finite = torch.isfinite(want)
        assert bool(((logs[s, :n].double() - want).abs()[finite] <= 4 * size[finite]).all()) and torch.equal(logs[s, :n].double()[~finite], want[~finite])
        assert bool((logs[s, n:] == 0).all())


def _verify_case(new, vocab, seed, probs, trees=None, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    n = sum(new)
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    z = _rows(n, vocab, g, spread)
    q = torch.softmax((z + torch.randn(n, vocab, generator=g)) / 0.9, 1) if probs else None
    t, k, p, m = _settings(len(new), vocab, seed + 1)
    u, accept = torch.rand(n, generator=g), torch.rand(n, generator=g)
    ids = torch.zeros(n, dtype=torch.int64)
    for s in range(len(new)):
        for i in range(1, new[s]):
            up = cu[s] + (i - 1 if trees is None else trees[s][i])
            ids[cu[s] + i] = int(torch.multinomial(q[up], 1, generator=g)) if probs else int(z[up].topk(min(2, vocab)).indices[min(vocab - 1, int(torch.randint(0, 4, (1,), generator=g) == 3))])
    seq = [s for s, x in enumerate(new) for _ in range(x)]
    args = dict(logits=z.cuda(), ids=ids.int().cuda(), cu_q=_i32(cu), token_seq=_i32(seq), most=max(new), uniform=u.cuda(), temperature=t.cuda(), top_k=k.cuda(), top_p=p.cuda(),
                min_p=m.cuda())
    if probs:
        args.update(draft_probs=q.cuda(), accept=accept.cuda())
    if trees is not None:
        args.update(parents=_i32([x for tree in trees for x in tree]))
    return args, dict(z=z, ids=ids.tolist(), cu=cu, u=u, settings=(t, k, p, m), parents=trees, probs=q, accept=accept if probs else None)


@pytest.mark.parametrize("vocab", [1, 7, 300, 2047, 9001])
@pytest.mark.parametrize("kind", ["chain", "probs", "tree"])
def test_verify(vocab, kind):
    ops = _ops("bfloat16")
    new = [5, 1, 2, 33, 8, 64, 3, 1, 17]
    trees = _trees(new, vocab) if kind == "tree" else None
    args, want = _verify_case(new, vocab, vocab + 11, kind == "probs", trees)
    _check_verify(ops.verify_drafts(**args), **want)


@pytest.mark.parametrize("vocab,sequences,kind", [(73448, 3, "probs"), (73448, 3, "tree"), (32000, 40, "probs"), (160001, 2, "probs")])
def test_verify_large_rows(vocab, sequences, kind):
    ops = _ops("bfloat16")
    new = [3] * sequences
    trees = _trees(new, 1) if kind == "tree" else None
    args, want = _verify_case(new, vocab, 5, kind == "probs", trees, spread=2.0)
    _check_verify(ops.verify_drafts(**args), **want)


def test_verify_rows_of_few_levels_and_edges():
    """Equal logits, rows with nothing above -inf, infinities and NaN; drafted tokens outside the vocabulary; probabilities that are no numbers, zero, or above the model's."""
    ops = _ops("bfloat16")
    vocab, new = 500, [4] * 12
    args, want = _verify_case(new, vocab, 3, True)
    z, q = want["z"], want["probs"]
    z[:8] = (z[:8] / 3).round()
    z[9], z[12, 3], z[17, 100], z[21, :250] = -math.inf, math.inf, math.nan, -math.inf
    q[2], q[5], q[8, 30], q[25] = 0.0, 1.0, math.nan, 2.0
    want["ids"][30], want["ids"][34] = -3, vocab
    args.update(logits=z.cuda(), draft_probs=q.cuda(), ids=_i32(want["ids"]))
    want["settings"][0][:6] = 0.8
    args["temperature"] = want["settings"][0].cuda()
    _check_verify(ops.verify_drafts(**args), **want)
    # the same as a chain without probabilities
    plain_args = {k: v for k, v in args.items() if k not in ("draft_probs", "accept")}
    _check_verify(ops.verify_drafts(**plain_args), **{**want, "probs": None, "accept": None})


def test_verify_rows_in_place_and_of_no_sequence():
    """Probabilities with rows apart, room behind the last sequence, sequences without tokens, and a most that is more than any brings."""
    ops = _ops("bfloat16")
    args, want = _verify_case([3, 4], 777, 2, True)
    wide = torch.full((9, 800), math.nan).cuda()
    wide[:7, 9:786] = args["draft_probs"]
    pad = lambda t, value: torch.cat((t, torch.full((2, *t.shape[1:]), value, dtype=t.dtype).cuda()))  # noqa: E731
    more = dict(args, logits=pad(args["logits"], math.nan), ids=pad(args["ids"], 5), token_seq=pad(args["token_seq"], -1), uniform=pad(args["uniform"], 0.5),
                accept=pad(args["accept"], 0.5), draft_probs=wide[:, 9:786], most=9, cu_q=_i32([0, 3, 3, 7]))
    three = lambda t: torch.stack((t[0], t[0], t[1]))  # noqa: E731
    more.update({n: three(args[n]) for n in ("temperature", "top_k", "top_p", "min_p")})
    more["token_seq"] = _i32([0] * 3 + [2] * 4 + [-1] * 2)
    tokens, count, path, logs = ops.verify_drafts(**more)
    assert int(count[1]) == 0 and bool((tokens[1] == -1).all()) and bool((path[1] == -1).all()) and bool((logs[1] == 0).all())
    pick = torch.tensor([0, 2]).cuda()
    _check_verify((tokens[pick], count[pick], path[pick], logs[pick]), **want)


def test_verify_by_keys_draws_what_single_steps_draw():
    """Without given numbers, the tokens of a chain are those that ``sample_filtered`` gives one step after the other."""
    ops = _ops("bfloat16")
    new, vocab = [6, 6, 6], 1000
    args, want = _verify_case(new, vocab, 8, False)
    keys, steps = _i32([5, 9, 2]), _i32([7, 0, 40])
    t, k, p, m = (args[n] for n in ("temperature", "top_k", "top_p", "min_p"))
    t.fill_(0.9)
    tokens = torch.zeros(18, dtype=torch.int32).cuda()
    for i in range(6):
        rows = args["logits"].view(3, 6, vocab)[:, i].contiguous()
        got, _ = ops.sample_filtered(rows, None, t, k, p, m, 123, keys, steps + i)
        if i < 5:
            tokens.view(3, 6)[:, i + 1] = got
    wrong = tokens.clone()
    wrong[6 + 3] += 1                                        # the second's third drafted token is another
    positions = _i32([100 + i for i in range(6)] + list(range(6)) + [7 + i for i in range(6)])
    more = {**args, "uniform": None, "seed": 123, "seq_key": keys, "step_key": steps, "positions": positions}
    got, count, _, _ = ops.verify_drafts(**{**more, "ids": wrong})
    assert count.tolist() == [6, 3, 6]
    assert torch.equal(got[0, :5], tokens[1:6]) and torch.equal(got[1, :3], tokens[7:10]) and torch.equal(got[2, :5], tokens[13:18])


def test_verify_is_distributed_as_the_model():
    """Whatever the drafter proposes, the first token out of a step is distributed as the model's: 40,000 sequences of one drafted token."""
    ops = _ops("bfloat16")
    n, vocab = 40000, 6
    g = torch.Generator().manual_seed(0)
    p = torch.tensor([0.4, 0.05, 0.25, 0.1, 0.15, 0.05])
    q = torch.tensor([0.1, 0.3, 0.05, 0.35, 0.1, 0.1])
    x = torch.multinomial(q, n, replacement=True, generator=g)
    ids = torch.stack((torch.zeros(n, dtype=torch.int64), x), 1).flatten().int().cuda()
    seq = torch.arange(n, dtype=torch.int32).repeat_interleave(2).cuda()
    tokens, count, _, _ = ops.verify_drafts(p.log().repeat(2 * n, 1).cuda(), ids, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32).cuda(), seq, 2, torch.rand(2 * n, generator=g).cuda(),
                                            torch.ones(n).cuda(), draft_probs=q.repeat(2 * n, 1).cuda(), accept=torch.rand(2 * n, generator=g).cuda())
    seen = torch.bincount(tokens[:, 0].cpu().long(), minlength=vocab).double()
    # each count is binomial: five deviations
    assert bool(((seen - n * p.double()).abs() <= 5 * (n * p.double() * (1 - p.double())).sqrt()).all())
    share = float((count == 2).float().mean())
    assert abs(share - float(torch.minimum(p, q).sum())) <= 5 * 0.5 / n ** 0.5


def test_refusals_of_verify():
    ops = _ops("bfloat16")
    args, _ = _verify_case([3, 2], 50, 2, True)
    ops.verify_drafts(**args)
    for bad in (dict(logits=args["logits"].half()), dict(logits=args["logits"][0]), dict(ids=args["ids"][:4]), dict(ids=args["ids"].long()), dict(cu_q=_i32([0, 5])), dict(token_seq=_i32([0])),
                dict(most=0), dict(most=65), dict(uniform=args["uniform"][:3]), dict(uniform=None), dict(accept=None), dict(top_k=_i32([1])), dict(min_p=args["min_p"].double()),
                dict(draft_probs=args["draft_probs"][:4]), dict(draft_probs=args["draft_probs"].t().contiguous().t()), dict(draft_probs=args["draft_probs"].double()),
                dict(parents=_i32([-1, 0, 1, -1, 0])), dict(draft_probs=None, accept=None, uniform=None), dict(draft_probs=None, accept=None, parents=_i32([0])),
                dict(logits=args["logits"].cpu())):
        with pytest.raises(ValueError):
            ops.verify_drafts(**{**args, **bad})
    none = torch.zeros(0).cuda()
    got = ops.verify_drafts(torch.zeros(0, 50).cuda(), _i32([]), _i32([0]), _i32([]), 4, none, none)
    assert [tuple(x.shape) for x in got] == [(0, 4), (0,), (0, 4), (0, 4)]
    got = ops.verify_drafts(torch.zeros(0, 50).cuda(), _i32([]), _i32([0, 0]), _i32([]), 4, none, torch.ones(1).cuda())          # a sequence that brings nothing
    assert got[1].tolist() == [0] and got[0].tolist() == [[-1] * 4]


# ---------------------------------------------------------------------------
# the step's tables
# ---------------------------------------------------------------------------

def _plain_tables(lengths, new, slots, table, n_tokens, trees, free):
    table = table.clone()
    cu, seq, pos, place, words, smap, taken = [0], [], [], [], [], [], 0
    for s, (h, n) in enumerate(zip(lengths, new)):
        have, want = (h + 63) // 64, (h + n + 63) // 64 - (h + 63) // 64
        fits = free is None or taken + want <= len(free)
        if free is not None:
            for i in range(want):
                if fits and have + i < table.shape[1]:
                    table[slots[s], have + i] = free[taken + i]
            taken += want
        word, depth = plain.ancestors(trees[s]) if trees is not None else ([0] * n, list(range(n)))
        for i in range(n):
            seq.append(s)
            place.append(h + i)
            pos.append(h + depth[i])
            words.append(plain.signed(word[i]))
            c = (h + i) // 64
            smap.append(int(table[slots[s], c]) * 64 + (h + i) % 64 if c < table.shape[1] and (fits or c < have) else -1)
        cu.append(cu[-1] + n)
    pad = n_tokens - len(seq)
    return cu, [h + n for h, n in zip(lengths, new)], seq + [-1] * pad, pos + [-1] * pad, place + [-1] * pad, smap + [-1] * pad, words + [0] * pad, taken, table


@pytest.mark.parametrize("sequences,most", [(1, 1), (3, 5), (64, 5), (300, 64), (4096, 3)])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("pages", ["held", "free", "short"])
def test_step_tables(sequences, most, tree, pages):
    ops = _ops("bfloat16")
    g = torch.Generator().manual_seed(sequences + most)
    lengths = torch.randint(0, 700, (sequences,), generator=g).tolist()
    new = torch.randint(0, most + 1, (sequences,), generator=g).tolist()
    trees = _trees([max(1, n) for n in new], 3, 9) if tree else None
    if tree:
        trees = [t[:n] for t, n in zip(trees, new)]
    table, slots, total = _tables([x + (n if pages == "held" else 0) for x, n in zip(lengths, new)], 4)
    if pages != "held":
        table = torch.cat((table, torch.full((table.shape[0], 1), 77, dtype=torch.int32)), 1)
    want = sum((h + n + 63) // 64 - (h + 63) // 64 for h, n in zip(lengths, new))
    free = None if pages == "held" else [1000 + i for i in range(want if pages == "free" else max(0, want // 2))]
    n_tokens = sum(new) + 3
    parents = None if trees is None else _i32([p for t in trees for p in t] + [0] * 3)
    on_device = table.cuda()
    got = ops.step_tables(_i32(lengths), _i32(new), _i32(slots), on_device, n_tokens, parents=parents, free=None if free is None else _i32(free))
    cu, kv_len, seq, pos, place, smap, words, taken, after = _plain_tables(lengths, new, slots, table, n_tokens, trees, free)
    for name, x in (("cu_q", cu), ("kv_len", kv_len), ("token_seq", seq), ("positions", pos), ("places", place), ("slot_map", smap)):
        assert getattr(got, name).tolist() == x, name
    assert (got.ancestors is None) == (not tree) and (not tree or got.ancestors.tolist() == words)
    assert (got.taken is None) == (free is None) and (free is None or got.taken.tolist() == [taken])
    assert torch.equal(on_device.cpu(), after)


def test_step_tables_of_parents_that_are_none():
    """A parent that is not before its child is none; a sequence of more than 64 tokens has no ancestors behind the 64th."""
    ops = _ops("bfloat16")
    table = torch.zeros(1, 4, dtype=torch.int32).cuda()
    got = ops.step_tables(_i32([10]), _i32([70]), _i32([0]), table, 70, parents=_i32([-1, 0, 2, 7, -5, 1] + [5] * 64))
    words = [1, 3, 4, 8, 16, 0b100011] + [0b100011 | 1 << i for i in range(6, 64)] + [0] * 6
    assert got.ancestors.tolist() == [plain.signed(w) for w in words]
    assert got.positions.tolist() == [10, 11, 10, 10, 10, 12] + [13] * 58 + [10] * 6


def test_refusals_of_step_tables():
    ops = _ops("bfloat16")
    table = torch.zeros(2, 4, dtype=torch.int32).cuda()
    args = dict(lengths=_i32([3, 70]), new=_i32([1, 2]), slots=_i32([0, 1]), page_table=table, n_tokens=3, parents=None, free=None)
    ops.step_tables(**args)
    for bad in (dict(lengths=_i32([3])), dict(new=_i32([1, 2]).long()), dict(slots=_i32([0])), dict(page_table=table[0]), dict(n_tokens=-1), dict(parents=_i32([0, 0])),
                dict(free=_i32([1]).long()), dict(lengths=_i32([]), new=_i32([]), slots=_i32([])), dict(new=_i32([1, 2]).cpu()),
                dict(lengths=_i32([0] * 4097), new=_i32([0] * 4097), slots=_i32([0] * 4097))):
        with pytest.raises(ValueError):
            ops.step_tables(**{**args, **bad})
    none = ops.step_tables(_i32([3, 70]), _i32([0, 0]), _i32([0, 1]), table, 0, parents=_i32([]), free=_i32([]))
    assert none.cu_q.tolist() == [0, 0, 0] and none.kv_len.tolist() == [3, 70] and none.ancestors.shape == (0,) and none.taken.tolist() == [0]
    # a slot that is none changes nothing and has no places
    got = ops.step_tables(_i32([3, 70]), _i32([1, 60]), _i32([5, -1]), table, 61, free=_i32([9, 9, 9]))
    assert bool((table == 0).all()) and bool((got.slot_map == -1).all())


# ---------------------------------------------------------------------------
# keeping accepted tokens
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,dv,kv", [(32, 32, 1), (64, 64, 2), (96, 96, 2), (128, 128, 2), (128, 64, 3), (20, 12, 2), (250, 7, 1), (256, 256, 1)])
def test_keep_drafts(dtype, d, dv, kv):
    ops = _ops(dtype)
    g = torch.Generator().manual_seed(d)
    held, new = [0, 60, 127, 1000, 5, 64], [64, 64, 20, 7, 1, 33]
    table, slots, total = _tables([h + n for h, n in zip(held, new)], 2)
    most = 64
    path = torch.full((6, most), -1, dtype=torch.int32)
    counts = [40, 64, 3, 7, 1, 20]
    for s, c in enumerate(counts):
        path[s, 1:c] = (torch.randperm(new[s] - 1, generator=g)[:c - 1] + 1).sort().values.int()
        path[s, 0] = 0
    pairs = [(torch.randn(lanes, total, kv, PAGE, d, generator=g).to(DT[dtype]), None if lanes == 3 else torch.randn(lanes, total, kv, dv, PAGE, generator=g).to(DT[dtype]))
             for lanes in (1, 4, 3)]
    on_device = [(k.cuda(), None if v is None else v.cuda()) for k, v in pairs]
    ops.keep_drafts(on_device, _i32(held), path.cuda(), _i32(counts), _i32(slots), table.cuda())
    for (k, v), (kd, vd) in zip(pairs, on_device):
        for s, c in enumerate(counts):
            for j in range(1, c):
                x, y = held[s] + int(path[s, j]), held[s] + j
                a, b = int(table[slots[s], x // PAGE]), int(table[slots[s], y // PAGE])
                k[:, b, :, y % PAGE] = k[:, a, :, x % PAGE].clone()
                if v is not None:
                    v[:, b, :, :, y % PAGE] = v[:, a, :, :, x % PAGE].clone()
        assert torch.equal(kd.cpu(), k) and (v is None or torch.equal(vd.cpu(), v))


def test_keep_drafts_leaves_out_what_is_no_place():
    ops = _ops("bfloat16")
    k = torch.randn(2, 3, 1, PAGE, 8).bfloat16().cuda()
    before = k.clone()
    table = _i32([[0, 7, 1], [2, -1, 1]])
    path = _i32([[0, 60], [0, 60], [0, 3], [0, 3], [0, 200]])
    ops.keep_drafts([(k, None)], _i32([10, 10, 10, -50, 10]), path, _i32([2, 2, 2, 2, 2]), _i32([0, 1, 9, 0, 0]), table)      # pages, slots and lengths that are none
    assert torch.equal(k, before)
    ops.keep_drafts([(k, None)], _i32([10]), _i32([[0, 3]]), _i32([0]), _i32([0]), table)                                     # nothing accepted
    assert torch.equal(k, before)


def test_refusals_of_keep_drafts():
    ops = _ops("bfloat16")
    k, v = torch.zeros(2, 3, 1, PAGE, 8).bfloat16().cuda(), torch.zeros(2, 3, 1, 8, PAGE).bfloat16().cuda()
    args = dict(pairs=[(k, v)], lengths=_i32([0]), path=_i32([[0, 1]]), count=_i32([2]), slots=_i32([0]), page_table=_i32([[0]]))
    ops.keep_drafts(**args)
    for bad in (dict(path=_i32([0, 1])), dict(path=_i32([[0] * 65])), dict(path=_i32([[]])), dict(lengths=_i32([0, 1])), dict(count=_i32([2]).long()), dict(slots=_i32([])),
                dict(page_table=_i32([0])), dict(pairs=[(k, k)]), dict(pairs=[(k.float(), v)]), dict(pairs=[(k.double(), None)]), dict(pairs=[(k[:, :, :, :32], None)]),
                dict(pairs=[(k[0], None)]), dict(pairs=[(k.cpu(), None)])):
        with pytest.raises(ValueError):
            ops.keep_drafts(**{**args, **bad})
    ops.keep_drafts([], _i32([0]), _i32([[0, 1]]), _i32([2]), _i32([0]), _i32([[0]]))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,rot_dim", [(64, 64), (48, 16), (20, 20)])
def test_rope_store_at_places(dtype, d, rot_dim):
    """A token that lies elsewhere than at its position is turned by the position and stored at the place, to the same bits."""
    ops = _ops(dtype)
    g = torch.Generator().manual_seed(d)
    qkv = torch.randn(6, 8 * d, generator=g).to(DT[dtype]).cuda()
    positions, places, seq = _i32([70, 71, 71, 72, 5, 6]), _i32([70, 71, 72, 73, 63, 64]), _i32([0, 0, 0, 0, 1, 1])
    table, slots = _i32([[2, 5], [4, 1]]), _i32([1, 0])
    inv_freq = (1.0 / 10000.0 ** (torch.arange(0, rot_dim, 2).float() / rot_dim)).cuda()
    make = lambda: (torch.zeros(6, 2, PAGE, d, dtype=DT[dtype]).cuda(), torch.zeros(6, 2, d, PAGE, dtype=DT[dtype]).cuda())  # noqa: E731
    (k, v), (k1, v1) = make(), make()
    q = ops.rope_store(qkv, 4, 2, d, positions, seq, slots, table, k, v, inv_freq, 1.1, rot_dim, places=places)
    for t in range(6):                                       # one at a time, so that no place is taken twice
        one = make()
        at = slice(t, t + 1)
        want = ops.rope_store(qkv[at].contiguous(), 4, 2, d, positions[at].contiguous(), seq[at].contiguous(), slots, table, *one, inv_freq, 1.1, rot_dim)
        assert torch.equal(q[at], want)
        row = table[int(slots[int(seq[t])])]
        x, y = int(positions[t]), int(places[t])
        k1[row[y // PAGE], :, y % PAGE] = one[0][row[x // PAGE], :, x % PAGE]
        v1[row[y // PAGE], :, :, y % PAGE] = one[1][row[x // PAGE], :, :, x % PAGE]
    assert torch.equal(k, k1) and torch.equal(v, v1)
    with pytest.raises(ValueError):
        ops.rope_store(qkv, 4, 2, d, positions, seq, slots, table, k, v, inv_freq, 1.1, rot_dim, places=places[:3].contiguous())
