"""Operators of drafted tokens put together as their documentation allows: room left on the token axis, too few pages, sequences without keys."""
import pytest
import torch

from tests.test_gpu_drafts import DT, PAGE, _attention_case, _check_attention, _i32, _ops, _weight_bits

pytestmark = pytest.mark.gpu


def _short_step(ops, dtype, d, room=5):
    """Three sequences of which the free list has pages for the first alone, the second having some of its tokens' places and the third none, and ``room`` more tokens
    than they bring.  The table's columns behind what a sequence holds name pages of others.  Returns the tables, the rows of the tokens that are to be stored
    (token, page, place), and what ``rope_store`` takes."""
    lengths, new = [64, 100, 128], [3, 70, 4]
    table = torch.tensor([[5, 0, 1], [2, 3, 5], [7, 8, 2]], dtype=torch.int32)          # (sequence 2's slot is 0)
    slots = [1, 2, 0]
    n = sum(new) + room
    on_device = table.cuda()
    free = _i32([9])
    tables = ops.step_tables(_i32(lengths), _i32(new), _i32(slots), on_device, n, free=free)
    rows, t = [], 0
    for s, (held, count) in enumerate(zip(lengths, new)):
        for i in range(count):
            place = held + i
            if s == 0:
                rows.append((t, 9, place % PAGE))
            elif place // PAGE < (held + PAGE - 1) // PAGE:
                rows.append((t, int(table[slots[s], place // PAGE]), place % PAGE))
            t += 1
    g = torch.Generator().manual_seed(d)
    qkv = torch.randn(n, 8 * d, generator=g).to(DT[dtype]).cuda()
    k = torch.randn(10, 2, PAGE, d, generator=g).to(DT[dtype]).cuda()
    v = torch.randn(10, 2, d, PAGE, generator=g).to(DT[dtype]).cuda()
    return tables, rows, dict(qkv=qkv, n_heads=4, n_kv=2, d=d, positions=tables.positions, token_seq=tables.token_seq, slots=_i32(slots), page_table=on_device, k_cache=k,
                              v_cache=v, inv_freq=None, magnitude=1.0, rot_dim=d)


def _stored(k, v, qkv, rows, d):
    """The caches with the tokens' own keys and values (which are not turned) at their rows."""
    k, v = k.clone(), v.clone()
    for t, page, place in rows:
        k[page, :, place] = qkv[t, 4 * d:6 * d].view(2, d)
        v[page, :, :, place] = qkv[t, 6 * d:].view(2, d)
    return k, v


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [64, 20])
def test_what_has_no_page_is_not_stored(dtype, d):
    """By the slot map, tokens of no sequence and of sequences that got no pages leave every other row of the cache as it was."""
    ops = _ops(dtype)
    tables, rows, args = _short_step(ops, dtype, d)
    assert tables.taken.tolist() == [3] and len(rows) == 3 + 28 and tables.slot_map.tolist().count(-1) == 82 - len(rows)
    want = _stored(args["k_cache"], args["v_cache"], args["qkv"], rows, d)
    q = ops.rope_store(**args, slot_map=tables.slot_map)
    assert torch.equal(args["k_cache"], want[0]) and torch.equal(args["v_cache"], want[1])
    assert torch.equal(q[:77], args["qkv"][:77, :4 * d].view(77, 4, d))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [64, 20])
def test_tokens_of_no_sequence_are_not_stored_at_places(dtype, d):
    """Room behind the last sequence, as ``step_tables`` describes it, and places, slots and pages that are none."""
    ops = _ops(dtype)
    table = _i32([[5, 0], [2, 3], [-1, 40]])
    got = ops.step_tables(_i32([64, 10]), _i32([3, 2]), _i32([1, 0]), table, 9)
    g = torch.Generator().manual_seed(d)
    qkv = torch.randn(9, 8 * d, generator=g).to(DT[dtype]).cuda()
    k = torch.randn(10, 2, PAGE, d, generator=g).to(DT[dtype]).cuda()
    v = torch.randn(10, 2, d, PAGE, generator=g).to(DT[dtype]).cuda()
    args = dict(n_heads=4, n_kv=2, d=d, page_table=table, inv_freq=None, magnitude=1.0, rot_dim=d)
    want = _stored(k, v, qkv, [(0, 3, 0), (1, 3, 1), (2, 3, 2), (3, 5, 10), (4, 5, 11)], d)
    ops.rope_store(qkv=qkv, positions=got.positions, token_seq=got.token_seq, slots=_i32([1, 0]), k_cache=k, v_cache=v, places=got.places, **args)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    # sequences, slots, places and pages that are none
    seq, places = _i32([0, 0, 1, 2, 3, 4, 5, -7, 0]), _i32([128, -1, 3, 3, 70, 3, 3, 3, 2 ** 31 - 1])
    ops.rope_store(qkv=qkv, positions=_i32([0] * 9), token_seq=seq, slots=_i32([0, -1, 3, 2, 2]), k_cache=k, v_cache=v, places=places, **args)
    ops.rope_store(qkv=qkv, positions=_i32([0] * 9), token_seq=_i32([0] * 9), slots=_i32([0]), k_cache=k, v_cache=v,
                   slot_map=torch.tensor([-1, 640, 2 ** 40, -2 ** 62, -64, 641, 1000, -1, -1]).cuda(), **args)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_refusals_of_storing_at_rows():
    ops = _ops("bfloat16")
    tables, _, args = _short_step(ops, "bfloat16", 64)
    for bad in (dict(slot_map=tables.slot_map[:5]), dict(slot_map=tables.places), dict(slot_map=tables.slot_map.cpu()), dict(slot_map=tables.slot_map, places=tables.places),
                dict(slot_map=tables.slot_map, positions=tables.positions[:7].contiguous()), dict(places=tables.places, token_seq=tables.token_seq.long()),
                dict(slot_map=tables.slot_map, k_cache=args["k_cache"][:, :, :32].contiguous()), dict(places=tables.places, v_cache=args["v_cache"][:9]),
                dict(places=tables.places, slots=args["slots"].long()), dict(places=tables.places, page_table=args["page_table"][0].contiguous()),
                dict(places=tables.places, page_table=args["page_table"][:, :2])):
        with pytest.raises(ValueError):
            ops.rope_store(**{**args, **bad})


def test_accepted_tokens_without_pages_move_nothing():
    """After a step with too few pages: the table's columns behind what a sequence holds name others' pages, which accepted tokens must not be moved in."""
    ops = _ops("bfloat16")
    tables, rows, args = _short_step(ops, "bfloat16", 64)
    k, v = args["k_cache"][None].contiguous(), args["v_cache"][None].contiguous()
    want_k, want_v = k.clone(), v.clone()
    # the second's accepted tokens lie in its own page and behind it, the third's all behind it
    path, count = [[0, 2, -1, -1], [0, 3, 27, 60], [0, 1, 3, -1]], [2, 4, 3]
    where = {t: (page, place) for t, page, place in rows}
    for first, accepted, n in zip((0, 3, 73), path, count):
        for j in range(n):
            if first + accepted[j] in where and first + j in where:
                (a, x), (b, y) = where[first + accepted[j]], where[first + j]
                want_k[0, b, :, y] = want_k[0, a, :, x].clone()
                want_v[0, b, :, :, y] = want_v[0, a, :, :, x].clone()
    assert not torch.equal(k, want_k)
    ops.keep_drafts([(k, v)], _i32([64, 100, 128]), _i32(path), _i32(count), args["slots"], args["page_table"], slot_map=tables.slot_map, cu_q=tables.cu_q)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    # places behind a sequence's own tokens, and offsets behind the slot map
    ops.keep_drafts([(k, v)], _i32([64, 100, 128]), _i32([[0, 3], [0, 75], [0, 63]]), _i32([2, 2, 2]), args["slots"], args["page_table"], slot_map=tables.slot_map[:74].contiguous(),
                    cu_q=tables.cu_q)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    more = dict(pairs=[(k, v)], lengths=_i32([64]), path=_i32([[0, 1]]), count=_i32([2]), slots=_i32([0]), page_table=args["page_table"])
    for bad in (dict(slot_map=tables.slot_map), dict(cu_q=_i32([0, 3])), dict(slot_map=tables.slot_map.int(), cu_q=_i32([0, 3])), dict(slot_map=tables.slot_map, cu_q=_i32([0]))):
        with pytest.raises(ValueError):
            ops.keep_drafts(**more, **bad)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_accepted_tokens_move_by_the_slot_map_as_by_the_table(dtype):
    ops = _ops(dtype)
    g = torch.Generator().manual_seed(3)
    held, new = [0, 60, 127, 500], [64, 30, 20, 7]
    pages = torch.randperm(24, generator=g).int()
    table = torch.cat((pages[:20].view(4, 5), pages[20:].expand(4, 4)), 1)               # (one sequence alone has more than five)
    slots = [2, 0, 3, 1]
    path, counts = torch.full((4, 64), -1, dtype=torch.int32), [40, 30, 3, 5]
    for s, c in enumerate(counts):
        path[s, 1:c] = (torch.randperm(new[s] - 1, generator=g)[:c - 1] + 1).sort().values.int()
        path[s, 0] = 0
    on_device = table.contiguous().cuda()
    tables = ops.step_tables(_i32(held), _i32(new), _i32(slots), on_device, sum(new) + 2)
    make = lambda *shape: torch.randn(2, 24, 2, *shape, generator=torch.Generator().manual_seed(8)).to(DT[dtype]).cuda()  # noqa: E731
    (k, v), (k1, v1) = (make(PAGE, 32), make(32, PAGE)), (make(PAGE, 32), make(32, PAGE))
    args = (_i32(held), path.cuda(), _i32(counts), _i32(slots), on_device)
    ops.keep_drafts([(k, v)], *args)
    ops.keep_drafts([(k1, v1)], *args, slot_map=tables.slot_map, cu_q=tables.cu_q)
    assert torch.equal(k, k1) and torch.equal(v, v1) and not torch.equal(k, make(PAGE, 32))


@pytest.mark.parametrize("mask", [None, 63])
@pytest.mark.parametrize("d", [64, 128, 48])
def test_tables_and_storing_launched_one_behind_the_other(mask, d):
    """The description that a step makes itself is there when its tokens are turned and stored, whichever kernels may start early; another description each time, in the
    same tensors."""
    ops = _ops("bfloat16")
    g = torch.Generator().manual_seed(d)
    n_seqs, most, heads = 512, 8, 2
    n, pages = n_seqs * most, n_seqs * 4
    table = torch.randperm(pages, generator=g).view(n_seqs, 4).int().cuda()
    slots, new = _i32(list(range(n_seqs))), _i32([most] * n_seqs)
    qkv = torch.randn(n, 3 * heads * d, generator=g).bfloat16().cuda()
    room = torch.zeros(wide := 4 * n + 3 * n + 2 * n_seqs + 2, dtype=torch.int32).cuda()
    ops.empty, make = (lambda *shape, **kw: room if shape == (wide,) else make(*shape, **kw)), ops.empty
    inv_freq = (1.0 / 10000.0 ** (torch.arange(0, d, 2).float() / d)).cuda()
    shape = (pages, heads, PAGE, d), (pages, heads, d, PAGE)
    parents = _i32([-1, 0, 0, 1, 1, 2, 3, 4] * n_seqs)
    try:
        if mask is not None:
            ops.lib.cpm_set_pdl(mask)
        for turn in range(12):
            lengths = torch.randint(0, 240, (n_seqs,), generator=g).int().cuda()
            k, v = torch.zeros(shape[0], dtype=torch.bfloat16, device="cuda"), torch.zeros(shape[1], dtype=torch.bfloat16, device="cuda")
            room.fill_(0)
            t = ops.step_tables(lengths, new, slots, table, n, parents=parents)
            q = ops.rope_store(qkv, heads, heads, d, t.positions, t.token_seq, slots, table, k, v, inv_freq, 1.0, d, places=t.places)
            torch.cuda.synchronize()
            # the same with everything of the description in place
            k1, v1 = torch.zeros_like(k), torch.zeros_like(v)
            positions, seq, places = t.positions.clone(), t.token_seq.clone(), t.places.clone()
            torch.cuda.synchronize()
            q1 = ops.rope_store(qkv, heads, heads, d, positions, seq, slots, table, k1, v1, inv_freq, 1.0, d, places=places)
            assert torch.equal(places.view(n_seqs, most)[:, 0], lengths) and torch.equal(q, q1) and torch.equal(k, k1) and torch.equal(v, v1), turn
    finally:
        ops.lib.cpm_set_pdl(-1)


@pytest.mark.parametrize("form", ["tcgen05", "plain"])
@pytest.mark.parametrize("sequences", [5, 40])
def test_attention_of_sequences_whose_slot_is_none(form, sequences):
    """A sequence without a row of the page table has no keys: its rows are zero, and the others' are what they are without it."""
    ops = _ops("bfloat16")
    ops.use_tcgen05_draft = form == "tcgen05"
    new, lengths = [2 + i % 3 for i in range(sequences)], [20 + 61 * i for i in range(sequences)]
    args, rows, cu = _attention_case("bfloat16", 64, 4, 2, lengths, new, None, seed=7)
    slots = args["slots"].clone()
    slots[1], slots[3], slots[4] = -1, args["page_table"].shape[0], 2 ** 31 - 1
    got = ops.draft_attention(**{**args, "slots": slots})
    none = [1, 3, 4]
    for s in none:
        assert bool((got[cu[s]:cu[s + 1]] == 0).all())
    for s in [s for s in range(sequences) if s not in none]:
        _check_attention("bfloat16", args, rows[s:s + 1], cu[s:s + 2], None, _weight_bits(ops, "bfloat16", 64, 4, 2), got)


@pytest.mark.parametrize("form", ["tcgen05", "plain"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_no_numbers_between_sequences_without_keys(form, bad):
    """Every eighth piece of work of a block has such a value among its own tokens' and those between have no keys at all: each reaches the rows that see it."""
    ops = _ops("bfloat16")
    ops.use_tcgen05_draft = form == "tcgen05"
    new, lengths = [4, 48] * 256, [30, 0] * 256                   # 2 pieces with a page, and 6 without, of 16 tokens and a key-value head each
    args, rows, cu = _attention_case("bfloat16", 64, 32, 2, lengths, new, None, seed=5)
    clean = ops.draft_attention(**args).view(-1, 32, 64).clone()
    table, slots = args["page_table"].cpu(), args["slots"].cpu()
    for s in range(0, 512, 2):
        page = int(table[int(slots[s]), 0])
        for head in range(2):
            args["v_cache"][page, head, (s // 2 + 7 * head) % 64, 27] = bad            # of the second of four tokens
    got = ops.draft_attention(**args).view(-1, 32, 64)
    want = clean.clone()
    for s in range(0, 512, 2):
        for head in range(2):
            want[cu[s] + 1:cu[s + 1], 16 * head:16 * head + 16, (s // 2 + 7 * head) % 64] = bad
    assert bool(torch.isfinite(clean).all())
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite) and torch.equal(got.isnan(), want.isnan()) and torch.equal(got[finite], want[finite])


def test_the_dry_run_counts_as_much_room_for_parts_as_the_library():
    from cpmcu_b200.ops.dry import DryOps

    ops = _ops("bfloat16")
    dry = DryOps(torch.bfloat16, ops.sm_count)
    for heads, kv in ((1, 1), (4, 2), (32, 2), (32, 8), (21, 1), (40, 1), (128, 1), (129, 1), (256, 1)):
        for d in (32, 64, 96, 128):
            for most in range(1, 65):
                assert ops.lib.cpm_draft_attention_scratch_floats(heads, kv, d, most) == dry.lib.cpm_draft_attention_scratch_floats(heads, kv, d, most), (heads, kv, d, most)
