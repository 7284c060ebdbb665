"""The 4-bit cache's kernels, the copying of pages and the filtered sampling against the definitions (tests/plain/kv4_plain.py)."""
import math

import pytest
import torch

from tests.plain import kv4_plain as plain

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
PAGE = 64


def _ops(dtype):
    from cpmcu_b200.ops.ops import Ops
    return Ops(DT[dtype], "cuda:0")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def _tables(lengths, seed, spare=3):
    """Page table [slots, pages], slots and the number of pages for sequences of the given lengths; pages and slots in no order."""
    g = torch.Generator().manual_seed(seed)
    pages = [(n + PAGE - 1) // PAGE for n in lengths]
    total = sum(pages) + spare
    order = torch.randperm(total, generator=g).tolist()
    slots = torch.randperm(len(lengths) + 2, generator=g)[:len(lengths)].tolist()
    table = torch.zeros(len(lengths) + 2, max(pages + [1]) + 1, dtype=torch.int32)
    for s, n in zip(slots, pages):
        table[s, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table.cuda(), slots, total


def _every_position(lengths):
    pos = [p for n in lengths for p in range(n)]
    seq = [i for i, n in enumerate(lengths) for _ in range(n)]
    return _i32(pos), _i32(seq)


def _filled(ops, lengths, kv, d, seed, loud=1.0, v_scale=1.0):
    """A cache that holds random keys and values; returns its parts and the values they stand for (fp32, on the host)."""
    table, slots, total = _tables(lengths, seed)
    g = torch.Generator().manual_seed(seed + 1)
    records = torch.randint(0, 256, (total, kv, ops.kv4_page_bytes(d)), generator=g, dtype=torch.uint8).cuda()
    records[..., 64 * d:] = 255                       # parameters that are no numbers wherever nothing is stored
    n = sum(lengths)
    pos, seq = _every_position(lengths)
    k = torch.randn(n, kv, d, generator=g) * (1 + (loud - 1) * (torch.rand(1, kv, d, generator=g) > 0.9))
    v = torch.randn(n, kv, d, generator=g) * v_scale + 0.2 * v_scale
    f32 = _ops("float32")
    if n:
        qkv = torch.cat((torch.zeros(n, kv, d), k, v), 1).flatten(1).cuda()
        f32.rope_store_kv4(qkv, kv, kv, d, pos, seq, _i32(slots), table, records, None, 1.0, 0)
        kk, vv = f32.kv4_values(records, pos, seq, _i32(slots), table, kv, d)
        kk, vv = kk.cpu(), vv.cpu()
    else:
        kk = vv = torch.zeros(0, kv, d)
    at = [0]
    for x in lengths:
        at.append(at[-1] + x)
    rows = [(kk[a:b], vv[a:b]) for a, b in zip(at, at[1:])]
    return table, slots, records, rows


# ---------------------------------------------------------------------------
# store and read back
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,kv", [(4, 1), (6, 2), (3, 3)])
def test_store_and_read_without_rotation(dtype, d, heads, kv):
    """Without a rotation every step of the definition is a rounding to 32 bits, so that the values are the same numbers."""
    ops = _ops(dtype)
    lengths = [1, 63, 64, 65, 200]
    table, slots, total = _tables(lengths, 3)
    pos, seq = _every_position(lengths)
    g = torch.Generator().manual_seed(d + heads)
    n = sum(lengths)
    qkv = (torch.randn(n, heads + 2 * kv, d, generator=g) * torch.rand(n, heads + 2 * kv, 1, generator=g).mul(12).sub(6).exp()).to(DT[dtype])
    qkv[5] = 0.75                                    # rows whose channels are all equal
    qkv[6, :, :d // 2] = 0
    qkv[7, :, 3] = 1e30 if dtype == "float32" else 1e20
    records = torch.randint(0, 256, (total, kv, ops.kv4_page_bytes(d)), generator=g, dtype=torch.uint8).cuda()
    before = records.clone()
    q = ops.rope_store_kv4(qkv.flatten(1).cuda(), heads, kv, d, pos, seq, _i32(slots), table, records, None, 1.0, 0)
    assert torch.equal(q.cpu(), qkv[:, :heads])
    k, v = ops.kv4_values(records, pos, seq, _i32(slots), table, kv, d)
    for got, x in ((k, qkv[:, heads:heads + kv]), (v, qkv[:, heads + kv:])):
        want, s = plain.quantised(x)
        assert torch.equal(got.cpu(), want.to(DT[dtype]))
        # and the definition keeps what it says: half a step, and the roundings of s (15 steps of 2^-9) and of the middle
        h = x.float().unflatten(-1, (2, -1))
        off = (want.unflatten(-1, (2, -1)) - h).abs().amax(-1)
        assert bool((off <= s * (0.5 + 16 / 512) + h.abs().amax(-1) * 2.0 ** -8).all())
    # pages that nothing was stored into are as they were
    used = torch.zeros(total, dtype=torch.bool)
    for s, x in zip(slots, lengths):
        used[table.cpu()[s, :(x + 63) // 64].long()] = True
    assert torch.equal(records.cpu()[~used], before.cpu()[~used])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("tokens", [1, 5, 70])
def test_store_rotates(dtype, d, tokens):
    heads, kv, first = 5, 5, 1003
    ops = _ops(dtype)
    g = torch.Generator().manual_seed(d)
    table, slots, total = _tables([first + tokens, first + tokens], 4)
    pos = torch.arange(first, first + tokens).repeat(2)
    qkv = torch.randn(2 * tokens, heads + 2 * kv, d, generator=g).to(DT[dtype])
    inv_freq = 1.0 / 10000.0 ** (torch.arange(0, d, 2).float() / d)
    records = torch.zeros(total, kv, ops.kv4_page_bytes(d), dtype=torch.uint8).cuda()
    seq = torch.arange(2).repeat_interleave(tokens)
    args = (_i32(pos.tolist()), _i32(seq.tolist()), _i32(slots), table)
    q = ops.rope_store_kv4(qkv.flatten(1).cuda(), heads, kv, d, *args, records, inv_freq.cuda(), 1.19, d)
    want = plain.rotated(qkv, pos, inv_freq, 1.19)
    # an angle of about 1,000 is rounded to 2^-15, its sine moves by as much; bf16: half the spacing of its 8 bits besides
    spacing = 2.0 ** (torch.log2(want[:, :heads].abs().clamp_min(1e-9)).floor() - 7) if dtype == "bfloat16" else 0.0
    assert bool(((q.cpu().double() - want[:, :heads]).abs() <= 2e-3 + 0.5 * spacing).all())
    k, v = _ops("float32").kv4_values(records, *args, kv, d)
    _, s = plain.quantised(want[:, heads:heads + kv].float())
    off = (k.cpu().double() - want[:, heads:heads + kv]).abs().unflatten(-1, (2, -1)).amax(-1)
    assert bool((off <= s * (0.5 + 16 / 512) + 6 * 2.0 ** -8 + 2e-3).all())
    assert torch.equal(v.cpu(), plain.quantised(qkv[:, heads + kv:])[0])


def test_rows_that_are_no_numbers_stay_alone():
    """A channel that is no number makes its half row one, and no other."""
    ops, d, kv = _ops("float32"), 64, 2
    table, slots, total = _tables([130], 5)
    pos, seq = _every_position([130])
    qkv = torch.randn(130, 3 * kv, d, generator=torch.Generator().manual_seed(1))
    qkv[17, 2, 40] = math.nan
    qkv[18, 5, 3] = math.inf
    records = torch.zeros(total, kv, ops.kv4_page_bytes(d), dtype=torch.uint8).cuda()
    ops.rope_store_kv4(qkv.flatten(1).cuda(), kv, kv, d, pos, seq, _i32(slots), table, records, None, 1.0, 0)
    k, v = (t.cpu() for t in ops.kv4_values(records, pos, seq, _i32(slots), table, kv, d))
    bad_k, bad_v = torch.zeros(130, kv, d, dtype=torch.bool), torch.zeros(130, kv, d, dtype=torch.bool)
    bad_k[17, 0, 32:] = True
    bad_v[18, 1, :32] = True
    assert torch.equal(k.isnan(), bad_k) and torch.equal(v.isnan(), bad_v)
    assert torch.equal(k[~bad_k], plain.quantised(qkv[:, 2:4])[0][~bad_k])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _check(got, want, rows, dtype):
    """bf16: one rounding of the output (2^-9, doubled for the sum's own) and weights of 11 bits (2^-11 of the largest value, doubled);
    fp32: queries and weights of 22 bits and scores of up to about 100: 2^-22 * 100 of the largest value."""
    assert got.shape == (want.shape[0], want.shape[1] * want.shape[2])
    got = got.cpu().double().view(want.shape)
    big = max([float(v.abs().nan_to_num(0).max()) for _, v in rows if v.numel()] + [0.0])
    tol = want.abs() * 2.0 ** -8 + big * 2.0 ** -10 if dtype == "bfloat16" else torch.full_like(want, big * 100 * 2.0 ** -22)
    assert bool(torch.isfinite(got).all())
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol.clamp_min(1e-30)).max())


SHAPES = [(1, 1), (2, 1), (6, 2), (5, 1), (16, 2), (16, 1), (24, 1), (40, 2)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,kv", SHAPES)
def test_one_token_a_sequence(dtype, d, heads, kv):
    ops = _ops(dtype)
    lengths = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 700]
    table, slots, records, rows = _filled(ops, lengths, kv, d, 11, loud=4.0)
    q = torch.randn(len(lengths), heads, d, generator=torch.Generator().manual_seed(7)).to(DT[dtype])
    for window in (0, 1, 16, 100):
        got = ops.kv4_attention(q.cuda(), records, _i32(lengths), _i32(slots), table, kv, d ** -0.5, window=window)
        want = torch.cat([plain.attention(q[i:i + 1], k, v, n - 1, d ** -0.5, window) for i, (n, (k, v)) in enumerate(zip(lengths, rows))])
        _check(got, want, rows, dtype)
        assert float(got[0].abs().max()) == 0.0           # no keys


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,n", [(8, 2, 1), (8, 2, 2), (8, 2, 18), (8, 2, 19), (24, 1, 18), (24, 1, 19), (3, 3, 12), (3, 3, 13), (8, 2, 70), (2, 1, 200)])
def test_batches_of_unequal_sequences(dtype, heads, kv, n):
    """Few rows of pages have blocks of their own, many are shared out by their cost: batches on both sides of the rule."""
    ops, d = _ops(dtype), 64
    g = torch.Generator().manual_seed(n)
    lengths = (2500 * torch.rand(n, generator=g) ** 3).int().tolist()
    lengths[0] = 4000 if n < 100 else 9000
    if n > 2:
        lengths[n // 2] = 0
    table, slots, records, rows = _filled(ops, lengths, kv, d, 31)
    q = torch.randn(n, heads, d, generator=g).to(DT[dtype])
    for window in (0, 200):
        got = ops.kv4_attention(q.cuda(), records, _i32(lengths), _i32(slots), table, kv, d ** -0.5, window=window)
        want = torch.cat([plain.attention(q[i:i + 1], k, v, m - 1, d ** -0.5, window) for i, (m, (k, v)) in enumerate(zip(lengths, rows))])
        _check(got, want, rows, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,n,length", [(4, 2, 20, 700), (4, 2, 72, 300), (4, 2, 74, 300), (2, 1, 148, 130), (2, 1, 149, 130), (24, 1, 74, 65)])
def test_batches_of_like_sequences(dtype, heads, kv, n, length):
    """Rows of pages of like length, up to as many as a device of 148 multiprocessors has blocks and one more."""
    ops, d = _ops(dtype), 64
    lengths = [length + i % 3 for i in range(n)]
    table, slots, records, rows = _filled(ops, lengths, kv, d, 37)
    q = torch.randn(n, heads, d, generator=torch.Generator().manual_seed(n)).to(DT[dtype])
    got = ops.kv4_attention(q.cuda(), records, _i32(lengths), _i32(slots), table, kv, d ** -0.5)
    want = torch.cat([plain.attention(q[i:i + 1], k, v, m - 1, d ** -0.5, 0) for i, (m, (k, v)) in enumerate(zip(lengths, rows))])
    _check(got, want, rows, dtype)


@pytest.mark.parametrize("tcgen05,shares", [(False, 0), (True, 1), (True, 3), (True, 0)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,heads,kv", [(32, 3, 1), (64, 8, 1), (64, 6, 2), (96, 4, 2), (128, 16, 1), (128, 2, 2), (64, 4, 2), (128, 5, 1), (64, 40, 2)])
def test_several_tokens_a_sequence(dtype, d, heads, kv, tcgen05, shares):
    ops = _ops(dtype)
    ops.KV4_PROMPT_BLOCKS = 0 if tcgen05 else 1 << 30         # either kernel, whatever the number of tokens
    if shares:
        ops.kv4_prompt_shares = lambda *a: shares
    assert ops.kv4_prompt_ok(295, heads, kv, d, 1.0) == (tcgen05 and dtype == "bfloat16" and d in (64, 128))
    new = [1, 5, 0, 64, 65, 130, 30]
    lengths = [1, 5, 40, 64, 200, 130, 161]
    table, slots, records, rows = _filled(ops, lengths, kv, d, 13)
    q = torch.randn(sum(new), heads, d, generator=torch.Generator().manual_seed(7)).to(DT[dtype])
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    tiles = [(i, r) for i, n in enumerate(new) for r in range(0, n, 64)] + [(2, 0)]       # a tile of a sequence that brings nothing
    args = dict(cu_q=_i32(cu), tiles=(_i32([t[0] for t in tiles]), _i32([t[1] for t in tiles]), len(tiles)))
    for window in (0, 3, 90):
        got = ops.kv4_attention(q.cuda(), records, _i32(lengths), _i32(slots), table, kv, d ** -0.5, window=window, **args)
        want = torch.cat([plain.attention(q[cu[i]:cu[i + 1]], k, v, lengths[i] - new[i], d ** -0.5, window) for i, (k, v) in enumerate(rows)])
        _check(got, want, rows, dtype)


@pytest.mark.parametrize("q_scale,v_scale", [(30.0, 1.0), (1e-6, 1e-6), (1.0, 1e6), (0.0, 1.0)])
def test_magnitudes_of_a_prompt(q_scale, v_scale):
    """The same for prompt tokens on the tcgen05 kernel, with pages of very different values."""
    ops, d, heads, kv, n, new = _ops("bfloat16"), 128, 4, 2, 400, 100
    ops.KV4_PROMPT_BLOCKS = 0
    table, slots, records, rows = _filled(ops, [n], kv, d, 17, v_scale=v_scale)
    f32 = _ops("float32")
    pos, seq = _every_position([n])
    k, v = rows[0]
    v = v * torch.where(torch.arange(n) % 130 < 64, 1.0, 1e-3)[:, None, None]
    f32.rope_store_kv4(torch.cat((torch.zeros(n, kv, d), k, v), 1).flatten(1).cuda(), kv, kv, d, pos, seq, _i32(slots), table, records, None, 1.0, 0)
    rows = [tuple(t.cpu() for t in f32.kv4_values(records, pos, seq, _i32(slots), table, kv, d))]
    q = (torch.randn(new, heads, d, generator=torch.Generator().manual_seed(7)) * q_scale).bfloat16()
    got = ops.kv4_attention(q.cuda(), records, _i32([n]), _i32(slots), table, kv, d ** -0.5, cu_q=_i32([0, new]), tiles=(_i32([0, 0]), _i32([0, 64]), 2))
    _check(got, plain.attention(q, *rows[0], n - new, d ** -0.5, 0), rows, "bfloat16")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("q_scale,v_scale", [(30.0, 1.0), (1e-6, 1e-6), (1.0, 1e6), (0.0, 1.0)])
def test_magnitudes(dtype, q_scale, v_scale):
    """Sharp and flat distributions, values of any size: what is kept in 16 bits is divided by powers of two first."""
    ops, d, heads, kv = _ops(dtype), 64, 4, 2
    lengths = [300, 77]
    table, slots, records, rows = _filled(ops, lengths, kv, d, 17, v_scale=v_scale)
    q = (torch.randn(2, heads, d, generator=torch.Generator().manual_seed(7)) * q_scale).to(DT[dtype])
    got = ops.kv4_attention(q.cuda(), records, _i32(lengths), _i32(slots), table, kv, d ** -0.5)
    want = torch.cat([plain.attention(q[i:i + 1], k, v, n - 1, d ** -0.5, 0) for i, (n, (k, v)) in enumerate(zip(lengths, rows))])
    _check(got, want, rows, dtype)


@pytest.mark.parametrize("form", ["single", "prompt"])
@pytest.mark.parametrize("keys", [100, 8000, 40000])
@pytest.mark.parametrize("d,heads,kv", [(64, 16, 2), (128, 4, 2)])
def test_many_keys_in_fp32(d, heads, kv, keys, form):
    """Most of many weights are far below the largest, and each keeps its 22 bits: errors of 2^-23 of a query and of a weight, and of scores below 8 whose last
    bit is 2^-21, are independent and move the result by about 2^-22 of its norm; twice that is tolerated."""
    ops, new = _ops("float32"), 1 if form == "single" else 20
    table, slots, records, rows = _filled(ops, [keys, keys // 2], kv, d, 41)
    q = torch.randn(2 * new, heads, d, generator=torch.Generator().manual_seed(7)) * 0.8
    prompt = {} if form == "single" else dict(cu_q=_i32([0, new, 2 * new]), tiles=(_i32([0, 1]), _i32([0, 0]), 2))
    got = ops.kv4_attention(q.cuda(), records, _i32([keys, keys // 2]), _i32(slots), table, kv, d ** -0.5, **prompt).cpu().double().view(2 * new, heads, d)
    want = torch.cat([plain.attention(q[i * new:(i + 1) * new], k, v, k.shape[0] - new, d ** -0.5, 0) for i, (k, v) in enumerate(rows)])
    assert float((got - want).norm() / want.norm()) < 2.0 ** -21


def test_many_keys_whose_values_average_to_nothing_in_fp32():
    """Codes less 8 average to -1/2 and middles make up for it: the sums of both are some 20 times the result of 40,000 keys.  A warp adds about ten parts
    of 2^-24 to them, which moves the result by about 2^-19 of its norm."""
    ops, d, heads, kv, keys = _ops("float32"), 128, 32, 2, 40000
    table, slots, records, rows = _filled(ops, [keys], kv, d, 43)
    k, v = rows[0][0], torch.randn(keys, kv, d, generator=torch.Generator().manual_seed(9))
    pos, seq = _every_position([keys])
    ops.rope_store_kv4(torch.cat((torch.zeros(keys, kv, d), k, v), 1).flatten(1).cuda(), kv, kv, d, pos, seq, _i32(slots), table, records, None, 1.0, 0)
    k, v = (t.cpu() for t in ops.kv4_values(records, pos, seq, _i32(slots), table, kv, d))
    q = torch.randn(1, heads, d, generator=torch.Generator().manual_seed(7)) * 0.8
    got = ops.kv4_attention(q.cuda(), records, _i32([keys]), _i32(slots), table, kv, d ** -0.5).cpu().double().view(1, heads, d)
    want = plain.attention(q, k, v, keys - 1, d ** -0.5, 0)
    assert float((got - want).norm() / want.norm()) < 2.0 ** -19


@pytest.mark.parametrize("tcgen05", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("poison", [math.nan, math.inf, 1e30])
def test_tokens_that_are_not_seen_have_no_part(dtype, poison, tcgen05):
    """Keys and values behind a prompt's token, or before its window, that are no numbers or very large, do not reach it."""
    ops, d, heads, kv = _ops(dtype), 64, 4, 2
    ops.KV4_PROMPT_BLOCKS = 0 if tcgen05 else 1 << 30
    n, new = 150, 40
    table, slots, total = _tables([n], 5)
    pos, seq = _every_position([n])
    g = torch.Generator().manual_seed(3)
    kvs = torch.randn(n, 2 * kv, d, generator=g)
    records = torch.zeros(total, kv, ops.kv4_page_bytes(d), dtype=torch.uint8).cuda()
    f32 = _ops("float32")
    store = lambda x: f32.rope_store_kv4(torch.cat((torch.zeros(n, kv, d), x), 1).flatten(1).cuda(), kv, kv, d, pos, seq, _i32(slots), table,  # noqa: E731
                                         records, None, 1.0, 0)
    q = torch.randn(new, heads, d, generator=g).to(DT[dtype]).cuda()
    tiles = (_i32([0]), _i32([0]), 1)
    run = lambda w: ops.kv4_attention(q, records, _i32([n]), _i32(slots), table, kv, d ** -0.5, window=w, cu_q=_i32([0, new]), tiles=tiles)  # noqa: E731
    store(kvs)
    clean = {w: run(w).cpu() for w in (0, 20)}
    bad = kvs.clone()
    bad[130] = poison                                  # position of the prompt's token 20
    bad[60] = poison                                   # before every window
    store(bad)
    windowed = run(20).cpu()
    assert torch.equal(windowed[:20], clean[20][:20])
    bad[60] = kvs[60]
    store(bad)
    assert torch.equal(run(0).cpu()[:20], clean[0][:20])


@pytest.mark.parametrize("form", ["single", "prompt", "tcgen05", "shared"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,heads,kv", [(64, 4, 2), (128, 24, 1), (32, 2, 2)])
@pytest.mark.parametrize("half", [0, 1])
def test_half_a_value_that_is_no_number(half, d, heads, kv, dtype, form):
    """A value of which half a row is no number makes that half of the output none for the queries that see it, and leaves the other half: in the last,
    partial slice, in a whole one, and at a prompt's causal edge, whichever kernel reads it.  A key that is none makes all of the output none."""
    ops = _ops(dtype)
    ops.KV4_PROMPT_BLOCKS = 0 if form in ("tcgen05", "shared") else 1 << 30
    if form == "shared":
        ops.kv4_prompt_shares = lambda *a: 3
    n, new = 275, 1 if form == "single" else 40
    table, slots, total = _tables([n], 5)
    pos, seq = _every_position([n])
    g = torch.Generator().manual_seed(3)
    kvs = torch.randn(n, 2 * kv, d, generator=g)
    records = torch.zeros(total, kv, ops.kv4_page_bytes(d), dtype=torch.uint8).cuda()
    f32 = _ops("float32")
    q = torch.randn(new, heads, d, generator=g).to(DT[dtype])
    prompt = {} if form == "single" else dict(cu_q=_i32([0, new]), tiles=(_i32([0]), _i32([0]), 1))
    for what, at in (("value", 273), ("value", 260), ("value", 100), ("key", 273), ("key", 100), ("value", 250)):
        x = kvs.clone()
        x[at, (kv if what == "value" else 0) + kv - 1, half * (d // 2) + 5] = math.nan
        f32.rope_store_kv4(torch.cat((torch.zeros(n, kv, d), x), 1).flatten(1).cuda(), kv, kv, d, pos, seq, _i32(slots), table, records, None, 1.0, 0)
        k, v = (t.cpu() for t in f32.kv4_values(records, pos, seq, _i32(slots), table, kv, d))
        for window in (0, 30):
            got = ops.kv4_attention(q.cuda(), records, _i32([n]), _i32(slots), table, kv, d ** -0.5, window=window, **prompt).cpu().view(new, heads, d)
            want = plain.attention(q, k, v, n - new, d ** -0.5, window)
            assert torch.equal(got.isnan(), want.isnan()), (what, at, window)
            whole = want.isfinite()
            _check(torch.where(whole, got, 0).flatten(1), torch.where(whole, want, 0), [(k, v)], dtype)


def test_shares_do_not_depend_on_neighbours():
    """However a batch is cut among the blocks, a sequence's result stays within the tolerance, and one call gives the same bits twice."""
    ops, d, heads, kv = _ops("bfloat16"), 128, 16, 1
    lengths = [3000, 1, 64, 5000, 700, 0, 129] + [200] * 30
    table, slots, records, rows = _filled(ops, lengths, kv, d, 23)
    q = torch.randn(len(lengths), heads, d, generator=torch.Generator().manual_seed(7)).bfloat16()
    got = ops.kv4_attention(q.cuda(), records, _i32(lengths), _i32(slots), table, kv, d ** -0.5)
    again = ops.kv4_attention(q.cuda(), records, _i32(lengths), _i32(slots), table, kv, d ** -0.5)
    assert torch.equal(got, again)
    want = torch.cat([plain.attention(q[i:i + 1], k, v, n - 1, d ** -0.5, 0) for i, (n, (k, v)) in enumerate(zip(lengths, rows))])
    _check(got, want, rows, "bfloat16")
    for i in (0, 3, 4):
        alone = ops.kv4_attention(q[i:i + 1].cuda(), records, _i32(lengths[i:i + 1]), _i32(slots[i:i + 1]), table, kv, d ** -0.5)
        _check(alone, want[i:i + 1], rows, "bfloat16")


def test_more_tiles_than_a_launch_takes():
    ops, d, heads, kv = _ops("bfloat16"), 32, 2, 1
    lengths = [(i * 7) % 5 for i in range(4500)]
    table, slots, records, rows = _filled(ops, lengths, kv, d, 29)
    q = torch.randn(len(lengths), heads, d, generator=torch.Generator().manual_seed(7)).bfloat16()
    got = ops.kv4_attention(q.cuda(), records, _i32(lengths), _i32(slots), table, kv, d ** -0.5)
    want = torch.cat([plain.attention(q[i:i + 1], k, v, n - 1, d ** -0.5, 0) for i, (n, (k, v)) in enumerate(zip(lengths, rows))])
    _check(got, want, rows, "bfloat16")


def test_offsets_beyond_32_bits():
    """A page that begins behind 4 GB of records."""
    ops, d, heads, kv = _ops("bfloat16"), 128, 16, 2
    size = kv * ops.kv4_page_bytes(d)
    total = (1 << 32) // size + 40
    records = torch.empty(total, kv, size // kv, dtype=torch.uint8, device="cuda")
    table = _i32([[total - 1, total - 7, 2, total - 3]])
    n = 210
    g = torch.Generator().manual_seed(2)
    k, v = torch.randn(n, kv, d, generator=g), torch.randn(n, kv, d, generator=g)
    pos, seq = _every_position([n])
    f32 = _ops("float32")
    f32.rope_store_kv4(torch.cat((torch.zeros(n, kv, d), k, v), 1).flatten(1).cuda(), kv, kv, d, pos, seq, _i32([0]), table, records, None, 1.0, 0)
    got_k, got_v = f32.kv4_values(records, pos, seq, _i32([0]), table, kv, d)
    assert torch.equal(got_k.cpu(), plain.quantised(k)[0]) and torch.equal(got_v.cpu(), plain.quantised(v)[0])
    q = torch.randn(1, heads, d, generator=g).bfloat16()
    got = ops.kv4_attention(q.cuda(), records, _i32([n]), _i32([0]), table, kv, d ** -0.5)
    _check(got, plain.attention(q, got_k.cpu(), got_v.cpu(), n - 1, d ** -0.5, 0), [(got_k.cpu(), got_v.cpu())], "bfloat16")


def test_another_stream_and_views():
    """Calls on a stream of their own, of tensors that are parts of larger ones."""
    ops, d, heads, kv = _ops("bfloat16"), 64, 8, 2
    lengths = [100, 333]
    table, slots, records, rows = _filled(ops, lengths, kv, d, 31)
    q = torch.randn(2, heads, d, generator=torch.Generator().manual_seed(7)).bfloat16()
    want = torch.cat([plain.attention(q[i:i + 1], k, v, n - 1, d ** -0.5, 0) for i, (n, (k, v)) in enumerate(zip(lengths, rows))])
    larger = torch.zeros(5, heads, d, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        larger[1:3].copy_(q.cuda())
        got = ops.kv4_attention(larger[1:3], records, _i32([7] + lengths)[1:], _i32([1] + slots)[1:], table, kv, d ** -0.5)
    side.synchronize()
    _check(got, want, rows, "bfloat16")


def test_refusals_of_the_4_bit_cache():
    ops, d, kv = _ops("bfloat16"), 64, 2
    records = torch.zeros(4, kv, ops.kv4_page_bytes(d), dtype=torch.uint8).cuda()
    table, one = torch.zeros(1, 4, dtype=torch.int32).cuda(), _i32([1])
    zero = _i32([0])
    q = torch.zeros(1, 4, d, dtype=torch.bfloat16).cuda()
    call = lambda **k: ops.kv4_attention(**{**dict(q=q, records=records, kv_len=one, slots=zero, page_table=table, n_kv=kv, scale=1.0), **k})  # noqa: E731
    call()
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=torch.zeros(1, 3, d, dtype=torch.bfloat16).cuda()), dict(records=records[:, :1]),
                dict(records=records.float()), dict(n_kv=1), dict(kv_len=_i32([1, 1])), dict(slots=_i32([0, 0])), dict(kv_len=one.long()),
                dict(window=-1), dict(cu_q=_i32([0, 1])), dict(cu_q=_i32([0]), tiles=(zero, zero, 1)), dict(cu_q=_i32([0, 1]), tiles=(zero, zero, 2)),
                dict(page_table=table[0]), dict(q=torch.zeros(1, 4, 48, dtype=torch.bfloat16).cuda())):
        with pytest.raises(ValueError):
            call(**bad)
    qkv = torch.zeros(1, 8 * d, dtype=torch.bfloat16).cuda()
    inv = torch.ones(d // 2).cuda()
    store = lambda **k: ops.rope_store_kv4(**{**dict(qkv=qkv, n_heads=4, n_kv=kv, d=d, positions=zero, token_seq=zero, slots=zero, page_table=table,  # noqa: E731
                                                    records=records, inv_freq=inv, magnitude=1.0, rot_dim=d), **k})
    store()
    off = torch.zeros(8 * d + 1, dtype=torch.bfloat16).cuda()[1:].view(1, -1)
    for bad in (dict(qkv=qkv[:, :-8]), dict(qkv=off), dict(rot_dim=d // 2), dict(inv_freq=inv[1:]), dict(positions=_i32([0, 1])), dict(token_seq=_i32([])),
                dict(records=records[..., :-16]), dict(n_heads=5), dict(qkv=qkv.float())):
        with pytest.raises(ValueError):
            store(**bad)
    with pytest.raises(ValueError):
        ops.kv4_values(records, zero, _i32([0, 0]), zero, table, kv, d)
    with pytest.raises(ValueError):
        ops.kv4_values(records, zero, zero, zero, table, kv, 48)
    assert ops.kv4_attention(q[:0], records, one[:0], zero[:0], table, kv, 1.0).shape == (0, 4 * d)


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("shapes", [[(3, 20, 2, 64, 32)], [(2, 20, 5), (4, 20, 3), (1, 20, 7, 16)], [(1, 20, 1)] * 11, [(2, 20, 4096), (0, 20, 4), (5, 20, 9000)]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8])
def test_copy_pages(shapes, dtype):
    ops = _ops("bfloat16")
    g = torch.Generator().manual_seed(1)
    tensors = [torch.randint(0, 200, s, generator=g).to(dtype) for s in shapes]
    here = [t.cuda() for t in tensors]
    src, dst = [3, 3, 19, 0, 25, 4, -1], [1, 2, 18, 5, 6, 40, 7]           # one page twice; numbers that are no page
    ops.copy_pages(here, _i32(src), _i32(dst))
    for t in tensors:
        for a, b in zip(src[:4], dst[:4]):
            t[:, b] = t[:, a]
    for got, want in zip(here, tensors):
        assert torch.equal(got.cpu(), want)


def test_copy_pages_of_unaligned_tensors_and_refusals():
    ops = _ops("bfloat16")
    t = torch.arange(4 * 8 * 6 + 1, dtype=torch.int16).to(torch.uint8).cuda()[1:].view(4, 8, 6)
    want = t.cpu().clone()
    want[:, 7] = want[:, 2]
    ops.copy_pages([t], _i32([2]), _i32([7]))
    assert torch.equal(t.cpu(), want)
    ops.copy_pages([], _i32([2]), _i32([7]))
    ops.copy_pages([t], _i32([]), _i32([]))
    for bad in (lambda: ops.copy_pages([t], _i32([2]), _i32([7, 1])), lambda: ops.copy_pages([t[:, :4]], _i32([2]), _i32([1])),
                lambda: ops.copy_pages([t.cpu()], _i32([2]), _i32([1])), lambda: ops.copy_pages([t], _i32([2]).long(), _i32([1])),
                lambda: ops.copy_pages([t.view(-1)], _i32([2]), _i32([1]))):
        with pytest.raises(ValueError):
            bad()
    assert torch.equal(t.cpu(), want)


# ---------------------------------------------------------------------------
# filtered sampling
# ---------------------------------------------------------------------------

def _settings(rows, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda: torch.rand(rows, generator=g)  # noqa: E731
    t = torch.where(r() < 0.2, torch.zeros(rows), 0.3 + 1.5 * r())
    k = torch.where(r() < 0.4, torch.zeros(rows), (vocab * r() ** 3).ceil()).int()
    p = torch.where(r() < 0.4, torch.ones(rows), r())
    m = torch.where(r() < 0.5, torch.zeros(rows), 0.2 * r())
    return r(), t, k, p, m


def _compare(ops, z, u, t, k, p, m):
    tok, lp = ops.sample_filtered(z.cuda(), u.cuda(), t.cuda(), k.cuda(), p.cuda(), m.cuda())
    for i in range(z.shape[0]):
        want, logp = plain.sampled(z[i], float(u[i]), float(t[i]), int(k[i]), float(p[i]), float(m[i]))
        assert int(tok[i]) == want, (i, int(tok[i]), want, float(t[i]), int(k[i]), float(p[i]), float(m[i]))
        # two roundings of a difference of up to 100, and a logarithm of up to 30
        assert float(lp[i]) == logp or abs(float(lp[i]) - logp) < 2e-5, (float(lp[i]), logp)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (7, 31), (5, 333), (40, 1000), (2, 5001), (150, 1030), (3, 20000)])
def test_sample_filtered(rows, vocab):
    z = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab)) * 3
    _compare(_ops("bfloat16"), z, *_settings(rows, vocab, rows))


@pytest.mark.parametrize("levels", [1, 2, 5])
def test_sample_filtered_ties(levels):
    """Rows of a few different logits: borders fall among equal ones, of which the first by index stay."""
    rows, vocab = 60, 700
    g = torch.Generator().manual_seed(levels)
    z = torch.randint(0, levels, (rows, vocab), generator=g).float() * 0.5
    _compare(_ops("bfloat16"), z, *_settings(rows, vocab, 5))


def test_sample_filtered_edges():
    vocab = 1500
    z = torch.randn(16, vocab, generator=torch.Generator().manual_seed(3))
    z[0] = -math.inf                                   # nothing to draw
    z[1] = math.nan
    z[2, :] = -math.inf
    z[2, 700] = -5.0                                   # a single token
    z[3, 10:] = -math.inf
    z[4, ::2] = math.nan
    z[5, [7, 900]] = math.inf
    z[6] = torch.finfo(torch.float32).min              # masks of the type's lowest value
    z[6, 1499] = 3.0
    z[7] = torch.finfo(torch.float32).min
    z[8] *= 1e4
    u = torch.full((16,), 0.5)
    u[9], u[10] = 0.0, 1.0 - 2.0 ** -24
    t = torch.full((16,), 0.9)
    t[11], t[12], t[13] = 1e-30, -1.0, math.nan
    k = torch.zeros(16, dtype=torch.int32)
    k[14], k[15] = vocab + 5, 1
    p, m = torch.ones(16), torch.zeros(16)
    p[3], p[4] = 0.0, 0.5
    m[14] = 2.0
    _compare(_ops("bfloat16"), z, u, t, k, p, m)


@pytest.mark.parametrize("ratio", [-0.0, -0.1, -math.inf, math.nan])
def test_sample_filtered_takes_a_min_p_of_no_more_than_zero_as_none(ratio):
    """Alone, with few and with many tokens left by top-k, and with top-p: the token is the one without min-p."""
    vocab = 1500
    z = torch.randn(5, vocab, generator=torch.Generator().manual_seed(8))
    k = torch.tensor([0, 20, 1000, 0, 1000], dtype=torch.int32)
    p = torch.tensor([1.0, 1.0, 1.0, 0.7, 0.7])
    _compare(_ops("bfloat16"), z, torch.full((5,), 0.6), torch.ones(5), k, p, torch.full((5,), ratio))


@pytest.mark.parametrize("rows,vocab", [(1, 73448), (64, 73448), (200, 40000), (1, 500000)])
def test_sample_filtered_large_rows(rows, vocab):
    """The largest vocabularies, against the definition in whole numbers on the device; the last does not fit in shared memory."""
    ops = _ops("bfloat16")
    z = (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(1)) * 2).cuda()
    u, t, k, p, m = (x.cuda() for x in _settings(rows, vocab, 9))
    t = t.clamp_min(0.5)
    tok, lp = ops.sample_filtered(z, u, t, k, p, m)
    again, _ = ops.sample_filtered(z, u, t, k, p, m)
    assert torch.equal(tok, again)
    w = torch.exp((z - z.amax(1, keepdim=True)) / t[:, None])
    units = (w.double() * plain.UNIT).long()
    ranked, order = torch.sort(w, dim=1, descending=True, stable=True)
    mass = units.gather(1, order).cumsum(1)
    n = torch.where(k > 0, k, vocab).long()
    within = mass.gather(1, n[:, None] - 1)
    n = torch.where(p < 1, torch.minimum(n, (mass.double() < p.double()[:, None] * within.double()).sum(1) + 1), n)
    n = torch.where(m > 0, torch.minimum(n, (ranked >= m[:, None]).sum(1)), n).clamp_min(1)
    keep = torch.zeros_like(z, dtype=torch.bool).scatter(1, order, torch.arange(vocab, device="cuda") < n[:, None])
    c = torch.where(keep, units, 0).cumsum(1)
    target = (u.double() * c[:, -1].double()).long()
    assert torch.equal(tok.long(), (c <= target[:, None]).sum(1))
    want = (z.double().gather(1, tok.long()[:, None])[:, 0] - z.double().amax(1)) / t.double() - torch.log(c[:, -1].double() / plain.UNIT)
    assert float((lp.double() - want).abs().max()) < 2e-5


def _defined(z, u, t, k, p, m):
    """Token of each row by the definition in whole numbers, on the device."""
    vocab = z.shape[1]
    w = torch.exp((z - z.amax(1, keepdim=True)) / t[:, None])
    units = (w.double() * plain.UNIT).long()
    ranked, order = torch.sort(w, dim=1, descending=True, stable=True)
    mass = units.gather(1, order).cumsum(1)
    n = torch.where(k > 0, k, vocab).long().clamp_max(vocab)
    within = mass.gather(1, n[:, None] - 1)
    n = torch.where(p < 1, torch.minimum(n, (mass.double() < p.double()[:, None] * within.double()).sum(1) + 1), n)
    n = torch.where(m > 0, torch.minimum(n, (ranked >= m[:, None]).sum(1)), n).clamp_min(1)
    keep = torch.zeros_like(z, dtype=torch.bool).scatter(1, order, torch.arange(vocab, device="cuda") < n[:, None])
    c = torch.where(keep, units, 0).cumsum(1)
    return (c <= (u.double() * c[:, -1].double()).long()[:, None]).sum(1)


@pytest.mark.parametrize("rows,vocab", [(70, 73448), (6, 73448), (300, 19000), (2, 300000)])
@pytest.mark.parametrize("spread", ["narrow", "wide", "tail"])
def test_sample_filtered_where_bins_are_full_or_tiny(rows, vocab, spread):
    """Weights that all lie in one or two bins, with every bit below the bin's number in use (sums beyond 32 bits); weights over 200 octaves; and
    a few large ones before a tail in which most of the mass lies below 2^-17 of the largest."""
    ops, g = _ops("bfloat16"), torch.Generator().manual_seed(rows)
    r = lambda *n: torch.rand(*n, generator=g)  # noqa: E731
    z = {"narrow": -0.02 * r(rows, vocab), "wide": 70 * torch.randn(rows, vocab, generator=g), "tail": -11.5 - 4 * r(rows, vocab)}[spread]
    if spread == "tail":
        z[:, ::vocab // 3] = 0.0
    p = torch.where(r(rows) < 0.3, torch.ones(rows), r(rows))
    p[0] = 1 - 2.0 ** -20
    k = torch.where(r(rows) < 0.6, torch.zeros(rows), (vocab * r(rows)).ceil()).int()
    m = torch.where(r(rows) < 0.8, torch.zeros(rows), 1e-6 * r(rows))
    args = [x.cuda() for x in (z, r(rows), torch.ones(rows), k, p, m)]
    assert torch.equal(ops.sample_filtered(*args)[0].long(), _defined(*args))


@pytest.mark.parametrize("vocab,of_one", [(1 << 20, 1.0), (1 << 21, 1.0), (1 << 19, 2.0 ** -12 * (1 - 2.0 ** -20)), (1 << 21, 2.0 ** -12 * (1 - 2.0 ** -20)),
                                          (350000, math.exp(-1)), (300000, 2.0 ** -39)])
def test_sample_filtered_of_flat_rows_above_2_18_tokens(vocab, of_one):
    """One token of weight 1 and all others of one weight: the blocks of a cluster find them in a single bin, whose mass needs more than 32 bits in every limb."""
    ops = _ops("bfloat16")
    z = torch.full((6, vocab), math.log(of_one))
    z[:, vocab // 3] = 0.0
    u = torch.tensor([0.1, 0.5, 0.9, 1 - 2.0 ** -24, 0.7, 0.0])
    p = torch.tensor([0.9, 0.3, 0.99999, 1 - 2.0 ** -20, 0.5, 0.9])
    k = torch.tensor([0, 0, 0, 0, vocab - 7, vocab // 2], dtype=torch.int32)
    args = [x.cuda() for x in (z, u, torch.ones(6), k, p, torch.zeros(6))]
    assert torch.equal(ops.sample_filtered(*args)[0].long(), _defined(*args))


def test_sample_filtered_is_distributed_as_it_should():
    """Frequencies over many given numbers against the kept probabilities: with 200,000 draws a share moves by 0.0011 (one sigma at one half)."""
    ops, vocab, n = _ops("bfloat16"), 50, 200000
    z = torch.randn(1, vocab, generator=torch.Generator().manual_seed(4)) * 1.5
    u = torch.rand(n, generator=torch.Generator().manual_seed(5))
    full = lambda x, dt=torch.float32: torch.full((n,), x, dtype=dt).cuda()  # noqa: E731
    tok, lp = ops.sample_filtered(z.expand(n, vocab).contiguous().cuda(), u.cuda(), full(0.8), full(12, torch.int32), full(0.9), full(0.03))
    share = torch.bincount(tok.long().cpu(), minlength=vocab).double() / n
    prob = torch.softmax(z[0].double() / 0.8, 0)
    ranked, order = torch.sort(prob, descending=True)
    ranked = ranked[:12]
    count = int((ranked.cumsum(0) < 0.9 * ranked.sum()).sum()) + 1
    count = min(count, int((ranked >= 0.03 * ranked[0]).sum()))
    want = torch.zeros(vocab, dtype=torch.float64)
    want[order[:count]] = prob[order[:count]] / prob[order[:count]].sum()
    assert float((share - want).abs().max()) < 6 * 0.0011
    assert float((lp.cpu().double().exp() - want[tok.long().cpu()]).abs().max()) < 1e-5


def test_sample_filtered_with_keys_draws_what_sample_draws():
    """The numbers made from seed and keys are those of ``sample``: without filters both draw from the same distribution at the same place."""
    ops = _ops("bfloat16")
    rows, vocab = 300, 90
    z = (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(6))).cuda()
    keys, steps = torch.arange(rows, dtype=torch.int32).cuda(), torch.full((rows,), 3, dtype=torch.int32).cuda()
    t = torch.full((rows,), 1.1).cuda()
    a = ops.sample(z, t, None, 77, keys, steps)
    b, _ = ops.sample_filtered(z, None, t, seed=77, seq_key=keys, step_key=steps)
    # masses are rounded differently: a draw within 1e-6 of a border may fall on its other side
    assert int((a != b).sum()) <= 1


def test_sample_filtered_leaves_other_rows_alone():
    ops = _ops("bfloat16")
    rows, vocab = 9, 5000
    z = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(6)).cuda()
    u, t, k = torch.rand(rows, generator=torch.Generator().manual_seed(7)).cuda(), torch.ones(rows).cuda(), torch.full((rows,), 900, dtype=torch.int32).cuda()
    want, logp = ops.sample_filtered(z, u, t, k)
    drawn = _i32([1, 0, 0, 1, 1, 0, 1, 0, 5])
    out = torch.arange(100, 100 + rows, dtype=torch.int32).cuda()
    got, lp = ops.sample_filtered(z, u, t, k, out=out, drawn=drawn)
    assert got is out and torch.equal(got, torch.where(drawn > 0, want, torch.arange(100, 100 + rows, dtype=torch.int32).cuda()))
    assert torch.equal(lp.isnan(), drawn == 0) and torch.equal(lp[drawn > 0], logp[drawn > 0])
    for bad in (dict(drawn=drawn), dict(drawn=drawn[1:], out=out), dict(drawn=drawn.long(), out=out)):
        with pytest.raises(ValueError):
            ops.sample_filtered(z, u, t, k, **bad)


def test_refusals_of_sample_filtered():
    ops = _ops("bfloat16")
    z, one = torch.zeros(2, 5).cuda(), torch.ones(2).cuda()
    ops.sample_filtered(z, one * 0.5, one)
    for bad in (dict(logits=z.bfloat16()), dict(logits=z[0]), dict(uniform=None), dict(temperature=None), dict(temperature=one[:1]),
                dict(top_k=one), dict(top_p=one[:1]), dict(min_p=one.double()), dict(logits=torch.zeros(2, 10).cuda()[:, ::2])):
        with pytest.raises(ValueError):
            ops.sample_filtered(**{**dict(logits=z, uniform=one * 0.5, temperature=one), **bad})
    assert ops.sample_filtered(z[:0], one[:0], one[:0])[0].numel() == 0
