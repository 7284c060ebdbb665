"""Forking and compacting the cache, several answers to a prompt, and the settings of the 4-bit cache and of the filters, without a device."""
import random

import pytest
import torch

from cpmcu_b200.cache import Cache, CacheFull, FreeList, HandleError, pages_for
from cpmcu_b200.config.base import ConfigError
from cpmcu_b200.config.minicpm import MiniCPMConfig
from cpmcu_b200.engine.generate import Request, plan_batches, run_requests
from cpmcu_b200.models.minicpm4 import model_spec
from cpmcu_b200.models.model import Model
from cpmcu_b200.ops.dry import measure_workspace
from cpmcu_b200.parts.base import CacheNeeds
from cpmcu_b200.sampling import SamplingParams
from tests.configs import tiny_a, tiny_b, tiny_e


def test_free_list_shares_and_moves():
    f = FreeList(6, "page")
    f.take(4)
    f.share([1, 2])
    f.give_back([1, 2, 3])
    assert f.n_free == 3 and f.is_held(1) and not f.is_held(3) and f.times_held(2) == 1
    with pytest.raises(HandleError):
        f.share([3])
    f.share([2])
    f.move([(2, 5), (1, 3)])
    assert f.times_held(5) == 2 and not f.is_held(2) and f.take(3) == [1, 2, 4]
    for bad in ([(4, 5)], [(0, 9)]):
        with pytest.raises(HandleError):
            f.move(bad)


def test_free_list_given_back_in_one_call():
    """A number in the list as often as it is held is free once; more often is an error, and nothing is given back."""
    f = FreeList(4, "page")
    f.take(3)
    f.share([1])
    for bad in ([0, 0], [2, 1, 1, 1], [1, 3]):
        with pytest.raises(HandleError):
            f.give_back(bad)
    assert f.n_free == 1 and f.times_held(1) == 2 and f.times_held(0) == 1
    f.give_back([1, 2, 1])
    assert f.n_free == 3 and f.take(3) == [1, 2, 3]


def _cache(n_pages=40, n_slots=8):
    needs = [CacheNeeds(kv_heads=2, head_dim=16), CacheNeeds(kv_heads=2, head_dim=32, bits=4), CacheNeeds(kv_heads=1, head_dim=32, window=70),
             CacheNeeds(kv_heads=1, head_dim=16, pooled_stride=16, pooled_kernel=32), CacheNeeds(state={"acc": ((8,), torch.float32)})]
    return Cache(needs, max_tokens=64 * n_pages, dtype=torch.float32, device="cpu", n_slots=n_slots)


def _write(c, slot, start, length, mark):
    """Marks the tokens [start, length) of a sequence in every lane, as a step would store them."""
    for lane in c.lanes:
        g = lane.group
        for t in range(start, length):
            page = g.pages_of_slot.get(slot, [None] * (t // 64 + 1))[t // 64]
            if g.k is not None and page != -1:
                lane.k[page, :, t % 64] = mark * 1000 + t
            if g.records is not None:
                lane.records[page, :, t % 64] = (mark * 7 + t) % 251
        for s in lane.state.values():
            s[slot] += mark


def _read(c, slot, length):
    out = []
    for lane in c.lanes:
        g = lane.group
        row = g.page_table[slot]
        for t in range(length):
            if g.k is not None and (not g.needs.window or t > length - g.needs.window):
                out.append(float(lane.k[row[t // 64], 0, t % 64, 0]))
            if g.records is not None:
                out.append(int(lane.records[row[t // 64], 0, t % 64]))
        out.extend(float(s[slot][0]) for s in lane.state.values())
    return out


def test_records_of_a_group_in_4_bits():
    c = _cache()
    lane = c.lane(1)
    assert lane.k is None and lane.v is None and lane.records.shape == (40, 2, 64 * 32 + 1024) and lane.records.dtype == torch.uint8
    assert lane.n_pages == 40 and c.lane(0).n_pages == 40 and c.lane(4).n_pages == 0
    assert lane.group.bytes_per_token() == 2 * (32 + 16) and c.lane(0).group.bytes_per_token() == 2 * 2 * 16 * 4


@pytest.mark.parametrize("length", [1, 63, 64, 65, 128, 200])
def test_forked_sequences_go_on_by_themselves(length):
    c = _cache()
    a = c.open_sequence()
    c.reserve(a, length)
    _write(c, a, 0, length, 1)
    c.set_length(a, length)
    c.sync()
    before = _read(c, a, length)
    children = c.fork_sequence(a, 3)
    c.sync()
    c.check_consistent()
    assert [c.length(s) for s in children] == [length] * 3
    # the full pages are there once
    assert c.groups[0].pages.n_held == length // 64 + 4 * (pages_for(length) - length // 64)
    for s in children:
        assert _read(c, s, length) == before
    want = {}
    for i, s in enumerate([a] + children):                      # every one of them grows, and none sees the others
        c.reserve(s, length + 70)
        _write(c, s, length, length + 70, 10 + i)
        c.set_length(s, length + 70)
        c.sync()
        want[s] = _read(c, s, length + 70)
    for s in [a] + children:
        assert _read(c, s, length + 70) == want[s]
    c.check_consistent()
    c.close_sequence(a)
    c.check_consistent()
    for s in children:
        assert _read(c, s, length + 70) == want[s]
        c.close_sequence(s)
        c.check_consistent()
    assert c.tokens_held() == 0


def test_fork_is_all_or_nothing_and_refuses():
    c = _cache(n_pages=5, n_slots=4)
    a = c.open_sequence()
    c.reserve(a, 100)
    c.set_length(a, 100)
    with pytest.raises(CacheFull, match="slots"):
        c.fork_sequence(a, 4)
    c.reserve(a, 200)                                            # four pages: no room for two more partial ones
    c.set_length(a, 200)
    with pytest.raises(CacheFull, match="forking"):
        c.fork_sequence(a, 2)
    assert c.slots.n_held == 1 and c.groups[0].pages.n_held == 4
    assert c.fork_sequence(a, 0) == []
    with pytest.raises(HandleError):
        c.fork_sequence(3, 1)
    c.check_consistent()


def test_random_open_fork_grow_close_compact():
    rng = random.Random(3)
    c = _cache(n_pages=60, n_slots=10)
    live, mark = {}, 0
    for _ in range(400):
        op = rng.random()
        try:
            if op < 0.25:
                s = c.open_sequence()
                live[s] = []
            elif op < 0.45 and live:
                s = rng.choice(list(live))
                for child in c.fork_sequence(s, rng.randint(1, 2)):
                    live[child] = list(live[s])
            elif op < 0.8 and live:
                s = rng.choice(list(live))
                n, more = c.length(s), rng.randint(1, 90)
                c.reserve(s, n + more)
                mark += 1
                _write(c, s, n, n + more, mark)
                c.set_length(s, n + more)
                live[s].append(mark)
            elif op < 0.9 and live:
                s = rng.choice(list(live))
                c.close_sequence(s)
                del live[s]
            else:
                held = [g.pages.n_held for g in c.groups]
                c.sync()
                want = {s: _read(c, s, c.length(s)) for s in live}
                c.compact()
                c.sync()
                for g, n in zip(c.groups, held):
                    assert g.pages.n_held == n and all(g.pages.is_held(p) for p in range(n))
                for s in live:
                    assert _read(c, s, c.length(s)) == want[s]
        except CacheFull:
            pass
        c.check_consistent()
    assert mark > 50


class ForkingBackend:
    """Scripted tokens: sequence with key k produces k*100 + n as its n-th token."""

    def __init__(self, pages=100, batch=5):
        self.pages, self.batch, self.ran, self.open = pages, batch, [], {}

    def capacity_pages(self): return self.pages
    def max_batch(self): return self.batch

    def prefill(self, prompts, keys, sampling):
        return self.prefill_forked(prompts, list(range(len(prompts))), keys, sampling)

    def prefill_forked(self, prompts, which, keys, sampling):
        assert not self.open and len(which) == len(keys) == len(sampling)
        self.ran.append([list(p) for p in prompts])
        self.open = {i: k for i, k in enumerate(keys)}
        self.prompt_of = [tuple(prompts[w]) for w in which]
        return [k * 100 for k in keys]

    def decode(self, live, last, keys, steps, sampling, changed):
        return [k * 100 + n for k, n in zip(keys, steps)]

    def finish(self, index):
        del self.open[index]

    def abort(self):
        self.open = {}


def test_answers_of_a_group_run_their_prompt_once_a_batch():
    reqs = [Request([1, 2, 3], 3, key=j, group=7) for j in range(3)] + [Request([9], 2, key=3), Request([4, 4], 2, key=4, group=8)] + \
           [Request([4, 4], 1, key=5, group=8)]
    b = ForkingBackend()
    out, stats = run_requests(b, reqs)
    assert [f.tokens for f in out] == [[0, 1, 2], [100, 101, 102], [200, 201, 202], [300, 301], [400, 401], [500]]
    assert b.ran == [[[1, 2, 3], [9], [4, 4]], [[4, 4]]]           # five a batch: the last group is cut
    assert stats.prompt_tokens == 3 + 1 + 2 + 2 and not b.open
    with pytest.raises(ValueError, match="another prompt"):
        run_requests(b, [Request([1], 1, group=0), Request([2], 1, group=0)])


def test_plan_batches_counts_shared_pages_once():
    reqs = [Request([0] * 130, 20, group=0) for _ in range(4)]      # three pages each, two of them shared
    assert plan_batches(reqs, 8, 6) == [[0, 1, 2, 3]]
    assert plan_batches(reqs, 8, 5) == [[0, 1, 2], [3]]
    assert plan_batches([Request([0] * 130, 20) for _ in range(4)], 8, 6) == [[0, 1], [2, 3]]


class CacheBackend(ForkingBackend):
    """Scripted tokens over a cache whose sequences grow by a token a step."""

    def __init__(self, cache):
        super().__init__(cache.n_pages - 1, 8)
        self.cache = cache
        pad = cache.open_sequence()
        cache.reserve(pad, 1)

    def shared_pages(self, length):
        return self.cache.shared_pages(length)

    def _grow(self, slot, length):
        self.cache.reserve(slot, length)
        self.cache.set_length(slot, length)

    def prefill_forked(self, prompts, which, keys, sampling):
        firsts = self.cache.open_sequences(len(prompts))
        slots_of = []
        for i, (s, p) in enumerate(zip(firsts, prompts)):
            self._grow(s, len(p))
            slots_of.append([s] + self.cache.fork_sequence(s, which.count(i) - 1))
        self.slots = [slots_of[w].pop(0) for w in which]
        return super().prefill_forked(prompts, which, keys, sampling)

    def decode(self, live, *args):
        for p in live:
            self._grow(self.slots[p], self.cache.length(self.slots[p]) + 1)
        self.cache.check_consistent()
        return super().decode(live, *args)

    def finish(self, index):
        super().finish(index)
        self.cache.close_sequence(self.slots[index])


@pytest.mark.parametrize("kernel,stride", [(0, 0), (32, 16), (128, 32)])
@pytest.mark.parametrize("length", [1, 63, 64, 94, 95, 96, 128, 130, 159, 191, 192])
def test_groups_that_are_planned_can_be_forked(length, kernel, stride):
    """Every cache that holds one request alone runs a group of four, in as many batches as its pages allow: with pooled keys forks share
    fewer pages than the prompt fills."""
    need = pages_for(length + 20)
    for pages in range(need, 4 * need + 1):
        c = Cache([CacheNeeds(kv_heads=1, head_dim=16), CacheNeeds(kv_heads=1, head_dim=16, pooled_stride=stride, pooled_kernel=kernel)],
                  max_tokens=64 * (pages + 1), dtype=torch.float32, device="cpu", n_slots=9)
        b = CacheBackend(c)
        out, stats = run_requests(b, [Request([1] * length, 20, key=j, group=0) for j in range(4)])
        assert [len(f.tokens) for f in out] == [20] * 4 and c.slots.n_held == 1
        assert stats.batches == 1 or pages < 4 * need - 3 * c.shared_pages(length)


def test_sampling_params():
    assert not SamplingParams(0.7, 0.9).filtered and not SamplingParams(0.0, 1.0, 5, 0.1).filtered
    assert SamplingParams(0.7, 1.0, 5).filtered and SamplingParams(0.7, min_p=0.1).filtered
    for bad in (dict(top_k=-1), dict(min_p=-0.1), dict(min_p=1.5)):
        with pytest.raises(ValueError):
            SamplingParams(0.5, **bad)


def test_configuration_of_the_cache():
    cfg = MiniCPMConfig.from_dict(dict(tiny_e(), cache_bits=4))
    assert cfg.cache_bits == 4 and MiniCPMConfig.from_dict(cfg.to_dict()) == cfg
    plain = MiniCPMConfig.from_dict(tiny_e())
    assert plain.cache_bits == 16 and "cache_bits" not in plain.to_dict()
    needs = Model(model_spec(cfg), None).cache_needs()
    assert all(n.bits == 4 and n.kv_heads == 2 and n.head_dim == 128 for n in needs)
    assert all(n.bits == 0 for n in Model(model_spec(plain), None).cache_needs())
    with pytest.raises(ConfigError):
        MiniCPMConfig.from_dict(dict(tiny_e(), cache_bits=8))
    with pytest.raises(ValueError, match="4 bits"):
        Model(model_spec(MiniCPMConfig.from_dict(dict(tiny_a(), cache_bits=4))), None)          # heads of 16 channels
    with pytest.raises(ValueError, match="4 bits"):
        Model(model_spec(MiniCPMConfig.from_dict(dict(tiny_b(), cache_bits=4))), None)          # sparse attention


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_workspace_is_measured_for_the_4_bit_cache(dtype):
    cfg = MiniCPMConfig.from_dict(dict(tiny_e(), cache_bits=4))
    persistent, frame, notes = measure_workspace(model_spec(cfg), dtype, 512, 8, 4096)
    assert persistent > 0 and frame > 0 and notes == []


def test_errors_of_the_prompt_kernel_are_asked_for_once_it_ran():
    from cpmcu_b200.ops.dry import DryOps

    class Library(type(DryOps(torch.bfloat16).lib)):
        def __init__(self):
            self.asked, self.code, self.checked_files = [], 0, ()

        def cpm_kv4_prompt_error(self):
            self.asked.append(self.code)
            return self.code

    ops = DryOps(torch.bfloat16)
    ops.lib = Library()
    ops.raise_on_kernel_error()
    assert ops.lib.asked == []
    meta = lambda *shape, dtype=torch.int32: torch.empty(*shape, dtype=dtype, device="meta")  # noqa: E731
    ops.kv4_attention(meta(700, 32, 128, dtype=torch.bfloat16), meta(20, 2, ops.kv4_page_bytes(128), dtype=torch.uint8), meta(1), meta(1), meta(1, 20), 2, 0.1,
                      cu_q=meta(2), tiles=(meta(11), meta(11), 11))
    ops.raise_on_kernel_error()
    ops.lib.code = 3
    with pytest.raises(RuntimeError, match="4-bit cache"):
        ops.raise_on_kernel_error()
    assert ops.lib.asked == [0, 3]


def test_cli_options():
    from cpmcu_b200.cli import create_cli_parser
    args = create_cli_parser().parse_args(["--model-path", "x", "--cache-bits", "4", "--samples", "3", "--top-k", "20", "--min-p", "0.05"])
    assert (args.cache_bits, args.samples, args.top_k, args.min_p) == (4, 3, 20, 0.05)
    args = create_cli_parser().parse_args(["--model-path", "x"])
    assert (args.cache_bits, args.samples, args.top_k, args.min_p) == (None, 1, 0, 0.0)
