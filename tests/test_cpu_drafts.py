"""Drafting by lookup, the generation loop with steps of several tokens, and what takes drafted tokens, without a device."""
import random

import pytest
import torch

from cpmcu_b200.cli import create_cli_parser
from cpmcu_b200.config.minicpm import MiniCPMConfig
from cpmcu_b200.engine.drafts import Lookup, tokens_of_step
from cpmcu_b200.engine.generate import Request, run_requests
from cpmcu_b200.models.minicpm4 import model_spec
from cpmcu_b200.models.model import Model
from cpmcu_b200.ops.dry import DryOps, measure_workspace
from tests import configs


def test_lookup_finds_what_followed():
    look = Lookup([1, 2, 3, 4, 5, 9, 1, 2])
    assert look.propose(3) == ([3, 4, 5], [0, 1, 2])
    look.extend([3])
    assert look.propose(2) == ([4, 5], [0, 1])
    look.extend([7])
    assert look.propose(4) == ([], [])
    assert Lookup([5]).propose(3) == ([], []) and Lookup().propose(3) == ([], [])


def test_lookup_merges_continuations_into_a_tree():
    # after 1 2 came 3 4, then 3 5, and last 6
    look = Lookup([1, 2, 3, 4, 0, 1, 2, 3, 5, 0, 1, 2, 6, 8, 1, 2])
    ids, parents = look.propose(6)
    assert (ids[:2], parents[:2]) == ([6, 8], [0, 1])                        # the latest first
    paths = set()
    for i in range(len(ids)):
        path, at = (), i + 1
        while at:
            path, at = (ids[at - 1],) + path, parents[at - 1]
        paths.add(path)
    assert (3, 5) in paths and (6, 8) in paths
    assert len({(p, t) for p, t in zip(parents, ids)}) == len(ids)            # no two children alike


@pytest.mark.parametrize("seed", range(20))
def test_lookup_gives_trees(seed):
    rng = random.Random(seed)
    look = Lookup()
    for _ in range(60):
        look.extend([rng.randrange(3) for _ in range(rng.randrange(4))])
        n = rng.randrange(1, 20)
        ids, parents = look.propose(n)
        assert len(ids) == len(parents) <= n
        assert all(0 <= p <= i for i, p in enumerate(parents))               # a parent comes before its child
        assert len({(p, t) for p, t in zip(parents, ids)}) == len(ids)


def test_tokens_of_a_step():
    assert [tokens_of_step(size, 7, 64) for size in (1, 4, 8, 16, 64, 128)] == [8, 8, 8, 4, 1, 1]


class Backend:
    """Tokens are numbered from the prompt's length on; a drafted step gives up to four of them where it likes to."""

    def __init__(self, several):
        self.several, self.calls, self.ended = several, [], []

    def capacity_pages(self):
        return 100

    def max_batch(self):
        return 8

    def prefill(self, prompts, keys, sampling):
        self.base = [len(p) for p in prompts]
        return list(self.base)

    def decode(self, live, last_tokens, keys, steps_done, sampling, changed):
        self.calls.append(("one", list(live), changed))
        assert last_tokens == [self.base[p] + n - 1 for p, n in zip(live, steps_done)]
        return [t + 1 for t in last_tokens]

    def decode_drafted(self, live, texts, keys, steps_done, sampling, room):
        n = self.several(len(self.calls))
        for p, (prompt, so_far), done, left in zip(live, texts, steps_done, room):
            assert len(prompt) == self.base[p] and so_far == [self.base[p] + i for i in range(done)] and left > 0
        if n is None or min(room) < n:
            return None
        self.calls.append(("some", list(live), n))
        return [[so_far[-1] + 1 + i for i in range(1 + (p + n) % n)] for p, (_, so_far) in zip(live, texts)]

    def finish(self, index):
        self.ended.append(index)


@pytest.mark.parametrize("several", [lambda i: 3, lambda i: None, lambda i: 4 if i % 2 else None, lambda i: 1])
def test_the_loop_takes_several_tokens_a_step(several):
    b = Backend(several)
    requests = [Request([0] * n, new, stop_token_ids=stop) for n, new, stop in ((3, 10, ()), (5, 7, (9,)), (4, 1, ()), (2, 12, ()))]
    seen = []
    results, stats = run_requests(b, requests, on_token=lambda i, t, last: seen.append((i, t, last)))
    assert [r.tokens for r in results] == [list(range(3, 13)), [5, 6, 7, 8, 9], [4], list(range(2, 14))]
    assert [r.reason for r in results] == ["length", "stop", "length", "length"]
    assert stats.generated_tokens == 28 and sorted(b.ended) == [0, 1, 2, 3]
    for i, r in enumerate(results):
        assert [t for j, t, _ in seen if j == i] == r.tokens and [last for j, _, last in seen if j == i] == [False] * (len(r.tokens) - 1) + [True]
    for before, call in zip(b.calls, b.calls[1:]):                           # an ordinary step after another kind starts anew
        if call[0] == "one" and before[0] == "some":
            assert call[2]


def _spec(make, **more):
    return model_spec(MiniCPMConfig.from_dict({**make, **more}))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_takes_drafts(dtype):
    takes = lambda spec: Model(spec, DryOps(dtype)).takes_drafts()  # noqa: E731
    assert takes(_spec(configs.tiny_a())) and takes(_spec(configs.tiny_b(False))) and takes(_spec(configs.tiny_e()))
    assert not takes(_spec(configs.tiny_b())) and not takes(_spec(configs.tiny_b(False), cache_bits=4))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("make", [configs.tiny_a, lambda: configs.tiny_b(False), configs.tiny_e])
def test_the_workspace_is_measured_for_drafts(make, dtype):
    spec = _spec(make())
    plain = measure_workspace(spec, dtype, 64, 4, 512)
    drafts = measure_workspace(spec, dtype, 64, 4, 512, drafts=15)
    assert not drafts[2] and drafts[0] >= plain[0] and drafts[1] >= plain[1]
    if dtype == torch.bfloat16 and make is configs.tiny_e:
        # 15 drafted tokens at two heads of 128 channels: two places of 32 rows for each of 148 blocks
        assert drafts[1] >= 148 * 2 * 32 * 130 * 4


def test_cli_option():
    parse = create_cli_parser().parse_args
    assert parse(["--model-path", "x"]).draft_tokens == 0
    assert parse(["--model-path", "x", "--draft-tokens", "7"]).draft_tokens == 7 == parse(["--model-path", "x", "--draft_tokens", "7"]).draft_tokens


@pytest.mark.parametrize("chunk,max_batch", [(16, 64), (64, 4), (1, 9), (100, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_of_drafts_fit_the_workspace_that_is_measured(chunk, max_batch, dtype):
    """As many tokens as the runner brings at every bucket size, with prompts' chunks smaller than a batch too."""
    from cpmcu_b200.cache import Cache
    from cpmcu_b200.engine.decode import bucket_size
    from cpmcu_b200.engine.drafts import DraftRunner, draft_step
    from cpmcu_b200.engine.storage import make_storage

    spec = _spec(configs.tiny_e())
    persistent, frame, _ = measure_workspace(spec, dtype, chunk, max_batch, 512, drafts=63)
    model = Model(spec, DryOps(dtype))
    model.loaded, model.ops.device = True, torch.device("cpu")
    make_storage(model, chunk, max_batch, max_tokens=512, max_seq_tokens=512, drafts=63)
    runner = DraftRunner.__new__(DraftRunner)
    runner.drafts, runner.ops = 63, model.ops                    # (with the storage's workspace)
    assert runner.ops.workspace.sized_tokens > 0
    meta = lambda n, **kw: torch.empty(n, device="meta", **{"dtype": torch.int32, **kw})  # noqa: E731
    size = 1
    while size <= bucket_size(max_batch):
        tokens = runner.tokens(size)
        if tokens > 1:
            ops = DryOps(dtype)
            model = Model(spec, ops)
            model.load_weights({name: torch.empty(w.shape, device="meta", dtype=torch.int32 if w.role == "table" else dtype) for name, w in model.weight_specs().items()})
            cache = Cache(model.cache_needs(), max_tokens=512, dtype=dtype, device="meta", n_slots=max_batch + 1, max_seq_tokens=512)
            n = size * tokens
            ops.workspace.begin_step()
            draft_step(model, cache, tokens, meta(n), meta(n), meta(size), meta(size), meta(size), 0, meta(size), meta(size), *(meta(size, dtype=torch.float32) for _ in range(3)),
                       meta(size), meta(n), 512, False)
            needs = ops.workspace.peaks()
            assert needs[0] <= persistent and needs[1] <= frame, (size, tokens, needs, frame)
        size *= 2


@pytest.mark.parametrize("sms", [20, 148, 160])
def test_rooms_for_parts_go_by_the_devices_multiprocessors(sms):
    ops = DryOps(torch.bfloat16, sms)
    # a block's entry of 6 numbers, and two places of 5 rows times 16 heads: two blocks a multiprocessor at 64 channels, one at 128
    assert ops.lib.cpm_draft_attention_scratch_floats(32, 2, 64, 5) == sms * 2 * (6 + 2 * 5 * 16 * 66)
    assert ops.lib.cpm_draft_attention_scratch_floats(32, 2, 128, 5) == sms * (6 + 2 * 5 * 16 * 130)
    assert ops.lib.cpm_kv4_attention_scratch_floats(128) == sms * (8 + 32 * 132)


def test_a_cache_leaves_room_for_the_logits_of_drafts(monkeypatch):
    """What a memory limit leaves for the cache is less by the logits of every bucket's recorded step, 1 to 8 sequences of 16 tokens (and of 8, where a step has no more room),
    and of the largest once more."""
    from cpmcu_b200.engine.storage import draft_logit_bytes, make_storage

    assert draft_logit_bytes(900, 64, 8, 15) == (16 + 32 + 64 + 64 + 64) * 900 * 4
    assert draft_logit_bytes(900, 64, 5, 63) == (64 * 4 + 64) * 900 * 4 and draft_logit_bytes(900, 16, 64, 1) == (2 + 4 + 8 + 16 + 32 + 64 + 64) * 900 * 4
    assert draft_logit_bytes(900, 64, 8, 0) == draft_logit_bytes(900, 1, 1, 15) == 0
    free = 96 << 20
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (free, free))
    spec = _spec(configs.tiny_e())
    left = {}
    for drafts in (0, 15):
        model = Model(spec, DryOps(torch.bfloat16))
        model.loaded, model.ops.device = True, torch.device("cpu")
        storage = make_storage(model, 64, 8, memory_limit=1.0, reserve_bytes=1 << 20, max_seq_tokens=4096, drafts=drafts)
        left[drafts] = free - (1 << 20) - storage.arena.total
    assert left[0] >= 0 and left[15] >= 240 * 900 * 4
