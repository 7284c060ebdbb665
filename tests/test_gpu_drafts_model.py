"""Generation with drafted tokens through the Python entry point and the command line, and a run of the operators together."""
import os
import subprocess
import sys

import pytest
import torch

from cpmcu_b200.engine.drafts import Lookup
from tests import configs, helpers

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _llm(folder, dtype, graph=False, **kw):
    from cpmcu_b200 import LLM
    return LLM(folder, dtype=dtype, cuda_graph=graph, max_tokens=64 * 64, chunk_length=kw.pop("chunk_length", 128), **kw)


def _repeating(vocab, n, seed):
    """A text that says things again, so that there is something to look up."""
    some = helpers.random_ids(vocab, 9, seed)
    return (some * (n // 9 + 1))[:n]


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("settings", [dict(temperature=0.0), dict(temperature=0.8, top_k=3), dict(temperature=0.6, top_k=20, top_p=0.8, min_p=0.05)])
@pytest.mark.parametrize("name,make", [("tiny_a", configs.tiny_a), ("tiny_b_dense", lambda: configs.tiny_b(False)), ("tiny_e", configs.tiny_e)])
def test_drafts_change_no_token(model_folders, name, make, settings, graph, monkeypatch):
    """In 32 bits a batch with drafted tokens generates what it does without, in no more steps."""
    cfgd = make()
    folder = model_folders(name, cfgd, 3, "float32", std=0.08)
    prompts = [_repeating(cfgd["vocab_size"], n, n) for n in (70, 33, 5, 64)]
    plain = _llm(folder, "float32", graph, random_seed=5)
    want = [r.tokens for r in plain.generate_batch(prompts, generation_length=60, **settings)]
    steps = plain.last_stats.decode_steps
    llm = _llm(folder, "float32", graph, random_seed=5, draft_tokens=7)
    got = [r.tokens for r in llm.generate_batch(prompts, generation_length=60, **settings)]
    assert got == want
    if settings["temperature"] == 0:
        assert llm.backend.drafter.accepted > 0 and llm.last_stats.decode_steps <= steps
    # and with drafts that are right for some tokens, beside others that are not
    texts = [p + w for p, w in zip(prompts, want)]

    def propose(self, n):
        text = next(t for t in texts if t[:len(self.tokens)] == self.tokens)
        right = text[len(self.tokens):][:len(self.tokens) % (n - 1)]
        ids, parents, at = [], [], 0
        for t in right:
            if len(ids) + 2 > n:
                break
            ids += [(t + 1) % cfgd["vocab_size"], t]
            parents += [at, at]
            at = len(ids)
        return ids, parents

    monkeypatch.setattr(Lookup, "propose", propose)
    before = llm.backend.drafter.accepted
    assert [r.tokens for r in llm.generate_batch(prompts, generation_length=60, **settings)] == want          # on slots and pages used before
    assert llm.backend.drafter.accepted > before + 100 and llm.last_stats.decode_steps < 50
    llm.ops.raise_on_kernel_error()
    llm.cache.check_consistent()
    assert llm.cache.slots.n_held == 1 and not llm.backend.lookups


@pytest.mark.parametrize("graph", [False, True])
def test_drafts_in_bf16_and_several_answers(model_folders, graph):
    """Answers forked from one prompt, with drafts: every answer's tokens are likely under the model that a step of one token would have been drawn from."""
    cfgd = configs.tiny_e()
    folder = model_folders("tiny_e", cfgd, 3, "bfloat16", std=0.08)
    prompt = _repeating(cfgd["vocab_size"], 100, 4)
    llm = _llm(folder, "bfloat16", graph, random_seed=2, draft_tokens=15, max_batch=8)
    got = llm.generate_batch([prompt, prompt[:31]], generation_length=40, samples=3, temperature=0.5, top_k=4)
    assert [len(r.tokens) for r in got] == [40] * 6
    assert len({tuple(r.tokens) for r in got}) > 1
    cfg, w = helpers.read_folder(folder)
    from tests.plain import minicpm4_plain
    for r, p in zip(got, [prompt] * 3 + [prompt[:31]] * 3):
        logits = minicpm4_plain.forward(cfg, w, list(p) + r.tokens[:-1])[len(p) - 1:]
        rank = (logits > logits.gather(1, torch.tensor(r.tokens)[:, None])).sum(1)
        # of four tokens that may be drawn; bf16 changes the order of near ones
        assert int((rank >= 4).sum()) <= 2 and int(rank.max()) < 12
    llm.ops.raise_on_kernel_error()
    llm.cache.check_consistent()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_step_of_drafts_gives_the_logits_of_single_steps(model_folders, dtype):
    """Tables, model, attention and the moving of accepted tokens in a row: after an accepted path through a tree, the cache holds what steps of its tokens one
    after the other leave."""
    from cpmcu_b200.engine.drafts import draft_step
    from cpmcu_b200.engine.step import SequenceStep

    cfgd = configs.tiny_e()
    folder = model_folders("tiny_e", cfgd, 3, dtype, std=0.08)
    llm = _llm(folder, dtype, draft_tokens=7)
    llm._ready()
    vocab, cache = cfgd["vocab_size"], llm.cache
    ids = helpers.random_ids(vocab, 62, 9)
    a, b = llm.stepper.open(2)
    logits = llm.step([SequenceStep(a, ids, [len(ids) - 1]), SequenceStep(b, ids, [])])
    path = [int(logits[0].argmax())]
    for _ in range(3):                                       # the greedy continuation, one token a step
        logits = llm.step([SequenceStep(a, path[-1:], [0])])
        path.append(int(logits[0].argmax()))
    # a tree that holds it between other tokens: root, two wrong ones, right, wrong, right, wrong, right
    wrong = lambda t: (t + 1) % vocab  # noqa: E731
    tree = [path[0], wrong(path[1]), wrong(wrong(path[1])), path[1], wrong(path[2]), path[2], 0, path[3]]
    parents = [-1, 0, 0, 0, 3, 3, 1, 5]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    f32 = lambda v: torch.tensor(v, dtype=torch.float32).cuda()  # noqa: E731
    cache.reserve(b, 62 + 8)
    cache.sync()
    llm.ops.begin_step()
    seen = {}
    forward = llm.model.forward
    llm.model.forward = lambda ctx, rows: seen.setdefault("logits", forward(ctx, rows))
    tokens, count, places, _ = draft_step(llm.model, cache, 8, i32(tree), i32(parents), i32([62]), i32([8]), i32([b]), 0, i32([0]), i32([0]), f32([0.0]), f32([1.0]),
                                          f32([0.0]), i32([0]), i32(list(range(8))), cache.max_pages_per_seq * 64, False)
    llm.model.forward = forward
    cache.set_length(b, 62 + int(count))
    assert places[0, :4].tolist() == [0, 3, 5, 7] and tokens[0, :3].tolist() == path[1:] and int(count) == 4
    tol = 1e-4 if dtype == "float32" else helpers.TOL["bfloat16"]
    assert helpers.rel_err(seen["logits"][5:6].cpu(), logits.cpu()) < tol
    # the next step of one token from both caches
    last = int(tokens[0, 3])
    both = llm.step([SequenceStep(a, [path[3]], [0]), ])
    both = torch.cat((both, llm.step([SequenceStep(a, [last], [0])])))
    again = llm.step([SequenceStep(b, [last], [0])])
    assert cache.length(a) == cache.length(b)
    assert helpers.rel_err(again.cpu(), both[1:].cpu()) < tol
    k = lambda s: cache.lanes[0].k[cache.groups[0].page_table[s, :2].long()][:, :, :].transpose(1, 2).flatten(0, 1)[:cache.length(s)]  # noqa: E731
    assert helpers.rel_err(k(b).float().cpu(), k(a).float().cpu()) < (1e-5 if dtype == "float32" else 0.02)
    llm.ops.raise_on_kernel_error()
    for s in (a, b):
        llm.stepper.close(s)
    cache.check_consistent()


@pytest.mark.parametrize("settings", [dict(temperature=0.9), dict(temperature=0.7, top_p=0.9)])
def test_drafts_beside_steps_without_filters(model_folders, settings, monkeypatch):
    """Steps of one token draw by sums in fp32 where there is no top-k and no min-p, steps of drafts by whole units: the same number falls on the same token unless it
    lies within the sums' error of a border (2^-20 of the mass at 512 tokens, 4 x 40 draws: a chance of one in some thousand, and the numbers are fixed)."""
    cfgd = configs.tiny_a()
    folder = model_folders("tiny_a", cfgd, 3, "float32", std=0.08)
    prompts = [_repeating(cfgd["vocab_size"], n, n) for n in (70, 33, 5, 64)]
    want = [r.tokens for r in _llm(folder, "float32", random_seed=5).generate_batch(prompts, generation_length=40, **settings)]
    llm = _llm(folder, "float32", random_seed=5, draft_tokens=7)
    texts = [p + w for p, w in zip(prompts, want)]

    def propose(self, n):
        right = next(t for t in texts if t[:len(self.tokens)] == self.tokens)[len(self.tokens):][:2]
        return right, list(range(len(right)))

    monkeypatch.setattr(Lookup, "propose", propose)
    assert [r.tokens for r in llm.generate_batch(prompts, generation_length=40, **settings)] == want
    assert llm.backend.drafter.accepted > 80


def test_a_kernel_that_gave_up_ends_the_generation(model_folders, monkeypatch):
    """The step's error is read with its tokens, none of which is then given, and nothing of the batch stays held."""
    cfgd = configs.tiny_a()
    llm = _llm(model_folders("tiny_a", cfgd, 3, "float32", std=0.08), "float32", draft_tokens=7)
    prompt = _repeating(cfgd["vocab_size"], 70, 1)
    want = llm.generate_batch([prompt], generation_length=30, temperature=0.0)[0].tokens
    assert llm.backend.drafter.steps > 0
    with monkeypatch.context() as m:
        m.setattr(llm.ops, "draft_attention_ran", True)
        before, found = llm.backend.drafter.steps, []
        real = llm.backend.drafter._bucket
        m.setattr(llm.backend.drafter, "_bucket", lambda n: (m.setattr(llm.ops.lib, "cpm_draft_attention_error", lambda: 3), real(n))[1])
        with pytest.raises(RuntimeError, match="drafted tokens gave up"):
            llm.generate_batch([prompt], generation_length=30, temperature=0.0, on_token=lambda i, t, last: found.append(t))
        assert llm.backend.drafter.steps == before and found == want[:len(found)] and len(found) < 30
    assert llm.cache.slots.n_held == 1 and not llm.backend.lookups
    assert llm.generate_batch([prompt], generation_length=30, temperature=0.0)[0].tokens == want
    llm.cache.check_consistent()


def test_refusals(model_folders):
    from cpmcu_b200 import LLM

    folder = model_folders("tiny_b", configs.tiny_b(), 3, "float32", std=0.08)
    with pytest.raises(ValueError):
        LLM(folder, dtype="float32", max_tokens=4096, draft_tokens=3)                            # block-sparse attention
    dense = model_folders("tiny_b_dense", configs.tiny_b(False), 3, "float32", std=0.08)
    for bad in (dict(draft_tokens=64), dict(draft_tokens=-1), dict(draft_tokens=2, cache_bits=4)):
        with pytest.raises(ValueError):
            LLM(dense, dtype="float32", max_tokens=4096, **bad)
    LLM(folder, dtype="float32", max_tokens=4096, draft_tokens=3, apply_sparse=False)


def test_cli(model_folders):
    folder = model_folders("tiny_a", configs.tiny_a(), 3, "float32", std=0.08)
    prompt = ",".join(str(i) for i in _repeating(512, 40, 1))
    run = lambda *more: subprocess.run([sys.executable, "-m", "cpmcu_b200.cli", "--model-path", folder, "--dtype", "float32", "--prompt-ids", prompt, "--max-tokens", "2048",  # noqa: E731
                                        "--num-generate", "24", *more], cwd=ROOT, capture_output=True, text=True, timeout=300)
    one, two = run(), run("--draft-tokens", "5")
    assert one.returncode == 0 and two.returncode == 0, two.stderr[-2000:]
    assert one.stdout == two.stdout and len(one.stdout.split()) == 24
