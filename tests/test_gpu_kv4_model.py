"""Models on a cache in 4 bits, several answers to a prompt and the filters, through the Python entry point and the command line."""
import os
import subprocess
import sys

import pytest
import torch

from tests import configs, helpers
from tests.plain import kv4_plain
from tests.plain import minicpm4_plain as plain

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _llm(folder, dtype, graph=False, **kw):
    from cpmcu_b200 import LLM
    return LLM(folder, dtype=dtype, cuda_graph=graph, max_tokens=64 * 64, chunk_length=kw.pop("chunk_length", 64), cache_bits=4, **kw)


def _quantised_forward(folder, ids, monkeypatch):
    """The plain implementation's logits with keys (after rotation) and values as a 4-bit cache holds them."""
    cfg, w = helpers.read_folder(folder)
    dense = plain.dense_attention
    with monkeypatch.context() as m:
        m.setattr(plain, "dense_attention", lambda q, k, v, scale, window=0: dense(q, kv4_plain.quantised(k)[0], kv4_plain.quantised(v)[0], scale, window))
        return plain.forward(cfg, w, list(ids))


def _run(folder, dtype, ids, chunk):
    """Logits of a prompt of 300 tokens in chunks and of steps of one token, and the keys and values that every layer's cache then holds."""
    from cpmcu_b200.engine.step import SequenceStep
    from cpmcu_b200.ops.ops import Ops

    llm = _llm(folder, dtype, chunk_length=chunk)
    llm.init_storage()
    llm.load_from_hf()
    slot = llm.stepper.open(1)[0]
    rows = [llm.step([SequenceStep(slot, ids[:300], list(range(300)))])]
    for t in range(300, len(ids)):
        rows.append(llm.step([SequenceStep(slot, ids[t:t + 1], [0])]))
    llm.ops.raise_on_kernel_error()
    f32, i32 = Ops(torch.float32), lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    held = []
    for lane in llm.cache.lanes:
        k, v = f32.kv4_values(lane.records, i32(list(range(len(ids)))), i32([0] * len(ids)), i32([slot]), lane.page_table, llm.config.num_key_value_heads,
                              llm.config.head_dim)
        held.append((k.cpu(), v.cpu()))
    llm.stepper.close(slot)
    llm.cache.check_consistent()
    return torch.cat(rows).cpu(), held


@pytest.mark.parametrize("name,make", [("tiny_b", lambda: configs.tiny_b(False)), ("tiny_e", configs.tiny_e)])
def test_logits_are_those_of_quantised_keys_and_values(model_folders, name, make, monkeypatch):
    """The 32-bit path against the plain implementation on quantised keys and values.  A key that lies at the border of two codes may take the
    other one, which is a step of 1/15 of its half row: tolerated is a fifth of what the 4 bits themselves change."""
    cfgd = make()
    folder = model_folders(name + "_dense", cfgd, 3, "float32", std=0.08)
    ids = helpers.random_ids(cfgd["vocab_size"], 330, 5)
    want = _quantised_forward(folder, ids, monkeypatch)
    cfg, w = helpers.read_folder(folder)
    change = float((want - plain.forward(cfg, w, list(ids))).norm() / want.norm())
    assert change > 1e-3
    got, _ = _run(folder, "float32", ids, 128)
    err = float((got - want).norm() / want.norm())
    assert err < change / 5, (err, change)


@pytest.mark.parametrize("chunk", [64, 512])
@pytest.mark.parametrize("name,make", [("tiny_b", lambda: configs.tiny_b(False)), ("tiny_e", configs.tiny_e)])
def test_logits_of_the_bf16_path(model_folders, name, make, chunk, monkeypatch):
    """The bf16 path against the plain implementation on the very keys and values that the engine's cache holds (a rounding of activations to
    bf16 moves about one code of a hundred, so that codes of other activations say little), within the rounding of bf16."""
    cfgd = make()
    folder = model_folders(name + "_dense", cfgd, 3, "bfloat16", std=0.08)
    ids = helpers.random_ids(cfgd["vocab_size"], 330, 5)
    got, held = _run(folder, "bfloat16", ids, chunk)
    cfg, w = helpers.read_folder(folder)
    dense, layers = plain.dense_attention, iter(held)
    monkeypatch.setattr(plain, "dense_attention", lambda q, k, v, scale, window=0: dense(q, *next(layers), scale, window))
    want = plain.forward(cfg, w, list(ids))
    assert helpers.rel_err(got, want) < helpers.TOL["bfloat16"]


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("settings", [dict(temperature=0.0), dict(temperature=1.0, top_k=20, top_p=0.9), dict(temperature=0.7, min_p=0.05)])
def test_several_answers_are_those_of_separate_requests(model_folders, settings, graph):
    """Answers that were forked from one prompt draw what requests of their own with the same keys draw, and leave nothing behind."""
    from cpmcu_b200.engine.generate import Request, run_requests
    from cpmcu_b200.sampling import SamplingParams

    cfgd = configs.tiny_b(False)
    folder = model_folders("tiny_b_dense", cfgd, 3, "float32", std=0.08)
    llm = _llm(folder, "float32", graph, random_seed=11, max_batch=8)
    prompts = [helpers.random_ids(cfgd["vocab_size"], n, n) for n in (70, 64, 5)]
    together = llm.generate_batch(prompts, generation_length=12, samples=3, **settings)
    assert len(together) == 9 and llm.last_stats.prompt_tokens == 70 + 64 + 5 + 5          # eight a batch: the last prompt's group is cut
    sp = SamplingParams(settings["temperature"], settings.get("top_p", 1.0), settings.get("top_k", 0), settings.get("min_p", 0.0))
    alone, _ = run_requests(llm.backend, [Request(prompts[i // 3], 12, sp, key=i) for i in range(9)])
    assert [r.tokens for r in together] == [r.tokens for r in alone]
    if settings["temperature"] > 0:
        assert len({tuple(r.tokens) for r in together[:3]}) > 1
    llm.cache.check_consistent()
    assert llm.cache.slots.n_held == 1                                                      # the decode runner's padding


@pytest.mark.parametrize("graph", [False, True])
def test_a_sequence_draws_the_same_whatever_its_batch_is_drawn_by(model_folders, graph, monkeypatch):
    """Logits of a few levels, among whose equal tokens the two kernels draw differently (``sample`` keeps all of them at top-p's border): sequences
    with filters, with top-p or a temperature alone, and greedy ones give the same tokens together, while others leave, and alone."""
    from cpmcu_b200.engine.generate import Request, run_requests
    from cpmcu_b200.sampling import SamplingParams

    cfgd = configs.tiny_e()
    folder = model_folders("tiny_e_dense", cfgd, 3, "float32", std=0.08)
    llm = _llm(folder, "float32", graph, random_seed=11, max_batch=8)
    llm.init_storage()
    forward = llm.model.forward
    monkeypatch.setattr(llm.model, "forward", lambda ctx, rows: None if rows is None else torch.round(forward(ctx, rows) * 2) / 2)
    kinds = [SamplingParams(1.0, 0.6), SamplingParams(1.0, 0.8, 30), SamplingParams(0.0), SamplingParams(0.8), SamplingParams(1.2, 0.7),
             SamplingParams(0.9, min_p=0.1)]
    reqs = [Request(helpers.random_ids(cfgd["vocab_size"], 9 + i, i), 6 + 3 * i, kinds[i], key=i) for i in range(6)]
    together, _ = run_requests(llm._ready(), reqs)
    pairs = [run_requests(llm.backend, reqs[i:i + 2])[0] for i in range(0, 6, 2)]
    alone = [run_requests(llm.backend, [r])[0][0] for r in reqs]
    assert [r.tokens for r in together] == [r.tokens for r in alone] == [r.tokens for p in pairs for r in p]


def test_filters_alone_change_nothing_where_they_keep_everything(model_folders):
    """A batch drawn by the filtered kernel with limits that keep all gives the tokens that the other kernel draws from the same numbers."""
    cfgd = configs.tiny_e()
    folder = model_folders("tiny_e_dense", cfgd, 3, "float32", std=0.08)
    llm = _llm(folder, "float32", random_seed=5)
    prompts = [helpers.random_ids(cfgd["vocab_size"], n, n) for n in (9, 30)]
    a = llm.generate_batch(prompts, generation_length=10, temperature=1.0)
    b = llm.generate_batch(prompts, generation_length=10, temperature=1.0, top_k=cfgd["vocab_size"])
    assert [r.tokens for r in a] == [r.tokens for r in b]


@pytest.mark.parametrize("bits", [4, 16])
def test_a_cache_is_forked_and_compacted_between_steps(model_folders, bits):
    """Steps after a fork and after pages have moved give the logits that they give without."""
    from cpmcu_b200 import LLM
    from cpmcu_b200.engine.step import SequenceStep

    cfgd = configs.tiny_b(False)
    folder = model_folders("tiny_b_dense", cfgd, 3, "bfloat16", std=0.08)
    llm = LLM(folder, dtype="bfloat16", max_tokens=64 * 40, chunk_length=64, cache_bits=bits, max_batch=8)
    llm.init_storage()
    llm.load_from_hf()
    cache = llm.cache
    cache.copy_pages = llm.ops.copy_pages
    ids = helpers.random_ids(cfgd["vocab_size"], 200, 5)
    first, second, third = llm.stepper.open(3)
    for s, n in ((first, 190), (second, 150), (third, 150)):
        llm.step([SequenceStep(s, ids[:n], [])])
    llm.stepper.close(first)                                     # its pages are holes in front of the others'
    child = cache.fork_sequence(second, 1)[0]
    cache.sync()
    want = llm.step([SequenceStep(third, ids[150:160], [9])])
    assert cache.compact() > 0
    cache.sync()
    got = llm.step([SequenceStep(child, ids[150:160], [9])])
    assert torch.equal(got, want)
    assert torch.equal(llm.step([SequenceStep(second, ids[150:160], [9])]), want)
    for g in cache.groups:
        assert all(g.pages.is_held(p) for p in range(g.pages.n_held))
    cache.check_consistent()
    llm.ops.raise_on_kernel_error()


def test_command_line(tmp_path):
    import json

    cfg_path, folder = str(tmp_path / "config.json"), str(tmp_path / "model")
    with open(cfg_path, "w") as f:
        json.dump(configs.tiny_e(), f)
    prompt = ",".join(map(str, helpers.random_ids(900, 70, 4)))
    run = lambda *more: subprocess.run([sys.executable, "-m", "cpmcu_b200.cli", "--model-path", folder, "--prompt-ids", prompt, "--num-generate", "6",  # noqa: E731
                                        "--ignore-eos", "true", "--max-tokens", "1024", "--cache-bits", "4", *more], cwd=ROOT, capture_output=True,
                                       text=True, timeout=300)
    out = run("--random-weights", "9", "--config", cfg_path, "--samples", "3", "--temperature", "1.0", "--top-k", "50", "--min-p", "0.01", "--random-seed", "3")
    assert out.returncode == 0, out.stderr
    lines = out.stdout.strip().splitlines()
    assert [ln.split("] ")[0] for ln in lines] == ["[0", "[1", "[2"] and all(len(ln.split("] ")[1].split()) == 6 for ln in lines)
    assert run("--samples", "3", "--temperature", "1.0", "--top-k", "50", "--min-p", "0.01", "--random-seed", "3").stdout == out.stdout
    bad = run("--samples", "0", "--use-stream", "false")
    assert bad.returncode == 1 and "samples" in bad.stderr


def test_an_architecture_without_a_4_bit_cache_says_so(tmp_path):
    from cpmcu_b200 import LLM
    from tests import dinutar_cases as cases

    cfg = cases.config_a()
    folder = cases.write_folder(cfg, cases.random_weights(cfg, 1), str(tmp_path / "d"))
    with pytest.raises(ValueError, match="4 bits"):
        LLM(folder, cache_bits=4)


def test_an_architecture_without_a_4_bit_cache_takes_16(tmp_path):
    from cpmcu_b200 import LLM
    from tests import dinutar_cases as cases

    cfg = cases.config_a()
    folder = cases.write_folder(cfg, cases.random_weights(cfg, 1), str(tmp_path / "d"))
    a, b = [LLM(folder, max_tokens=64 * 8, **kw).generate([3, 1, 4], 5)[0] for kw in ({}, dict(cache_bits=16))]
    assert a == b and len(a) == 5
    with pytest.raises(ValueError, match="4 or 16"):
        LLM(folder, cache_bits=8)


CHECKED = r'''
import os, tempfile
from cpmcu_b200 import LLM
from tests import configs, helpers
with tempfile.TemporaryDirectory() as tmp:
    for dtype in ("bfloat16", "float32"):
        cfgd = configs.tiny_e()
        folder = helpers.make_folder(cfgd, os.path.join(tmp, dtype), 1, dtype)
        llm = LLM(folder, dtype=dtype, cuda_graph=True, max_tokens=64 * 40, chunk_length=64, max_batch=8, cache_bits=4)
        res = llm.generate_batch([helpers.random_ids(cfgd["vocab_size"], n, n) for n in (100, 7, 300)], generation_length=8, samples=2, temperature=1.0, top_k=30)
        assert all(len(r.tokens) == 8 for r in res)
        llm.ops.raise_on_kernel_error()
print("CLEAN OK")
'''


def test_checked_build():
    """Page numbers and the arena's guard words under the checked build."""
    env = dict(os.environ, CPMCU_CHECK_BOUNDS="1", PYTHONPATH=ROOT)
    out = subprocess.run([sys.executable, "-c", CHECKED], cwd=ROOT, env=env, capture_output=True, text=True, timeout=600)
    assert out.returncode == 0 and "CLEAN OK" in out.stdout, out.stdout + out.stderr
