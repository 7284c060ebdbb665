"""Several answers to a prompt on every architecture: caches with windows, pooled keys, latents and per-sequence states are forked."""
import importlib

import pytest
import torch

from tests import configs, helpers

pytestmark = pytest.mark.gpu

CASES = [("minicpm", "tiny_a"), ("minicpm", "tiny_b")] + [(arch, c) for arch in ("dinutar", "kipizen", "lukelorn", "mufevik", "rabadra", "reravik")
                                                         for c in ("a", "b", "c", "d")]


@pytest.fixture(scope="module")
def folders(model_folders, tmp_path_factory):
    made = {}

    def get(arch, which):
        if arch == "minicpm":
            return model_folders(which, getattr(configs, which)(), 3, "float32", std=0.08)
        if (arch, which) not in made:
            cases = importlib.import_module(f"tests.{arch}_cases")
            cfg = getattr(cases, f"config_{which}")()
            made[arch, which] = cases.write_folder(cfg, cases.random_weights(cfg, 3), str(tmp_path_factory.mktemp(f"{arch}-{which}")))
        return made[arch, which]

    return get


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("arch,which", CASES)
def test_answers_are_those_of_separate_requests(folders, arch, which, graph):
    """Prompts that end inside a page, at its end and within a pooled window of it; nine sequences, eight a batch."""
    from cpmcu_b200 import LLM
    from cpmcu_b200.engine.generate import Request, run_requests
    from cpmcu_b200.sampling import SamplingParams

    folder = folders(arch, which)
    llm = LLM(folder, dtype="float32", cuda_graph=graph, max_tokens=64 * 40, chunk_length=48, max_batch=8, random_seed=11)
    prompts = [helpers.random_ids(llm._ready().vocab_size(), n, n) for n in (70, 64, 5)]
    together = llm.generate_batch(prompts, generation_length=12, samples=3, temperature=1.0, top_k=20)
    llm.cache.check_consistent()
    alone, _ = run_requests(llm.backend, [Request(prompts[i // 3], 12, SamplingParams(1.0, 1.0, 20), key=i) for i in range(9)])
    assert [r.tokens for r in together] == [r.tokens for r in alone]
    llm.cache.check_consistent()
    assert llm.cache.slots.n_held == 1
    llm.ops.raise_on_kernel_error()


@pytest.mark.parametrize("arch,which", CASES)
def test_forks_hold_what_their_sequence_held(folders, arch, which):
    """Steps of a fork give the logits, to the bit, that the same steps of the sequence itself give."""
    from cpmcu_b200 import LLM
    from cpmcu_b200.engine.step import SequenceStep

    folder = folders(arch, which)
    llm = LLM(folder, dtype="bfloat16", max_tokens=64 * 40, chunk_length=48, max_batch=8)
    llm.init_storage()
    llm.load_from_hf()
    llm.cache.copy_pages = llm.ops.copy_pages
    ids = helpers.random_ids(llm.stepper.vocab_size, 200, 5)
    for n in (64, 91, 150):
        slot = llm.stepper.open(1)[0]
        llm.step([SequenceStep(slot, ids[:n], [])])
        children = llm.cache.fork_sequence(slot, 2)
        llm.cache.sync()
        rows = []
        for s in (children[0], slot, children[1]):          # a child goes first: what it writes is its own
            out = [llm.step([SequenceStep(s, ids[n:n + 20], [19])]), llm.step([SequenceStep(s, ids[n + 20:n + 21], [0])])]
            rows.append(torch.cat(out).cpu())
        assert torch.equal(rows[0], rows[1]) and torch.equal(rows[2], rows[1])
        for s in (slot, *children):
            llm.stepper.close(s)
        llm.cache.check_consistent()
    llm.ops.raise_on_kernel_error()
