"""The generation loop's backend on the device: prompts through the step function,
decode steps through the decode runner, sampling by the library's kernel."""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import torch

from ..sampling import SamplingParams
from .decode import DecodeRunner
from .drafts import DraftRunner, Lookup
from .step import SequenceStep, Stepper


class EngineBackend:
    drafter: Optional[DraftRunner] = None
    lookups: Dict[int, Lookup] = {}             # by slot, of the current batch's sequences (a backend with a drafter has its own)

    def __init__(self, stepper: Stepper, max_batch: int = 64, use_graph: bool = True, seed: int = 0, draft_tokens: int = 0):
        """``draft_tokens`` > 0: steps check that many looked-up tokens a sequence where they can (see ``DraftRunner``)."""
        self.stepper = stepper
        self.ops = stepper.ops
        self.seed = int(seed)
        stepper.cache.copy_pages = self.ops.copy_pages
        self.runner = DecodeRunner(stepper, use_graph=use_graph, seed=seed)
        self._max_batch = int(max_batch)
        self.drafter = DraftRunner(self.runner, draft_tokens) if draft_tokens else None
        self.lookups = {}
        self.slots: List[int] = []
        self.open: set = set()              # slots of the current batch that are not finished yet
        self.h2d_bytes = 0
        self.d2h_bytes = 0

    def capacity_pages(self) -> int:
        return self.stepper.cache.n_pages - 1          # one page belongs to the decode runner's padding

    def max_batch(self) -> int:
        return min(self._max_batch, self.stepper.cache.n_slots - 1)

    def _sample(self, logits: torch.Tensor, keys: Sequence[int], steps: Sequence[int],
                sampling: Sequence[SamplingParams]) -> List[int]:
        n = len(keys)
        if all(p.greedy for p in sampling):
            out = self.ops.sample(logits)
        elif any(p.filtered for p in sampling):
            i = torch.tensor(list(keys) + list(steps) + [p.top_k for p in sampling], dtype=torch.int32).view(3, n).to(self.ops.device)
            f = torch.tensor([p.temperature for p in sampling] + [p.top_p for p in sampling] + [p.min_p for p in sampling],
                             dtype=torch.float32).view(3, n).to(self.ops.device)
            out = drawn = None
            if any(p.unfiltered for p in sampling):          # these as they would be drawn without the others
                drawn = torch.tensor([not p.unfiltered for p in sampling], dtype=torch.int32).to(self.ops.device)
                out = self.ops.sample(logits, f[0] * (1 - drawn), f[1], self.seed, i[0], i[1])
            out, _ = self.ops.sample_filtered(logits, None, f[0], i[2], f[1], f[2], self.seed, i[0], i[1], out=out, drawn=drawn)
        else:
            i = torch.tensor(list(keys) + list(steps), dtype=torch.int32).view(2, n).to(self.ops.device)
            f = torch.tensor([p.temperature for p in sampling] + [p.top_p for p in sampling],
                             dtype=torch.float32).view(2, n).to(self.ops.device)
            out = self.ops.sample(logits, f[0].contiguous(), f[1].contiguous(), self.seed, i[0].contiguous(),
                                  i[1].contiguous())
        self.d2h_bytes += 4 * n
        return out.cpu().tolist()

    def max_sequence_pages(self) -> int:
        return self.stepper.cache.max_pages_per_seq

    def shared_pages(self, length: int) -> int:
        return self.stepper.cache.shared_pages(length)

    def vocab_size(self) -> int:
        return self.stepper.vocab_size

    def prefill(self, prompts, keys, sampling) -> List[int]:
        self.slots = self.stepper.open(len(prompts))
        self.open = set(self.slots)
        try:
            batch = [SequenceStep(s, list(p), [len(p) - 1]) for s, p in zip(self.slots, prompts)]
            self.h2d_bytes += 4 * sum(len(p) for p in prompts)
            logits = self.stepper.step(batch)
            tokens = self._sample(logits, keys, [0] * len(prompts), sampling)
            self.ops.raise_on_kernel_error()            # the host has just waited for the tokens anyway
        except BaseException:
            self.abort()
            raise
        return tokens

    def prefill_forked(self, prompts, which, keys, sampling) -> List[int]:
        """As ``prefill`` for sequences that begin alike: sequence j has the prompt ``prompts[which[j]]``.  Every prompt runs once
        and is forked for its further sequences, each of which draws its own first token from the prompt's logits."""
        firsts = self.stepper.open(len(prompts))
        self.open = set(firsts)
        try:
            batch = [SequenceStep(s, list(p), [len(p) - 1]) for s, p in zip(firsts, prompts)]
            self.h2d_bytes += 4 * sum(len(p) for p in prompts)
            logits = self.stepper.step(batch)
            cache = self.stepper.cache
            slots_of = []
            for i, s in enumerate(firsts):
                more = cache.fork_sequence(s, sum(1 for w in which if w == i) - 1)
                self.open.update(more)
                slots_of.append([s] + more)
            cache.sync()
            self.slots = [slots_of[w].pop(0) for w in which]
            rows = logits[torch.tensor(list(which), dtype=torch.int64).to(logits.device)].contiguous()
            tokens = self._sample(rows, keys, [0] * len(which), sampling)
            self.ops.raise_on_kernel_error()
        except BaseException:
            self.abort()
            raise
        return tokens

    def abort(self) -> None:
        """Closes every sequence of the current batch that is still open (a step failed)."""
        for s in sorted(self.open):
            self.stepper.close(s)
        self.open = set()
        self.lookups.clear()

    def decode(self, live, last_tokens, keys, steps_done, sampling, changed) -> List[int]:
        if changed:
            self.runner.start([self.slots[p] for p in live], last_tokens, keys, steps_done, sampling)
            self.h2d_bytes += 4 * 7 * len(live)
        else:
            self.runner.feed(last_tokens)               # the step's inputs: host tokens, pinned, every step
            self.h2d_bytes += 4 * len(live)
        self.runner.step()
        self.d2h_bytes += 4 * len(live)
        return self.runner.read_tokens()

    def decode_drafted(self, live, texts, keys, steps_done, sampling, room):
        """A step of drafted tokens for the live sequences; None where there are none: without a drafter, where nothing was found for any sequence, where one may
        not get as many tokens any more, or where so many sequences leave no room in a step."""
        if self.drafter is None:
            return None
        tokens = self.drafter.tokens(len(live))
        if tokens < 2 or min(room) < tokens:
            return None
        drafted = []
        for p, (prompt, so_far) in zip(live, texts):
            slot = self.slots[p]
            lookup = self.lookups.get(slot)
            if lookup is None:
                lookup = self.lookups[slot] = Lookup(prompt)
            lookup.extend(so_far[len(lookup.tokens) - len(prompt):])
            drafted.append(lookup.propose(tokens - 1))
        if not any(ids for ids, _ in drafted):
            return None
        out = self.drafter.step([self.slots[p] for p in live], [so_far[-1] for _, so_far in texts], drafted, keys, steps_done, sampling)
        self.h2d_bytes += 4 * len(live) * (2 * tokens + 8)
        self.d2h_bytes += 4 * len(live) * (tokens + 1)
        return out

    def finish(self, index: int) -> None:
        self.stepper.close(self.slots[index])
        self.open.discard(self.slots[index])
        self.lookups.pop(self.slots[index], None)
