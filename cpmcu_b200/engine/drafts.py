"""Steps of drafted tokens: several tokens per sequence run through the model together, and those that it would have drawn itself stay.

A sequence's last tokens have often been followed by something before, in the prompt or in what was generated (:class:`Lookup`): what
followed is drafted, several continuations as a tree.  One step then gives every sequence between one token and as many as were drafted and
one more.  A row of the logits draws its token as a step of its own would (the same random number), and a drafted token is
accepted where it is that token, so that drafts change how many tokens a step gives and not which: as far as a step of several tokens computes the logits of
single steps (in bf16 other kernels round otherwise), and but for numbers that fall on the very border of two tokens where an ordinary step
draws with sums in fp32 (no top-k and no min-p).

Every sequence brings the same number of tokens, what is not drafted being filled with tokens that nothing leads to, so that one recording per bucket size
serves all steps.  The reference drafts with a small model of its own and verifies a tree in the same way
(src/model/tree_drafter.cuh, src/model/model.cuh:20-22); it has one sequence.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from ..parts.base import StepContext
from ..sampling import SamplingParams
from .decode import DecodeRunner, bucket_size


class Lookup:
    """What followed earlier occurrences of a text's last tokens, as a tree.

    ``propose(n)`` gives up to ``n`` tokens and their parents (0 is the text's last token, the first drafted one is 1, ...; a parent comes before its
    children, and no two children of one parent are the same token): continuations of the latest earlier occurrences of the last ``LONGEST``
    tokens, then of shorter runs down to two, merged where they begin alike.  Looked at are the ``LOOKED_AT`` latest occurrences of the last two tokens, each of which
    knows the one before it, so that a prompt's token costs the host a third of a microsecond (the runs themselves as keys: 7 to 11)."""

    LONGEST, OCCURRENCES, LOOKED_AT = 4, 4, 64

    def __init__(self, tokens: Sequence[int] = ()):
        self.tokens: List[int] = []
        self.latest: Dict[int, int] = {}           # two tokens, as one number -> the place behind their latest occurrence
        self.before: List[int] = [0, 0]            # by place: the one behind the occurrence before, of the two tokens in front of it (0: none)
        self.extend(tokens)

    def extend(self, tokens: Sequence[int]) -> None:
        text, latest, before = self.tokens, self.latest, self.before
        for t in tokens:
            text.append(int(t))
            n = len(text)
            if n >= 2:
                pair = text[-2] << 32 | text[-1]
                before.append(latest.get(pair, 0))
                latest[pair] = n

    def propose(self, n: int) -> Tuple[List[int], List[int]]:
        text, length = self.tokens, len(self.tokens)
        ids: List[int] = []
        parents: List[int] = []
        if length < 2:
            return ids, parents
        found: List[Tuple[int, int]] = []          # places behind earlier occurrences, the latest first, and how many tokens are alike
        end = self.before[length]
        while end and len(found) < self.LOOKED_AT:
            alike = 2
            while alike < self.LONGEST and alike < end and text[end - alike - 1] == text[length - alike - 1]:
                alike += 1
            found.append((end, alike))
            end = self.before[end]
        child: Dict[Tuple[int, int], int] = {}
        seen = set()
        for size in range(self.LONGEST, 1, -1):
            for end in [e for e, alike in found if alike >= size][:self.OCCURRENCES]:
                if end in seen:
                    continue
                seen.add(end)
                at = 0
                for t in text[end:end + n]:
                    node = child.get((at, t))
                    if node is None:
                        if len(ids) == n:
                            break
                        ids.append(t)
                        parents.append(at)
                        node = child[(at, t)] = len(ids)
                    at = node
            if len(ids) == n:
                break
        return ids, parents


def tokens_of_step(size: int, drafts: int, room: int) -> int:
    """Tokens that each of ``size`` sequences brings to a step: its last one and ``drafts`` more, or as many as the step has room for."""
    return max(1, min(int(drafts) + 1, room // size))


def draft_step(model, cache, tokens: int, ids, parents, lengths, new, slots, seed: int, seq_key, step_key, temperature, top_p, min_p, top_k, want_rows,
               longest: int, captured: bool):
    """The work of one step on the device: its description, the model, the check of the drafted tokens, and the moving of the accepted ones' keys and
    values.  Returns what ``Ops.verify_drafts`` does."""
    ops = model.ops
    size, n = lengths.numel(), ids.numel()
    group = next(g for g in cache.groups if g.k is not None)
    t = ops.step_tables(lengths, new, slots, group.page_table, n, parents=parents)
    ctx = StepContext(
        n_tokens=n, n_seqs=size, is_decode=False, captured=captured, q_lens=[tokens] * size, kv_lens=[], slots=[], max_q_len=tokens, max_kv_len=longest,
        token_ids=ids, positions=t.positions, token_seq=t.token_seq, cu_q=t.cu_q, kv_len_dev=t.kv_len, slot_dev=slots, cache=cache,
        drafts=tokens, places=t.places, slot_map=t.slot_map, slot_table=group.page_table, ancestors=t.ancestors)
    ctx.extras["step_begun"] = True
    logits = model.forward(ctx, want_rows)
    got = ops.verify_drafts(logits, ids, t.cu_q, t.token_seq, tokens, None, temperature, top_k, top_p, min_p, parents=parents, seed=seed, seq_key=seq_key,
                            step_key=step_key, positions=t.positions)
    for g in cache.groups:
        if g.k is not None:
            known = dict(slot_map=t.slot_map, cu_q=t.cu_q) if g is group else {}
            ops.keep_drafts([(g.k, g.v)], lengths, got[2], got[1], slots, g.page_table, **known)
    return got


class _DraftBucket:
    def __init__(self, size: int, tokens: int, device: torch.device):
        i32 = dict(dtype=torch.int32, device=device)
        n = size * tokens
        self.size, self.tokens = size, tokens
        # what a step begins with lies in one tensor, so that one copy brings it
        self.block = torch.zeros(2 * n + 8 * size, **i32)
        self.ids, self.parents, rest = self.block[:n], self.block[n:2 * n], self.block[2 * n:].view(8, size)
        self.lengths, self.slots, self.seq_key, self.step_key, self.top_k = rest[:5]
        self.temperature, self.top_p, self.min_p = rest[5:].view(torch.float32)
        self.top_p.fill_(1.0)
        self.new = torch.full((size,), tokens, **i32)
        self.want_rows = torch.arange(n, **i32)
        self.out: Optional[tuple] = None
        self.graph: Optional[torch.cuda.CUDAGraph] = None
        self.warm = False


class DraftRunner:
    """Steps of drafted tokens for batches of sequences, beside a decode runner, whose scratch sequence pads them."""

    def __init__(self, runner: DecodeRunner, drafts: int):
        self.runner = runner
        self.model, self.cache, self.ops = runner.model, runner.cache, runner.ops
        if not self.model.takes_drafts():
            raise ValueError(f"{self.model.spec.architecture} has parts that take no drafted tokens (they keep something per sequence, or a cache that is not of "
                             "plain keys and values)")
        if not 1 <= int(drafts) < self.ops.MOST_DRAFTS:
            raise ValueError(f"a step takes 1 to {self.ops.MOST_DRAFTS - 1} drafted tokens a sequence, got {drafts}")
        self.drafts = int(drafts)
        self.cache.reserve(runner.pad_slot, self.drafts + 1)       # (a page, which it has)
        self.cache.sync()
        self.buckets: Dict[int, _DraftBucket] = {}
        self.steps = self.accepted = 0                # steps run, and drafted tokens that they accepted

    def tokens(self, n_seqs: int) -> int:
        """Tokens that each of ``n_seqs`` sequences brings; 1: there is no room for drafted ones."""
        size, ws = bucket_size(n_seqs), self.ops.workspace
        return tokens_of_step(size, self.drafts, ws.sized_tokens if ws is not None and ws.sized_tokens else 1 << 30)

    def _body(self, b: _DraftBucket, captured: bool) -> None:
        ws = self.ops.workspace
        if ws is not None:
            ws.require(b.ids.numel(), b.size)
        self.ops.begin_step()
        b.out = draft_step(self.model, self.cache, b.tokens, b.ids, b.parents, b.lengths, b.new, b.slots, self.runner.seed, b.seq_key, b.step_key, b.temperature,
                           b.top_p, b.min_p, b.top_k, b.want_rows, self.cache.max_pages_per_seq * 64, captured)

    def _bucket(self, n: int) -> _DraftBucket:
        size = bucket_size(n)
        b = self.buckets.get(size)
        if b is None:
            b = self.buckets[size] = _DraftBucket(size, self.tokens(n), self.ops.device)
        if not b.warm:
            # on the scratch sequence alone, so that no other is touched
            b.slots.fill_(self.runner.pad_slot)
            b.parents.fill_(-1)
            if self.runner.use_graph:
                torch.cuda.synchronize()
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    self._body(b, captured=True)
                torch.cuda.current_stream().wait_stream(side)
                torch.cuda.synchronize()
                b.graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(b.graph):
                    self._body(b, captured=True)
            b.warm = True
        return b

    def step(self, slots: Sequence[int], last_tokens: Sequence[int], drafted: Sequence[Tuple[Sequence[int], Sequence[int]]], seq_keys: Sequence[int],
             step_keys: Sequence[int], sampling: Sequence[SamplingParams]) -> List[List[int]]:
        """One step: sequence i (in the cache's slot slots[i], which holds all its tokens but the last) brings last_tokens[i] and the tokens drafted[i] = (ids,
        parents).  Returns each one's new tokens, and leaves the cache with all of them but the last."""
        n, cache = len(slots), self.cache
        b = self._bucket(n)
        pad = b.size - n
        lengths = [cache.length(s) for s in slots]
        cache.check_room([(s, length + b.tokens) for s, length in zip(slots, lengths)], b.tokens)
        for s, length in zip(slots, lengths):
            cache.reserve(s, length + b.tokens)
        cache.sync()
        ids: List[int] = []
        parents: List[int] = []
        for last, (tree, up) in zip(last_tokens, drafted):
            room = b.tokens - 1
            tree, up = list(tree)[:room], list(up)[:room]
            ids += [int(last)] + tree + [0] * (room - len(tree))
            parents += [-1] + up + [-1] * (room - len(tree))
        ids += [0] * (pad * b.tokens)
        parents += [-1] * (pad * b.tokens)
        ints = torch.tensor(ids + parents + lengths + [0] * pad + list(slots) + [self.runner.pad_slot] * pad + list(seq_keys) + [0] * pad + list(step_keys) + [0] * pad
                            + [p.top_k for p in sampling] + [0] * pad, dtype=torch.int32)
        reals = torch.tensor([p.temperature for p in sampling] + [0.0] * pad + [p.top_p for p in sampling] + [1.0] * pad + [p.min_p for p in sampling] + [0.0] * pad,
                             dtype=torch.float32)
        cache.staging.copy(torch.cat((ints, reals.view(torch.int32))), [b.block])
        if b.graph is not None:
            b.graph.replay()
        else:
            self._body(b, captured=False)
        tokens, count = b.out[0], b.out[1]
        host = torch.cat((count, tokens.reshape(-1))).cpu().tolist()        # (waits for the step)
        self.ops.raise_on_draft_error()
        out = []
        for i in range(n):
            m = host[i]
            out.append(host[b.size + i * b.tokens:b.size + i * b.tokens + m])
            cache.set_length(slots[i], lengths[i] + m)
        self.steps += 1
        self.accepted += sum(len(x) - 1 for x in out)
        return out
