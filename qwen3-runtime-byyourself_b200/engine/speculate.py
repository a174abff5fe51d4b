"""Greedy generation with drafted tokens: a drafter proposes how each sequence may go on, one step runs the whole tree of proposals
over the cache, and the tokens that the model itself would have chosen are kept.

A step reads weights and cache once for all tokens of its trees, and yields one token more than the drafted ones that stand.  The tokens are those that
greedy generation one by one chooses, but where the two largest logits lie within the arithmetic's rounding: a step of another shape takes other kernels, which
add up in another order, in 32 bits and, in a bfloat16 engine, with roundings to 16 bits in other places (as steps of other batch sizes do).  A chosen token that
differs changes all that follow.

Drafts pay where enough of them stand: a tree step is launched kernel by kernel, where a decode step is replayed from a graph (8B shape, 8 sequences of
4,096, bfloat16: 3.9 ms a decode step; 5.0, 5.3 and 6.0 with 4, 8 and 16 tokens a sequence).
"""
from __future__ import annotations

from typing import Callable, List, Optional, Sequence, Tuple

import torch

from .engine import Engine, TreeEntry
from .generate import MAX_NEW_TOKENS, STOP_TOKEN, GenerationResult, plan_batches

Tree = Tuple[List[int], List[int]]             # tokens, parents (-1: the token that the tree hangs on)


class PromptLookup:
    """Drafts from the sequence's own text: where its last few tokens stood before, they were followed by what may follow now.

    `longest` to `shortest` tokens are looked for, the longest match first and the latest places first; up to `branches` different continuations
    of up to `depth` tokens make a tree of at most `tokens` tokens.  The whole text is walked through on the host: without a match 1.5 ms for 4,096
    tokens and 14 for 32,000, a sequence and step; long texts want a drafter that keeps an index."""

    def __init__(self, tokens: int = 15, depth: int = 8, branches: int = 3, longest: int = 4, shortest: int = 1):
        if tokens < 0 or depth < 1 or branches < 1 or not 1 <= shortest <= longest:
            raise ValueError("a drafter takes tokens >= 0, depth and branches >= 1, 1 <= shortest <= longest")
        self.tokens, self.depth, self.branches, self.longest, self.shortest = tokens, depth, branches, longest, shortest

    def __call__(self, text: Sequence[int]) -> Tree:
        tokens, parents, found, text = [], [], 0, list(text)
        for n in range(min(self.longest, len(text) - 1), self.shortest - 1, -1):
            last = text[-n:]
            for at in range(len(text) - n - 1, -1, -1):
                if found == self.branches or len(tokens) >= self.tokens:
                    return tokens, parents
                if text[at:at + n] != last:
                    continue
                parent, new = -1, False
                for token in text[at + n:at + n + self.depth]:
                    child = next((i for i, (t, p) in enumerate(zip(tokens, parents)) if t == token and p == parent), None)
                    if child is None:
                        if len(tokens) >= self.tokens:
                            break
                        tokens.append(token)
                        parents.append(parent)
                        child, new = len(tokens) - 1, True
                    parent = child
                found += new
            if tokens:
                break
        return tokens, parents


def accepted(tokens: Sequence[int], parents: Sequence[int], chosen: Sequence[int]) -> List[int]:
    """The tree's tokens that stand: from token 0 on, which is no draft, always the child that the model chose (`chosen[i]`: what it puts
    behind token i)."""
    path, children = [0], {}
    for i, p in enumerate(parents):
        children.setdefault(p, []).append(i)
    while True:
        last = path[-1]
        follow = next((i for i in children.get(last, ()) if tokens[i] == chosen[last]), None)
        if follow is None:
            return path
        path.append(follow)


def generate_speculative(engine: Engine, prompts: Sequence[Sequence[int]], max_new_tokens: int = 128, stop_token_ids: Sequence[int] = (),
                         draft: Optional[Callable[[Sequence[int]], Tree]] = None, batch_size: Optional[int] = None) -> List[GenerationResult]:
    """Greedy generation for every prompt with drafted tokens.  `draft(text) -> (tokens, parents)` proposes continuations of a
    sequence's tokens (default: `PromptLookup()`)."""
    from ..csrc import ops
    from .engine import StepEntry
    draft = draft or PromptLookup()
    prompts = [[int(t) for t in p] for p in prompts]
    if any(not p for p in prompts):
        raise ValueError("a prompt needs at least one token")
    if max_new_tokens < 0 or any(len(p) + max_new_tokens > engine.max_seq_len for p in prompts):
        raise ValueError(f"prompt and new tokens exceed the context of {engine.max_seq_len} tokens")
    stops = {int(t) for t in stop_token_ids}
    results = [GenerationResult() for _ in prompts]
    if max_new_tokens == 0 or not prompts:
        return results

    def pages(tokens: int) -> int:
        return -(-tokens // engine.cache.page_tokens)

    def choose(logits: torch.Tensor) -> List[int]:
        ids = ops.argmax(logits, torch.empty(logits.shape[0], dtype=torch.int32, device=engine.device)).tolist()
        engine.check_kernels()                               # the device has been waited for: nothing of a step that a kernel gave up on is taken
        return ids

    for batch in plan_batches([len(p) for p in prompts], max_new_tokens, engine.cache.n_pages, engine.cache.n_slots, engine.cache.page_tokens,
                              batch_size):
        live = {}                                            # request -> slot
        try:
            for i in batch:
                live[i] = engine.new_sequence()

            def record(i: int, new: Sequence[int]) -> bool:
                """Adds the request's next tokens; True once it has ended."""
                for token in new:
                    results[i].token_ids.append(token)
                    if token in stops:
                        results[i].stop_reason = STOP_TOKEN
                        return True
                    if len(results[i].token_ids) == max_new_tokens:
                        results[i].stop_reason = MAX_NEW_TOKENS
                        return True
                return False

            def end(i: int) -> None:
                engine.release(live.pop(i))

            first = choose(engine.step([StepEntry(live[i], prompts[i], want=[len(prompts[i]) - 1]) for i in batch]))
            for i, token in zip(batch, first):
                if record(i, [token]):
                    end(i)
            while live:
                entries, order = [], list(live)
                for i in order:
                    text = prompts[i] + results[i].token_ids
                    # token 0 is the one chosen last; no draft goes beyond the tokens that are still wanted
                    left = max_new_tokens - len(results[i].token_ids)
                    tokens, parents = draft(text) if left > 1 else ([], [])
                    depth = []
                    for p in parents:
                        depth.append(depth[p] + 1 if p >= 0 else 1)
                    keep = [n for n, d in enumerate(depth) if d < left]
                    number = {n: k + 1 for k, n in enumerate(keep)}
                    room = engine.max_seq_len - len(text)    # places behind the last token
                    keep = keep[:max(room, 0)]
                    entries.append(TreeEntry(live[i], [text[-1]] + [int(tokens[n]) for n in keep],
                                             [-1] + [number[parents[n]] if parents[n] >= 0 else 0 for n in keep]))
                # a tree that the pages have no room for, beside the pages that the sequences' next tokens need, goes without its drafts
                free = min(g.n_free for g in engine.cache.groups)
                free -= sum(pages(engine.length(e.slot) + 1) - pages(engine.length(e.slot)) for e in entries)
                for e in entries:
                    length = engine.length(e.slot)
                    need = pages(length + len(e.tokens)) - pages(length + 1)
                    if need > free:
                        e.tokens, e.parents = e.tokens[:1], e.parents[:1]
                    else:
                        free -= need
                chosen, at, paths, ended = choose(engine.step_tree(entries)), 0, {}, []
                for i, e in zip(order, entries):
                    mine = chosen[at:at + len(e.tokens)]
                    at += len(e.tokens)
                    path = accepted(e.tokens, e.parents, mine)
                    paths[e.slot] = path
                    if record(i, [e.tokens[n] for n in path[1:]] + [mine[path[-1]]]):
                        ended.append(i)
                engine.keep(paths)
                for i in ended:
                    end(i)
        finally:
            for slot in list(live.values()):
                engine.release(slot)
    return results
