"""Drafts from a sequence's own text, and which drafted tokens stand."""
import pytest

import qwen3_b200 as q
from qwen3_b200.engine.speculate import accepted


def test_prompt_lookup_finds_what_followed_before():
    draft = q.PromptLookup(tokens=4, depth=3, branches=2, longest=2, shortest=1)
    assert draft([5, 6, 7, 8, 9, 5, 6]) == ([7, 8, 9], [-1, 0, 1])
    assert draft([1]) == ([], []) and draft([1, 2, 3]) == ([], [])
    # two continuations of the same tokens share what they have in common
    tokens, parents = q.PromptLookup(tokens=8, depth=3, branches=2, longest=1, shortest=1)([1, 2, 3, 4, 1, 2, 5, 6, 1])
    assert (tokens, parents) == ([2, 5, 6, 3, 4], [-1, 0, 1, 0, 3])
    # a longer match is taken before a shorter one, a later one before an earlier one
    assert q.PromptLookup(tokens=1, depth=1, branches=1, longest=2)([1, 2, 9, 2, 8, 1, 2])[0] == [9]
    assert q.PromptLookup(tokens=1, depth=1, branches=1, longest=1)([2, 9, 2, 8, 2])[0] == [8]
    assert q.PromptLookup(tokens=0)([1, 1, 1]) == ([], [])
    assert len(q.PromptLookup(tokens=3, depth=9)([1] * 30)[0]) == 3


@pytest.mark.parametrize("options", [dict(tokens=-1), dict(depth=0), dict(branches=0), dict(longest=1, shortest=2), dict(shortest=0)])
def test_a_drafter_refuses(options):
    with pytest.raises(ValueError):
        q.PromptLookup(**options)


def test_accepted_tokens_are_what_the_model_chose():
    tokens, parents = [9, 1, 2, 1, 3, 4], [-1, 0, 0, 2, 2, 4]
    assert accepted(tokens, parents, [7, 0, 0, 0, 0, 0]) == [0]
    assert accepted(tokens, parents, [1, 5, 0, 0, 0, 0]) == [0, 1]
    assert accepted(tokens, parents, [2, 0, 3, 0, 4, 8]) == [0, 2, 4, 5]
    assert accepted([9], [-1], [3]) == [0]


class _Book:
    """A stand-in for a cache that counts places and pages."""
    page_tokens, n_pages, n_slots = 4, 6, 3

    def __init__(self):
        self.groups = [self]
        self.held = 0

    @property
    def n_free(self):
        return self.n_pages - self.held


def test_the_loop_refuses():
    class Engine:
        max_seq_len, cache = 8, _Book()
    assert q.generate_speculative(Engine(), [], 3) == []
    assert [r.token_ids for r in q.generate_speculative(Engine(), [[1]], 0)] == [[]]
    for prompts, n in (([[]], 3), ([[1] * 6], 3), ([[1]], -1)):
        with pytest.raises(ValueError):
            q.generate_speculative(Engine(), prompts, n)
