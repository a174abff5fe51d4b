"""Generation with drafted tokens over a stand-in engine: what it asks of the engine beside its steps."""
import pytest
import torch

import qwen3_b200 as q


class Group:
    n_free = 100


class Cache:
    page_tokens, n_pages, n_slots, groups = 64, 100, 8, [Group()]


class Engine:
    """The token after t is t + 1.  `fails_at`: the number of the step after which a kernel says that it gave up."""
    max_seq_len, vocab_size, device, cache = 1000, 64, "cpu", Cache()

    def __init__(self, fails_at=None):
        self.fails_at, self.steps, self.checks, self.held, self.cached, self.kept = fails_at, 0, 0, {}, {}, []

    def new_sequence(self):
        slot = len(self.held)
        self.held[slot], self.cached[slot] = True, 0
        return slot

    def release(self, slot):
        assert self.held.pop(slot)

    def length(self, slot):
        return self.cached[slot]

    def check_kernels(self):
        from qwen3_b200.csrc import ops
        self.checks += 1
        if self.fails_at is not None and self.steps > self.fails_at:
            raise ops.KernelError("a wait ran out")

    def _logits(self, tokens):
        self.steps += 1
        return torch.nn.functional.one_hot((torch.tensor(tokens) + 1) % self.vocab_size, self.vocab_size).float()

    def step(self, entries):
        for e in entries:
            self.cached[e.slot] += len(e.tokens)
        return self._logits([e.tokens[i] for e in entries for i in e.want])

    def step_tree(self, entries):
        return self._logits([t for e in entries for t in e.tokens])

    def keep(self, paths):
        self.kept.append(paths)
        for slot, path in paths.items():
            self.cached[slot] += len(path)


@pytest.fixture(autouse=True)
def argmax_on_the_host(monkeypatch):
    from qwen3_b200.csrc import ops
    monkeypatch.setattr(ops, "argmax", lambda logits, out: out.copy_(logits.argmax(-1)))


def test_every_step_is_asked_whether_its_kernels_finished():
    engine = Engine()
    got = q.generate_speculative(engine, [[5], [9, 10]], 6, draft=lambda text: ([text[-1] + 1, text[-1] + 2], [-1, 0]))
    assert [r.token_ids for r in got] == [list(range(6, 12)), list(range(11, 17))]
    assert engine.checks >= engine.steps == 3 and not engine.held


@pytest.mark.parametrize("fails_at", [0, 1, 2])
def test_nothing_of_a_step_that_failed_is_taken(fails_at):
    from qwen3_b200.csrc import ops
    engine = Engine(fails_at)
    with pytest.raises(ops.KernelError):
        q.generate_speculative(engine, [[5], [9, 10]], 9, draft=lambda text: ([text[-1] + 1], [-1]))
    assert len(engine.kept) == max(fails_at - 1, 0) and not engine.held       # of the prompts' step nothing has to be kept


def test_drafts_that_need_no_page_run_where_none_is_free(monkeypatch):
    """The sequences' pages have room for their drafts; no other page is free."""
    monkeypatch.setattr(Group, "n_free", 0)
    engine = Engine()
    got = q.generate_speculative(engine, [[1] * 20, [2] * 30], 12, draft=lambda text: ([text[-1] + 1, text[-1] + 2], [-1, 0]))
    assert [r.token_ids for r in got] == [list(range(2, 14)), list(range(3, 15))] and engine.steps == 5


def test_drafts_leave_a_page_for_every_sequence(monkeypatch):
    """Three sequences stand at the end of their pages and two pages more than they need are free: two of the trees that ask for one more get it."""
    monkeypatch.setattr(Group, "n_free", 3 + 2)
    engine, asked = Engine(), []
    step_tree = engine.step_tree

    def counted(entries):
        asked.append([len(e.tokens) for e in entries])
        return step_tree(entries)
    engine.step_tree = counted
    q.generate_speculative(engine, [[1] * 64] * 3, 80, draft=lambda text: ([0] * 70, [-1] * 70))
    assert asked[0] == [71, 71, 1]
