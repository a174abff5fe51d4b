"""The pages of a step that reads a cache in 8 bits back: those that its sequences hold, packed."""
import pytest
import torch

import qwen3_b200 as q
from qwen3_b200.engine.context import Scratch, StepContext


def context(pos0, n_new, tables):
    i = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    start = [0]
    for n in n_new:
        start.append(start[-1] + n)
    N, B = start[-1], len(n_new)
    return StepContext(n_tokens=N, n_seqs=B, n_want=0, is_decode=False, max_new=max(n_new), max_context=max(a + b for a, b in zip(pos0, n_new)),
                       max_positions=10 ** 6, dtype=torch.float32, device=torch.device("cpu"), scratch=Scratch("cpu"), token_ids=i([0] * N), token_seq=i([0] * N),
                       token_pos=i([0] * N), seq_slots=i(list(range(B))), seq_start=i(start), seq_pos0=i(pos0), want_rows=i([0]), page_tables=tables,
                       host_slots=list(range(B)), host_n_new=list(n_new), host_pos0=list(pos0))


@pytest.mark.parametrize("pos0,n_new", [([0], [1]), ([64], [64]), ([0, 63, 500, 5], [1, 1, 600, 60]), ([0] * 40, list(range(1, 41))), ([32000] + [100] * 63, [1] * 63 + [513])])
def test_every_page_that_is_held_is_read_once(pos0, n_new):
    lengths = [a + b for a, b in zip(pos0, n_new)]
    held = [-(-n // q.PAGE_TOKENS) for n in lengths]
    width, tables = max(held) + 3, []
    for g in range(2):
        order = torch.randperm(sum(held), generator=torch.Generator().manual_seed(g)).to(torch.int32)
        table, at = torch.full((len(held), width), -1, dtype=torch.int32), 0
        for s, n in enumerate(held):
            table[s, :n] = order[at:at + n]
            at += n
        tables.append(table)
    ctx = context(pos0, n_new, tables)
    for g, table in enumerate(tables):
        numbers, rows, read = ctx.read_back(g)
        assert numbers.shape == (sum(held), 1) and rows.shape == (sum(held),) and read.shape == (len(held), max(held))
        assert all(t.dtype == torch.int32 and t.is_contiguous() for t in (numbers, rows, read)) and 0 <= int(read.min()) and int(read.max()) < sum(held)
        for s, n in enumerate(held):
            at = read[s, :n].long()
            assert torch.equal(numbers[at, 0], table[s, :n])
            assert rows[at].tolist() == [min(64, lengths[s] - 64 * j) for j in range(n)]
        assert sorted(numbers[:, 0].tolist()) == sorted(table[table >= 0].tolist())
