"""Attention of trees of drafted tokens, runs and single tokens over a cache in the compute type or in 8 bits, against 64 bits."""
import math

import pytest
import torch

import tree_cases as tc
from tree_cases import PAGE

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def tolerance(kind, size):
    """`size` is sum of p |v|.  bfloat16: the output is rounded (2^-8 of a value not above `size`), and so may the weights be
    (2^-8 of every term); scores, exponentials and sums in 32 bits add less than 2e-4 for scores below 100.  32-bit: the latter, smaller."""
    return size * (2 * 2.0 ** -8 + 2e-4 if kind == "bf16" else 2e-5) + 1e-30


def make(kind, store, d, kv, group, spans, seed=0, loud=1.0):
    from qwen3_b200.csrc import ops
    g, dtype = torch.Generator(device="cuda").manual_seed(seed + d), TYPES[kind]
    table, n_pages = tc.pages_for([a + b for a, b in spans], seed)
    n, heads = sum(b for _, b in spans), kv * group
    parts = []
    for _ in range(2):
        x = torch.randn(n_pages, kv, PAGE, d, generator=g, device="cuda") * torch.exp(loud * torch.randn(n_pages, kv, PAGE, 1, generator=g, device="cuda"))
        parts.append(tc.quantised(x) if store == "f8" else (x.to(dtype), None))
    q = torch.randn(n, heads * d, generator=g, device="cuda").to(dtype)
    return q, ops.CachePages(parts[0][0], parts[1][0], parts[0][1], parts[1][1]), table, heads


def attend(q, cache, table, spans, heads, scale, tree, fill=float("nan"), max_new=None):
    from qwen3_b200.csrc import ops
    old, new = [a for a, _ in spans], [b for _, b in spans]
    start = [0]
    for b in new:
        start.append(start[-1] + b)
    out = torch.full_like(q, fill)
    sizes = ops.attention_tree_scratch(len(spans), max_new or max(new), heads, cache.kv_heads, cache.d, q.device)
    parts = torch.full((sizes.parts,), float("nan"), device="cuda")
    counters = torch.zeros(sizes.counters, dtype=torch.int32, device="cuda")
    got = ops.attention_tree(q, cache, out, parts, counters, ints(start), ints(old), table.cuda(), max_new or max(new), heads, scale,
                             tree=None if tree is None else tree.cuda())
    assert not bool(counters.any()) and ops.tcgen05_status(q.device) == 0
    return got.view(q.shape[0], heads, cache.d)


def check(kind, store, d, kv, group, spans, masks, seed=0, words=None, loud=1.0):
    q, cache, table, heads = make(kind, store, d, kv, group, spans, seed, loud)
    old, new = [a for a, _ in spans], [b for _, b in spans]
    tree = None if masks is None else tc.masks_for(masks, new, words or -(-max(new) // 64), seed)
    scale = 1.7 * d ** -0.5
    want, size = tc.attention(q, tc.values_of(cache.keys, cache.key_scales), tc.values_of(cache.values, cache.value_scales), table, old, new, heads,
                              scale, tree)
    got = attend(q, cache, table, spans, heads, scale, tree)
    off = (got.double() - want).abs()
    assert bool((off <= tolerance(kind, size)).all()), float((off / (size + 1e-30)).max())
    return got


RAGGED = [(300, 5), (0, 1), (63, 8), (64, 2), (1, 3), (129, 7)]
KINDS = [("bf16", "bf16"), ("bf16", "f8"), ("f32", "f32"), ("f32", "f8")]


@pytest.mark.parametrize("kind,store", KINDS)
@pytest.mark.parametrize("d,kv,group", [(128, 2, 4), (64, 1, 5), (128, 1, 1), (128, 1, 8), (64, 3, 2), (48, 1, 3), (256, 1, 2), (16, 2, 7), (96, 1, 12)])
def test_single_tokens(kind, store, d, kv, group):
    check(kind, store, d, kv, group, [(a, 1) for a in (0, 1, 62, 63, 64, 65, 127, 128, 500, 1000)], None)


@pytest.mark.parametrize("kind,store", KINDS)
@pytest.mark.parametrize("d,kv,group", [(128, 2, 4), (64, 1, 5), (128, 1, 7), (64, 2, 1), (80, 1, 3)])
@pytest.mark.parametrize("masks", ["tree", "bits", None])
def test_few_new_tokens(kind, store, d, kv, group, masks):
    check(kind, store, d, kv, group, RAGGED, masks)


@pytest.mark.parametrize("kind,store", KINDS)
@pytest.mark.parametrize("d,kv,group", [(128, 1, 4), (64, 2, 3), (128, 1, 5)])
@pytest.mark.parametrize("masks", ["tree", "bits", None])
@pytest.mark.parametrize("spans", [[(500, 64), (0, 33), (77, 50), (64, 1)], [(130, 65), (3, 130), (200, 20)]])
def test_many_new_tokens(kind, store, d, kv, group, masks, spans):
    check(kind, store, d, kv, group, spans, masks)


@pytest.mark.parametrize("kind,store", KINDS[:2])
@pytest.mark.parametrize("spans", [[(9000, 1)], [(20000, 3)], [(9000, 40)], [(6000, 1)] * 3 + [(0, 1)] * 30, [(100 * i, 1 + i % 4) for i in range(40)], [(37 * (i % 9), 1 + i % 3) for i in range(70)],
                                   [(5000, 64), (1, 1)], [(900, 20)] * 9])
def test_long_contexts(kind, store, spans):
    check(kind, store, 128, 1, 4, spans, "tree", seed=5)


@pytest.mark.parametrize("kind,store", KINDS)
@pytest.mark.parametrize("b", [1, 7, 40])
def test_rows_that_see_nothing_are_zero(kind, store, b):
    spans = [(0, b), (0, 1), (70, b)]
    got = check(kind, store, 128, 1, 4, spans, "none")
    assert not bool(got[:b + 1].any())


@pytest.mark.parametrize("kind,store", KINDS)
def test_one_seen_key_is_its_value(kind, store):
    """A token that sees one key gets that key's value, to its last bit."""
    for d, group, b in ((128, 4, 5), (64, 2, 60), (48, 1, 3)):
        spans = [(0, b)]
        q, cache, table, heads = make(kind, store, d, 1, group, spans)
        tree = torch.tensor([[1 << (b - 1 - t)] for t in range(b)], dtype=torch.int64)
        got = attend(q, cache, table, spans, heads, 0.3, tree)
        want = tc.rows_of(tc.values_of(cache.values, cache.value_scales), table[0], b).flip(0).expand(b, heads, d)
        assert torch.equal(got.double(), want)


@pytest.mark.parametrize("kind,store", KINDS)
@pytest.mark.parametrize("d,group,b", [(128, 4, 1), (128, 4, 6), (64, 5, 20), (128, 4, 64), (48, 2, 5)])
def test_nothing_unseen_is_felt(kind, store, d, group, b):
    """Infinities and NaN in rows that a token does not see - behind the sequence's end, of drafts that are not its ancestors, in other
    pages - leave its output as it is, bit for bit; one that sees such a value has it in that place of its output."""
    spans = [(100, b), (0, b)]
    q, cache, table, heads = make(kind, store, d, 2, group, spans)
    tree = tc.masks_for("tree", [b, b], 1, 4)
    plain = attend(q, cache, table, spans, heads, d ** -0.5, tree)
    last = b - 1
    untouched = [t for t in range(2 * b) if not int(tree[t, 0]) >> last & 1]
    live = torch.zeros(cache.n_pages, PAGE, dtype=torch.bool, device="cuda")
    for s, (a, n) in enumerate(spans):
        for p in range(a + n):
            if p != a + last:
                live[table[s, p // PAGE], p % PAGE] = True
    bad = [math.nan, math.inf, -math.inf]
    for pages, scales in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
        wide = tc.values_of(pages, scales) if store != "f8" else pages.float()
        kind_of_bad = torch.tensor([bad[i % 3] for i in range(d)], device="cuda", dtype=wide.dtype)
        wide = torch.where(live[:, None, :, None], wide, kind_of_bad)
        pages.copy_(wide.to(pages.dtype))
        if scales is not None:
            scales.view(torch.uint8)[(~live)[:, None].expand(scales.shape)] = 187
    got = attend(q, cache, table, spans, heads, d ** -0.5, tree)
    assert torch.equal(got[untouched], plain[untouched])
    seen = [t for t in range(2 * b) if t not in untouched]
    assert bool(got[seen].isnan().all())                                # its score is no number, and so is all of the row


@pytest.mark.parametrize("kind,store", KINDS)
@pytest.mark.parametrize("d,group,b", [(128, 4, 1), (128, 4, 6), (64, 5, 20), (128, 4, 64), (48, 2, 5)])
def test_values_that_are_no_numbers_stay_in_their_column(kind, store, d, group, b):
    spans = [(100, b), (0, b)]
    q, cache, table, heads = make(kind, store, d, 2, group, spans)
    tree = tc.masks_for("tree", [b, b], 1, 4)
    plain = attend(q, cache, table, spans, heads, d ** -0.5, tree)
    for s, (a, n) in enumerate(spans):
        place = a + n - 1
        row = cache.values.view(torch.uint8) if store == "f8" else cache.values
        row[table[s, place // PAGE], :, place % PAGE, 7] = 0x7f if store == "f8" else math.nan
    got = attend(q, cache, table, spans, heads, d ** -0.5, tree)
    for t in range(2 * b):
        seen = int(tree[t, 0]) >> (b - 1) & 1
        where = torch.zeros(heads, d, dtype=torch.bool, device="cuda")
        where[:, 7] = bool(seen)
        assert torch.equal(got[t].isnan(), where) and torch.equal(got[t][~where], plain[t][~where])


@pytest.mark.parametrize("kind,store", KINDS)
@pytest.mark.parametrize("b", [1, 9, 50])
def test_loud_and_quiet_rows(kind, store, b):
    """Rows of very unequal size: values whose weights are small may be the largest, and the other way round."""
    spans = [(400, b), (30, b)]
    for loud in (3.0, 6.0):
        q, cache, table, heads = make(kind, store, 128, 1, 4, spans, seed=9, loud=loud)
        q = q * math.exp(-3 * loud)                                     # scores stay within the bound of `tolerance`
        keep = tc.values_of(cache.keys, cache.key_scales), tc.values_of(cache.values, cache.value_scales)
        new = [b, b]
        tree = tc.masks_for("tree", new, 1, 2)
        scale = 128 ** -0.5
        want, size = tc.attention(q, *keep, table, [400, 30], new, heads, scale, tree)
        got = attend(q, cache, table, spans, heads, scale, tree)
        assert bool(((got.double() - want).abs() <= tolerance(kind, size)).all())


def test_the_same_step_gives_the_same_bits():
    for spans in ([(3000, 1)] * 5, [(2000, 30), (10, 3)], [(70, 64)] * 3):
        q, cache, table, heads = make("bf16", "f8", 128, 2, 4, spans)
        tree = tc.masks_for("tree", [b for _, b in spans], 1, 1)
        first = attend(q, cache, table, spans, heads, 0.1, tree)
        for _ in range(5):
            assert torch.equal(attend(q, cache, table, spans, heads, 0.1, tree), first)


def test_on_another_stream():
    spans = [(500, 6), (90, 2)]
    q, cache, table, heads = make("bf16", "f8", 128, 2, 4, spans)
    want = attend(q, cache, table, spans, heads, 0.1, None)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = attend(q, cache, table, spans, heads, 0.1, None)
        torch.cuda.current_stream().synchronize()
    assert torch.equal(got, want)


def test_refusals():
    from qwen3_b200.csrc import ops
    q, cache, table, heads = make("bf16", "f8", 64, 2, 2, [(5, 3)])
    sizes = ops.attention_tree_scratch(1, 3, heads, 2, 64, q.device)
    parts, counters = torch.empty(max(sizes.parts, 1), device="cuda"), torch.zeros(max(sizes.counters, 1), dtype=torch.int32, device="cuda")
    start, pos0, tree = ints([0, 3]), ints([5]), torch.ones(3, 1, dtype=torch.int64, device="cuda")
    args = [q, cache, torch.empty_like(q), parts, counters, start, pos0, table.cuda(), 3, heads, 0.1]
    ops.attention_tree(*args, tree=tree)
    wrong = {0: [q[:, :-1], q.float(), q.half(), q.cpu()], 2: [q[:2], q.float()], 5: [start[:1], start.long()], 6: [pos0.float(), ints([5, 6])],
             7: [table[0].cuda(), table], 8: [0], 9: [3, 0]}
    for i, values in wrong.items():
        for v in values:
            with pytest.raises(ops.KernelError):
                ops.attention_tree(*args[:i], v, *args[i + 1:], tree=tree)
    for bad in (tree[:2], tree[:, 0], tree.int(), tree.cpu(), torch.ones(3, 2, dtype=torch.int64, device="cuda")[:, ::2]):
        with pytest.raises(ops.KernelError):
            ops.attention_tree(*args, tree=bad)
    with pytest.raises(ops.KernelError):
        ops.attention_tree(*args[:8], 65, *args[9:], tree=tree)


@pytest.mark.parametrize("store", ["bf16", "f8"])
@pytest.mark.parametrize("d,kv,group", [(128, 2, 4), (64, 3, 3), (128, 1, 8)])
@pytest.mark.parametrize("rows", [1, 10 ** 9])
@pytest.mark.parametrize("spans,masks", [([(200, 3), (61, 9), (0, 1), (130, 5)], "tree"), ([(900, 4)], None), ([(40, 30), (3, 64), (700, 1)], "tree"),
                                         ([(70 * (i % 5), 2 + i % 7) for i in range(45)], "tree")])
def test_each_form_takes_any_number_of_rows(monkeypatch, store, d, kv, group, rows, spans, masks):
    """The tcgen05 form where the mma.sync form would be taken, and the other way round: which is faster is all that the choice rests on."""
    from qwen3_b200.csrc import ops
    monkeypatch.setattr(ops, "tree_tc_rows", rows)
    monkeypatch.setattr(ops, "tree_tc_items", 10 ** 9)
    monkeypatch.setattr(ops, "tree_tc_pages", 10 ** 9)
    check("bf16", store, d, kv, group, spans, masks, seed=11)


def test_the_choice_of_a_form():
    from qwen3_b200.csrc import ops

    def form(rows, eight_bit=False, items=8, table=10, d=128, scale=0.1, dtype=torch.bfloat16, places=1000):
        return ops._tree_form(dtype, rows, d, scale, places, eight_bit, items, table)
    assert [form(r) for r in (1, 16, 17, 64)] == ["mma", "mma", "tc", "tc"]
    assert [form(32, items=200), form(32, items=200, table=17), form(33, items=200)] == ["mma", "tc", "tc"]
    assert [form(32, True, items=200, table=17), form(32, True, 100, 41), form(32, True, 100, 40), form(33, True, 200, 1000)] == ["mma", "mma", "tc", "tc"]
    assert [form(64, d=80), form(64, dtype=torch.float32), form(64, scale=0.0), form(64, places=2 ** 31)] == ["any", "any", "mma", "mma"]
