"""Rows of the paged cache on the GPU: appended (normed, rotated, quantised to 8 bits), read back, kept after drafts."""
import itertools
import math

import pytest
import torch

import tree_cases as tc
from tree_cases import PAGE

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def blank(n_pages, kv, d, dtype, eight_bit):
    """Pages that are filled with a value of their own, to see what was written."""
    from qwen3_b200.csrc import ops
    if not eight_bit:
        return ops.CachePages(*(torch.full((n_pages, kv, PAGE, d), 77.0, dtype=dtype, device="cuda") for _ in range(2)))
    codes = [torch.full((n_pages, kv, PAGE, d), 0x55, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.full((n_pages, kv, PAGE), 99, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    return ops.CachePages(*codes, *scales)


def raw(x):
    return x.view(torch.uint8) if x.element_size() == 1 else x


CASES = [  # type, 8 bits, head size, kv heads, query heads of each, rotated values, norm, rounded once, more columns
    ("bf16", True, 128, 2, 4, 128, True, True, 0), ("bf16", True, 128, 8, 5, 128, True, False, 0), ("bf16", False, 128, 1, 8, 128, True, False, 0),
    ("bf16", False, 64, 2, 2, 64, True, True, 0), ("bf16", True, 64, 3, 1, 64, False, True, 40), ("bf16", True, 256, 1, 3, 256, True, True, 0),
    ("bf16", True, 48, 2, 3, 48, True, True, 0), ("bf16", True, 80, 1, 2, 32, True, False, 3), ("bf16", True, 128, 2, 1, 64, True, True, 0),
    ("bf16", True, 128, 2, 2, 0, True, True, 0), ("bf16", False, 96, 1, 2, 0, False, False, 8), ("bf16", True, 16, 4, 2, 16, True, True, 0),
    ("bf16", True, 30, 2, 2, 20, True, True, 1), ("f32", True, 128, 2, 2, 128, True, True, 0), ("f32", True, 64, 1, 1, 64, True, False, 4),
    ("f32", False, 32, 1, 8, 32, True, True, 0), ("f32", False, 100, 1, 2, 50, False, True, 0), ("f32", True, 24, 2, 1, 24, True, True, 2),
    ("bf16", True, 112, 2, 7, 112, True, True, 0), ("bf16", True, 192, 1, 2, 192, True, False, 0)]


@pytest.mark.parametrize("kind,eight_bit,d,kv,group,rot,norm,once,more", CASES)
@pytest.mark.parametrize("spans", [[(0, 1)], [(63, 3), (0, 130), (64, 1), (700, 17)]])
def test_append(kind, eight_bit, d, kv, group, rot, norm, once, more, spans):
    from qwen3_b200.csrc import ops
    dtype, heads, g = TYPES[kind], kv * group, torch.Generator(device="cuda").manual_seed(d + rot + len(spans))
    old, new = [a for a, _ in spans], [b for _, b in spans]
    table, n_pages = tc.pages_for([a + b for a, b in spans], d)
    n, columns = sum(new), (heads + 2 * kv) * d
    qkv = (torch.randn(n, columns + more, generator=g, device="cuda") * torch.exp(torch.randn(n, 1, generator=g, device="cuda"))).to(dtype)
    qw, kw = (1 + 0.3 * torch.randn(d, generator=g, device="cuda") for _ in range(2)) if norm else (None, None)
    seq = [i for i, b in enumerate(new) for _ in range(b)]
    place = [a + t for a, b in spans for t in range(b)]
    pos = [a + t // 2 for a, b in spans for t in range(b)]              # several tokens at one position
    angle = torch.rand(max(pos) + 1, max(rot // 2, 1), generator=g, device="cuda") * 6.3
    cos, sin = (angle.cos(), angle.sin()) if rot else (None, None)
    cache, q = blank(n_pages, kv, d, dtype, eight_bit), torch.full((n, heads * d), 77.0, dtype=dtype, device="cuda")
    before = [raw(t).clone() for t in (cache.keys, cache.values)] + ([raw(t).clone() for t in (cache.key_scales, cache.value_scales)] if eight_bit else [])
    ops.cache_append(qkv, q, cache, qw, kw, cos, sin, 1e-5, ints(seq), ints(pos), ints(place), table.cuda(), heads, norm_once=once)

    x = qkv[:, :columns].double().view(n, heads + 2 * kv, d)
    # a value's error: a rounding to the type wherever one is made (half a unit: u), and some 32-bit operations
    u, f = (2.0 ** -8 if kind == "bf16" else 2.0 ** -24), 2.0 ** -20

    def made(y, w):
        """(exact, bound of the error before the last rounding)"""
        if w is not None:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-5) * w.double()
        size = y.abs()
        if rot:
            a, b, rest = y[..., :rot // 2], y[..., rot // 2:rot], y[..., rot:]
            c, s = (t.double()[torch.tensor(pos, device="cuda")][:, None] for t in (cos, sin))
            y = torch.cat([a * c - b * s, b * c + a * s, rest], -1)
            size = torch.cat([a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs(), rest.abs()], -1)
        return y, size * (f + (0 if once or w is None else 2.01 * u))

    def stored(got, exact, bound, rounded):
        assert bool(((got.double() - exact).abs() <= bound + rounded).all())

    want, bound = made(x[:, :heads], qw)
    stored(q.view(n, heads, d), want, bound, 1.01 * u * want.abs())
    page = table[torch.tensor(seq), torch.tensor(place) // PAGE].long().cuda()
    at = torch.tensor(place, device="cuda") % PAGE
    keys, bound = made(x[:, heads:heads + kv], kw)
    vals = x[:, heads + kv:]
    if not eight_bit:
        stored(cache.keys[page, :, at], keys, bound, 1.01 * u * keys.abs())
        assert torch.equal(cache.values[page, :, at], vals.to(dtype))
    else:
        codes, scales = tc.quantised(vals)                             # values are taken as they are: every bit is given
        assert torch.equal(raw(cache.values)[page, :, at], raw(codes)) and torch.equal(raw(cache.value_scales)[page, :, at], raw(scales))
        k = raw(cache.key_scales)[page, :, at].double() - 127
        one, top = torch.exp2(k)[..., None], keys.abs().amax(-1)
        slack = (bound + (0 if once else 1.01 * u * keys.abs())).amax(-1)
        assert bool((top - slack <= 448 * one[..., 0]).all()) and bool(((top + slack > 224 * one[..., 0]) | (k == -60)).all())
        got = cache.keys.view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn).float().double()
        v = (keys / one).abs()
        half_step = torch.where(v < 2.0 ** -6, torch.full_like(v, 2.0 ** -10), torch.exp2(torch.floor(torch.log2(v.clamp_min(1e-30) * 1.001)) - 4))
        off = (bound + (0 if once else 1.01 * u * keys.abs())) / one
        assert bool(((got - keys / one).abs() <= half_step + off).all())
    # nothing else was written
    touched = torch.zeros(n_pages, PAGE, dtype=torch.bool, device="cuda")
    touched[page, at] = True
    for t, was in zip((cache.keys, cache.values) + ((cache.key_scales, cache.value_scales) if eight_bit else ()), before):
        same = raw(t).transpose(1, 2) == was.transpose(1, 2)
        assert bool(same[~touched].all())


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_rows_of_every_size_and_no_numbers(kind, d):
    """Zeros, the smallest and largest numbers, infinities, NaN, and largest values on both sides of a scale's limit."""
    from qwen3_b200.csrc import ops
    dtype, g = TYPES[kind], torch.Generator(device="cuda").manual_seed(3)
    biggest, least = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    tops = [0.0, least, 2.0 ** -60, 448 * 2.0 ** -60, 224.0, 448.0, 450.0, 1.75, 1.7578125, 1.0, 3.5, 447.0, 448 * 2.0 ** 60, biggest]
    rows = torch.rand(len(tops), d, generator=g, device="cuda") * 2 - 1
    rows = (rows * torch.tensor(tops, device="cuda")[:, None]).to(dtype)
    rows[:, 5] = torch.tensor(tops, device="cuda").to(dtype)
    odd = rows[-6:].clone()
    odd[0, 1], odd[1, 2], odd[2, 3], odd[3, :], odd[4, ::2] = math.inf, -math.inf, math.nan, math.nan, math.inf
    rows = torch.cat([rows, odd])
    n = rows.shape[0]
    qkv = torch.cat([rows, rows, rows], 1).contiguous()
    cache, q = blank(2, 1, d, dtype, True), torch.empty(n, d, dtype=dtype, device="cuda")
    ops.cache_append(qkv, q, cache, None, None, None, None, 0.0, ints([0] * n), ints(list(range(n))), ints(list(range(n))), ints([[1]]), 1)
    codes, scales = tc.quantised(rows)
    for pages, held in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
        assert torch.equal(raw(held)[1, 0, :n], raw(scales))
        got, want = pages[1, 0, :n].float(), codes.float()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    assert torch.equal(q.nan_to_num(1.0), rows.nan_to_num(1.0))
    for out in (torch.float32, torch.bfloat16):                        # and what is read back is what they stand for
        back = torch.zeros(1, 1, 1, PAGE, d, dtype=out, device="cuda")
        also = torch.zeros_like(back)
        ops.cache_read(cache, ints([[1]]), ints([n]), back, also)
        want = tc.values_of(codes, scales)
        for x in (back, also):
            x = x[0, 0, 0, :n].double()
            assert torch.equal(x.isnan(), want.isnan()) and torch.equal(x.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("kind,eight_bit,d,kv,group", [("bf16", True, 128, 3, 3), ("bf16", False, 64, 1, 4), ("f32", True, 128, 2, 1), ("bf16", True, 80, 1, 5)])
@pytest.mark.parametrize("once", [True, False])
def test_a_prompt_is_what_its_tokens_are(kind, eight_bit, d, kv, group, once):
    """So many rows that heads are taken several at a time give the same bits as a few."""
    from qwen3_b200.csrc import ops
    dtype, heads, n = TYPES[kind], kv * group, 5000
    g = torch.Generator(device="cuda").manual_seed(d)
    qkv = torch.randn(n, (heads + 2 * kv) * d, generator=g, device="cuda").to(dtype)
    qw, kw = (1 + 0.3 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
    angle = torch.rand(n, d // 2, generator=g, device="cuda") * 6.3
    table, n_pages = tc.pages_for([n], 1)
    table, at = table.cuda(), torch.arange(n, dtype=torch.int32, device="cuda")
    whole, few = blank(n_pages, kv, d, dtype, eight_bit), blank(n_pages, kv, d, dtype, eight_bit)
    outs = [torch.empty(n, heads * d, dtype=dtype, device="cuda") for _ in range(2)]
    seq = torch.zeros_like(at)
    ops.cache_append(qkv, outs[0], whole, qw, kw, angle.cos(), angle.sin(), 1e-6, seq, at, at, table, heads, norm_once=once)
    for i in range(0, n, 250):
        s = slice(i, i + 250)
        ops.cache_append(qkv[s], outs[1][s], few, qw, kw, angle.cos(), angle.sin(), 1e-6, seq[s], at[s], at[s], table, heads, norm_once=once)
    assert torch.equal(*outs)
    for name in ("keys", "values") + (("key_scales", "value_scales") if eight_bit else ()):
        assert torch.equal(raw(getattr(whole, name)), raw(getattr(few, name)))


def test_tokens_without_a_page_are_not_written():
    from qwen3_b200.csrc import ops
    for d, eight_bit in itertools.product((128, 40), (True, False)):
        cache = blank(3, 2, d, torch.bfloat16, eight_bit)
        qkv = torch.randn(4, 8 * d, device="cuda").to(torch.bfloat16)
        q = torch.zeros(4, 4 * d, dtype=torch.bfloat16, device="cuda")
        table = ints([[1, -1], [3, 0]])                                # no page; a number beyond the pages
        was = raw(cache.keys).clone()
        ops.cache_append(qkv, q, cache, None, None, None, None, 0.0, ints([0, 0, 1, 1]), ints([0] * 4), ints([70, 130, 5, -1]), table, 4)
        assert torch.equal(raw(cache.keys), was) and torch.equal(q, qkv[:, :4 * d])


@pytest.mark.parametrize("d,kv", [(128, 8), (64, 3), (256, 1), (16, 2), (40, 2), (6, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_read(d, kv, dtype):
    from qwen3_b200.csrc import ops
    ends, g = [1, 64, 0, 65, 200, 63], torch.Generator(device="cuda").manual_seed(d)
    table, n_pages = tc.pages_for(ends, d)
    pages = [tc.quantised(torch.randn(n_pages, kv, PAGE, d, generator=g, device="cuda") * 9) for _ in range(2)]
    cache = ops.CachePages(pages[0][0], pages[1][0], pages[0][1], pages[1][1])
    P = table.shape[1] + 1
    outs = [torch.full((len(ends), P, kv, PAGE, d), 77.0, dtype=TYPES[dtype], device="cuda") for _ in range(2)]
    ops.cache_read(cache, table.cuda(), ints(ends), *outs)
    for out, (codes, scales) in zip(outs, pages):
        want = torch.full(out.shape, 77.0, dtype=torch.float64, device="cuda")
        stands = tc.values_of(codes, scales)
        for s, n in enumerate(ends):
            for j in range(-(-n // PAGE)):
                live = min(PAGE, n - j * PAGE)
                want[s, j] = 0
                want[s, j, :, :live] = stands[table[s, j]][:, :live]
        assert torch.equal(out.double(), want)


@pytest.mark.parametrize("kind,d,kv,lead", [("f8", 128, 8, (3, 2)), ("f8", 64, 1, (2,)), ("bf16", 128, 2, (5, 2)), ("bf16", 24, 3, ()), ("f32", 4, 1, (1, 2)),
                                            ("f8", 16, 5, (2, 2)), ("bf16", 256, 8, (2,))])
def test_keep(kind, d, kv, lead):
    from qwen3_b200.csrc import ops
    paths = [[0], [1], [0, 1, 2], [1, 2], [2, 5, 6, 60], [], [63], list(range(0, 64, 2)), list(range(1, 41)), [3, 64, 65, 120]]
    old = [0, 63, 10, 62, 64, 30, 1, 50, 127, 3]
    table, n_pages = tc.pages_for([a + 128 for a in old], d)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(*lead, n_pages, kv, PAGE, d, generator=g, device="cuda")
    store, scales = tc.quantised(x) if kind == "f8" else (x.to(TYPES[kind]), None)
    want, want_scales = raw(store).clone(), None if scales is None else raw(scales).clone()
    for s, path in enumerate(paths):
        for i, node in enumerate(path):
            a, b = old[s] + node, old[s] + i
            for t in [want] + ([] if scales is None else [want_scales]):
                t = t.view(-1, n_pages, kv, PAGE, d) if t is want else t.view(-1, n_pages, kv, PAGE)
                t[:, table[s, b // PAGE], :, b % PAGE] = t[:, table[s, a // PAGE], :, a % PAGE].clone()
    most = max(map(len, paths))
    path = ints([p + [-1] * (most - len(p)) for p in paths])
    ops.cache_keep(store, scales, table.cuda(), ints(old), path)
    assert torch.equal(raw(store), want) and (scales is None or torch.equal(raw(scales), want_scales))


def test_keep_leaves_what_is_no_path():
    """Numbers that do not ascend, or lie beyond the sequence's pages, move nothing."""
    from qwen3_b200.csrc import ops
    store = torch.randn(1, 2, 1, PAGE, 64, device="cuda").to(torch.bfloat16)
    was = store.clone()
    ops.cache_keep(store, None, ints([[0, 1], [0, -1]]), ints([10, 60]), ints([[0, 1, 1], [90, 20, 68]]))
    assert torch.equal(store, was)


def test_refusals():
    from qwen3_b200.csrc import ops
    bf = dict(dtype=torch.bfloat16, device="cuda")
    pages = torch.zeros(2, 2, PAGE, 32, **bf)
    codes, scales = torch.zeros(2, 2, PAGE, 32, device="cuda").to(torch.float8_e4m3fn), torch.ones(2, 2, PAGE, device="cuda").to(torch.float8_e8m0fnu)
    good = ops.CachePages(codes, codes.clone(), scales, scales.clone())
    for bad in [(pages, pages[:1]), (pages, pages.float()), (pages.half(), pages.half()), (pages, pages, scales, scales), (codes, codes),
                (codes, codes, scales[:1], scales), (codes, codes, scales.view(torch.uint8), scales), (pages.cpu(), pages.cpu()),
                (pages[:, :, :32], pages[:, :, :32]), (torch.zeros(1, 1, PAGE, 272, **bf),) * 2, (pages.transpose(0, 1), pages.transpose(0, 1))]:
        with pytest.raises(ops.KernelError):
            ops.CachePages(*bad)
    one, table = ints([0]), ints([[0]])
    qkv, q = torch.zeros(1, 6 * 32, **bf), torch.zeros(1, 2 * 32, **bf)
    args = [qkv, q, good, None, None, None, None, 0.0, one, one, one, table, 2]
    ops.cache_append(*args)
    wrong = {0: [qkv[:, :-1], qkv.half(), qkv.float(), qkv.cpu(), torch.zeros(1, 12 * 32, **bf)[:, ::2]], 1: [q[:, 1:], q.float()],
             2: [ops.CachePages(pages.float(), pages.float())], 3: [torch.ones(32, device="cuda"), torch.ones(31, device="cuda")], 5: [torch.zeros(4, 17, device="cuda")],
             8: [one.long()], 9: [one[:0]], 10: [one.cpu()], 11: [one], 12: [3, 0]}
    for i, values in wrong.items():
        for v in values:
            with pytest.raises((ops.KernelError, AttributeError)):
                ops.cache_append(*args[:i], v, *args[i + 1:])
    out = torch.zeros(1, 1, 2, PAGE, 32, **bf)
    for bad in [(ops.CachePages(pages, pages), table, one, out, out), (good, table, one, out[..., :16], out[..., :16]), (good, table, one, out, out.float()),
                (good, table, ints([1, 1]), out, out), (good, table, one, out.half(), out.half()), (good, one, one, out, out), (good, table, one.long(), out, out)]:
        with pytest.raises(ops.KernelError):
            ops.cache_read(*bad)
    path = ints([[0, -1]])
    for bad in [(codes, None, table, one, path), (pages, scales, table, one, path), (codes, scales[:1], table, one, path), (pages.half(), None, table, one, path),
                (pages, None, table, one, path[0]), (pages, None, table, one[:0], path), (pages, None, table, one, path.long()),
                (torch.zeros(1, 1, PAGE, 12, **bf), None, table, one, path)]:
        with pytest.raises(ops.KernelError):
            ops.cache_keep(*bad)
