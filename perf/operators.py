"""The operators of a cache that is kept in 8 bits and of steps that bring a tree of drafted tokens, and the work they do.

A server that drafts tokens runs, layer by layer of a step, these four:

  append   norms and rotates the new queries and keys and writes keys and values into the cache's pages, as 8-bit codes
           with one scale of a power of two for each row, or as they are;
  read     writes the cached rows of sequences out as bfloat16 pages again, for the attention of whole prompts;
  attend   attention of the new tokens - one a sequence, or a tree of drafted ones - over the cached pages;
  keep     after the step, moves the rows of the drafted tokens that stand to the places behind the sequence's old end.

A case names its operator and its sizes.  Head counts and sizes are those of this repository's models (32, 40 or 64
query heads over 8 of 128; the tests' small heads of 64).  Lengths of sequences are ragged and hang on the case alone;
values, trees and the order of pages hang on the seed.
"""
import math
import random

import torch

own = False

PAGE = 64
MOST_HELD = 1.5e8                          # values of a drawn case's pages of keys, where the whole pages are its output


def listed():
    return [
        # one chat's decode step, short context: latency alone
        _attend("attend_1_short", 1, 130, 1, 32, 8, 128, "f8"),
        # the benchmark's decode: 8 sequences of some thousand tokens
        _attend("attend_8", 8, 4000, 1, 32, 8, 128, "f8"),
        # a busy server: 64 sequences of very unequal context
        _attend("attend_64", 64, 9000, 1, 40, 8, 128, "f8"),
        # drafts of a few tokens over a cache that is not quantised
        _attend("attend_draft_8", 8, 3000, 7, 32, 8, 128, "bf16"),
        # one long document, a tree of odd size
        _attend("attend_tree_1_long", 1, 32000, 33, 64, 8, 128, "bf16"),
        # wide trees on every sequence: products as large as those of a prompt
        _attend("attend_tree_8_wide", 8, 8000, 64, 40, 8, 128, "f8"),
        # the rows of a decode step of 8 sequences
        _append("append_8", 8, 4000, 1, 32, 8, 128, "f8"),
        # a prompt's rows
        _append("append_prompt", 1, 0, 8000, 32, 8, 128, "f8"),
        # a follow-up of a chat: one sequence's pages read back
        _read("read_1", 1, 1500, 8, 128),
        # prompts that go on: 8 long sequences read back
        _read("read_8_long", 8, 8000, 8, 128),
        # one sequence's drafts kept in the layers of a small model
        _keep("keep_1", 1, 8, 12, 4, 128, "bf16"),
        # a batch's trees kept in the 36 layers of the 8B shape
        _keep("keep_8_deep", 8, 64, 36, 8, 128, "f8"),
    ]


def _attend(name, seqs, context, tokens, heads, kv_heads, d, store):
    return {"name": name, "op": "attend", "seqs": seqs, "context": context, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "d": d, "store": store}


def _append(name, seqs, context, tokens, heads, kv_heads, d, store):
    return {"name": name, "op": "append", "seqs": seqs, "context": context, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "d": d, "store": store}


def _read(name, seqs, context, kv_heads, d):
    return {"name": name, "op": "read", "seqs": seqs, "context": context, "kv_heads": kv_heads, "d": d}


def _keep(name, seqs, tokens, layers, kv_heads, d, store):
    return {"name": name, "op": "keep", "seqs": seqs, "tokens": tokens, "layers": layers, "kv_heads": kv_heads, "d": d,
            "store": store}


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    limit = [max(work(c)[what] for c in listed()) for what in ("bytes", "flops")]
    while True:
        d, kv = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 8])
        heads, store = kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8]), rng.choice(["f8", "f8", "bf16"])
        op = rng.choice(["attend", "attend", "attend", "append", "read", "keep"])
        if op == "attend":
            case = _attend("", log(1, 64), log(1, 32000), log(1, 64), heads, kv, d, store)
        elif op == "append":
            case = _append("", log(1, 64), log(1, 30000), log(1, 8000), heads, kv, d, store)
        elif op == "read":
            case = _read("", log(1, 64), log(1, 32000), kv, d)
        else:
            case = _keep("", log(1, 64), log(2, 64), rng.randint(1, 40), kv, d, store)
        del case["name"]
        cost = work(case)
        held = case["seqs"] * kv * d * (case["layers"] * 5 * PAGE if op == "keep" else case["context"] + case["tokens"] if op == "append" else 0)
        if cost["bytes"] <= limit[0] and cost["flops"] <= limit[1] and held <= MOST_HELD:
            return case


def _lengths(case):
    """Cached tokens and new tokens of every sequence: from a twelfth of the case's number up to it."""
    r = random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))
    n, context, tokens = case["seqs"], case.get("context", 250), case.get("tokens", 0)
    old = [context if i == 0 else r.randint(context // 12, context) for i in range(n)]
    new = [tokens if i == 0 else r.randint(max(1, tokens // 2), tokens) if tokens else 0 for i in range(n)]
    return old, new


def work(case):
    old, new = _lengths(case)
    kv, d, op = case["kv_heads"], case["d"], case["op"]
    row = kv * (d + 1 if case.get("store", "f8") == "f8" else 2 * d)         # a token's keys, or its values
    if op == "attend":
        n, h = sum(new), case["heads"]
        return {"bytes": 2 * row * sum(a + b for a, b in zip(old, new)) + 4 * n * h * d,
                "flops": 4 * h * d * sum(b * (a + 1) for a, b in zip(old, new))}
    if op == "append":
        n, h = sum(new), case["heads"]
        return {"bytes": n * (2 * (h + 2 * kv) * d + 2 * h * d + 2 * row + 4 * d), "flops": 8 * n * (h + kv) * d}
    if op == "read":
        return {"bytes": sum(old) * 2 * (row + kv * 2 * d), "flops": 2 * sum(old) * kv * d}
    rows = sum(_path_length(b) for b in new)
    return {"bytes": rows * 2 * case["layers"] * 2 * row, "flops": 0}


def _path_length(tokens):
    """How many drafted tokens of a tree stand, in a case of `keep`."""
    return max(1, min(tokens, 1 + tokens.bit_length()))


# ------------------------------------------------------------------ inputs
def _quantise(x):
    """Codes and scales of rows [..., d]: the smallest power of two by which the largest value fits into 448."""
    top = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)                                 # top = m * 2^e, m in [1/2, 1); 448 = 7/8 * 2^9
    k = torch.where(m > 0.875, e - 8, e - 9).clamp(-60, 60)
    k = torch.where(top == 0, torch.full_like(k, -60), k)
    codes = torch.ldexp(x, -k).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, (k + 127).squeeze(-1).to(torch.uint8).view(torch.float8_e8m0fnu)


def _tree(r, n):
    """Parents (-1: the sequence's last token) of n drafted tokens, each after its parent."""
    parent = [-1]
    for i in range(1, n):
        parent.append(r.choice([i - 1, i - 1, r.randrange(i)]))
    return parent


def _layout(case, r, dev):
    """The pages of the sequences in a mixed order, and the integers of the step."""
    old, new = _lengths(case)
    pages = [max(1, -(-(a + b) // PAGE)) for a, b in zip(old, new)]
    order = list(range(sum(pages)))
    r.shuffle(order)
    table = torch.full((len(old), max(pages)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    start = [0]
    for b in new:
        start.append(start[-1] + b)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    return {"old": old, "new": new, "table": table.to(dev), "pages": sum(pages), "start": ints(start), "pos0": ints(old)}


def prepare(case, seed):
    dev, op = "cuda", case["op"]
    r, g = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
    kv, d = case["kv_heads"], case["d"]
    s = dict(case, **_layout(case, r, dev))
    f8 = case.get("store", "f8") == "f8"
    randn = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731

    def stored(*lead):
        """Keys or values as a model leaves them: rows of unequal size, some channels larger than others."""
        x = randn(*lead, kv, PAGE, d) * torch.exp(0.5 * randn(*lead, kv, PAGE, 1)) * (1 + 2 * (randn(d) > 1.5))
        return _quantise(x) if f8 else (x.to(torch.bfloat16), None)

    n = sum(s["new"])
    if op in ("attend", "read"):
        s["keys"], s["key_scales"] = stored(s["pages"])
        s["values"], s["value_scales"] = stored(s["pages"])
    if op == "read":
        P = s["table"].shape[1]
        s["ends"] = s["pos0"]
        s["read_keys"], s["read_values"] = (torch.zeros(case["seqs"], P, kv, PAGE, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    if op == "attend":
        h = case["heads"]
        s["q"] = (randn(n, h * d) * 1.2).to(torch.bfloat16)
        s["out"] = torch.zeros(n, h * d, dtype=torch.bfloat16, device=dev)
        masks = []
        for b in s["new"]:
            parent, seen = _tree(r, b), []
            for i, p in enumerate(parent):
                seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            masks += [m - (1 << 64) if m >> 63 else m for m in seen]
        s["tree"] = torch.tensor(masks, dtype=torch.int64, device=dev).view(n, 1) if case["tokens"] > 1 else None
    if op == "append":
        h, longest = case["heads"], max(a + b for a, b in zip(s["old"], s["new"]))
        s["qkv"] = (randn(n, (h + 2 * kv) * d) * (0.5 + randn(1, (h + 2 * kv) * d).abs())).to(torch.bfloat16)
        s["q_norm"], s["k_norm"] = 1 + 0.1 * randn(d), 1 + 0.1 * randn(d)
        angle = torch.arange(longest, device=dev).double()[:, None] * 1e6 ** (-torch.arange(d // 2, device=dev).double() / (d // 2))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        seqs, pos, place = [], [], []
        for i, (a, b) in enumerate(zip(s["old"], s["new"])):
            depth = list(range(b))
            if 1 < b <= PAGE:                              # drafted tokens stand at their depth in the tree
                for j, p in enumerate(_tree(r, b)):
                    depth[j] = depth[p] + 1 if p >= 0 else 0
            seqs += [i] * b
            pos += [a + x for x in depth]
            place += range(a, a + b)
        s["seq"], s["pos"], s["place"] = (torch.tensor(v, dtype=torch.int32, device=dev) for v in (seqs, pos, place))
        s["q"] = torch.zeros(n, h * d, dtype=torch.bfloat16, device=dev)
        pool = (s["pages"], kv, PAGE, d)
        s["keys"], s["values"] = (torch.zeros(pool, device=dev).to(torch.float8_e4m3fn if f8 else torch.bfloat16) for _ in range(2))
        s["key_scales"], s["value_scales"] = ((torch.full(pool[:3], 67, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu) if f8 else None)
                                              for _ in range(2))
    if op == "keep":
        s["store"], s["scales"] = stored(case["layers"], 2, s["pages"])
        paths = []
        for b in s["new"]:
            paths.append(sorted(r.sample(range(b), _path_length(b))))
        most = max(map(len, paths))
        s["path"] = torch.tensor([p + [-1] * (most - len(p)) for p in paths], dtype=torch.int32, device=dev)
    if own:
        from qwen3_b200.csrc import ops
        if op == "keep":
            return s
        s["cache"] = ops.CachePages(s["keys"], s["values"], s["key_scales"], s["value_scales"])
        if op == "attend":
            sizes = ops.attention_tree_scratch(case["seqs"], max(s["new"]), case["heads"], kv, d, dev)
            s["parts"] = torch.empty(sizes.parts, dtype=torch.float32, device=dev)
            s["counters"] = torch.zeros(sizes.counters, dtype=torch.int32, device=dev)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


def _own_append(s):
    from qwen3_b200.csrc import ops
    ops.cache_append(s["qkv"], s["q"], s["cache"], s["q_norm"], s["k_norm"], s["cos"], s["sin"], 1e-6, s["seq"], s["pos"],
                     s["place"], s["table"], s["heads"], norm_once=True)
    return _appended(s)


def _appended(s):
    return [s["q"], s["keys"], s["values"]] + ([s["key_scales"], s["value_scales"]] if s["key_scales"] is not None else [])


def _own_read(s):
    from qwen3_b200.csrc import ops
    ops.cache_read(s["cache"], s["table"], s["ends"], s["read_keys"], s["read_values"])
    return [s["read_keys"], s["read_values"]]


def _own_attend(s):
    from qwen3_b200.csrc import ops
    return ops.attention_tree(s["q"], s["cache"], s["out"], s["parts"], s["counters"], s["start"], s["pos0"], s["table"],
                              max(s["new"]), s["heads"], s["d"] ** -0.5, tree=s["tree"])


def _own_keep(s):
    from qwen3_b200.csrc import ops
    ops.cache_keep(s["store"], s["scales"], s["table"], s["pos0"], s["path"])
    return [s["store"]] + ([s["scales"]] if s["scales"] is not None else [])


def _normed_rotated(x, weight, cos, sin):
    """x [n, heads, d] in 32 bits: every head normed, then its halves rotated by the token's angles [n, 1, d / 2]."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_append(s):
    h, kv, d = s["heads"], s["kv_heads"], s["d"]
    x = s["qkv"].float().view(-1, h + 2 * kv, d)
    pos, place = s["pos"].long(), s["place"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    s["q"].copy_(_normed_rotated(x[:, :h], s["q_norm"], cos, sin).reshape(-1, h * d))
    page, at = s["table"][s["seq"].long(), place // PAGE].long(), place % PAGE
    for rows, to, scales in ((_normed_rotated(x[:, h:h + kv], s["k_norm"], cos, sin), s["keys"], s["key_scales"]),
                             (x[:, h + kv:], s["values"], s["value_scales"])):
        if scales is None:
            to[page, :, at] = rows.to(to.dtype)
        else:
            codes, scale = _quantise(rows)
            to.view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
            scales.view(torch.uint8)[page, :, at] = scale.view(torch.uint8)
    return _appended(s)


def _rows(pages, scales, page_list, n):
    """The first n rows of a sequence, [kv_heads, n, d] in 32 bits."""
    if scales is None:
        x = pages[page_list].float()
    else:                                                  # codes are gathered as bytes
        x, e = (y.view(torch.uint8)[page_list].view(y.dtype).float() for y in (pages, scales))
        x = x * e[..., None]
    return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[-1])[:, :n]


def _plain_read(s):
    for i, n in enumerate(s["old"]):
        P = -(-n // PAGE)
        for pages, scales, to in ((s["keys"], s["key_scales"], s["read_keys"]), (s["values"], s["value_scales"], s["read_values"])):
            x = _rows(pages, scales, s["table"][i, :P].long(), n)
            x = torch.nn.functional.pad(x, (0, 0, 0, P * PAGE - n)).view(s["kv_heads"], P, PAGE, s["d"])
            to[i, :P] = x.transpose(0, 1).to(to.dtype)
    return [s["read_keys"], s["read_values"]]


def _seen(s, first, a, b):
    """[b, a + b]: which keys the new tokens of a sequence see."""
    seen = torch.ones(b, a + b, dtype=torch.bool, device=s["q"].device)
    if s["tree"] is not None:
        seen[:, a:] = (s["tree"][first:first + b] >> torch.arange(b, device=s["q"].device)) & 1 != 0
    return seen


def _plain_attend(s):
    h, kv, d, first = s["heads"], s["kv_heads"], s["d"], 0
    for i, (a, b) in enumerate(zip(s["old"], s["new"])):
        listed_pages = s["table"][i, :-(-(a + b) // PAGE)].long()
        k = _rows(s["keys"], s["key_scales"], listed_pages, a + b)
        v = _rows(s["values"], s["value_scales"], listed_pages, a + b)
        q = s["q"][first:first + b].float().view(b, kv, h // kv, d).permute(1, 2, 0, 3).reshape(kv, -1, d)
        score = (q @ k.transpose(1, 2)).view(kv, h // kv, b, a + b) * d ** -0.5
        score = score.masked_fill(~_seen(s, first, a, b), -math.inf)
        e = torch.exp(score - score.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
        x = p.view(kv, -1, a + b) @ v
        s["out"][first:first + b] = x.view(kv, h // kv, b, d).permute(2, 0, 1, 3).reshape(b, h * d).to(s["out"].dtype)
        first += b
    return s["out"]


def _plain_keep(s):
    path = s["path"].long()
    seq, to = torch.nonzero(path >= 0, as_tuple=True)
    came, goes = s["pos0"].long()[seq] + path[seq, to], s["pos0"].long()[seq] + to
    came_page, goes_page = s["table"][seq, came // PAGE].long(), s["table"][seq, goes // PAGE].long()
    for x in [s["store"]] + ([s["scales"]] if s["scales"] is not None else []):
        raw = x.view(torch.uint8) if x.dtype != torch.bfloat16 else x
        raw[:, :, goes_page, :, goes % PAGE] = raw[:, :, came_page, :, came % PAGE]
    return [s["store"]] + ([s["scales"]] if s["scales"] is not None else [])


_run_own = {"append": _own_append, "read": _own_read, "attend": _own_attend, "keep": _own_keep}
_run_plain = {"append": _plain_append, "read": _plain_read, "attend": _plain_attend, "keep": _plain_keep}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    """Codes are given as the numbers that were rounded to them."""
    s = prepare(case, seed)
    if case["op"] == "keep":
        return None                                        # bytes that move: nothing is computed
    kv, d = case["kv_heads"], case["d"]
    if case["op"] == "append":
        h = case["heads"]
        x = s["qkv"].double().view(-1, h + 2 * kv, d)
        half, pos = d // 2, s["pos"].long()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[pos].unsqueeze(1)

        def turned(y, w):
            y = y / (y.square().sum(-1, keepdim=True) / d + 1e-6).sqrt() * w.double()
            z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        out = [turned(x[:, :h], s["q_norm"]).flatten(1)]
        scales = []
        flat = s["table"].long()[s["seq"].long(), s["place"].long() // PAGE] * PAGE + s["place"].long() % PAGE
        for y in (turned(x[:, h:h + kv], s["k_norm"]), x[:, h + kv:]):
            pool = torch.zeros(s["pages"], kv, PAGE, d, dtype=torch.float64, device="cuda")
            scale = torch.full(pool.shape[:3], 2.0 ** -60, dtype=torch.float64, device="cuda")
            # (a largest value of 448 times a power of two fits, whatever the logarithm's last bit says)
            k = torch.ceil(torch.log2(y.abs().amax(-1) / 448) - 1e-12).clamp(-60, 60) if case["store"] == "f8" else torch.zeros(y.shape[:2], device="cuda")
            one = torch.exp2(k.double())
            for n in range(kv):                            # the rows of a head, by page and place
                rows = torch.zeros(s["pages"] * PAGE, d, dtype=torch.float64, device="cuda")
                rows[flat] = y[:, n] / one[:, n, None]
                pool[:, n] = rows.view(-1, PAGE, d)
                scale[:, n] = scale[:, n].reshape(-1).scatter(0, flat, one[:, n]).view(-1, PAGE)
            out.append(pool)
            scales.append(scale)
        return out + (scales if case["store"] == "f8" else [])
    wide = [x.double() if e is None else x.double() * torch.exp2(e.view(torch.uint8).double() - 127)[..., None]
            for x, e in ((s["keys"], s["key_scales"]), (s["values"], s["value_scales"]))]
    if case["op"] == "read":
        out = []
        for x in wide:
            y = torch.zeros(s["read_keys"].shape, dtype=torch.float64, device="cuda")
            for i, n in enumerate(s["old"]):
                for p in range(-(-n // PAGE)):
                    live = min(PAGE, n - p * PAGE)
                    y[i, p, :, :live] = x[int(s["table"][i, p]), :, :live]
            out.append(y)
        return out
    h, first, out = case["heads"], 0, []
    group = h // kv
    for i, (a, b) in enumerate(zip(s["old"], s["new"])):
        k, v = (torch.cat([x[int(p)] for p in s["table"][i, :-(-(a + b) // PAGE)]], dim=1)[:, :a + b] for x in wide)
        q = s["q"][first:first + b].double().view(b, kv, group, d)
        logit = torch.einsum("tngd,nkd->ngtk", q, k) / math.sqrt(d)
        for t in range(b):
            if s["tree"] is not None:
                bits = int(s["tree"][first + t, 0]) & (1 << 64) - 1
                hidden = [a + j for j in range(b) if not bits >> j & 1]
                logit[:, :, t, hidden] = -math.inf
        out.append(torch.einsum("ngtk,nkd->tngd", torch.softmax(logit, -1), v).reshape(b, h * d))
        first += b
    return torch.cat(out)
