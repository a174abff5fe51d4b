"""A cache in 8 bits and steps with drafted tokens: the definitions in 64 bits, and inputs for them."""
import math
import random

import torch

PAGE = 64


def scale_of(top):
    """The exponent of the smallest power of two by which rows whose largest values are `top` (float64) fit into 448."""
    m, e = torch.frexp(top)                                  # 448 = 7/8 * 2^9
    k = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(top == 0, torch.full_like(k, -60), k).clamp(-60, 60)


def quantised(x):
    """Rows [..., d] (any float type) as codes and scales."""
    x = x.double()
    fine = torch.isfinite(x)
    k = scale_of(torch.where(fine, x.abs(), torch.zeros_like(x)).amax(-1))
    y = torch.where(fine, torch.ldexp(x, -k[..., None]).clamp(-448, 448), torch.full_like(x, math.nan))
    return y.float().to(torch.float8_e4m3fn), (k + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def values_of(codes, scales):
    """What pages stand for, in 64 bits."""
    if scales is None:
        return codes.double()
    return codes.float().double() * torch.exp2(scales.view(torch.uint8).double() - 127)[..., None]


def pages_for(lengths, seed, spare=2):
    """A page table [sequences, most pages] in a mixed order (-1 behind a sequence's last), and the number of pages."""
    r, need = random.Random(seed), [-(-n // PAGE) for n in lengths]
    order = list(range(sum(need) + spare))
    r.shuffle(order)
    table, at = torch.full((len(lengths), max(max(need), 1)), -1, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, sum(need) + spare


def rows_of(pages, table_row, n):
    """The first n rows of a sequence, [n, kv heads, d]."""
    return pages[table_row[:-(-n // PAGE)].long()].transpose(1, 2).reshape(-1, pages.shape[1], pages.shape[-1])[:n]


def masks_for(kind, new, words, seed):
    """int64 [tokens, words]: 'tree' ancestors and oneself, 'bits' at random (some rows empty), 'none' all rows empty."""
    r, rows = random.Random(seed), []
    for b in new:
        seen = []
        for i in range(b):
            if kind == "tree":
                parent = r.choice([i - 1, r.randrange(i)]) if i else -1
                seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
            else:
                seen.append(0 if kind == "none" or r.random() < 0.2 else r.getrandbits(b))
        rows += seen
    signed = lambda w: w - (1 << 64) if w >> 63 else w  # noqa: E731
    return torch.tensor([[signed(m >> 64 * w & (1 << 64) - 1) for w in range(words)] for m in rows], dtype=torch.int64)


def attention(q, keys, values, table, old, new, heads, scale, tree):
    """(out, sum of p |v|) [tokens, heads, d] in 64 bits; keys, values: what the pages stand for."""
    d, kv, at, outs, sizes = keys.shape[-1], keys.shape[1], 0, [], []
    for i, (a, b) in enumerate(zip(old, new)):
        k, v = rows_of(keys, table[i], a + b), rows_of(values, table[i], a + b)
        x = q[at:at + b].double().view(b, kv, heads // kv, d)
        seen = torch.zeros(b, a + b, dtype=torch.bool)
        seen[:, :a] = True
        for t in range(b):
            for n in range(b):
                seen[t, a + n] = n <= t if tree is None else bool(int(tree[at + t, n // 64]) >> n % 64 & 1)
        seen = seen.to(q.device)
        out, size = torch.zeros(b, heads, d, dtype=torch.float64, device=q.device), torch.zeros(b, heads, d, dtype=torch.float64, device=q.device)
        for t in range(b):
            at_t = seen[t]
            if at_t.any():
                p = torch.softmax(torch.einsum("ghd,ngd->ghn", x[t], k[at_t]) * scale, -1)
                out[t] = torch.einsum("ghn,ngd->ghd", p, v[at_t]).reshape(heads, d)
                size[t] = torch.einsum("ghn,ngd->ghd", p, v[at_t].abs()).reshape(heads, d)
        outs.append(out)
        sizes.append(size)
        at += b
    return torch.cat(outs), torch.cat(sizes)
