"""The operators of a model whose projections are 8-bit integers with scales, and the work they do.

An engine with such weights runs, layer by layer of a step, these four:

  norm      adds a sublayer's output to the hidden state, norms the sum and hands it on as 8-bit codes with a scale a token;
  product   codes of tokens times codes of a matrix, summed in whole numbers, scaled by token and by channel: the
            projections of the attention and the second one of the feed-forward;
  gated     the same for the gate and up projections, with the activation and the gating: rows of both in turns of eight;
  quantise  rows as codes with a scale each: the attention's output, the gated activations, and the weights at load.

A row's scale is its largest magnitude over 127; a code is 127 times the value over that magnitude, rounded to the nearest, ties to
even.  Rows of codes begin 16 bytes apart or a multiple, whatever their length.

A case names its operator and its sizes.  Sizes are those of this repository's models and benchmark (hidden sizes of 4096 and
5120, feed-forwards of 12288, 17408 and 25600); drawn ones are of any width.  All inputs hang on the seed.
"""
import math

import torch

own = False


def listed():
    return [
        # the attention's output of one chat's decode step: latency alone
        _rows("quantise_1", "quantise", 1, 4096, "bf16"),
        # gated activations of a long prompt
        _rows("quantise_prompt", "quantise", 8000, 12288, "bf16"),
        # a matrix of a checkpoint that is stored in 32 bits, at load: a row is an output channel
        _rows("quantise_weights", "quantise", 10240, 5120, "f32"),
        # the norms of a decode step of 8 sequences
        _rows("norm_8", "norm", 8, 4096, "bf16"),
        # those of a prompt
        _rows("norm_prompt", "norm", 8000, 5120, "bf16"),
        # some short prompts of a 32-bit engine
        _rows("norm_527", "norm", 527, 4096, "f32"),
        # the output projection of one chat's decode step
        _product("product_1", "product", 1, 4096, 4096, "bf16"),
        # the feed-forward's second projection, decode of 8 sequences
        _product("product_8", "product", 8, 4096, 12288, "bf16"),
        # q, k and v of a busy server's decode step
        _product("product_64", "product", 64, 6144, 4096, "bf16"),
        # some short prompts
        _product("product_527", "product", 527, 5120, 17408, "bf16"),
        # gate and up of the benchmark's decode step
        _product("gated_8", "gated", 8, 24576, 4096, "bf16"),
        # of a long prompt: the largest product of a layer
        _product("gated_prompt", "gated", 8000, 24576, 4096, "bf16"),
    ]


def _rows(name, op, rows, width, dtype):
    return {"name": name, "op": op, "rows": rows, "width": width, "dtype": dtype}


def _product(name, op, rows, channels, width, out):
    return {"name": name, "op": op, "rows": rows, "channels": channels, "width": width, "out": out}


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    limit = [max(work(c)[what] for c in listed()) for what in ("bytes", "flops")]
    while True:
        op = rng.choice(["quantise", "norm", "product", "product", "gated"])
        if op in ("quantise", "norm"):
            case = _rows("", op, log(1, 8000), log(64, 25600), rng.choice(["bf16", "bf16", "f32"]))
        else:
            channels = 16 * log(4, 1600) if op == "gated" else log(64, 25600)
            case = _product("", op, log(1, 8000), channels, log(64, 25600), "bf16" if op == "gated" else rng.choice(["bf16", "bf16", "f32"]))
        del case["name"]
        cost = work(case)
        if cost["bytes"] <= limit[0] and cost["flops"] <= limit[1]:
            return case


def work(case):
    m, k = case["rows"], case["width"]
    if case["op"] in ("quantise", "norm"):
        size = 2 if case["dtype"] == "bf16" else 4
        if case["op"] == "norm":
            return {"bytes": m * (k * (3 * size + 1) + 4) + 4 * k, "flops": 8 * m * k}
        return {"bytes": m * (k * (size + 1) + 4), "flops": 4 * m * k}
    n = case["channels"]
    written = m * (n // 2 if case["op"] == "gated" else n) * (2 if case["out"] == "bf16" else 4)
    return {"bytes": (m + n) * (k + 4) + written, "flops": 2 * m * n * k}


# ------------------------------------------------------------------ inputs
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _padded(rows, width):
    """Room for codes [rows, width] whose rows begin at multiples of 16 bytes."""
    return torch.zeros(rows, -(-width // 16) * 16, dtype=torch.int8, device="cuda")[:, :width]


def _quantised(u):
    """Codes and scales of rows in 32 bits; the ratios in 64, in which what lies between two codes is told from what lies beside."""
    top = u.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top)
    codes = (127 * u.double() / top.double()).round()
    codes = torch.where(fine & (top > 0), codes, torch.zeros_like(codes)).to(torch.int8)
    return codes, torch.where(fine, top / 127, torch.full_like(top, math.nan)).squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    m, k = case["rows"], case["width"]

    def activations():
        """Tokens of unequal size, some channels larger than others."""
        return randn(m, k).mul_(torch.exp(0.5 * randn(m, 1)) * (1 + 6 * (randn(k) > 2)))

    def codes_of(x):
        codes = _padded(*x.shape)
        values, scales = _quantised(x)
        codes.copy_(values)
        return codes, scales

    s = dict(case)
    if case["op"] in ("quantise", "norm"):
        dtype = _TYPES[case["dtype"]]
        s["x"] = activations().to(dtype)
        s["codes"], s["scales"] = _padded(m, k), torch.zeros(m, device="cuda")
        if case["op"] == "norm":
            s["delta"] = (0.3 * randn(m, k)).to(dtype)
            s["total"] = torch.zeros_like(s["x"])
            s["weight"] = 1 + 0.1 * randn(k)
    else:
        s["x"], s["x_scales"] = codes_of(activations())
        s["w"], s["w_scales"] = codes_of(0.02 * randn(case["channels"], k))
        s["y"] = torch.zeros(m, case["channels"] // (2 if case["op"] == "gated" else 1), dtype=_TYPES[case["out"]], device="cuda")
    if own:
        from qwen3_b200.csrc import ops
        if case["op"] in ("quantise", "norm"):
            s["out"] = ops.Int8Rows(s["codes"], s["scales"])
        else:
            s["x8"], s["w8"] = ops.Int8Rows(s["x"], s["x_scales"]), ops.Int8Rows(s["w"], s["w_scales"])
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


def _own_quantise(s):
    from qwen3_b200.csrc import ops
    ops.quantize_rows(s["x"], s["out"])
    return [s["codes"], s["scales"]]


def _own_norm(s):
    from qwen3_b200.csrc import ops
    ops.rms_norm_int8(s["x"], s["weight"], 1e-6, s["out"], delta=s["delta"], total=s["total"])
    return [s["total"], s["codes"], s["scales"]]


def _own_product(s):
    from qwen3_b200.csrc import ops
    return ops.gemm_int8(s["x8"], s["w8"], s["y"])


def _own_gated(s):
    from qwen3_b200.csrc import ops
    return ops.gemm_int8(s["x8"], s["w8"], s["y"], activation="silu")


def _plain_quantise(s):
    codes, scales = _quantised(s["x"].float())
    s["codes"].copy_(codes)
    s["scales"].copy_(scales)
    return [s["codes"], s["scales"]]


def _plain_norm(s):
    s["total"].copy_(s["x"].float() + s["delta"].float())
    t = s["total"].float()
    inv = torch.rsqrt((t * t).mean(-1) + 1e-6)
    codes, scales = _quantised(t * s["weight"])            # the root is the same for a whole row: codes do not need it
    s["codes"].copy_(codes)
    s["scales"].copy_(scales * inv)
    return [s["total"], s["codes"], s["scales"]]


def _scaled_product(s):
    """Sums of these inputs' products stay far below 2^24, where 32 bits hold every whole number."""
    return s["x"].float() @ s["w"].float().t() * s["x_scales"][:, None] * s["w_scales"]


def _plain_product(s):
    return s["y"].copy_(_scaled_product(s))


def _plain_gated(s):
    m = s["rows"]
    pairs = _scaled_product(s).view(m, -1, 2, 8)
    gate, up = pairs[:, :, 0], pairs[:, :, 1]
    return s["y"].copy_((gate / (1 + torch.exp(-gate)) * up).reshape(m, -1))


_run_own = {"quantise": _own_quantise, "norm": _own_norm, "product": _own_product, "gated": _own_gated}
_run_plain = {"quantise": _plain_quantise, "norm": _plain_norm, "product": _plain_product, "gated": _plain_gated}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    """Codes have no value in 64 bits: they are whole numbers."""
    s = prepare(case, seed)
    if case["op"] in ("quantise", "norm"):
        x = s["x"].double()
        if case["op"] == "quantise":
            return [None, x.abs().max(dim=1).values / 127]
        total = x + s["delta"].double()
        stored = total.to(s["x"].dtype).double()           # the norm reads the sum as it is stored
        normed = stored / (stored.square().sum(1, keepdim=True) / case["width"] + 1e-6).sqrt() * s["weight"].double()
        return [total, None, normed.abs().max(dim=1).values / 127]
    sums = torch.zeros(case["rows"], case["channels"], dtype=torch.float64, device="cuda")
    for at in range(0, case["width"], 512):                # 512 products of codes are exact in 32 bits
        sums += s["x"][:, at:at + 512].float() @ s["w"][:, at:at + 512].float().t()
    y = sums.mul_(s["x_scales"].double()[:, None]).mul_(s["w_scales"].double())
    if case["op"] == "product":
        return y
    at = torch.arange(case["channels"], device="cuda").view(-1, 16)
    gate, up = y[:, at[:, :8].reshape(-1)], y[:, at[:, 8:].reshape(-1)]
    return gate * torch.sigmoid(gate) * up
