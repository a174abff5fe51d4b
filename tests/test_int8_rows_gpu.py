"""Rows as 8-bit integers with a scale each, quantised and normed, against the definition in 64 bits."""
import math

import pytest
import torch

import int8_cases as ic

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
WIDTHS = [1, 2, 7, 8, 16, 24, 63, 100, 127, 256, 1000, 1024, 1025, 2056, 4096, 5001, 9000, 25600, 33000, 70001]


def rows_for(rows, width, extra=0):
    """Int8Rows whose memory is full of a code of its own, beyond the rows too; the whole of that memory."""
    from qwen3_b200.csrc import ops
    memory = ic.padded(rows, width, extra=extra)
    return ops.Int8Rows(memory[:, :width], torch.full((rows,), 77.0, device="cuda")), memory


def special(x, g):
    """Rows of every kind that a scale can go wrong with, as far as there are rows."""
    rows, width = x.shape
    top = x.float().abs().amax(-1)
    for i in range(rows):
        kind = i % 12
        if kind == 1:
            x[i] = 0
        elif kind == 2:
            x[i, width // 2] = math.nan
        elif kind == 3:
            x[i, width - 1] = -math.inf
        elif kind == 4:                                    # halves of the largest value: ties at 63.5
            x[i] = top[i] * torch.randint(-2, 3, (width,), generator=g, device="cuda") / 2
        elif kind == 5:
            x[i] = x[i].float() * 1e-39
        elif kind == 6:
            x[i] = (x[i].float() / top[i].clamp(min=1e-30) * 3.3e38).to(x.dtype)
        elif kind == 7:                                    # every value a tie where the largest is 254 units
            x[i] = torch.randint(-127, 128, (width,), generator=g, device="cuda") * 2 - 1
            x[i, 0] = 254
        elif kind == 8:
            x[i] = -x[i].float().abs() * 1e30
    return x


def same_rows(got, memory, u, scale_bound):
    """Codes equal, scales within a relative bound, and nothing written beyond the rows."""
    codes, scales = ic.quantised(u)
    assert torch.equal(got.codes.long(), codes)
    nan = scales.isnan()
    assert torch.equal(got.scales.isnan(), nan)
    assert bool(((got.scales.double() - scales).abs() <= scale_bound * scales.abs() + 2.0 ** -149)[~nan].all())
    assert bool((memory[:, u.shape[1]:] == 77).all())


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 13, 700])
@pytest.mark.parametrize("width", WIDTHS)
def test_quantize(kind, rows, width):
    from qwen3_b200.csrc import ops
    if rows * width > 1 << 25:
        rows = 13
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    x = torch.randn(rows, width, generator=g, device="cuda") * torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))
    x = special(x.to(TYPES[kind]), g)
    out, memory = rows_for(rows, width)
    ops.quantize_rows(x, out)
    same_rows(out, memory, x.double(), 2.0 ** -24)        # one division, half a unit


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("width,first,row", [(64, 0, 72), (64, 1, 70), (100, 8, 133), (4096, 0, 6144), (4096, 3, 4101), (33000, 2, 33002)])
def test_quantize_rows_apart(kind, width, first, row):
    from qwen3_b200.csrc import ops
    g = torch.Generator(device="cuda").manual_seed(width + first)
    for rows in (1, 5, 400):
        x = torch.randn(rows, row, generator=g, device="cuda").to(TYPES[kind])[:, first:first + width]
        out, memory = rows_for(rows, width, extra=32)
        ops.quantize_rows(x, out)
        same_rows(out, memory, x.double(), 2.0 ** -24)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("delta,apart", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("rows", [1, 13, 700])
@pytest.mark.parametrize("width", WIDTHS)
def test_norm(kind, delta, apart, rows, width):
    """Scales: a sum of at most 110 roundings in a row (each half a unit, and half of that in the root), then a root, a product and a division."""
    from qwen3_b200.csrc import ops
    if rows * width > 1 << 24:
        rows = 13
    dtype, g = TYPES[kind], torch.Generator(device="cuda").manual_seed(rows + width + delta)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    x = (randn(rows, width) * torch.exp(randn(rows, 1))).to(dtype)
    for i in range(rows):
        if i % 8 == 1:
            x[i] = 0
        elif i % 8 == 2:
            x[i, width // 2] = math.nan
        elif i % 8 == 3:
            x[i, 0] = math.inf
        elif i % 8 == 4:
            x[i] = x[i].float() * 1e-12
        elif i % 8 == 5:
            x[i] = 1e25                                   # squares beyond 32 bits
    w = 1 + 0.3 * randn(width)
    d = (0.5 * randn(rows, width)).to(dtype) if delta else None
    stored = (x.float() + d.float()).to(dtype) if delta else x.clone()
    before = x.clone()
    total = torch.full_like(x, 77.0) if apart else None
    out, memory = rows_for(rows, width)
    ops.rms_norm_int8(x, w, 1e-6, out, delta=d, total=total)
    got = total if apart else x
    assert torch.equal(got.nan_to_num(nan=-5.0), stored.nan_to_num(nan=-5.0))
    if apart:
        assert torch.equal(x.nan_to_num(nan=-5.0), before.nan_to_num(nan=-5.0))
    u = ic.normed(stored, w)
    squares = stored.double().square()
    beyond = ~(squares.sum(-1) < 3.4e38)
    u[beyond] = math.nan
    codes, tops = ic.quantised(u)
    assert torch.equal(out.codes.long(), codes)
    scales = tops / (squares.mean(-1) + 1e-6).sqrt()
    assert torch.equal(out.scales.isnan(), scales.isnan())
    fine = ~scales.isnan()
    assert bool(((out.scales.double() - scales).abs() <= 2.0 ** -18 * scales + 2.0 ** -140)[fine].all())
    assert bool((memory[:, width:] == 77).all())


def test_norm_rows_apart_and_no_rows():
    from qwen3_b200.csrc import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(40, 300, generator=g, device="cuda").to(torch.bfloat16)
    x, d, t = wide[:, 3:131], wide[:, 140:268], torch.zeros(40, 200, dtype=torch.bfloat16, device="cuda")
    w = torch.rand(129, generator=g, device="cuda")[1:]
    out, _ = rows_for(40, 128)
    ops.rms_norm_int8(x, w, 1e-5, out, delta=d, total=t[:, 72:])
    stored = (x.float() + d.float()).to(torch.bfloat16)
    assert torch.equal(t[:, 72:], stored) and not bool(t[:, :72].any())
    assert torch.equal(out.codes.long(), ic.quantised(ic.normed(stored, w))[0])
    none, _ = rows_for(0, 128)
    ops.rms_norm_int8(x[:0], w, 1e-5, none, delta=d[:0])
    ops.quantize_rows(x[:0], none)


def test_values_of_rows():
    from qwen3_b200.csrc import ops
    x = torch.randn(5, 77, generator=torch.Generator().manual_seed(1)).cuda()
    out = ops.quantize_rows(x, ops.Int8Rows.empty(5, 77, "cuda"))
    assert out.shape == (5, 77) and bool(((out.float() - x).abs() <= 0.5001 * out.scales[:, None]).all())


def test_refusals():
    from qwen3_b200.csrc import ops
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(64, device="cuda")
    out = ops.Int8Rows.empty(4, 64, "cuda")
    scales = torch.zeros(4, device="cuda")
    memory = torch.zeros(4, 80, dtype=torch.int8, device="cuda")
    for codes, s in ((memory[:, :64].to(torch.uint8), scales), (memory[:, :64], scales[:3]), (memory[:, 1:65], scales), (memory[:, :64].double(), scales),
                     (torch.zeros(4, 72, dtype=torch.int8, device="cuda")[:, :64], scales), (memory[:, :64], scales.double()),
                     (memory.t()[:4, :4], scales), (memory[:, ::2], scales), (memory[:, :64].cpu(), scales.cpu()),
                     (torch.zeros(4, dtype=torch.int8, device="cuda"), scales),
                     (torch.zeros(4 * 64 - 3, dtype=torch.int8, device="cuda").as_strided((4, 61), (64, 1)), scales)):
        with pytest.raises(ops.KernelError):
            ops.Int8Rows(codes, s)
    for bad in (x[:3], x[:, :60], x.to(torch.float16), x.cpu(), x.t().contiguous().t(), x[:1].expand(4, 64)):
        with pytest.raises(ops.KernelError):
            ops.quantize_rows(bad, out)
        with pytest.raises(ops.KernelError):
            ops.rms_norm_int8(bad, w, 1e-6, out)
    for more in ({"delta": x[:3]}, {"delta": x.float()}, {"total": x}, {"delta": x, "total": x.float()}, {"delta": x, "total": x[:, :32]}):
        with pytest.raises(ops.KernelError):
            ops.rms_norm_int8(x, w, 1e-6, out, **more)
    for weight in (w[:60], w.double(), w.cpu(), torch.zeros(128, device="cuda")[::2]):
        with pytest.raises(ops.KernelError):
            ops.rms_norm_int8(x, weight, 1e-6, out)


def test_every_pair_of_bfloat16_magnitudes():
    """Every largest magnitude of a binade beside every value of the eleven binades below it: ties, and what lies closest to them."""
    from qwen3_b200.csrc import ops
    tops = torch.arange(128, 256, device="cuda").double()
    values = torch.cat([tops * 2.0 ** -e for e in range(11)])
    for scale in (1.0, 2.0 ** -90, 2.0 ** 100):
        x = torch.cat([tops[:, None], torch.where(values[None] <= tops[:, None], values[None], torch.zeros((), device="cuda").double())], dim=1) * scale
        x = torch.cat([x, -x], dim=1).to(torch.bfloat16)
        out, memory = rows_for(*x.shape)
        ops.quantize_rows(x, out)
        same_rows(out, memory, x.double(), 2.0 ** -24)


@pytest.mark.parametrize("width", [8192, 8191])
def test_offsets_beyond_32_bits(width):
    """2.2 billion values: the last rows as by themselves."""
    from qwen3_b200.csrc import ops
    rows = 270000
    x = torch.randn(1000, width, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(torch.bfloat16).repeat(rows // 1000, 1)
    w, out = torch.rand(width, device="cuda") + 0.5, ops.Int8Rows.empty(rows, width, "cuda")
    ops.quantize_rows(x, out)
    codes, scales = ic.quantised(x[:1000])
    for first in (0, 135000, 269000):
        assert torch.equal(out.codes[first:first + 1000].long(), codes)
    ops.rms_norm_int8(x, w, 1e-6, out, delta=x, total=x)
    stored = (2 * x[:1000].float() / 2).to(torch.bfloat16)           # (x was doubled, which rounds nothing)
    codes = ic.quantised(ic.normed(stored, w))[0]
    for first in (0, 135000, 269000):
        assert torch.equal(x[first:first + 1000], stored) and torch.equal(out.codes[first:first + 1000].long(), codes)
    del x, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,width", [(3, 64), (3, 65), (700, 65), (2, 40000)])
def test_rows_of_zeros_without_an_epsilon(rows, width):
    from qwen3_b200.csrc import ops
    x = torch.zeros(rows, width, device="cuda")
    x[0, 0] = 3.0
    out, _ = rows_for(rows, width)
    ops.rms_norm_int8(x, torch.ones(width, device="cuda"), 0.0, out)
    assert int(out.codes[0, 0]) == 127 and abs(float(out.scales[0]) * 127 / width ** 0.5 - 1) < 1e-6
    assert not bool(out.codes[1:].any()) and bool((out.scales[1:] == 0).all())
