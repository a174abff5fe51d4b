"""Products of 8-bit integers with scales against the definition in 64 bits."""
import pytest
import torch

import int8_cases as ic

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
U = 2.0 ** -24
HALF = {"f32": U, "bf16": 2.0 ** -8}                       # half a step of the output


def operands(M, N, K, seed):
    """Codes of the whole range, with other memory full of other codes behind every row."""
    from qwen3_b200.csrc import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for rows in (M, N):
        memory = torch.randint(-128, 128, (rows, -(-K // 16) * 16 + 16), generator=g, device="cuda", dtype=torch.int64).to(torch.int8)
        scales = torch.exp(0.3 * torch.randn(rows, generator=g, device="cuda")) / (74.0 * K ** 0.25)
        out.append(ops.Int8Rows(memory[:, :K], scales))
    return out


def check(x, w, y, kind, activation):
    """A sum of whole numbers has no error; it becomes 32 bits (half a unit) and is scaled twice (half a unit each); then the last rounding.  With a gate:
    both errors, some units of the activation and a product, all beside |gate| |up|."""
    want = ic.product(x.codes, x.scales, w.codes, w.scales, activation)
    got = y.double()
    if activation is None:
        assert bool(((got - want).abs() <= want.abs() * (3.01 * U + HALF[kind] * (1 + 4 * U)) + 2.0 ** -140).all())
    else:
        want, gate, up = want
        bound = 16 * U * gate.abs() * up.abs()
        assert bool(((got - want).abs() <= bound + (want.abs() + bound) * HALF[kind] + 2.0 ** -120).all())


SHAPES = [(1, 16, 64), (1, 64, 1), (2, 33, 15), (3, 100, 17), (7, 48, 100), (8, 4096, 4096), (8, 1000, 2050), (9, 160, 129), (16, 512, 1000), (17, 96, 640),
          (31, 2000, 333), (33, 48, 4100), (64, 6144, 512), (65, 80, 63), (100, 272, 127), (128, 1024, 2048), (129, 1040, 500), (200, 4096, 1024),
          (257, 272, 640), (300, 6144, 4096), (527, 1001, 777), (700, 512, 12288), (1024, 2048, 2048), (1500, 4096, 1008), (2100, 80, 96), (3001, 1072, 1500)]


@pytest.mark.parametrize("kind,activation", [("bf16", None), ("f32", None), ("bf16", "silu"), ("f32", "silu"), ("bf16", "gelu_tanh")])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(M, N, K, kind, activation):
    from qwen3_b200.csrc import ops
    if activation:
        N = -(-N // 16) * 16
    x, w = operands(M, N, K, M + N + K)
    columns = N // 2 if activation else N
    memory = torch.full((M + 2, columns), 77.0, dtype=TYPES[kind], device="cuda")
    y = memory[1:1 + M] if columns * memory.element_size() % 16 == 0 else memory[:M]
    ops.gemm_int8(x, w, y, activation=activation)
    assert ops.tcgen05_status("cuda") == 0
    check(x, w, y, kind, activation)
    rest = memory[M + 1:] if y.data_ptr() != memory.data_ptr() else memory[M:]
    assert bool((rest == 77).all()) and (y.data_ptr() == memory.data_ptr() or bool((memory[0] == 77).all()))


@pytest.mark.parametrize("form,splits", [("few", 0), ("mid", 0), ("mid", 1), ("mid", 2), ("mid", 3), ("mid", 5), ("mid", 8), ("pair", 0)]
                         + [("pair", tile) for tile in (32, 64, 96, 128, 160, 192, 224, 256)])
@pytest.mark.parametrize("M,N,K", [(1, 272, 200), (31, 96, 1500), (130, 560, 1024), (417, 1056, 900)])
def test_forms(M, N, K, form, splits):
    """Whatever form takes a product: the same bits, written to rows that lie at whole words and beside them, and no others."""
    from qwen3_b200.csrc import ops
    x, w = operands(M, N, K, M)
    for kind, activation, columns in (("bf16", None, N), ("f32", None, N), ("bf16", "silu", N // 2), ("f32", "gelu_tanh", N // 2)):
        outs = []
        for first, use in ((0, form), (1, form), (0, "few")):
            memory = torch.full((M * columns + 9,), 77.0, dtype=TYPES[kind], device="cuda")
            y = memory[first:first + M * columns].view(M, columns)
            ops.gemm_int8(x, w, y, activation=activation, form=use, splits=splits if use == form else 0)
            assert bool((memory[:first] == 77).all()) and bool((memory[first + M * columns:] == 77).all())
            outs.append(y)
        assert ops.tcgen05_status("cuda") == 0
        check(x, w, outs[0], kind, activation)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("form", ["few", "mid", "pair"])
@pytest.mark.parametrize("M,N,K", [(40, 33, 100), (300, 1001, 300), (5, 7, 16)])
def test_forms_of_odd_channels(M, N, K, form):
    from qwen3_b200.csrc import ops
    x, w = operands(M, N, K, M)
    for kind in TYPES:
        y = ops.gemm_int8(x, w, torch.zeros(M, N, dtype=TYPES[kind], device="cuda"), form=form)
        check(x, w, y, kind, None)


@pytest.mark.parametrize("M", [1, 5, 40, 150, 300, 1200])
def test_a_token_does_not_hang_on_the_batch(M):
    """Every form gives the same bits."""
    from qwen3_b200.csrc import ops
    x, w = operands(M, 528, 1111, 5)
    for activation, columns in ((None, 528), ("silu", 264)):
        y = ops.gemm_int8(x, w, torch.zeros(M, columns, device="cuda"), activation=activation)
        for row in (0, M // 2, M - 1):
            one = ops.Int8Rows(x.codes[row:row + 1], x.scales[row:row + 1])
            assert torch.equal(ops.gemm_int8(one, w, torch.zeros(1, columns, device="cuda"), activation=activation)[0], y[row])


@pytest.mark.parametrize("M", [1, 20, 140, 600])
def test_largest_sums(M):
    """-128 times -128 over the widest rows: 2^31 - 2^14; and the sum of opposite signs."""
    from qwen3_b200.csrc import ops
    K = ops.INT8_MAX_WIDTH
    x, w = ops.Int8Rows.empty(M, K, "cuda"), ops.Int8Rows.empty(32, K, "cuda")
    x.codes.fill_(-128), w.codes.fill_(-128)
    w.codes[16:].fill_(127)
    x.scales.fill_(0.5), w.scales.fill_(2.0)
    y = ops.gemm_int8(x, w, torch.zeros(M, 32, device="cuda"))
    assert bool((y[:, :16].double() == float(torch.tensor(float(K * 16384), dtype=torch.float32))).all())
    assert bool((y[:, 16:].double() == float(torch.tensor(float(-K * 128 * 127), dtype=torch.float32))).all())


@pytest.mark.parametrize("M", [1, 3, 50, 200, 600])
def test_scales_that_are_no_numbers_and_zeros(M):
    from qwen3_b200.csrc import ops
    x, w = operands(M, 96, 200, 7)
    x.scales[M - 1], w.scales[5], w.scales[6] = float("nan"), float("nan"), 0.0
    y = ops.gemm_int8(x, w, torch.zeros(M, 96, dtype=torch.bfloat16, device="cuda"))
    assert bool(y[M - 1].isnan().all()) and bool(y[:, 5].isnan().all()) and bool((y[:M - 1, 6] == 0).all())
    assert not bool(y[:M - 1, :5].isnan().any())


def test_no_rows():
    from qwen3_b200.csrc import ops
    x, w = operands(4, 32, 64, 1)
    y = torch.full((4, 32), 77.0, device="cuda")
    ops.gemm_int8(ops.Int8Rows(x.codes[:0], x.scales[:0]), w, y[:0])
    ops.gemm_int8(x, ops.Int8Rows(w.codes[:0], w.scales[:0]), torch.zeros(4, 0, device="cuda"))
    assert bool((y == 77).all())


def test_on_another_stream_and_in_a_graph():
    from qwen3_b200.csrc import ops
    for M in (2, 100, 300, 900):
        x, w = operands(M, 272, 500, M)
        want = ops.gemm_int8(x, w, torch.zeros(M, 272, device="cuda"))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            y = ops.gemm_int8(x, w, torch.zeros(M, 272, device="cuda"))
        side.synchronize()
        assert torch.equal(y, want)
        graphs, outs = [], []
        for _ in range(2):
            graph, y = torch.cuda.CUDAGraph(), torch.zeros(M, 272, device="cuda")
            with torch.cuda.graph(graph):
                ops.gemm_int8(x, w, y)
            graphs.append(graph), outs.append(y)
        for _ in range(3):
            for graph in graphs:
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in outs) and ops.tcgen05_status("cuda") == 0


def test_refusals():
    from qwen3_b200.csrc import ops
    x, w = operands(4, 40, 64, 1)
    good = torch.zeros(4, 40, device="cuda")
    for out in (good[:3], good[:, :39], good.half(), good.cpu(), good.t().contiguous().t(), torch.zeros(4, 80, device="cuda")[:, ::2]):
        with pytest.raises(ops.KernelError):
            ops.gemm_int8(x, w, out)
    with pytest.raises(ops.KernelError):                   # gates and ups in turns of eight
        ops.gemm_int8(x, w, torch.zeros(4, 20, device="cuda"), activation="silu")
    wide = operands(4, 48, 64, 1)[1]
    for activation, out in (("relu", torch.zeros(4, 24, device="cuda")), ("silu", torch.zeros(4, 48, device="cuda"))):
        with pytest.raises(ops.KernelError):
            ops.gemm_int8(x, wide, out, activation=activation)
    for form, splits in (("many", 0), ("mid", 9), ("mid", -1), ("pair", 16), ("pair", 48), ("pair", 288)):
        with pytest.raises(ops.KernelError):
            ops.gemm_int8(x, w, good, form=form, splits=splits)
    with pytest.raises(ops.KernelError):
        ops.gemm_int8(x, operands(4, 40, 65, 1)[1], good)
    a, b = ops.Int8Rows.empty(1, ops.INT8_MAX_WIDTH + 1, "cuda"), ops.Int8Rows.empty(4, ops.INT8_MAX_WIDTH + 1, "cuda")
    with pytest.raises(ops.KernelError):
        ops.gemm_int8(a, b, torch.zeros(1, 4, device="cuda"))


@pytest.mark.parametrize("M", [1, 16, 64, 200, 700])
def test_weights_that_were_written_just_before(M):
    """Quantised one launch before the product, over and over into the same memory: a product that starts before the kernel ahead of it has ended
    may not read its weights until then."""
    from qwen3_b200.csrc import ops
    N, K = 2048, 1000
    g = torch.Generator(device="cuda").manual_seed(M)
    x = operands(M, N, K, M)[0]
    matrices = [torch.randn(N, K, generator=g, device="cuda") for _ in range(3)]
    settled = [ops.quantize_rows(m, ops.Int8Rows.empty(N, K, "cuda")) for m in matrices]
    torch.cuda.synchronize()
    want = [ops.gemm_int8(x, w, torch.zeros(M, N, device="cuda")) for w in settled]
    w, outs = ops.Int8Rows.empty(N, K, "cuda"), [torch.zeros(M, N, device="cuda") for _ in range(30)]
    torch.cuda.synchronize()
    for i, y in enumerate(outs):
        ops.quantize_rows(matrices[i % 3], w)
        ops.gemm_int8(x, w, y)
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(outs))


@pytest.mark.parametrize("form", ["few", "mid", "pair"])
def test_offsets_beyond_32_bits(form):
    """Codes of 2.2 GB, and 2.3 billion outputs: the last rows are those of the rows alone."""
    from qwen3_b200.csrc import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    for M, N, K in ((270000, 16, 8192), (143000, 16400, 64)):
        x, w = ops.Int8Rows.empty(M, K, "cuda"), ops.Int8Rows.empty(N, K, "cuda")
        x.codes.random_(-127, 128, generator=g), w.codes.random_(-127, 128, generator=g)
        x.scales.fill_(0.01), w.scales.fill_(0.02)
        y = ops.gemm_int8(x, w, torch.zeros(M, N, dtype=torch.bfloat16, device="cuda"), form=form)
        assert ops.tcgen05_status("cuda") == 0
        for first in (0, M // 2, M - 40):
            some = ops.Int8Rows(x.codes[first:first + 40], x.scales[first:first + 40])
            assert torch.equal(ops.gemm_int8(some, w, torch.zeros(40, N, dtype=torch.bfloat16, device="cuda")), y[first:first + 40])
            check(some, w, y[first:first + 40], "bf16", None)
        del x, w, y
        torch.cuda.empty_cache()


FIRST_CALL = """
import sys
sys.path.insert(0, {root!r})
import torch
from qwen3_b200.csrc import ops
x, w = torch.randn({M}, 200, device="cuda"), torch.randn(272, 200, device="cuda")
x8, w8, y = ops.Int8Rows.empty({M}, 200, "cuda"), ops.Int8Rows.empty(272, 200, "cuda"), torch.zeros({M}, 272, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.quantize_rows(x, x8), ops.quantize_rows(w, w8)
    ops.gemm_int8(x8, w8, y)
assert ops.tcgen05_status("cuda") == 0
graph.replay()
torch.cuda.synchronize()
want = ops.gemm_int8(x8, w8, torch.zeros({M}, 272, device="cuda"))
assert torch.equal(y, want) and bool(y.any()) and ops.tcgen05_status("cuda") == 0
print("captured")
"""


@pytest.mark.parametrize("M", [3, 100, 700])
def test_first_call_of_a_process_inside_a_capture(M):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=root, M=M)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_another_current_device_is_refused(monkeypatch):
    from qwen3_b200.csrc import ops
    x, w = operands(4, 32, 64, 1)
    a = torch.zeros(4, 64, device="cuda")
    y = torch.zeros(4, 32, device="cuda")
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    for call in (lambda: ops.gemm_int8(x, w, y), lambda: ops.quantize_rows(a, x), lambda: ops.rms_norm_int8(a, a[0].contiguous(), 1e-6, x)):
        with pytest.raises(ops.KernelError, match="current device"):
            call()
