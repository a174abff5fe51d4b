"""Calls of the 8-bit operators as programs make them: one kernel right behind the other, forms that the sizes alone would not ask for, edges of the sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def drawn(rows, width, seed):
    return torch.randn(rows, width, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("activation", [None, "silu", "gelu_tanh"])
@pytest.mark.parametrize("form,M,N,K", [("few", 1, 2048, 1000), ("few", 8, 6144, 8200), ("few", 5, 9600, 500), ("few", 16, 2048, 1000), ("few", 12, 6144, 500),
                                        ("few", 32, 2048, 1000), ("few", 70, 4000, 200), ("mid", 16, 2048, 1000), ("mid", 64, 4096, 4096),
                                        ("mid", 200, 1024, 640), ("pair", 40, 2048, 512), ("pair", 700, 2048, 1000)])
def test_weights_and_tokens_written_just_before(form, M, N, K, activation, kind):
    """Weights and tokens are quantised one and two launches before the product, over and over into the same memory: what a product reads before the kernel
    ahead has ended is the round before's.  All variants of the form for few tokens, every output and gate."""
    from qwen3_b200.csrc import ops
    columns = N // 2 if activation else N
    matrices, tokens = [drawn(N, K, 3 + i) for i in range(3)], [drawn(M, K, 13 + i) for i in range(3)]
    want = []
    for w, x in zip(matrices, tokens):
        w8, x8 = ops.quantize_rows(w, ops.Int8Rows.empty(N, K, "cuda")), ops.quantize_rows(x, ops.Int8Rows.empty(M, K, "cuda"))
        torch.cuda.synchronize()
        want.append(ops.gemm_int8(x8, w8, torch.zeros(M, columns, dtype=kind, device="cuda"), activation=activation, form="mid" if form != "mid" else "pair"))
        torch.cuda.synchronize()
    w8, x8 = ops.Int8Rows.empty(N, K, "cuda"), ops.Int8Rows.empty(M, K, "cuda")
    outs = [torch.zeros(M, columns, dtype=kind, device="cuda") for _ in range(12)]
    torch.cuda.synchronize()
    for i, y in enumerate(outs):
        for which in ((0, 1), (1, 0))[i % 2]:              # either of them last
            if which:
                ops.quantize_rows(matrices[i % 3], w8)
            else:
                ops.quantize_rows(tokens[i % 3], x8)
        ops.gemm_int8(x8, w8, y, activation=activation, form=form)
    torch.cuda.synchronize()
    assert ops.tcgen05_status("cuda") == 0
    assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(outs))


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("rows,width", [(6, 1), (12, 64), (13, 65), (1, 4096), (700, 1000), (400, 1001), (13, 5001), (12, 40000)])
def test_norm_of_small_rows_without_an_epsilon(rows, width, delta, kind):
    """Squares that 32 bits lose, wholly or in part, between rows that they hold: beside an eps of 0 the scale is that of 64 bits but for the rounding of
    some sums of at most 110 terms in a row, a root, a product and a division (2^-18), and a step of the smallest scales."""
    import int8_cases as ic
    from qwen3_b200.csrc import ops
    x = drawn(rows, width, rows + width)
    for i in range(rows):
        x[i] *= (1.0, 1e-10, 1e-18, 1e-20, 1e-22, 1e-25, 1e-30, 1e-36, 1e-38, 1e-40)[i % 10]
    x[rows // 2] = 0
    x, w = x.to(kind), 1 + 0.3 * drawn(1, width, 7)[0]
    d = (0.5 * x.float().roll(1, 1)).to(kind) if delta else None
    stored = (x.float() + d.float()).to(kind) if delta else x.clone()
    u = ic.normed(stored, w)
    codes, tops = ic.quantised(u)
    for eps in (0.0, 1e-42, 2.0 ** -127):
        mean = stored.double().square().mean(-1) + float(torch.tensor(eps, dtype=torch.float32))
        want = torch.where(tops > 0, tops / mean.sqrt(), torch.zeros_like(tops))
        t, total, out = x.clone(), torch.full_like(x, 77.0), ops.Int8Rows.empty(rows, width, "cuda")
        ops.rms_norm_int8(t, w, eps, out, **({"delta": d, "total": total} if delta else {}))
        assert torch.equal(out.codes.long(), codes)
        assert bool(((out.scales.double() - want).abs() <= 2.0 ** -18 * want + 2.0 ** -149).all()), (eps, out.scales, want)
        if delta:
            assert torch.equal(total, stored) and torch.equal(t, x)
            ops.rms_norm_int8(t, w, eps, out, delta=d)     # in place
            assert torch.equal(t, stored) and bool(((out.scales.double() - want).abs() <= 2.0 ** -18 * want + 2.0 ** -149).all())


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 5, 700])
def test_rows_of_no_values(rows, kind):
    """As rows of zeros: the scale 0.  A product over no values is refused."""
    from qwen3_b200.csrc import ops
    x, w = torch.zeros(rows, 0, dtype=kind, device="cuda"), torch.zeros(0, device="cuda")
    memory = torch.full((rows, 16), 77, dtype=torch.int8, device="cuda")
    for out in (ops.Int8Rows(memory[:, :0], torch.full((rows,), 77.0, device="cuda")), ops.Int8Rows.empty(rows, 0, "cuda")):
        for call in (lambda: ops.quantize_rows(x, out), lambda: ops.rms_norm_int8(x, w, 1e-6, out), lambda: ops.rms_norm_int8(x, w, 0.0, out, delta=x)):
            out.scales.fill_(77.0)
            call()
            assert bool((out.scales == 0).all()) and out.float().shape == (rows, 0)
        with pytest.raises(ops.KernelError):
            ops.gemm_int8(out, out, torch.zeros(rows, rows, device="cuda"))
    assert bool((memory == 77).all())


def test_tensors_of_rows_stay_those_they_were_made_with():
    """Other tensors in their place would not reach the kernels: assigning them is an error."""
    from qwen3_b200.csrc import ops
    a, b = (ops.quantize_rows(drawn(4, 64, seed), ops.Int8Rows.empty(4, 64, "cuda")) for seed in (1, 2))
    before = a.float()
    for name in ("codes", "scales"):
        with pytest.raises(AttributeError):
            setattr(a, name, getattr(b, name))
    assert torch.equal(a.float(), before)
    a.scales.mul_(2)                                       # (values in place are felt)
    assert torch.equal(a.float(), 2 * before)


@pytest.mark.parametrize("width,apart", [(8192, True), (8191, False)])
def test_scales_and_sums_beyond_32_bit_offsets(width, apart):
    """2.2 billion values of x, delta and total: three runs of rows, of their own values each, against 64 bits: codes, scales (rounded once; under the norm as in the
    tests of widths, 2^-18) and sums; and the rows between them, which are zeros."""
    import int8_cases as ic
    from qwen3_b200.csrc import ops
    rows, runs = 270000, (0, 135000, 269000)
    x, d = (torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for i, first in enumerate(runs):
        x[first:first + 1000] = (drawn(1000, width, 3 + i) * (1 + i)).to(torch.bfloat16)
        d[first:first + 1000] = (drawn(1000, width, 33 + i) * 0.5).to(torch.bfloat16)
    w, out = 0.5 + drawn(1, width, 9)[0].abs(), ops.Int8Rows.empty(rows, width, "cuda")
    out.codes.fill_(77), out.scales.fill_(77.0)
    ops.quantize_rows(x, out)
    for first in runs:
        part = slice(first, first + 1000)
        codes, scales = ic.quantised(x[part])
        assert torch.equal(out.codes[part].long(), codes)
        assert bool(((out.scales[part].double() - scales).abs() <= 2.0 ** -24 * scales).all())
        assert bool((out.scales[first + 1000:first + 1010] == 0).all()) and not bool(out.codes[first + 1000:first + 1010].any())
    stored = [(x[f:f + 1000].float() + d[f:f + 1000].float()).to(torch.bfloat16) for f in runs]
    before = [x[f:f + 1000].clone() for f in runs]
    total = torch.full_like(x, 77.0) if apart else x
    out.codes.fill_(77), out.scales.fill_(77.0)
    ops.rms_norm_int8(x, w, 1e-6, out, delta=d, **({"total": total} if apart else {}))
    for first, sums, old in zip(runs, stored, before):
        part = slice(first, first + 1000)
        assert not torch.equal(sums, old) and torch.equal(total[part], sums) and (not apart or torch.equal(x[part], old))
        u = ic.normed(sums, w)
        codes, tops = ic.quantised(u)
        scales = tops / (sums.double().square().mean(-1) + 1e-6).sqrt()
        assert torch.equal(out.codes[part].long(), codes)
        assert bool(((out.scales[part].double() - scales).abs() <= 2.0 ** -18 * scales).all())
        assert bool((out.scales[first + 1000:first + 1010] == 0).all()) and not bool(total[first + 1000:first + 1010].any())
    del x, d, total, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,width", [(3, 4096), (700, 65), (20, 40000)])
def test_norm_of_small_rows_on_another_stream_and_in_graphs(rows, width):
    """Two launches: the second reads what the first has noted, also from a graph, and where a product follows."""
    from qwen3_b200.csrc import ops
    x = drawn(rows, width, 5).mul_(1e-30)
    x[::2] *= 1e30
    w, matrix = 1 + 0.3 * drawn(1, width, 7)[0], ops.quantize_rows(drawn(48, width, 6), ops.Int8Rows.empty(48, width, "cuda"))
    want = ops.rms_norm_int8(x.clone(), w, 0.0, ops.Int8Rows.empty(rows, width, "cuda"))
    torch.cuda.synchronize()
    product = ops.gemm_int8(want, matrix, torch.zeros(rows, 48, device="cuda"))
    assert bool(product.isfinite().all()) and bool((want.scales > 0).all())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = ops.rms_norm_int8(x, w, 0.0, ops.Int8Rows.empty(rows, width, "cuda"))
        y = ops.gemm_int8(out, matrix, torch.zeros(rows, 48, device="cuda"))
    side.synchronize()
    assert torch.equal(out.codes, want.codes) and torch.equal(out.scales, want.scales) and torch.equal(y, product)
    graph, out, y = torch.cuda.CUDAGraph(), ops.Int8Rows.empty(rows, width, "cuda"), torch.zeros(rows, 48, device="cuda")
    with torch.cuda.graph(graph):
        ops.rms_norm_int8(x, w, 0.0, out)
        ops.gemm_int8(out, matrix, y)
    for _ in range(3):
        out.scales.fill_(77.0), y.fill_(77.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.scales, want.scales) and torch.equal(y, product)


def test_graphs_replayed_at_once_and_threads():
    """Products on the same weights from graphs on two streams at once, and from two threads, each with outputs of its own."""
    import threading
    from qwen3_b200.csrc import ops
    w = ops.quantize_rows(drawn(2048, 1000, 1), ops.Int8Rows.empty(2048, 1000, "cuda"))
    tokens = [ops.quantize_rows(drawn(M, 1000, M), ops.Int8Rows.empty(M, 1000, "cuda")) for M in (4, 60, 200, 700)]
    want = [ops.gemm_int8(x, w, torch.zeros(x.rows, 2048, device="cuda")) for x in tokens]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for _ in streams:
        graph, ys = torch.cuda.CUDAGraph(), [torch.zeros_like(y) for y in want]
        with torch.cuda.graph(graph):
            for x, y in zip(tokens, ys):
                ops.gemm_int8(x, w, y)
        graphs.append(graph), outs.append(ys)
    for _ in range(10):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, z) for ys in outs for y, z in zip(ys, want))
    failed = []

    def work(stream):
        with torch.cuda.stream(stream):
            for _ in range(30):
                ys = [ops.gemm_int8(x, w, torch.empty(x.rows, 2048, device="cuda")) for x in tokens]
                stream.synchronize()
                if not all(torch.equal(y, z) for y, z in zip(ys, want)):
                    failed.append(stream)
    threads = [threading.Thread(target=work, args=(s,)) for s in streams]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and ops.tcgen05_status("cuda") == 0


@pytest.mark.parametrize("form", ["few", "mid", "pair"])
@pytest.mark.parametrize("rows,width", [(37, 100), (300, 1000)])
def test_rows_multiplied_with_themselves_and_slices_of_rows(rows, width, form):
    from qwen3_b200.csrc import ops
    x = ops.quantize_rows(drawn(rows, width, 2), ops.Int8Rows.empty(rows, width, "cuda"))
    y = ops.gemm_int8(x, x, torch.zeros(rows, rows, device="cuda"), form=form)
    want = (x.codes.double() @ x.codes.double().t() * x.scales.double()[:, None] * x.scales.double())
    assert bool(((y.double() - want).abs() <= 3.01 * 2.0 ** -24 * want.abs()).all())
    a, b = (ops.Int8Rows(x.codes[s], x.scales[s].contiguous()) for s in (slice(3, 20), slice(1, None, 2)))
    assert b.stride == 2 * x.stride
    part = ops.gemm_int8(a, b, torch.zeros(a.rows, b.rows, device="cuda"), form=form)
    assert torch.equal(part, y[3:20, 1::2])
