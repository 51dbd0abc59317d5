"""quantize_rows, swiglu_quantize_rows and linear_i8 against their 64-bit forms.

Bars. Plain rows: 127 x / max|x| of 16-bit x is a border between two integers or further from one than f32 can miss, so elements are the
64-bit ones, and scales f32 quotients. Gated rows: e^-g is off by (|g| + 4) 2^-23 of itself (the product with log2 e and the exponential),
the rest of a = g / (1 + e^-g) u by 6 roundings of 2^-23; an element by that of itself and of the row's largest, and half a step.
Products: the integer sum is exact; three factors and the bias round by 2^-24 each, then half a step of the type (and half of f16's
smallest subnormal)."""
import pytest
import torch

import intent_amd as intent
from intent_amd.examples.kernels.contraction import linear_i8
from intent_amd.examples.kernels.normalization import quantize_rows
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def kernel(name, **options):
    return intent.jit(getattr(linear_i8 if name.startswith("linear") else quantize_rows, name), backend="hip", **options)


def quantised(x):
    """(elements, scales) of rows, in 64 bits and rounded to f32."""
    x = x.double()
    most = x.abs().amax(-1) if x.shape[-1] else x.new_zeros(x.shape[0])
    elements = torch.round(127 * x / torch.where(most > 0, most, 1)[:, None])
    return elements, (most.float() / 127)


def gated(gate, up):
    """(rows, what each element may be off by) in 64 bits."""
    gate, up = gate.double(), up.double()
    a = gate / (1 + torch.exp(-gate)) * up
    return a, a.abs() * (gate.abs() + 10) * 2.0 ** -23


def check_gated(elements, scales, gate, up):
    a, off = gated(gate, up)
    most, at = a.abs().max(-1, keepdim=True)
    share = off.gather(-1, at) / most
    assert ((scales.double().cpu()[:, None] - most / 127).abs() <= (share + 2.0 ** -23) * most / 127).all()
    quotient = 127 * a / most
    assert ((elements.double().cpu() - quotient).abs() <= 0.5 + 127 * off / most + quotient.abs() * share + 1e-6).all()


SIZES = [(1, 1), (3, 8), (5, 63), (4, 512), (9, 520), (6, 1000), (70, 96), (2, 2048), (3, 2056), (5, 4096), (2, 8192), (3, 8200), (2, 14336),
         (2, 14333), (2, 32768)]


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_rows(device, dtype, rows, d):
    announce("quantize rows", dtype, rows, d)
    g = torch.Generator().manual_seed(rows + d)
    x, up = ((torch.randn((rows, d), generator=g) * 3).to(TYPES[dtype]) for _ in range(2))
    elements, scales = kernel("quantize_rows_" + dtype).run(x.to(device))
    want, want_scales = quantised(x)
    assert torch.equal(elements.cpu().double(), want) and torch.equal(scales.cpu(), want_scales)
    check_gated(*kernel("swiglu_quantize_rows_" + dtype).run(x.to(device), up.to(device)), x, up)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_every_value(device, dtype):
    """Rows of every finite value up to a largest one, for largest ones over the whole type: subnormals, borders and ties."""
    announce("quantize every value", dtype)
    values = torch.arange(2 ** 15, dtype=torch.int32).to(torch.int16).view(TYPES[dtype])
    values = values[values.isfinite()]
    run = kernel("quantize_rows_" + dtype)
    for last in (1, 2, 3, 100, 255, 1024, 4097, len(values) // 2 + 1, len(values) - 1):
        x = values[max(0, last - 4000):last + 1].clone()
        x[::3] *= -1
        spread = torch.cat((x, values[torch.linspace(0, last, 3000).long()]))[None]
        elements, scales = run.run(spread.to(device))
        want, want_scales = quantised(spread)
        assert torch.equal(elements.cpu().double(), want), last
        assert torch.equal(scales.cpu(), want_scales), last


def test_rows_special_and_layouts(device):
    """Zeros, infinities and NaN in a row, halves of one projection's rows, odd strides and starts, empty extents."""
    announce("quantize rows special")
    g = torch.Generator().manual_seed(2)
    halves = torch.randn((7, 2 * 96), generator=g).half().to(device)
    gate, up = halves[:, :96], halves[:, 96:]
    run, run_gated = kernel("quantize_rows_f16"), kernel("swiglu_quantize_rows_f16")
    check_gated(*run_gated.run(gate, up), gate.cpu(), up.cpu())
    want = run.run(gate.contiguous())
    odd = torch.zeros((7, 101), dtype=torch.float16, device=device)
    odd[:, 3:99] = gate
    inner = torch.zeros((7, 96, 2), dtype=torch.float16, device=device)
    inner[..., 1] = gate
    for x in (gate, odd[:, 3:99], inner[..., 1]):
        held = torch.full((7, 99), 55, dtype=torch.int8, device=device)
        scales = torch.full((14,), 5.0, device=device)
        run(x, held[:, 1:97], scales[::2])
        assert torch.equal(held[:, 1:97], want[0]) and torch.equal(scales[::2], want[1])
        assert (held[:, 0] == 55).all() and (held[:, 97:] == 55).all() and (scales[1::2] == 5).all()
    x = gate.clone()
    x[0], x[1, 5], x[2, 95], x[3, 0] = 0, float("nan"), float("inf"), float("-inf")
    elements, scales = run.run(x)
    assert (elements[:4] == 0).all() and scales[0] == 0 and scales[1:4].isnan().all()
    assert torch.equal(elements[4:], want[0][4:]) and torch.equal(scales[4:], want[1][4:])
    wild = torch.tensor([[-30000.0, 2.0, 60000.0, -60000.0]], device=device).half()
    elements, scales = run_gated.run(wild, torch.ones_like(wild))
    assert torch.equal(elements.cpu(), torch.tensor([[0, 0, 127, 0]], dtype=torch.int8)) and scales.isfinite().all()
    assert run.run(x[:0])[0].shape == (0, 96) and (run.run(x[:, :0])[1] == 0).all()
    with pytest.raises(intent.CompilationStageError, match="32768"):
        run.run(torch.zeros((1, 32769), dtype=torch.float16, device=device))
    with pytest.raises(ValueError):
        run_gated.run(gate, up[:, :8])
    with pytest.raises(TypeError):
        run.run(gate.float())


def case(seed, m, n, k, biased, low=-128):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(low, 128, (m, k), generator=g, dtype=torch.int8), torch.randint(low, 128, (n, k), generator=g, dtype=torch.int8),
            torch.rand((m,), generator=g) / 64 + 1e-3, torch.rand((n,), generator=g) / 64 + 1e-3,
            torch.randn((n if biased else 0,), generator=g))


def check(got, x, weight, x_scales, weight_scales, bias, dtype):
    want = (x.double() @ weight.double().t()) * x_scales.double()[:, None] * weight_scales.double()
    size = want.abs()
    if bias.numel():
        want, size = want + bias.double(), size + bias.double().abs()
    got = got.double().cpu()
    assert not got.isnan().any()
    bound = HALF_STEP[dtype] * want.abs() + 4 * 2.0 ** -24 * size + 2.0 ** -25
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"off by {(got - want).abs().flatten()[over.argmax()]} of {want.flatten()[over.argmax()]}"


SHAPES = [(1, 1, 16), (1, 16, 64), (1, 17, 144), (3, 100, 160), (16, 33, 1024), (17, 64, 512), (5, 4096, 128), (31, 127, 544), (1, 7000, 80),
          (33, 130, 272), (64, 512, 2048), (65, 257, 1056), (1, 300, 14336), (100, 96, 4096), (127, 1000, 320), (128, 256, 256), (2, 6200, 2064),
          (129, 513, 512), (200, 77, 96), (256, 512, 1024), (300, 1024, 736), (1021, 320, 288), (513, 4100, 208), (700, 8190, 1184)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(device, dtype, m, n, k):
    announce("linear i8", dtype, m, n, k)
    given = case(m + n + k, m, n, k, (m + n) % 2 == 0)
    check(kernel("linear_i8_" + dtype).run(*(t.to(device) for t in given)), *given, dtype)


@pytest.mark.parametrize("m,n,k", [(9, 70, 6176), (16, 6152, 160), (40, 8200, 2080), (161, 2058, 6176), (250, 4100, 3840), (1500, 14000, 96),
                                   (1024, 4096, 4096), (2048, 6144, 528), (24, 48, 131056), (3000, 3000, 16), (600, 2050, 4112)])
def test_every_tile(device, m, n, k):
    """Sizes that each take another kernel, tile or division of K, whose last stage, row and column tiles are partial."""
    announce("linear i8 tile", m, n, k)
    given = case(m + n + k, m, n, k, True)
    check(kernel("linear_i8_bf16").run(*(t.to(device) for t in given)), *given, "bf16")


@pytest.mark.parametrize("dtype,m,n,k", [
    ("f16", 1466, 775, 25120), ("bf16", 473, 5273, 4992), ("f16", 6285, 263, 11456), ("bf16", 142, 18518, 7168), ("f16", 954, 5812, 6160),
    ("bf16", 1834, 329, 6976), ("f16", 82, 2834, 2256), ("bf16", 385, 12290, 4112), ("f16", 2866, 6617, 1104)])
def test_parts_of_k_and_partial_tiles(device, dtype, m, n, k):
    """K divided over each kind of tile, rows of sums that are not whole fours, last parts that are shorter than the others, rounds of
    whole and halved tiles."""
    announce("linear i8 parts", dtype, m, n, k)
    given = case(m + n + k, m, n, k, m % 2 == 0)
    check(kernel("linear_i8_" + dtype).run(*(t.to(device) for t in given)), *given, dtype)


@pytest.mark.parametrize("m", [1, 9, 40, 300])
def test_largest_sums(device, m):
    """Every element -128 at the largest K: sums just below 2^31."""
    announce("linear i8 largest sums", m)
    k = 131056
    given = (torch.full((m, k), -128, dtype=torch.int8), torch.full((24, k), -128, dtype=torch.int8), torch.full((m,), 2.0 ** -20),
             torch.full((24,), 2.0 ** -5), torch.zeros(0))
    check(kernel("linear_i8_bf16").run(*(t.to(device) for t in given)), *given, "bf16")


@pytest.mark.parametrize("m", [1, 20, 130, 520])
def test_layouts(device, m):
    """x with an odd start, odd and inner strides (staged), a weight inside a larger one, scales with a stride, an output with odd rows:
    the values of contiguous ones bit for bit; nothing is written beside the output."""
    announce("linear i8 layouts", m)
    n, k = 70, 160
    x, weight, xs, ws, bias = (t.to(device) for t in case(m, m, n, k, True))
    run = kernel("linear_i8_f16")
    want = run.run(x, weight, xs, ws, bias)
    wide = torch.zeros((m, k + 5), dtype=torch.int8, device=device)
    wide[:, 3:3 + k] = x
    spread = torch.zeros((m, k, 2), dtype=torch.int8, device=device)
    spread[..., 0] = x
    held = torch.full((n, k + 32), 77, dtype=torch.int8, device=device)
    held[:, 16:16 + k] = weight
    twice = lambda t: torch.stack((t, t), 1).flatten()[::2]  # noqa: E731
    for rows in (wide[:, 3:3 + k], spread[..., 0]):
        out = torch.full((m, n + 3), 7.0, dtype=torch.float16, device=device)
        run(rows, held[:, 16:16 + k], twice(xs), twice(ws), twice(bias), out[:, 1:1 + n])
        assert torch.equal(out[:, 1:1 + n], want)
        assert (out[:, 0] == 7).all() and (out[:, 1 + n:] == 7).all()
    out = torch.full((m, n, 2), 7.0, dtype=torch.float16, device=device)
    run(x, weight, xs, ws, bias, out[..., 0])
    assert torch.equal(out[..., 0], want) and (out[..., 1] == 7).all()


def test_special_scales_and_empty_extents(device):
    announce("linear i8 special scales")
    run = kernel("linear_i8_bf16")
    x, weight, xs, ws, bias = (t.to(device) for t in case(5, 40, 48, 64, True))
    want = run.run(x, weight, xs, ws, bias)
    xs[3], ws[7] = float("nan"), 0
    got = run.run(x, weight, xs, ws, bias)
    keep = torch.ones((40, 48), dtype=torch.bool, device=device)
    keep[3], keep[:, 7] = False, False
    assert torch.equal(got[keep], want[keep]) and got[3].isnan().all()
    assert torch.equal(got[4:, 7], bias[7].bfloat16().expand(36))
    assert run.run(x[:0], weight, xs[:0], ws, bias).shape == (0, 48)
    assert run.run(x, weight[:0], xs, ws[:0], bias[:0]).shape == (40, 0)
    for m in (1, 8, 40):
        assert torch.equal(run.run(x[:m, :0], weight[:, :0], torch.ones(m, device=device), ws, bias), bias.bfloat16().expand(m, 48))


def test_streams_and_graphs(device):
    announce("linear i8 streams, graphs")
    for m, n, k in ((1, 256, 8192), (33, 192, 4096), (600, 512, 512)):
        given = [t.to(device) for t in case(m, m, n, k, True)]
        run = kernel("linear_i8_f16")
        want = run.run(*given)
        call = run.prepare(*given)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call.launch()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(call.result(), want)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                call.launch()
            graphs.append(graph)
        for step in range(4):
            call.result().zero_()
            graphs[step % 2].replay()
            again = run.run(*given)
            torch.cuda.synchronize()
            assert torch.equal(call.result(), want) and torch.equal(again, want)


def test_refusals(device):
    x, weight, xs, ws, bias = (t.to(device) for t in case(1, 4, 8, 64, True))
    run = kernel("linear_i8_f16")
    with pytest.raises(TypeError):
        run.run(x.to(torch.uint8), weight, xs, ws, bias)
    with pytest.raises(ValueError, match="multiples of 16"):
        run.run(x[:, :40], weight[:, :40], xs, ws, bias)
    with pytest.raises(ValueError, match="bias holds"):
        run.run(x, weight, xs, ws, bias[:3])
    with pytest.raises(ValueError, match="16 bytes"):
        run.run(x, torch.zeros((8, 72), dtype=torch.int8, device=device)[:, :64], xs, ws, bias)
    with pytest.raises(ValueError):
        run.run(x, weight, xs[:3], ws, bias)
    with pytest.raises(intent.CompilationStageError, match="131072"):
        run.run(*(t.to(device) for t in case(1, 2, 4, 131072, False)))
    static = kernel("linear_i8_f16", backend_options={"workspace": "static"})
    static.run(x, weight, xs, ws, bias)
    with pytest.raises(intent.CompilationStageError, match="workspace"):
        static.run(*(t.to(device) for t in case(2, 100, 64, 4096, True)))


@pytest.mark.parametrize("m", [1, 20, 300])
def test_weights_beyond_32_bits(device, m):
    announce("linear i8 beyond 32 bits", m)
    n, k = 2 ** 18 + 70, 16384
    x, few, xs, few_scales, _ = case(m, m, 64, k, False)
    weight, ws = torch.zeros((n, k), dtype=torch.int8, device=device), torch.ones(n, device=device)
    assert weight.numel() > 2 ** 32
    rows = torch.cat((torch.arange(16), torch.arange(n - 48, n)))
    weight[rows.to(device)], ws[rows.to(device)] = few.to(device), few_scales.to(device)
    out = kernel("linear_i8_f16").run(x.to(device), weight, xs.to(device), ws, torch.zeros(0, device=device))
    check(out[:, rows.to(device)], x, few, xs, few_scales, torch.zeros(0), "f16")
    assert (out[:, 16:n - 48] == 0).all()
