"""linear_mxfp4 against its 64-bit form.

Bar. Every product of an element of x and one of W is exact in f32 (11 or 8 bits times 2), so a result is an f32 sum of K
terms in some order: at most K * 2^-24 of the sum of their magnitudes (the matrix instructions and the joins add in chains far
shorter than K), then half a step of the type (and half of f16's smallest subnormal)."""
import pytest
import torch

import intent_amd as intent
from intent_amd.examples.kernels.contraction import linear_mxfp4
from tests import plain64
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def kernel(dtype):
    return intent.jit(getattr(linear_mxfp4, "linear_mxfp4_" + dtype), backend="hip")


def case(seed, dtype, m, n, k, low=115, high=125):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((m, k), generator=g).to(TYPES[dtype]), torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8),
            torch.randint(low, high, (n, k // 32), generator=g, dtype=torch.uint8))


def check(got, x, weight, exponents, dtype):
    w = plain64.unpack_e2m1(weight, exponents)
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    got = got.double().cpu()
    assert not got.isnan().any()
    bound = HALF_STEP[dtype] * want.abs() + x.shape[1] * 2.0 ** -24 * size + 2.0 ** -25
    worst = (got - want).abs() - bound
    assert (worst <= 0).all(), f"off by {(got - want).abs().flatten()[worst.argmax()]} of {want.flatten()[worst.argmax()]}"


SHAPES = [(1, 1, 32), (1, 16, 64), (1, 17, 96), (3, 100, 160), (16, 33, 1024), (17, 64, 512), (5, 4096, 128), (31, 127, 544),
          (33, 130, 256), (64, 512, 2048), (65, 257, 1056), (1, 300, 14336), (100, 96, 4096), (127, 1000, 320), (128, 256, 256),
          (129, 513, 512), (200, 77, 96), (256, 512, 1024), (300, 1024, 736), (1021, 320, 288)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matches_plain_form(device, dtype, m, n, k):
    announce("linear mxfp4", dtype, m, n, k)
    x, weight, exponents = case(m + n + k, dtype, m, n, k)
    check(kernel(dtype).run(x.to(device), weight.to(device), exponents.to(device)), x, weight, exponents, dtype)


@pytest.mark.parametrize("m,n,k", [(9, 70, 6176), (16, 6152, 160), (16, 12296, 96), (40, 8200, 2080), (161, 2058, 6176),
                                   (250, 4100, 3840), (513, 4128, 96), (1500, 14000, 96), (700, 8190, 1184)])
def test_every_tile(device, m, n, k):
    """Sizes that each take another kernel, tile or division of K, whose last stage, row and column tiles are partial."""
    announce("linear mxfp4 tile", m, n, k)
    x, weight, exponents = case(m + n + k, "bf16", m, n, k)
    check(kernel("bf16").run(x.to(device), weight.to(device), exponents.to(device)), x, weight, exponents, "bf16")


@pytest.mark.parametrize("m", [1, 40, 150])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_every_element_and_exponent(device, dtype, m):
    """The unit rows of x pick single weights: each element at each exponent, rounded to the type as a value of it is (f16:
    subnormals, infinity beyond its range); NaN at exponent 255 reaches its weight row and no other."""
    announce("linear mxfp4 every element", dtype, m)
    code = torch.arange(32, dtype=torch.uint8) % 16
    packed = (code[0::2] | code[1::2] << 4).repeat(255, 1)
    exponents = torch.arange(255, dtype=torch.uint8)[:, None]
    x = torch.zeros((m, 32), dtype=TYPES[dtype])
    for i in range(m):
        x[i, i % 32] = 1
    w = plain64.unpack_e2m1(packed, exponents).to(TYPES[dtype]).double()
    finite = w.isfinite().all(1)               # an infinite weight times the zeros of x is NaN
    got = kernel(dtype).run(x.to(device), packed.to(device), exponents.to(device)).cpu()
    assert torch.equal(got[:, finite].double(), w[finite].t()[torch.arange(m) % 32])
    assert got[:, ~finite].isnan().any() or bool(finite.all())
    exponents[7] = 255
    got = kernel(dtype).run(x.to(device), packed.to(device), exponents.to(device)).cpu()
    finite[7] = False
    assert got[:, 7].isnan().all() and torch.equal(got[:, finite].double(), w[finite].t()[torch.arange(m) % 32])


@pytest.mark.parametrize("m", [1, 20, 130])
def test_layouts(device, m):
    """x with an odd start, odd and inner strides (staged), a weight and exponents inside larger ones, an output with odd
    rows: the values of contiguous ones bit for bit; nothing is written beside the output."""
    announce("linear mxfp4 layouts", m)
    n, k = 70, 160
    x, weight, exponents = (a.to(device) for a in case(m, "f16", m, n, k))
    run = kernel("f16")
    want = run.run(x, weight, exponents)
    wide = torch.zeros((m, k + 5), dtype=torch.float16, device=device)
    wide[:, 3:3 + k] = x
    spread = torch.zeros((m, k, 2), dtype=torch.float16, device=device)
    spread[..., 0] = x
    held = torch.full((n, k // 2 + 32), 0x77, dtype=torch.uint8, device=device)
    held[:, 16:16 + k // 2] = weight
    powers = torch.full((n, k // 32 + 3), 255, dtype=torch.uint8, device=device)
    powers[:, 1:1 + k // 32] = exponents
    for rows in (wide[:, 3:3 + k], spread[..., 0]):
        out = torch.full((m, n + 3), 7.0, dtype=torch.float16, device=device)
        run(rows, held[:, 16:16 + k // 2], powers[:, 1:1 + k // 32], out[:, 1:1 + n])
        assert torch.equal(out[:, 1:1 + n], want)
        assert (out[:, 0] == 7).all() and (out[:, 1 + n:] == 7).all()
    out = torch.full((m, n, 2), 7.0, dtype=torch.float16, device=device)
    run(x, weight, exponents, out[..., 0])
    assert torch.equal(out[..., 0], want) and (out[..., 1] == 7).all()


def test_special_rows_and_empty_extents(device):
    """NaN and infinities of x stay in their rows; no row or column is fine, and K = 0 gives 0."""
    announce("linear mxfp4 special rows")
    run = kernel("bf16")
    x, weight, exponents = (a.to(device) for a in case(5, "bf16", 40, 48, 64))
    want = run.run(x, weight, exponents)
    x[3, 5], x[38, 63] = float("nan"), float("inf")
    got = run.run(x, weight, exponents)
    keep = torch.ones(40, dtype=torch.bool, device=device)
    keep[3] = keep[38] = False
    assert torch.equal(got[keep], want[keep]) and got[3].isnan().all() and not got[38].isfinite().any()
    assert run.run(x[:0], weight, exponents).shape == (0, 48) and run.run(x, weight[:0], exponents[:0]).shape == (40, 0)
    assert (run.run(x[:, :0], weight[:, :0], exponents[:, :0]) == 0).all()


def test_streams_and_graphs(device):
    announce("linear mxfp4 streams, graphs")
    for m, n, k in ((1, 256, 8192), (33, 192, 4096), (200, 512, 512)):
        x, weight, exponents = (a.to(device) for a in case(m, "f16", m, n, k))
        run = kernel("f16")
        want = run.run(x, weight, exponents)
        call = run.prepare(x, weight, exponents)
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
            again = run.run(x, weight, exponents)
            torch.cuda.synchronize()
            assert torch.equal(call.result(), want) and torch.equal(again, want)


def test_refusals(device):
    x, weight, exponents = (a.to(device) for a in case(1, "f16", 4, 8, 64))
    run = kernel("f16")
    with pytest.raises(TypeError):
        run.run(x.bfloat16(), weight, exponents)
    with pytest.raises(ValueError, match="blocks of 32"):
        run.run(x[:, :48], weight[:, :24], exponents)
    with pytest.raises(ValueError, match="blocks of 32"):
        run.run(x, weight, exponents[:, :1])
    with pytest.raises(ValueError, match="blocks of 32"):
        run.run(x, weight[:, :16], exponents)
    with pytest.raises(ValueError, match="16 bytes"):
        run.run(x, torch.zeros((8, 40), dtype=torch.uint8, device=device)[:, :32], exponents)
    with pytest.raises(ValueError, match="unit inner stride"):
        run.run(x, weight, torch.zeros((2, 8), dtype=torch.uint8, device=device).t())
    with pytest.raises(ValueError):
        run.run(x, weight, exponents[:7])
    static = intent.jit(linear_mxfp4.linear_mxfp4_f16, backend="hip", backend_options={"workspace": "static"})
    static.run(x, weight, exponents)
    with pytest.raises(intent.CompilationStageError, match="workspace"):
        static.run(*(a.to(device) for a in case(2, "f16", 100, 64, 4096)))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,k", [(1, 32), (6143, 96), (6145, 96), (6150, 4128), (33, 8224), (100, 4064), (7000, 64)])
def test_one_row(device, dtype, n, k):
    """A single row of x: both sizes of its kernel, runs of K that end inside a step, weight rows behind the last."""
    announce("linear mxfp4 one row", dtype, n, k)
    x, weight, exponents = case(n + k, dtype, 1, n, k)
    check(kernel(dtype).run(x.to(device), weight.to(device), exponents.to(device)), x, weight, exponents, dtype)


@pytest.mark.parametrize("m", [1, 20])
def test_weights_beyond_32_bits(device, m):
    announce("linear mxfp4 beyond 32 bits", m)
    n, k = 2 ** 19 + 70, 16384
    x, few, powers = case(m, "f16", m, 64, k)
    weight = torch.zeros((n, k // 2), dtype=torch.uint8, device=device)
    exponents = torch.full((n, k // 32), 120, dtype=torch.uint8, device=device)
    assert weight.numel() > 2 ** 32
    rows = torch.cat((torch.arange(16), torch.arange(n - 48, n)))
    weight[rows.to(device)], exponents[rows.to(device)] = few.to(device), powers.to(device)
    out = kernel("f16").run(x.to(device), weight, exponents)
    check(out[:, rows.to(device)], x, few, powers, "f16")
    assert (out[:, 16:n - 48] == 0).all()
