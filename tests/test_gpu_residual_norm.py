"""residual_norm, residual_norm_i8 and residual_norm_backward against their 64-bit forms.

Bars. A row's sum is formed in f32 from at most 16 elements a thread, 6 steps of a wave and 16 waves, each rounding by 2^-24 of the sum of
magnitudes; a reciprocal root takes half of that and adds 2^-23, and a result a handful of products. So every quantity is within 2^-18 (64
roundings) of the magnitudes that it is formed from, where a norm also passes on what its own mean is off by, and is then rounded to its
type by half a step (or half of f16's smallest subnormal, 2^-25). An 8-bit element is within that (in steps) of its quotient and half a step."""
import pytest
import torch

import intent_amd as intent
from intent_amd.examples.kernels.backward import residual_norm as backward
from intent_amd.examples.kernels.normalization import residual_norm as forward
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f16": 2.0 ** -25, "bf16": 1e-40}
NUMBERS = (0.75, 1.25, 1e-6)
TINY = 2.0 ** -18


def kernel(name, **options):
    return intent.jit(getattr(backward if "backward" in name else forward, name), backend="hip", **options)


def case(seed, dtype, tokens, d, gated, post):
    """block, residual, gate, post_weight, weight, grad_sum, grad_output on the CPU."""
    g = torch.Generator().manual_seed(seed)
    rows = [(torch.randn((tokens, d), generator=g) * s).to(TYPES[dtype]) for s in (1, 2, 1, 1)]
    gate = torch.rand((tokens if gated else 0,), generator=g) * 2 - 0.5
    weights = [1 + 0.3 * torch.randn((n,), generator=g) for n in (d if post else 0, d)]
    return (*rows[:2], gate, *weights, *rows[2:])


def unit(x, size, eps):
    """x over its root mean square in 64 bits; the share it may be off by for what its elements (formed from `size`) are off by."""
    square = x.pow(2).mean(-1, keepdim=True) + eps
    return 1 / square.sqrt(), 2 + (x.abs() * size).mean(-1, keepdim=True) / square


def plain(block, residual, gate, post, weight, numbers=NUMBERS):
    """(sum, magnitudes, output, magnitudes) in 64 bits."""
    rs, bs, eps = numbers
    x = block.double()
    u, size = x, x.abs()
    if post.numel():
        r, off = unit(x, x.abs(), eps)
        u = x * r * post.double()
        size = u.abs() * off
    factor = bs * (gate.double()[:, None] if gate.numel() else 1.0)
    h, h_size = rs * residual.double() + factor * u, (rs * residual.double()).abs() + (factor * size).abs()
    r, off = unit(h, h_size, eps)
    y = h * r * weight.double()
    return h, h_size, y, h_size * r * weight.double().abs() + y.abs() * off


def plain_backward(block, total, gate, post, weight, grad_sum, grad_output, numbers=NUMBERS):
    """((value, magnitudes) of grad_block, grad_residual, grad_gate, grad_post_weight, grad_weight) in 64 bits."""
    rs, bs, eps = numbers

    def through(x, w, g, g_size):
        r, off = unit(x, x.abs(), eps)
        x1, inner, inner_size = x * r, g * w, g_size * w.abs()
        along, along_size = (inner * x1).mean(-1, keepdim=True), (inner_size * x1.abs()).mean(-1, keepdim=True)
        size = r * (inner_size + x1.abs() * along_size) * off
        return r * (inner - x1 * along), size, (g * x1).sum(0), (g_size * x1.abs() * off).sum(0), x1 * w, (x1 * w).abs() * off

    gy = grad_output.double()
    d, d_size, gw, gw_size, _, _ = through(total.double(), weight.double(), gy, gy.abs())
    d, d_size = d + grad_sum.double(), d_size + grad_sum.double().abs()
    grad_residual = (rs * d, abs(rs) * d_size)
    g = bs * (gate.double()[:, None] if gate.numel() else torch.ones((1, 1), dtype=torch.float64))
    u = block.double()
    u_size, down, down_size = u.abs(), g * d, g.abs() * d_size
    empty = torch.zeros(0, dtype=torch.float64)
    grad_post = (empty, empty)
    if post.numel():
        down, down_size, gp, gp_size, u, u_size = through(u, post.double(), down, down_size)
        grad_post = (gp, gp_size)
    grad_gate = (bs * (d * u).sum(-1), abs(bs) * (d_size * u_size).sum(-1)) if gate.numel() else (empty, empty)
    return (down, down_size), grad_residual, grad_gate, grad_post, (gw, gw_size)


def close(got, want, size, dtype, share=TINY):
    got = got.double().cpu()
    assert got.shape == want.shape and not got.isnan().any()
    bound = HALF_STEP.get(dtype, 2.0 ** -24) * want.abs() + share * size + LEAST.get(dtype, 1e-37)
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"off by {(got - want).abs().flatten()[over.argmax()]} of {want.flatten()[over.argmax()]}"


def check_i8(elements, scales, want, size, tokens):
    """8-bit rows within half a step and what the quotient is off by; scales within a share."""
    elements, scales = elements.double().cpu(), scales.double().cpu()
    most, at = want.abs().max(-1, keepdim=True)
    share = (size / want.abs().clamp_min(1e-300)).gather(-1, at) * TINY
    assert ((scales[:, None] - most / 127).abs() <= (share + 2.0 ** -22) * most / 127).all()
    quotient = 127 * want / most
    off = 127 * TINY * size / most + quotient.abs() * share
    assert ((elements - quotient).abs() <= 0.5 + off + 1e-6).all()
    assert (elements.abs().max(-1).values == 127).all()


SHAPES = [(1, 8), (3, 1), (5, 7), (4, 64), (9, 257), (2, 511), (6, 512), (5, 520), (7, 1021), (33, 768), (3, 2048), (2, 2056), (5, 2304),
          (4, 4095), (3, 4096), (2, 4104), (3, 8192), (2, 8200), (2, 16383), (2, 16384)]


@pytest.mark.parametrize("tokens,d", SHAPES)
@pytest.mark.parametrize("dtype,gated,post", [("f16", False, False), ("bf16", True, True), ("f16", False, True), ("bf16", True, False)])
def test_matches_plain_form(device, dtype, tokens, d, gated, post):
    announce("residual_norm", dtype, tokens, d, gated, post)
    given = case(tokens + d, dtype, tokens, d, gated, post)
    on = [t.to(device) for t in given]
    h, h_size, y, y_size = plain(*given[:5])
    total, out = kernel("residual_norm_" + dtype).run(*on[:5], *NUMBERS)
    close(total, h, h_size, dtype)
    close(out, y, y_size, dtype)
    total8, elements, scales = kernel("residual_norm_i8_" + dtype).run(*on[:5], *NUMBERS)
    assert torch.equal(total8, total)
    check_i8(elements, scales, y, y_size, tokens)
    run = kernel("residual_norm_backward_" + dtype)
    got = run.run(on[0], total, *on[2:], *NUMBERS)
    for a, b in zip(got, run.run(on[0], total, *on[2:], *NUMBERS)):
        assert torch.equal(a, b)                                       # sums in a fixed order
    want = plain_backward(given[0], total.cpu(), *given[2:])
    for i, (value, size) in enumerate(want):
        close(got[i], value, size, dtype if i < 2 else "f32")


@pytest.mark.parametrize("tokens,d", [(700, 512), (1500, 72), (2100, 1000), (600, 4096)])
def test_many_tokens(device, tokens, d):
    """More tokens than the backward's slots: each walks several rows. A weight's sum of T terms is off by T roundings at most; the slots
    and the second kernel add in short chains, and T is below 2^12."""
    announce("residual_norm many tokens", tokens, d)
    given = case(d, "bf16", tokens, d, True, True)
    on = [t.to(device) for t in given]
    total, out = kernel("residual_norm_bf16").run(*on[:5], *NUMBERS)
    h, h_size, y, y_size = plain(*given[:5])
    close(total, h, h_size, "bf16")
    close(out, y, y_size, "bf16")
    got = kernel("residual_norm_backward_bf16").run(on[0], total, *on[2:], *NUMBERS)
    for i, (value, size) in enumerate(plain_backward(given[0], total.cpu(), *given[2:])):
        close(got[i], value, size, "bf16" if i < 2 else "f32")


@pytest.mark.parametrize("tokens,d", [(5000, 512), (2501, 1000), (9001, 72), (1301, 2049), (700, 8191), (300, 8201)])
def test_workgroups_take_several_turns(device, tokens, d):
    """More tokens than all workgroups of the backward take at a time, and a last turn that not all of them fill. A weight's sum goes
    through a chain of 3 turns, 8 rows, 8 workgroups and a tree of 6 at most, 25 roundings, which the share (64 of them) holds."""
    announce("residual_norm several turns", tokens, d)
    given = case(tokens, "bf16", tokens, d, True, True)
    on = [t.to(device) for t in given]
    total, _ = kernel("residual_norm_bf16").run(*on[:5], *NUMBERS)
    run = kernel("residual_norm_backward_bf16")
    got = run.run(on[0], total, *on[2:], *NUMBERS)
    for a, b in zip(got, run.run(on[0], total, *on[2:], *NUMBERS)):
        assert torch.equal(a, b)
    for i, (value, size) in enumerate(plain_backward(given[0], total.cpu(), *given[2:])):
        close(got[i], value, size, "bf16" if i < 2 else "f32")


@pytest.mark.parametrize("tokens,d", [(1, 64), (5, 64), (3, 520), (9, 7)])
def test_no_epsilon(device, tokens, d):
    """Without an epsilon the rows behind the last token, which workgroups of several rows have, must not become NaN."""
    announce("residual_norm no epsilon", tokens, d)
    numbers = (*NUMBERS[:2], 0.0)
    given = case(tokens, "f16", tokens, d, True, True)
    on = [t.to(device) for t in given]
    total, _ = kernel("residual_norm_f16").run(*on[:5], *numbers)
    got = kernel("residual_norm_backward_f16").run(on[0], total, *on[2:], *numbers)
    for i, (value, size) in enumerate(plain_backward(given[0], total.cpu(), *given[2:], numbers)):
        close(got[i], value, size, "f16" if i < 2 else "f32")


@pytest.mark.parametrize("d", [9, 255, 4095])
def test_in_place_rows_of_any_alignment(device, d):
    """Rows whose last piece is read together with elements of the piece before it, which another thread may have written by then."""
    announce("residual_norm in place, any alignment", d)
    for post in (False, True):
        given = [t.to(device) for t in case(d, "bf16", 300, d, True, post)]
        forward_run, back = kernel("residual_norm_bf16"), kernel("residual_norm_backward_bf16")
        want = forward_run.run(*given[:5], *NUMBERS)
        block, stream = given[0].clone(), given[1].clone()
        forward_run(block, stream, *given[2:5], stream, block, *NUMBERS)
        assert torch.equal(stream, want[0]) and torch.equal(block, want[1])
        rows = (given[0], want[0], *given[2:])
        want = back.run(*rows, *NUMBERS)
        block, grad_sum = given[0].clone(), given[5].clone()
        rest = [torch.empty_like(t) for t in want[2:]]
        back(block, rows[1], *given[2:5], grad_sum, given[6], block, grad_sum, *rest, *NUMBERS)
        for a, b in zip((block, grad_sum, *rest), want):
            assert torch.equal(a, b)


def test_gradients_against_differences(device):
    """Along random directions, the gradients give the change of sum(sum * grad_sum + output * grad_output) that the 64-bit forward has
    between x - s v and x + s v: a central difference, off by s^2 times a third derivative. The backward is given the sum as it is stored,
    so that adds what a half step of the sum changes: its norm's gradient by 2^-11 of its own size."""
    announce("residual_norm gradients against differences")
    given = case(5, "f16", 6, 64, True, True)
    on = [t.to(device) for t in given]
    total, _ = kernel("residual_norm_f16").run(*on[:5], *NUMBERS)
    got = [t.double().cpu() for t in kernel("residual_norm_backward_f16").run(on[0], total, *on[2:], *NUMBERS)]
    sizes = [size for _, size in plain_backward(given[0], total.cpu(), *given[2:])]
    inputs = [t.double() for t in given[:5]]

    def value(at, v, s):
        moved = list(inputs)
        moved[at] = moved[at] + s * v
        h, _, y, _ = plain(*moved)
        return (h * given[5].double()).sum() + (y * given[6].double()).sum()

    g = torch.Generator().manual_seed(9)
    for at in range(5):
        v = torch.randn(inputs[at].shape, generator=g, dtype=torch.float64)
        slope = (value(at, v, 1e-4) - value(at, v, -1e-4)) / 2e-4
        # rounding of the gradient and of the sum it is formed from (both at most half a step of magnitudes), and the third derivative
        bound = (4 * 2.0 ** -11 * sizes[at] * v.abs()).sum() + 1e-5 * v.abs().pow(3).sum()
        assert abs((got[at] * v).sum() - slope) <= bound, (at, (got[at] * v).sum(), slope)
        # the direction is not one that a wrong gradient would pass: half of it does not
        assert abs(0.5 * (got[at] * v).sum() - slope) > 0 or abs(slope) <= bound


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 2304])
def test_layouts(device, dtype, d):
    """Odd starts and strides, an inner stride of 2, rows of a wider buffer and a broadcast gate: the contiguous values, but for the order
    of a row's sum; nothing is written beside the outputs."""
    announce("residual_norm layouts", dtype, d)
    given = [t.to(device) for t in case(3, dtype, 19, d, True, True)]
    given[2] = given[2][:1].expand(19)
    names = ("residual_norm_", "residual_norm_i8_", "residual_norm_backward_")
    want = [kernel(names[i] + dtype).run(*given[:5], *NUMBERS) for i in range(2)]
    rows = (given[0], want[0][0], *given[2:])
    want.append(kernel(names[2] + dtype).run(*rows, *NUMBERS))

    def shifted(x):
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 3), 7, dtype=x.dtype, device=device)
        wide[..., 1:1 + x.shape[-1]] = x
        return wide[..., 1:1 + x.shape[-1]]

    def spread(x):
        wide = torch.full((*x.shape, 2), 7, dtype=x.dtype, device=device)
        wide[..., 0] = x
        return wide[..., 0]

    def padded(x):
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 32), 7, dtype=x.dtype, device=device)
        wide[..., 16:16 + x.shape[-1]] = x
        return wide[..., 16:16 + x.shape[-1]]

    for change in (shifted, spread, padded):
        for name, inputs, exact in zip(names, (given[:5], given[:5], rows), want):
            moved = [change(t) if t.dim() == 2 or t.shape[0] == d else t for t in inputs]
            outs = [change(torch.zeros_like(t)) for t in exact]
            kernel(name + dtype)(*moved, *outs, *NUMBERS)
            for got, value in zip(outs, exact):
                if value.dtype == torch.int8:
                    assert (got.int() - value.int()).abs().max() <= 1 and (got != value).float().mean() < 0.01
                else:
                    loose = dict(rtol=2 * HALF_STEP[dtype], atol=1e-5) if value.dim() == 2 else dict(rtol=1e-4, atol=1e-4)
                    torch.testing.assert_close(got.float(), value.float(), **loose)
                if change is not padded and got._base is not None:
                    beside = got._base.clone()
                    beside.as_strided(got.shape, got.stride(), got.storage_offset()).fill_(7)
                    assert (beside == 7).all()


@pytest.mark.parametrize("d", [96, 100, 4096])
def test_in_place(device, d):
    """The stream and the norm written over what was read, gradients over the rows they come from."""
    announce("residual_norm in place", d)
    given = [t.to(device) for t in case(8, "bf16", 300, d, True, True)]
    run, run8, back = (kernel(n + "bf16") for n in ("residual_norm_", "residual_norm_i8_", "residual_norm_backward_"))
    want, want8 = run.run(*given[:5], *NUMBERS), run8.run(*given[:5], *NUMBERS)
    grads = back.run(given[0], want[0], *given[2:], *NUMBERS)
    for at in ((1, 0), (0, 1)):
        moved = [t.clone() for t in given]
        run(*moved[:5], moved[at[0]], moved[at[1]], *NUMBERS)
        assert torch.equal(moved[at[0]], want[0]) and torch.equal(moved[at[1]], want[1])
    moved = [t.clone() for t in given]
    run8(*moved[:5], moved[1], torch.empty_like(want8[1]), torch.empty_like(want8[2]), *NUMBERS)
    assert torch.equal(moved[1], want8[0])
    for into in ((0, 5), (6, 1), (5, 6)):
        moved = [t.clone() for t in (given[0], want[0], *given[2:])]
        back(*moved, moved[into[0]], moved[into[1]], *(torch.empty_like(t) for t in grads[2:]), *NUMBERS)
        assert torch.equal(moved[into[0]], grads[0]) and torch.equal(moved[into[1]], grads[1])


def test_special_rows(device):
    """Rows of zeros, infinities, NaN and sizes at the ends of the type stay by themselves."""
    announce("residual_norm special rows")
    given = [t.to(device) for t in case(4, "bf16", 8, 256, False, False)]
    run, run8 = kernel("residual_norm_bf16"), kernel("residual_norm_i8_bf16")
    want, want8 = run.run(*given[:5], *NUMBERS), run8.run(*given[:5], *NUMBERS)
    block, residual = given[0].clone(), given[1].clone()
    block[0], residual[0] = 0, 0
    block[1, 5], block[2, 7], residual[3, 9] = float("nan"), float("inf"), float("-inf")
    block[4], residual[4] = 1e-30, 0
    total, out = run.run(block, residual, *given[2:5], *NUMBERS)
    total8, elements, scales = run8.run(block, residual, *given[2:5], *NUMBERS)
    assert torch.equal(total[5:], want[0][5:]) and torch.equal(out[5:], want[1][5:]) and torch.equal(elements[5:], want8[1][5:])
    assert (total[0] == 0).all() and (out[0] == 0).all() and (elements[0] == 0).all() and scales[0] == 0
    assert out[1].isnan().all() and not total[2].isfinite().all()
    assert scales[1:4].isnan().all() and (elements[1:4] == 0).all() and scales[4:].isfinite().all()
    assert not out[4].isnan().any()
    none = run.run(block[:0], residual[:0], *given[2:5], *NUMBERS)
    assert none[0].shape == (0, 256)
    grads = kernel("residual_norm_backward_bf16").run(block[:0], total[:0], given[2], given[4], given[4], block[:0], block[:0], *NUMBERS)
    assert (grads[3] == 0).all() and (grads[4] == 0).all()
    narrow = run.run(block[:, :0], residual[:, :0], given[2], given[3], given[4][:0], *NUMBERS)
    assert narrow[1].shape == (8, 0)


def test_rows_beyond_32_bits(device):
    announce("residual_norm beyond 32 bits")
    given = case(6, "f16", 3, 64, True, True)
    far = [torch.zeros(2 * 2 ** 31 + 64, dtype=torch.float16, device=device).as_strided((3, 64), (2 ** 31, 1)) for _ in range(2)]
    far[0].copy_(given[0])
    on = [t.to(device) for t in given]
    want = kernel("residual_norm_f16").run(*on[:5], *NUMBERS)
    out = torch.empty_like(want[1])
    kernel("residual_norm_f16")(far[0], *on[1:5], far[1], out, *NUMBERS)
    assert torch.equal(far[1], want[0]) and torch.equal(out, want[1])
    got = kernel("residual_norm_backward_f16").run(far[0], far[1], *on[2:], *NUMBERS)
    for a, b in zip(got, kernel("residual_norm_backward_f16").run(on[0], want[0], *on[2:], *NUMBERS)):
        assert torch.equal(a, b)


def test_refusals(device):
    given = [t.to(device) for t in case(1, "f16", 6, 64, True, True)]
    run, run8, back = (kernel(n + "f16") for n in ("residual_norm_", "residual_norm_i8_", "residual_norm_backward_"))
    with pytest.raises(ValueError, match="gate holds"):
        run.run(*given[:2], given[2][:3], *given[3:5], *NUMBERS)
    with pytest.raises(ValueError, match="post_weight holds"):
        run.run(*given[:3], given[3][:8], given[4], *NUMBERS)
    with pytest.raises(TypeError):
        run.run(given[0].bfloat16(), *given[1:5], *NUMBERS)
    with pytest.raises(ValueError):
        run.run(given[0][:, :32], *given[1:5], *NUMBERS)
    out, square = torch.empty_like(given[0]), torch.empty((64, 64), dtype=torch.float16, device=device)
    with pytest.raises(ValueError, match="overlap"):
        run(*given[:5], given[1], given[1], *NUMBERS)
    with pytest.raises(ValueError, match="overlap"):
        run(*given[:5], square[1:7], square[4:10], *NUMBERS)
    elements = given[0].view(torch.int8)[:, :64]
    with pytest.raises(ValueError, match="overlap"):
        run8(*given[:5], out, elements, torch.empty(6, device=device), *NUMBERS)
    many = [t.to(device) for t in case(1, "f16", 64, 64, True, True)]
    with pytest.raises(ValueError, match="overlap"):                    # scales of 64 tokens over the weights of 64 columns
        run8(*many[:5], torch.empty_like(many[0]), torch.empty((64, 64), dtype=torch.int8, device=device), many[4], *NUMBERS)
    wide = torch.zeros((2, 16385), dtype=torch.float16, device=device)
    with pytest.raises(intent.CompilationStageError, match="16384"):
        run.run(wide, wide, given[2][:0], given[3][:0], torch.ones(16385, device=device), *NUMBERS)
    with pytest.raises(intent.CompilationStageError, match="workspace"):
        kernel("residual_norm_backward_f16", backend_options={"workspace": "static"}).run(given[0], given[1], *given[2:], *NUMBERS)
    kernel("residual_norm_f16", backend_options={"workspace": "static"}).run(*given[:5], *NUMBERS)
    back.run(given[0], given[1], *given[2:], *NUMBERS)


def test_captured_and_other_stream(device):
    """The backward captured twice (its workspaces apart) and replayed between eager calls, and a launch on another stream than the one
    it was prepared on, give the eager results bit for bit."""
    announce("residual_norm captured")
    given = [t.to(device) for t in case(6, "bf16", 257, 512, True, True)]
    args = (given[0], given[1], *given[2:], *NUMBERS)
    run = kernel("residual_norm_backward_bf16")
    want = [a.clone() for a in run.run(*args)]
    call = run.prepare(*args)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call.launch()
        graphs.append(graph)
    side = torch.cuda.Stream()
    for step in range(4):
        for a in call.result():
            a.zero_()
        if step < 3:
            graphs[step % 2].replay()
        else:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                call.launch()
            torch.cuda.current_stream().wait_stream(side)
        run.run(*args)
        torch.cuda.synchronize()
        for a, b in zip(call.result(), want):
            assert torch.equal(a, b)


def test_autograd_registration(device):
    """Forward and authored backward as torch operators: a stream through two layers, whose leaves collect both layers' gradients. The
    64-bit gradients come from torch's own differentiation of the plain form. A layer rounds its sum, its output and four gradients by half
    a step each, of which the other layer's gradients are made, so 8 half steps of the largest magnitudes of a row."""
    announce("residual_norm autograd")
    block, residual, gate, post, weight, grad_sum, grad_output = case(7, "bf16", 12, 64, True, True)
    on = [t.to(device).requires_grad_(True) for t in (block, residual, gate, post, weight)]
    run, back = kernel("residual_norm_bf16"), kernel("residual_norm_backward_bf16")
    run.prepare(*(t.detach() for t in on), *NUMBERS)
    back.prepare(*(t.detach() for t in on), grad_sum.to(device), grad_output.to(device), *NUMBERS)
    operation = run.as_torch_op("intent_amd_tests::residual_norm")
    backward_operation = back.as_torch_op("intent_amd_tests::residual_norm_backward")

    def setup_context(ctx, inputs, output):
        ctx.save_for_backward(inputs[0], output[0], *inputs[2:5])
        ctx.numbers = inputs[5:]

    def backward_formula(ctx, grad_sum, grad_output):
        return (*backward_operation(*ctx.saved_tensors, grad_sum.contiguous(), grad_output.contiguous(), *ctx.numbers), None, None, None)

    operation.register_autograd(backward_formula, setup_context=setup_context)
    total, out = operation(*on, *NUMBERS)
    total, out = operation(out, total, *on[2:], *NUMBERS)
    ((total.float() * grad_sum.to(device).float()).sum() + (out.float() * grad_output.to(device).float()).sum()).backward()
    leaves = [t.double().requires_grad_(True) for t in (block, residual, gate, post, weight)]

    def norm(x, w):
        return x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + NUMBERS[2]) * w

    def layer(x, s):
        h = NUMBERS[0] * s + NUMBERS[1] * leaves[2][:, None] * norm(x, leaves[3])
        return h, norm(h, leaves[4])

    h, y = layer(leaves[0], leaves[1])
    h, y = layer(y, h)
    ((h * grad_sum.double()).sum() + (y * grad_output.double()).sum()).backward()
    for got, want in zip(on, leaves):
        error = (got.grad.double().cpu() - want.grad).abs()
        scale = want.grad.abs().amax(-1, keepdim=True) if want.dim() == 2 else want.grad.abs().max() + want.grad.abs().mean() * 12 ** 0.5
        assert (error <= 8 * 2.0 ** -8 * scale).all(), (error / scale).max()
