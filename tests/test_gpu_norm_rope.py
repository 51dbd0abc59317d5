"""qk_norm_rope and qk_norm_rope_backward against their 64-bit forms, and the gradients against differences.

Bars. The kernels work in f32 and round once. A row's sum of squares has at most 16 + 10 additions in a chain and the rsqrt
two units in the last place, the products and the turn five more roundings: below 40 * 2^-24 < 2^-18 of the magnitudes that
an element is formed from; then half a step of the storage type, 2^-11 (f16) or 2^-8 (bf16) of the value, or half the
smallest f16 subnormal. A gradient element passes through a second such sum: 2^-17. The weights' gradients add to the terms'
2^-18 a chain of at most 300 additions: 2^-15 of the sum of magnitudes."""
import pytest
import torch

import intent_amd as intent
from intent_amd.examples.kernels.backward import qk_norm_rope as backward
from intent_amd.examples.kernels.normalization import qk_norm_rope as forward
from tests import plain64
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
EPS = 1e-6


def kernel(name, interleaved=False):
    module = backward if "backward" in name else forward
    return intent.jit(getattr(module, name), backend="hip", constexprs={"INTERLEAVED": interleaved})


def tables(pairs, rows=4096):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(1, pairs))
    return angle.cos().float(), angle.sin().float()


def case(seed, dtype, tokens, q_heads, kv_heads, d, pairs):
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn((tokens, q_heads + 2 * kv_heads, d), generator=g).mul(2).to(TYPES[dtype])
    weights = 1 + 0.3 * torch.randn((2, d), generator=g)
    positions = torch.randint(0, 4096, (tokens,), generator=g, dtype=torch.int32)
    grads = [torch.randn((tokens, h, d), generator=g).to(TYPES[dtype]) for h in (q_heads, kv_heads)]
    return rows, weights, positions, *tables(pairs), *grads


def close(got, want, size, dtype, units):
    got = got.double().cpu()
    assert not got.isnan().any()
    bound = HALF_STEP[dtype] * want.abs() + units * size + (2.0 ** -25 if dtype == "f16" else 0)
    worst = (got - want).abs() - bound
    assert (worst <= 0).all(), f"off by {(got - want).abs().flatten()[worst.argmax()]} against {want.flatten()[worst.argmax()]}"


SHAPES = [(1, 1, 1, 64, 32, False), (8, 32, 8, 128, 64, False), (8, 32, 8, 128, 64, True), (33, 4, 4, 64, 16, True),
          (33, 5, 1, 64, 16, False), (7, 3, 2, 80, 40, False), (7, 15, 5, 96, 24, True), (5, 2, 2, 256, 128, False),
          (3, 2, 1, 256, 32, True), (2, 1, 1, 1024, 512, False), (2, 1, 1, 1024, 100, True), (9, 2, 1, 20, 3, False),
          (9, 2, 1, 21, 10, True), (4, 2, 2, 1, 0, False), (6, 2, 2, 128, 0, False), (6, 2, 2, 48, 24, False),
          (6, 3, 2, 128, 12, True), (301, 64, 8, 128, 64, False), (1021, 16, 16, 64, 32, True)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,d,pairs,interleaved", SHAPES)
def test_forward_and_backward(device, dtype, tokens, q_heads, kv_heads, d, pairs, interleaved):
    announce("qk_norm_rope", dtype, tokens, q_heads, kv_heads, d, pairs, interleaved)
    rows, weights, positions, cos, sin, grad_q, grad_k = case(tokens + d, dtype, tokens, q_heads, kv_heads, d, pairs)
    on = rows.to(device)
    q, k = on[:, :q_heads], on[:, q_heads:q_heads + kv_heads]          # slices of the projection
    common = (q, k, *weights.to(device), positions.to(device), cos.to(device), sin.to(device))
    out = kernel(f"qk_norm_rope_{dtype}", interleaved).run(*common, EPS)
    got = kernel(f"qk_norm_rope_backward_{dtype}", interleaved).run(*common, grad_q.to(device), grad_k.to(device), EPS)
    again = kernel(f"qk_norm_rope_backward_{dtype}", interleaved).run(*common, grad_q.to(device), grad_k.to(device), EPS)
    for a, b in zip(got, again):
        assert torch.equal(a, b)                                       # sums in a fixed order
    for i, (x, grad) in enumerate(((rows[:, :q_heads], grad_q), (rows[:, q_heads:q_heads + kv_heads], grad_k))):
        want, size = plain64.norm_rope(x, weights[i], positions, cos, sin, EPS, interleaved)
        close(out[i], want, size, dtype, 2.0 ** -18)
        dx, dx_size, dw, dw_size = plain64.norm_rope_backward(x, weights[i], grad, positions, cos, sin, EPS, interleaved)
        close(got[i], dx, dx_size, dtype, 2.0 ** -17)
        error = (got[2 + i].double().cpu() - dw).abs()
        assert (error <= 2.0 ** -15 * dw_size + 1e-37).all(), error.max()


def test_gradients_against_differences(device):
    """Along random directions, the gradients give the change of sum(out * grad) that the 64-bit forward has between
    x - h v and x + h v: a central difference, off by its third derivative (h^2) and the rounding of grad_x."""
    announce("qk_norm_rope gradients against differences")
    rows, weights, positions, cos, sin, grad_q, grad_k = case(5, "f16", 6, 3, 2, 64, 24)
    on = rows.to(device)
    got = kernel("qk_norm_rope_backward_f16").run(on[:, :3], on[:, 3:5], *weights.to(device), positions.to(device), cos.to(device),
                                                  sin.to(device), grad_q.to(device), grad_k.to(device), EPS)
    g = torch.Generator().manual_seed(9)
    for i, (x, grad) in enumerate(((rows[:, :3], grad_q), (rows[:, 3:5], grad_k))):
        def value(x, w):
            return (plain64.norm_rope(x, w, positions, cos, sin, EPS, False)[0] * grad.double()).sum()
        h = 1e-4
        v = torch.randn(x.shape, generator=g, dtype=torch.float64)
        slope = (value(x.double() + h * v, weights[i]) - value(x.double() - h * v, weights[i])) / (2 * h)
        dx = got[i].double().cpu()
        # half a step of each element times |v|, and h^2 times a third derivative of order sum |v|^3
        assert abs((dx * v).sum() - slope) <= (2.0 ** -11 * dx.abs() * v.abs()).sum() + 1e-6 * v.abs().pow(3).sum()
        v = torch.randn(weights[i].shape, generator=g, dtype=torch.float64)
        slope = value(x.double(), weights[i].double() + v) - value(x.double(), weights[i].double())    # linear in the weight
        dw = got[2 + i].double().cpu()
        assert abs((dw * v).sum() - slope) <= 2.0 ** -15 * (plain64.norm_rope_backward(
            x, weights[i], grad, positions, cos, sin, EPS, False)[3] * v.abs()).sum()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_layouts(device, dtype):
    """Head-major rows, a start that is no multiple of 16 bytes, a stride that is no multiple of 8, an inner stride of 2,
    padded outputs and tables, and odd weights give the values of contiguous ones bit for bit."""
    announce("qk_norm_rope layouts", dtype)
    rows, weights, positions, cos, sin, grad_q, grad_k = (a.to(device) for a in case(3, dtype, 19, 4, 2, 64, 16))
    q, k = rows[:, :4].contiguous(), rows[:, 4:6].contiguous()
    run = lambda q, k, w, c, s: kernel(f"qk_norm_rope_{dtype}").run(q, k, *w, positions, c, s, EPS)  # noqa: E731
    back = lambda q, k, w, c, s, gq, gk: kernel(f"qk_norm_rope_backward_{dtype}").run(  # noqa: E731
        q, k, *w, positions, c, s, gq, gk, EPS)
    want, grads = run(q, k, weights, cos, sin), back(q, k, weights, cos, sin, grad_q, grad_k)

    def head_major(x):
        return x.transpose(0, 1).contiguous().transpose(0, 1)

    def shifted(x):
        wide = torch.zeros((*x.shape[:-1], x.shape[-1] + 3), dtype=x.dtype, device=device)
        wide[..., 1:1 + x.shape[-1]] = x
        return wide[..., 1:1 + x.shape[-1]]

    def spread(x):
        wide = torch.zeros((*x.shape, 2), dtype=x.dtype, device=device)
        wide[..., 0] = x
        return wide[..., 0]

    for change in (head_major, shifted, spread):
        odd = change(weights[:, None])[:, 0] if change is not head_major else weights
        table = (cos, sin) if change is head_major else (change(cos), change(sin))
        # a layout may change the kernel, and with it the order of a row's sum: a step of the storage type at most
        for got, exact in zip(run(change(q), change(k), odd, *table), want):
            torch.testing.assert_close(got.float(), exact.float(), rtol=2 * HALF_STEP[dtype], atol=1e-6)
        outs = [change(torch.zeros_like(a)) for a in want]
        kernel(f"qk_norm_rope_{dtype}")(change(q), change(k), *odd, positions, *table, *outs, EPS)
        for got, exact in zip(outs, want):
            torch.testing.assert_close(got.float(), exact.float(), rtol=2 * HALF_STEP[dtype], atol=1e-6)
        for i, (got, exact) in enumerate(zip(back(change(q), change(k), odd, *table, change(grad_q), change(grad_k)), grads)):
            loose = dict(rtol=2 * HALF_STEP[dtype], atol=1e-5) if i < 2 else dict(rtol=1e-4, atol=1e-4)
            torch.testing.assert_close(got.float(), exact.float(), **loose)


def test_positions_clamped_and_special_values(device):
    """Positions outside the tables take the nearest row; zero rows stay zero; a NaN or infinity stays in its row; the
    other head kind may be absent."""
    announce("qk_norm_rope special values")
    rows, weights, positions, cos, sin, grad_q, grad_k = (a.to(device) for a in case(4, "f16", 6, 4, 2, 128, 64))
    run = lambda q, k, p: kernel("qk_norm_rope_f16").run(q, k, *weights, p, cos, sin, EPS)  # noqa: E731
    q, k = rows[:, :4], rows[:, 4:6]
    far = torch.tensor([-1, -2 ** 31, 4096, 2 ** 31 - 1, 0, 4095], dtype=torch.int32, device=device)
    near = torch.tensor([0, 0, 4095, 4095, 0, 4095], dtype=torch.int32, device=device)
    for a, b in zip(run(q, k, far), run(q, k, near)):
        assert torch.equal(a, b)
    want = run(q, k, positions)
    odd = rows.clone()
    odd[0, 0], odd[1, 1, 5], odd[2, 2, 7], odd[3, 3] = 0, float("nan"), float("inf"), 6e-8
    got = run(odd[:, :4], odd[:, 4:6], positions)[0]
    same = torch.ones((6, 4), dtype=torch.bool, device=device)
    same[0, 0] = same[1, 1] = same[2, 2] = same[3, 3] = False
    assert torch.equal(got[same], want[0][same])
    assert (got[0, 0] == 0).all() and got[1, 1].isnan().all() and not got[3, 3].isnan().any()
    assert got[2, 2].isnan().sum() == 2              # inf * 0 turns its pair NaN; the rest of the row is 0
    empty = rows[:, :0]
    assert torch.equal(run(q, empty, positions)[0], want[0]) and torch.equal(run(empty, k, positions)[1], want[1])
    none = kernel("qk_norm_rope_backward_f16").run(q[:0], k[:0], *weights, positions[:0], cos, sin, grad_q[:0], grad_k[:0], EPS)
    assert (none[2] == 0).all() and (none[3] == 0).all()
    only = kernel("qk_norm_rope_backward_f16").run(q, empty, *weights, positions, cos, sin, grad_q, grad_k[:, :0], EPS)
    assert (only[3] == 0).all() and only[2].abs().max() > 0


def test_refusals(device):
    rows, weights, positions, cos, sin, grad_q, grad_k = (a.to(device) for a in case(4, "f16", 6, 4, 2, 64, 32))
    q, k = rows[:, :4], rows[:, 4:6]
    forward_ = kernel("qk_norm_rope_f16")
    with pytest.raises(ValueError, match="do not fit"):
        forward_.run(q, k, *weights, positions, *(a.to(device) for a in tables(33)), EPS)
    with pytest.raises(ValueError, match="hold no position"):
        forward_.run(q, k, *weights, positions, cos[:0], sin[:0], EPS)
    with pytest.raises(ValueError):
        forward_.run(q, k[..., :32], *weights, positions, cos, sin, EPS)
    with pytest.raises(TypeError):
        forward_.run(q.bfloat16(), k, *weights, positions, cos, sin, EPS)
    with pytest.raises(ValueError, match="overlap"):
        forward_(q, k, *weights, positions, cos, sin, q, torch.empty_like(k), EPS)
    wide = torch.zeros((2, 1, 1088), dtype=torch.float16, device=device)
    with pytest.raises(intent.CompilationStageError, match="1024"):
        forward_.run(wide, wide.clone(), *torch.ones((2, 1088), device=device), positions[:2], cos, sin, EPS)
    with pytest.raises(intent.CompilationStageError, match="INTERLEAVED"):
        intent.jit(forward.qk_norm_rope_f16, backend="hip", constexprs={"INTERLEAVED": 2}).run(q, k, *weights, positions, cos, sin, EPS)
    static = intent.jit(backward.qk_norm_rope_backward_f16, backend="hip", constexprs={"INTERLEAVED": False},
                        backend_options={"workspace": "static"})
    with pytest.raises(intent.CompilationStageError, match="workspace"):
        static.run(q, k, *weights, positions, cos, sin, grad_q, grad_k, EPS)


def test_captured_and_other_stream(device):
    """The backward captured twice (its workspaces apart) and replayed between eager calls, and a launch on another stream
    than the one it was prepared on, give the eager results bit for bit."""
    announce("qk_norm_rope captured")
    rows, weights, positions, cos, sin, grad_q, grad_k = (a.to(device) for a in case(6, "bf16", 257, 8, 2, 128, 64))
    args = (rows[:, :8], rows[:, 8:10], *weights, positions, cos, sin, grad_q, grad_k, EPS)
    run = kernel("qk_norm_rope_backward_bf16")
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
    """Forward and authored backward as torch operators: leaves used by two calls, of which one shares a packed projection,
    collect the sum of both calls' gradients."""
    announce("qk_norm_rope autograd")
    rows, weights, positions, cos, sin, grad_q, grad_k = case(5, "bf16", 12, 4, 2, 64, 32)
    forward_kernel, backward_kernel = kernel("qk_norm_rope_bf16"), kernel("qk_norm_rope_backward_bf16")
    packed = rows.to(device).requires_grad_(True)
    leaves = [w.to(device).requires_grad_(True) for w in weights]
    tables_on = (positions.to(device), cos.to(device), sin.to(device))
    grads = (grad_q.to(device), grad_k.to(device))
    split = lambda t: (t[:, :4], t[:, 4:6])          # noqa: E731
    forward_kernel.prepare(*split(packed.detach()), *(w.detach() for w in leaves), *tables_on, EPS)
    backward_kernel.prepare(*split(packed.detach()), *(w.detach() for w in leaves), *tables_on, *grads, EPS)
    operation = forward_kernel.as_torch_op("intent_amd_tests::qk_norm_rope")
    backward_operation = backward_kernel.as_torch_op("intent_amd_tests::qk_norm_rope_backward")

    def setup_context(ctx, inputs, output):
        ctx.save_for_backward(*inputs[:7])
        ctx.eps = inputs[7]

    def backward_formula(ctx, dq, dk):
        return (*backward_operation(*ctx.saved_tensors, dq.contiguous(), dk.contiguous(), ctx.eps), None, None, None, None)

    operation.register_autograd(backward_formula, setup_context=setup_context)
    total = 0
    for _ in range(2):
        q, k = operation(*split(packed), *leaves, *tables_on, EPS)
        total = total + (q.float() * grads[0].float()).sum() + (k.float() * grads[1].float()).sum()
    total.backward()
    assert (packed.grad[:, 6:] == 0).all()
    for i, grad in enumerate((grad_q, grad_k)):
        x = split(rows)[i]
        dx, dx_size, dw, dw_size = plain64.norm_rope_backward(x, weights[i], grad, positions, cos, sin, EPS, False)
        # twice the gradient, each call's and their sum rounded to bf16
        close(split(packed.grad)[i] / 2, dx, dx_size, "bf16", 2.0 ** -17 + 2 * 2.0 ** -8)
        bound = 2.0 ** -15 * dw_size + 2.0 ** -23 * dw.abs()
        assert ((leaves[i].grad.double().cpu() / 2 - dw).abs() <= bound).all()
