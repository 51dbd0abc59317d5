"""What a decode step on an 8-bit paged cache with 4-bit weights is measured on, and the training pass of its norm: the calls
that a user's program makes of the operators, and the same in elementary torch operations.

The step's parts: the norm of every query and key head with the rotation of its position (and its gradients, for training),
the cache pages of e4m3 elements with a shared power of two per 32 of them, written as tokens come and read back, the
attention of one new token over those pages, and the products with e2m1 weights.
"""
import functools
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
TABLE = 32768          # positions of the rotation tables
BLOCK = 32             # elements that share an exponent


def listed():
    return [
        # One decode step of 8 sequences: the smallest call, latency is all of it.
        {"name": "norm_step", "op": "norm", "dtype": "f16", "tokens": 8, "heads": 32, "kv_heads": 8, "dim": 128, "pairs": 64,
         "interleaved": False},
        # A training batch of 4 sequences of 4096 tokens.
        {"name": "norm_batch", "op": "norm", "dtype": "bf16", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "pairs": 64, "interleaved": False},
        # Its backward pass.
        {"name": "norm_backward_batch", "op": "norm_backward", "dtype": "bf16", "tokens": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "pairs": 64, "interleaved": False},
        # A fine-tuning step over a ragged number of tokens: narrow heads, of which half is rotated, pairs side by side.
        {"name": "norm_backward_ragged", "op": "norm_backward", "dtype": "f16", "tokens": 1021, "heads": 16, "kv_heads": 16,
         "dim": 64, "pairs": 16, "interleaved": True},
        # The new tokens of a step of 32 sequences go into the cache.
        {"name": "append_step", "op": "append", "dtype": "f16", "sequences": 32, "longest": 2048, "new": 1, "kv_heads": 8,
         "dim": 128, "page": 64, "head_major": True},
        # Packed prompts of different lengths go into the cache.
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "sequences": 8, "longest": 8191, "new": 8191, "kv_heads": 8,
         "dim": 128, "page": 64, "head_major": True},
        # Cached prefixes come back in 16 bits, for a prompt that goes on from them.
        {"name": "read_prefixes", "op": "read", "dtype": "f16", "sequences": 8, "longest": 8191, "kv_heads": 8, "dim": 128,
         "page": 64, "head_major": True},
        # One step over 8 long sequences (about 7300 tokens each).
        {"name": "decode_long", "op": "decode", "dtype": "f16", "sequences": 8, "longest": 8191, "even": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "head_major": True},
        # One step of a full server: 64 sequences from one token to 8191, pages with their heads side by side.
        {"name": "decode_server", "op": "decode", "dtype": "bf16", "sequences": 64, "longest": 8191, "even": False, "heads": 64,
         "kv_heads": 8, "dim": 128, "page": 16, "head_major": False},
        # A feed-forward projection of one token.
        {"name": "linear_row", "op": "linear", "dtype": "f16", "m": 1, "n": 14336, "k": 4096},
        # The same of a step of 32 sequences, the way back.
        {"name": "linear_step", "op": "linear", "dtype": "bf16", "m": 32, "n": 4096, "k": 14336},
        # The same of a prompt.
        {"name": "linear_prompt", "op": "linear", "dtype": "f16", "m": 1021, "n": 14336, "k": 4096},
    ]


# ------------------------------------------------------------------------------------------ drawing
def _spread(rng, low, high, multiple=1):
    """A size between low and high, even over its logarithm, a multiple of `multiple`."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high // multiple, max(-(-low // multiple), round(value / multiple))) * multiple


def draw(rng):
    """One more case: token counts, lengths and batches are arbitrary, widths are those of models."""
    op = rng.choice(["norm", "norm_backward", "append", "read", "decode", "linear"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "linear":
        n, k = _spread(rng, 512, 16384, rng.choice([1, 8, 16])), _spread(rng, 512, 16384, BLOCK)
        most = max(1, 1021 * 14336 * 4096 // (n * k))
        return {"op": op, "dtype": dtype, "m": min(most, _spread(rng, 1, rng.choice([16, 128, 2048]))), "n": n, "k": k}
    kv_heads, group = rng.choice([(8, 4), (4, 8), (8, 8), (2, 4), (16, 1), (1, 16), (5, 3), (8, 1)])
    if op in ("norm", "norm_backward"):
        dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        heads = kv_heads * group
        tokens = min(_spread(rng, 1, 16384), 16384 * 40 * 128 // ((heads + kv_heads) * dim))
        return {"op": op, "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "pairs": dim // rng.choice([2, 2, 2, 4]), "interleaved": rng.random() < 0.4}
    case = {"op": op, "dtype": dtype, "sequences": _spread(rng, 1, 64), "longest": _spread(rng, 16, 8191),
            "kv_heads": kv_heads, "dim": rng.choice([64, 96, 128, 128, 256]), "page": rng.choice([16, 32, 64]),
            "head_major": rng.random() < 0.5}
    tokens = 64 * 8191 * 8 * 128 // 2 // (kv_heads * case["dim"])
    case["longest"] = max(16, min(case["longest"], tokens // case["sequences"]))
    if op == "append":
        case["longest"] = min(case["longest"], 65536 // case["sequences"])
        case["new"] = rng.choice([1, 1, rng.randint(2, 8), case["longest"]])
    if op == "read":
        case["longest"] = min(case["longest"], 65536 // case["sequences"])
    if op == "decode":
        case["heads"], case["even"] = kv_heads * group, rng.random() < 0.5
    return case


# ------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(DTYPES[dtype])


def _table(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


@functools.lru_cache(maxsize=None)
def _rotation(pairs):
    """Cosine and sine of position * 10000^(-i / pairs), formed in 64 bits (a program makes them once)."""
    rate = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    angle = torch.arange(TABLE, dtype=torch.float64)[:, None] * rate
    return angle.cos().float().to(DEVICE), angle.sin().float().to(DEVICE)


def _lengths(case):
    """Tokens of each sequence after the call, the longest among them: part of the case, not of its inputs."""
    count, longest = case["sequences"], case["longest"]
    if case.get("even"):     # sequences of similar age, from three quarters of the longest up
        return [longest - (longest // 4) * i // count for i in range(count)]
    rng = random.Random(count * 8191 + longest)
    return [longest] + [rng.randint(1, longest) for _ in range(count - 1)]


def _new(case):
    return [min(case["new"], n) for n in _lengths(case)]


def _sums(values):
    out = [0]
    for value in values:
        out.append(out[-1] + value)
    return out


def _pages(g, case):
    """Page tables of sequences whose pages are scattered over the cache."""
    offsets = _sums(-(-n // case["page"]) for n in _lengths(case))
    indices = torch.randperm(offsets[-1], generator=g, device=DEVICE).to(torch.int32)
    return offsets[-1], _table(offsets), indices


def _cache(g, case, pages):
    """Elements and exponents as earlier steps left them; [pages, page, heads, dim] views of pages that hold their heads
    one after another (head_major) or side by side."""
    hk, page, dim = case["kv_heads"], case["page"], case["dim"]
    shape = (pages, hk, page) if case["head_major"] else (pages, page, hk)
    elements = (torch.randn((*shape, dim), generator=g, device=DEVICE) * 96).clamp_(-448, 448).to(torch.float8_e4m3fn)
    exponents = torch.randint(118, 122, (*shape, dim // BLOCK), generator=g, device=DEVICE, dtype=torch.uint8)
    if case["head_major"]:
        return elements.transpose(1, 2), exponents.transpose(1, 2)
    return elements, exponents


def prepare(case, seed):
    g, op, dtype = _generator(seed), case["op"], case.get("dtype")
    s = dict(case)
    if op == "linear":
        n, k = case["n"], case["k"]
        s["x"] = _normal(g, (case["m"], k), dtype)
        s["weight"] = torch.randint(0, 256, (n, k // 2), generator=g, device=DEVICE, dtype=torch.uint8)
        s["exponents"] = torch.randint(117, 123, (n, k // BLOCK), generator=g, device=DEVICE, dtype=torch.uint8)
        return s
    hk, dim = case["kv_heads"], case["dim"]
    if op in ("norm", "norm_backward"):
        # Queries and keys are slices of one projection's rows, which hold the values too.
        t, hq = case["tokens"], case["heads"]
        projected = _normal(g, (t, hq + 2 * hk, dim), dtype, 2)
        s["q"], s["k"] = projected[:, :hq], projected[:, hq:hq + hk]
        s["q_weight"], s["k_weight"] = (1 + 0.2 * torch.randn((2, dim), generator=g, device=DEVICE)).unbind()
        s["positions"] = torch.randint(0, TABLE, (t,), generator=g, device=DEVICE, dtype=torch.int32)
        s["cos"], s["sin"] = _rotation(case["pairs"])
        if op == "norm_backward":
            s["grad_q"], s["grad_k"] = _normal(g, (t, hq, dim), dtype), _normal(g, (t, hk, dim), dtype)
        return s
    pages, s["page_offsets"], s["page_indices"] = _pages(g, case)
    s["key_cache"], s["key_exponents"] = _cache(g, case, pages)
    s["value_cache"], s["value_exponents"] = _cache(g, case, pages)
    s["lengths"] = _table(_lengths(case))
    if op == "append":
        new = _new(case)
        s["cu_seqlens"] = _table(_sums(new))
        s["k"], s["v"] = _normal(g, (sum(new), hk, dim), dtype, 2), _normal(g, (sum(new), hk, dim), dtype)
    if op == "read":
        s["cu_seqlens"] = _table(_sums(_lengths(case)))
        s["rows"] = sum(_lengths(case))
    if op == "decode":
        s["q"] = _normal(g, (case["sequences"], case["heads"], dim), dtype)
        s["scale"] = dim ** -0.5
        s["most"] = max(_lengths(case))
    return s


# ------------------------------------------------------------------------------------------ the framework's calls
@functools.lru_cache(maxsize=None)
def _kernel(name, **constexprs):
    """A program jits a definition once and keeps the kernel."""
    import intent_amd as intent
    from intent_amd.examples.kernels.backward import qk_norm_rope as backward
    from intent_amd.examples.kernels.contraction import linear_mxfp4
    from intent_amd.examples.kernels.normalization import qk_norm_rope
    from intent_amd.examples.kernels.streaming import mx_cache

    for module in (qk_norm_rope, backward, mx_cache, linear_mxfp4):
        if hasattr(module, name):
            return intent.jit(getattr(module, name), backend="hip", constexprs=constexprs)
    raise LookupError(name)


def _stepped(s, kernel, *arguments):
    """A decode loop prepares a call for its buffers once and launches it every step."""
    if "call" not in s:
        s["call"] = kernel.prepare(*arguments)
    s["call"].launch()
    return s["call"].result()


def _call(s):
    op, dtype = s["op"], s["dtype"]
    if op == "linear":
        kernel = _kernel("linear_mxfp4_" + dtype)
        if s["m"] > 128:             # a prompt comes once
            return kernel.run(s["x"], s["weight"], s["exponents"])
        return _stepped(s, kernel, s["x"], s["weight"], s["exponents"])
    if op == "norm":
        kernel = _kernel("qk_norm_rope_" + dtype, INTERLEAVED=s["interleaved"])
        arguments = (s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["cos"], s["sin"], EPS)
        return kernel.run(*arguments) if s["tokens"] > 128 else _stepped(s, kernel, *arguments)
    if op == "norm_backward":
        return _kernel("qk_norm_rope_backward_" + dtype, INTERLEAVED=s["interleaved"]).run(
            s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["cos"], s["sin"], s["grad_q"], s["grad_k"], EPS)
    cache = (s["key_cache"], s["key_exponents"], s["value_cache"], s["value_exponents"])
    if op == "append":
        kernel = _kernel("paged_cache_append_" + dtype)
        arguments = (s["k"], s["v"], *cache, s["cu_seqlens"], s["page_offsets"], s["page_indices"], s["lengths"])
        if s["new"] > 8:
            kernel.run(*arguments)
        else:
            _stepped(s, kernel, *arguments)
        return cache
    if op == "read":
        k, v = (torch.empty((s["rows"], s["kv_heads"], s["dim"]), dtype=DTYPES[dtype], device=DEVICE) for _ in range(2))
        _kernel("paged_cache_read_" + dtype)(*cache, s["cu_seqlens"], s["page_offsets"], s["page_indices"], k, v)
        return k, v
    return _stepped(s, _kernel("paged_gqa_decode_mx_" + dtype, HEAD_GROUP=s["heads"] // s["kv_heads"]), s["q"], *cache,
                    s["page_offsets"], s["page_indices"], s["lengths"], s["scale"])


# ------------------------------------------------------------------------------------------ the plain forms
def _apart(x, pairs, interleaved):
    """The two halves of the rotated pairs of x, and what is not rotated."""
    if interleaved:
        return x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2], x[..., 2 * pairs:]
    return x[..., :pairs], x[..., pairs:2 * pairs], x[..., 2 * pairs:]


def _together(a, b, rest, interleaved):
    return torch.cat((torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1), rest), -1)


def _rotated(x, s, sign):
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], sign * s["sin"][at][:, None]
    a, b, rest = _apart(x, s["pairs"], s["interleaved"])
    return _together(a * cos - b * sin, b * cos + a * sin, rest, s["interleaved"])


def _plain_norm(x, weight, s):
    x = x.float()
    inverse = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return _rotated(x * inverse * weight, s, 1).to(DTYPES[s["dtype"]])


def _plain_norm_backward(x, weight, grad, s):
    x, grad = x.float(), _rotated(grad.float(), s, -1)
    inverse = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    unit, inner = x * inverse, grad * weight
    grad_x = inverse * (inner - unit * (inner * unit).mean(-1, keepdim=True))
    # The weight's gradient sums over every token and head, so in 64 bits.
    return grad_x.to(DTYPES[s["dtype"]]), (grad * unit).sum((0, 1), dtype=torch.float64).float()


def _quantised(x):
    """Elements (as bytes) and exponent bytes of rows [..., D]: the smallest power of two that brings a block within 448."""
    blocks = x.float().unflatten(-1, (-1, BLOCK))
    size = torch.where(blocks.isfinite(), blocks.abs(), 0.0).amax(-1)
    mantissa, exponent = torch.frexp(size)
    exponent = torch.where(size > 0, (exponent - 9 + (mantissa > 0.875)).clamp_min(-127), -127)
    elements = torch.ldexp(blocks, -exponent[..., None]).to(torch.float8_e4m3fn).flatten(-2)
    return elements.view(torch.uint8), (exponent + 127).to(torch.uint8)


def _slots(sequence, position, s):
    """Page and place in it of tokens of sequences."""
    page = s["page_indices"].long()[s["page_offsets"].long()[sequence] + position // s["page"]]
    return page, position % s["page"]


def _packed(cu, rows):
    """Sequence of each of `rows` packed rows, and its place in the sequence."""
    row = torch.arange(rows, device=DEVICE)
    cu = cu.long()
    sequence = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    return sequence, row - cu[sequence]


def _plain_append(s):
    cu, rows = s["cu_seqlens"].long(), s["k"].shape[0]
    sequence, place = _packed(cu, rows)
    position = s["lengths"].long()[sequence] - (cu[1:] - cu[:-1])[sequence] + place
    at = _slots(sequence, position, s)
    for rows_, cache, exponents in ((s["k"], s["key_cache"], s["key_exponents"]),
                                    (s["v"], s["value_cache"], s["value_exponents"])):
        cache.view(torch.uint8)[at], exponents[at] = _quantised(rows_)
    return s["key_cache"], s["key_exponents"], s["value_cache"], s["value_exponents"]


def _values(cache, exponents, at):
    """What the cache holds at slots, in f32."""
    elements = cache.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
    return elements * torch.exp2(exponents[at].float() - 127).repeat_interleave(BLOCK, -1)


def _plain_read(s):
    at = _slots(*_packed(s["cu_seqlens"], s["rows"]), s)
    return tuple(_values(s[x + "_cache"], s[x + "_exponents"], at).to(DTYPES[s["dtype"]]) for x in ("key", "value"))


def _plain_decode(s):
    count, hk = s["sequences"], s["kv_heads"]
    position = torch.arange(s["most"], device=DEVICE)
    live = position < s["lengths"][:, None]
    sequence = torch.arange(count, device=DEVICE)[:, None].expand_as(live)
    at = _slots(sequence, torch.where(live, position, 0), s)
    keys = _values(s["key_cache"], s["key_exponents"], at).transpose(1, 2).contiguous()       # [B, HK, T, D]
    q = s["q"].float().unflatten(1, (hk, -1))
    scores = (keys @ q.transpose(2, 3).contiguous()).transpose(2, 3) * s["scale"]
    scores = scores.masked_fill(~live[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    values = _values(s["value_cache"], s["value_exponents"], at).transpose(1, 2).contiguous()
    out = (weights @ values) / weights.sum(-1, keepdim=True)
    return out.flatten(1, 2).to(DTYPES[s["dtype"]])


def _plain_linear(s):
    bits = torch.stack((s["weight"] & 15, s["weight"] >> 4), -1).flatten(-2)
    element = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=DEVICE)[bits.int()]
    weight = element * torch.exp2(s["exponents"].float() - 127).repeat_interleave(BLOCK, -1)
    return (s["x"].float() @ weight.t()).to(DTYPES[s["dtype"]])


def _plain(s):
    op = s["op"]
    if op == "norm":
        return _plain_norm(s["q"], s["q_weight"], s), _plain_norm(s["k"], s["k_weight"], s)
    if op == "norm_backward":
        grad_q, grad_q_weight = _plain_norm_backward(s["q"], s["q_weight"], s["grad_q"], s)
        grad_k, grad_k_weight = _plain_norm_backward(s["k"], s["k_weight"], s["grad_k"], s)
        return grad_q, grad_k, grad_q_weight, grad_k_weight
    return {"append": _plain_append, "read": _plain_read, "decode": _plain_decode, "linear": _plain_linear}[op](s)


def run(state):
    return _call(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k // 2 + n * k // BLOCK + 2 * m * (n + k), "flops": 2 * m * n * k}
    hk, dim = case["kv_heads"], case["dim"]
    if op in ("norm", "norm_backward"):
        elements = case["tokens"] * (case["heads"] + hk) * dim
        once = 4 * case["tokens"] + 8 * min(case["tokens"], TABLE) * case["pairs"]
        return {"bytes": elements * (4 if op == "norm" else 6) + once, "flops": elements * (10 if op == "norm" else 20)}
    held = 2 * hk * (dim + dim // BLOCK)                  # bytes of a token's keys and values in the cache
    if op == "append":
        return {"bytes": sum(_new(case)) * (4 * hk * dim + held), "flops": sum(_new(case)) * 4 * hk * dim}
    tokens = sum(_lengths(case))
    if op == "read":
        return {"bytes": tokens * (4 * hk * dim + held), "flops": tokens * 2 * hk * dim}
    return {"bytes": tokens * held + case["sequences"] * case["heads"] * dim * 4, "flops": 4 * tokens * case["heads"] * dim}


# ------------------------------------------------------------------------------------------ exact results
def _exact_turn(case, s, grad):
    """Cosine and sine of each token's angles as complex factors, conjugated for the way back."""
    at = s["positions"].long()
    factor = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
    return factor.conj().resolve_conj() if grad else factor


def _exact_rotate(case, x, factor):
    r = case["pairs"]
    turned = x.clone()
    if case["interleaved"]:
        z = torch.view_as_complex(x[..., :2 * r].unflatten(-1, (r, 2)).contiguous()) * factor
        turned[..., :2 * r] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :r].contiguous(), x[..., r:2 * r].contiguous()) * factor
        turned[..., :r], turned[..., r:2 * r] = z.real, z.imag
    return turned


def _exact_norm(case, s):
    outs = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x = x.double()
        unit = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS)
        outs.append(_exact_rotate(case, unit * w.double(), _exact_turn(case, s, False)))
    return tuple(outs)


def _exact_norm_backward(case, s):
    """Differentiated through the definition; the weight's gradient summed in 64 bits."""
    grads, weights = [], []
    for x, w, dy in ((s["q"], s["q_weight"], s["grad_q"]), (s["k"], s["k_weight"], s["grad_k"])):
        x, w = x.double(), w.double()
        g = _exact_rotate(case, dy.double(), _exact_turn(case, s, True))
        norm = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS)
        # d/dx of sum g w x / norm
        along = (g * w * x).sum(-1, keepdim=True)
        grads.append(g * w / norm - x * along / (case["dim"] * norm.pow(3)))
        weights.append((g * x / norm).flatten(0, 1).sum(0))
    return (*grads, *weights)


def _exact_cache(cache, exponents):
    scale = torch.pow(torch.full((), 2.0, dtype=torch.float64, device=DEVICE), exponents.double() - 127)
    return cache.float().double() * scale.repeat_interleave(BLOCK, -1)


def _exact_e4m3(x):
    """x rounded to four significant bits (a multiple of 2^-9 below 2^-6), halves to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(case, s):
    outs, starts, pages = [], s["page_offsets"].tolist(), s["page_indices"].tolist()
    lengths, new, page = _lengths(case), _new(case), case["page"]
    slots = [(pages[starts[b] + p // page], p % page) for b in range(case["sequences"])
             for p in range(lengths[b] - new[b], lengths[b])]
    at = torch.tensor(slots, device=DEVICE).unbind(1)
    for rows, cache in ((s["k"], s["key_cache"]), (s["v"], s["value_cache"])):
        held, x = cache.float().double(), rows.double().unflatten(-1, (-1, BLOCK))
        power = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True).clamp_min(1e-300) / 448)).clamp_min(-127)
        # log2 may be a rounding off next to a power of two: settle it with exact products
        fits = x.abs().amax(-1, keepdim=True) <= 448 * torch.exp2(power - 1)
        power = torch.where(fits & (power > -127), power - 1, power)
        power = torch.where(x.abs().amax(-1, keepdim=True) > 448 * torch.exp2(power), power + 1, power)
        held[at] = _exact_e4m3(x / torch.exp2(power)).flatten(-2)
        outs += [held, None]
    return tuple(outs)


def _exact_sequences(case, s, which):
    """Each sequence's rows of the cache, [tokens, heads, dim]."""
    held = _exact_cache(s[which + "_cache"], s[which + "_exponents"])
    for b, n in enumerate(_lengths(case)):
        first, last = s["page_offsets"][b].item(), s["page_offsets"][b + 1].item()
        yield held[s["page_indices"][first:last].long()].flatten(0, 1)[:n]


def _exact_decode(case, s):
    outs, hk = [], case["kv_heads"]
    for b, (k, v) in enumerate(zip(_exact_sequences(case, s, "key"), _exact_sequences(case, s, "value"))):
        q = s["q"][b].double().unflatten(0, (hk, -1))
        scores = q @ k.permute(1, 2, 0).contiguous() * s["scale"]
        outs.append((torch.softmax(scores, -1) @ v.transpose(0, 1).contiguous()).flatten(0, 1))
    return torch.stack(outs)


def _exact_linear(case, s):
    w = s["weight"].long()
    bits = torch.stack((w % 16, w // 16), -1).flatten(-2)
    sign, exponent, half = 1 - 2 * (bits // 8), bits // 2 % 4, bits % 2
    magnitude = torch.where(exponent == 0, half * 0.5, torch.exp2(exponent.double() - 1) * (1 + half * 0.5))
    scale = torch.exp2(s["exponents"].double() - 127)
    weight = (sign * magnitude).unflatten(-1, (-1, BLOCK)) * scale[..., None]
    return s["x"].double() @ weight.flatten(-2).t().contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "read":
        return tuple(torch.cat(list(_exact_sequences(case, s, which))) for which in ("key", "value"))
    return {"norm": _exact_norm, "norm_backward": _exact_norm_backward, "append": _exact_append, "decode": _exact_decode,
            "linear": _exact_linear}[op](case, s)
