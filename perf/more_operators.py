"""What the rest of a decoder layer is measured on when its products run in 8-bit integers and its batch shares a prompt's
prefix, and the training pass of the layer's norm: the calls that a user's program makes of the operators, and the same in
elementary torch operations.

The parts: the norm of the residual stream after a block's output has joined it (its own norm, gate and scales included) and its
gradients, the product of 8-bit integers with a scale for each token and channel, from rows that are given in 8 bits or made so
(a projection: plain rows, the norm's, or the gated product of a feed-forward block), and the attention of one new token per
sequence over a prefix that all sequences share and what each has of its own.
"""
import functools
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
RESIDUAL_SCALE, BLOCK_SCALE = 0.75, 1.25


def listed():
    return [
        # One decode step of 8 sequences, pre-norm: the smallest call, latency is all of it.
        {"name": "norm_step", "op": "norm", "dtype": "f16", "tokens": 8, "dim": 4096, "post": False, "gated": False},
        # A training batch of 4 sequences of 4096 tokens, norms on both sides of a gated block.
        {"name": "norm_batch", "op": "norm", "dtype": "bf16", "tokens": 16384, "dim": 4096, "post": True, "gated": True},
        # Its backward pass.
        {"name": "norm_backward_batch", "op": "norm_backward", "dtype": "bf16", "tokens": 16384, "dim": 4096, "post": True,
         "gated": True},
        # A fine-tuning step over a ragged number of tokens of a narrow model.
        {"name": "norm_backward_ragged", "op": "norm_backward", "dtype": "f16", "tokens": 1021, "dim": 2304, "post": False,
         "gated": True},
        # A feed-forward product of one token whose row is there in 8 bits.
        {"name": "product_row", "op": "product", "dtype": "f16", "m": 1, "n": 14336, "k": 4096, "bias": False},
        # The way back, of a step of 32 sequences.
        {"name": "product_step", "op": "product", "dtype": "bf16", "m": 32, "n": 4096, "k": 14336, "bias": True},
        # The same of a packed prompt.
        {"name": "product_prompt", "op": "product", "dtype": "f16", "m": 4096, "n": 14336, "k": 4096, "bias": False},
        # The attention's heads of 32 sequences, made 8 bits and projected.
        {"name": "project_heads", "op": "project", "source": "rows", "dtype": "f16", "m": 32, "n": 4096, "k": 4096,
         "bias": False},
        # Queries, keys and values of a prompt from the stream's norm.
        {"name": "project_norm", "op": "project", "source": "norm", "dtype": "bf16", "m": 1021, "n": 6144, "k": 4096,
         "bias": True, "post": True, "gated": False},
        # The way back of a prompt's feed-forward block from its gate and up halves.
        {"name": "project_gated", "op": "project", "source": "gated", "dtype": "bf16", "m": 1021, "n": 4096, "k": 14336,
         "bias": False},
        # One step of 8 sequences that share a long prompt and have a few hundred tokens of their own.
        {"name": "prefix_step", "op": "prefix", "dtype": "f16", "sequences": 8, "prefix": 8191, "longest": 512, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "head_major": False},
        # One step of a full server: 64 sequences from one token to 1000 of their own behind a prefix of 16384.
        {"name": "prefix_server", "op": "prefix", "dtype": "bf16", "sequences": 64, "prefix": 16384, "longest": 1000,
         "heads": 64, "kv_heads": 8, "dim": 128, "page": 16, "head_major": True},
    ]


# ------------------------------------------------------------------------------------------ drawing
def _spread(rng, low, high, multiple=1):
    """A size between low and high, even over its logarithm, a multiple of `multiple`."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high // multiple, max(-(-low // multiple), round(value / multiple))) * multiple


def draw(rng):
    """One more case: token counts, lengths and batches are arbitrary, widths are those of models."""
    op = rng.choice(["norm", "norm_backward", "product", "project", "prefix"])
    dtype = rng.choice(["f16", "bf16"])
    if op in ("norm", "norm_backward"):
        dim = _spread(rng, 256, 8192, rng.choice([1, 8, 64, 256]))
        tokens = min(_spread(rng, 1, 16384), 16384 * 4096 // dim)
        return {"op": op, "dtype": dtype, "tokens": tokens, "dim": dim, "post": rng.random() < 0.5, "gated": rng.random() < 0.5}
    if op in ("product", "project"):
        n, k = _spread(rng, 512, 16384, rng.choice([1, 8, 16])), _spread(rng, 512, 16384, rng.choice([16, 64]))
        most = max(1, 4096 * 14336 * 4096 // (n * k))
        case = {"op": op, "dtype": dtype, "m": min(most, _spread(rng, 1, rng.choice([16, 128, 4096]))), "n": n, "k": k,
                "bias": rng.random() < 0.5}
        if op == "project":
            case["source"] = rng.choice(["rows", "norm", "gated"])
            if case["source"] == "norm":
                case["post"], case["gated"] = rng.random() < 0.5, rng.random() < 0.5
        return case
    kv_heads, group = rng.choice([(8, 4), (4, 8), (8, 8), (2, 4), (16, 1), (1, 16), (5, 3), (8, 1)])
    case = {"op": op, "dtype": dtype, "sequences": _spread(rng, 1, 64), "prefix": _spread(rng, 16, 16384),
            "longest": _spread(rng, 1, 1000), "heads": kv_heads * group, "kv_heads": kv_heads,
            "dim": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 64]), "head_major": rng.random() < 0.5}
    return case


# ------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(DTYPES[dtype])


def _table(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _uniform(g, shape, low, high):
    return low + (high - low) * torch.rand(shape, generator=g, device=DEVICE)


def _lengths(case):
    """Own tokens of each sequence, the longest among them: part of the case, not of its inputs."""
    count, longest = case["sequences"], case["longest"]
    rng = random.Random(count * 8191 + longest)
    return [longest] + [rng.randint(1, longest) for _ in range(count - 1)]


def _sums(values):
    out = [0]
    for value in values:
        out.append(out[-1] + value)
    return out


def _norm_inputs(g, s, tokens, dim, dtype):
    """A block's output, the stream before it, the gates of its tokens (none: length 0) and the norms' weights."""
    s["block"], s["residual"] = _normal(g, (tokens, dim), dtype), _normal(g, (tokens, dim), dtype, 2)
    s["gate"] = torch.sigmoid(torch.randn((tokens if s["gated"] else 0,), generator=g, device=DEVICE))
    s["post_weight"] = 1 + 0.2 * torch.randn((dim if s["post"] else 0,), generator=g, device=DEVICE)
    s["weight"] = 1 + 0.2 * torch.randn((dim,), generator=g, device=DEVICE)


def prepare(case, seed):
    g, op, dtype = _generator(seed), case["op"], case["dtype"]
    s = dict(case)
    if op in ("norm", "norm_backward"):
        shape = (case["tokens"], case["dim"])
        _norm_inputs(g, s, *shape, dtype)
        if op == "norm_backward":
            s["sum"] = _plain_sum(s).to(DTYPES[dtype])
            s["grad_sum"], s["grad_output"] = _normal(g, shape, dtype), _normal(g, shape, dtype)
        return s
    if op in ("product", "project"):
        m, n, k = case["m"], case["n"], case["k"]
        s["weight_i8"] = torch.randint(-127, 128, (n, k), generator=g, device=DEVICE, dtype=torch.int8)
        s["weight_scales"] = _uniform(g, (n,), 0.5, 2) / (73 * math.sqrt(k))
        s["bias_values"] = torch.randn((n if case["bias"] else 0,), generator=g, device=DEVICE)
        if op == "product":
            s["x"] = torch.randint(-127, 128, (m, k), generator=g, device=DEVICE, dtype=torch.int8)
            s["x_scales"] = _uniform(g, (m,), 0.5, 2) / 73
        elif case["source"] == "rows":
            s["x"] = _normal(g, (m, k), dtype)
        elif case["source"] == "gated":
            s["halves"] = _normal(g, (m, 2 * k), dtype, 1.5)          # one projection's rows: gate, then up
        else:
            _norm_inputs(g, s, m, k, dtype)
        return s
    hk, dim, page = case["kv_heads"], case["dim"], case["page"]
    # Pages of the prefix and of the sequences are scattered over one cache; the prefix need not fill its last page.
    held = -(-case["prefix"] // page)
    offsets = _sums(-(-n // page) for n in _lengths(case))
    where = torch.randperm(held + offsets[-1], generator=g, device=DEVICE).to(torch.int32)
    s["prefix_indices"], s["page_indices"] = where[:held].clone(), where[held:].clone()
    s["prefix_length"], s["page_offsets"] = _table([case["prefix"]]), _table(offsets)
    s["lengths"] = _table(_lengths(case))
    shape = (held + offsets[-1], hk, page, dim) if case["head_major"] else (held + offsets[-1], page, hk, dim)
    for name in ("key_cache", "value_cache"):
        rows = _normal(g, shape, dtype)
        s[name] = rows.transpose(1, 2) if case["head_major"] else rows
    s["q"] = _normal(g, (case["sequences"], case["heads"], dim), dtype, 1.5)
    s["scale"] = dim ** -0.5
    s["most"] = max(_lengths(case))
    return s


# ------------------------------------------------------------------------------------------ the framework's calls
@functools.lru_cache(maxsize=None)
def _kernel(name, **constexprs):
    """A program jits a definition once and keeps the kernel."""
    import intent_amd as intent
    from intent_amd.examples.kernels.backward import residual_norm as backward
    from intent_amd.examples.kernels.contraction import linear_i8
    from intent_amd.examples.kernels.normalization import quantize_rows, residual_norm
    from intent_amd.examples.kernels.streaming import prefix_decode

    for module in (residual_norm, backward, quantize_rows, linear_i8, prefix_decode):
        if hasattr(module, name):
            return intent.jit(getattr(module, name), backend="hip", constexprs=constexprs)
    raise LookupError(name)


def _called(s, repeated, kernel, *arguments, name="call"):
    """A decode loop prepares a call for its buffers once and launches it every step; a batch or a prompt comes once."""
    if not repeated:
        return kernel.run(*arguments)
    if name not in s:
        s[name] = kernel.prepare(*arguments)
    s[name].launch()
    return s[name].result()


def _call(s):
    op, dtype = s["op"], s["dtype"]
    scales = (RESIDUAL_SCALE, BLOCK_SCALE, EPS)
    if op == "norm":
        return _called(s, s["tokens"] <= 128, _kernel("residual_norm_" + dtype), s["block"], s["residual"], s["gate"],
                       s["post_weight"], s["weight"], *scales)
    if op == "norm_backward":
        return _kernel("residual_norm_backward_" + dtype).run(
            s["block"], s["sum"], s["gate"], s["post_weight"], s["weight"], s["grad_sum"], s["grad_output"], *scales)
    if op == "prefix":
        return _called(s, True, _kernel("paged_gqa_decode_prefix_" + dtype, HEAD_GROUP=s["heads"] // s["kv_heads"]), s["q"],
                       s["key_cache"], s["value_cache"], s["prefix_indices"], s["prefix_length"], s["page_offsets"],
                       s["page_indices"], s["lengths"], s["scale"])
    repeated, outputs = s["m"] <= 128, ()
    if op == "product":
        rows, row_scales = s["x"], s["x_scales"]
    elif s["source"] == "rows":
        rows, row_scales = _called(s, repeated, _kernel("quantize_rows_" + dtype), s["x"], name="rows")
    elif s["source"] == "gated":
        halves = s["halves"]
        rows, row_scales = _called(s, repeated, _kernel("swiglu_quantize_rows_" + dtype), halves[:, :s["k"]], halves[:, s["k"]:],
                                   name="rows")
    else:
        total, rows, row_scales = _called(s, repeated, _kernel("residual_norm_i8_" + dtype), s["block"], s["residual"],
                                          s["gate"], s["post_weight"], s["weight"], *scales, name="rows")
        outputs = (total,)
    return (*outputs, _called(s, repeated, _kernel("linear_i8_" + dtype), rows, s["weight_i8"], row_scales, s["weight_scales"],
                              s["bias_values"]))


# ------------------------------------------------------------------------------------------ the plain forms
def _plain_unit(x):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _plain_branch(s):
    """The block's output under its own norm, and its factor."""
    branch = s["block"].float()
    if s["post"]:
        branch = _plain_unit(branch) * s["post_weight"]
    return branch, BLOCK_SCALE * s["gate"][:, None] if s["gated"] else BLOCK_SCALE


def _plain_sum(s):
    branch, factor = _plain_branch(s)
    return RESIDUAL_SCALE * s["residual"].float() + factor * branch


def _plain_norm(s):
    total, t = _plain_sum(s), DTYPES[s["dtype"]]
    return total.to(t), (_plain_unit(total) * s["weight"]).to(t)


def _unit_gradient(x, g):
    """The gradient of x that unit(x) passes on from g."""
    inverse = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    unit = x * inverse
    return inverse * (g - unit * (g * unit).mean(-1, keepdim=True))


def _plain_norm_backward(s):
    t, total, grad = DTYPES[s["dtype"]], s["sum"].float(), s["grad_output"].float()
    # The weights' gradients sum over every token, so in 64 bits.
    grad_weight = (grad * _plain_unit(total)).sum(0, dtype=torch.float64).float()
    grad_total = s["grad_sum"].float() + _unit_gradient(total, grad * s["weight"])
    branch, factor = _plain_branch(s)
    grad_gate = BLOCK_SCALE * (grad_total * branch).sum(-1) if s["gated"] else s["gate"]
    grad_block, grad_post = factor * grad_total, s["post_weight"]
    if s["post"]:
        block = s["block"].float()
        grad_post = (grad_block * _plain_unit(block)).sum(0, dtype=torch.float64).float()
        grad_block = _unit_gradient(block, grad_block * s["post_weight"])
    return grad_block.to(t), (RESIDUAL_SCALE * grad_total).to(t), grad_gate, grad_post, grad_weight


def _plain_quantised(x):
    """Whole numbers and the scale of each row; in 64 bits, since a value next to a border is a whole step."""
    x = x.double()
    most = x.abs().amax(-1, keepdim=True)
    return torch.round(x * 127 / torch.where(most > 0, most, 1)).float(), (most / 127).float()


def _plain_product(rows, row_scales, s):
    y = (rows @ s["weight_i8"].float().t()) * row_scales * s["weight_scales"]
    return (y + s["bias_values"] if s["bias"] else y).to(DTYPES[s["dtype"]])


def _plain_project(s):
    if s["op"] == "product":
        return (_plain_product(s["x"].float(), s["x_scales"][:, None], s),)
    if s["source"] == "rows":
        return (_plain_product(*_plain_quantised(s["x"]), s),)
    if s["source"] == "gated":
        gate, up = s["halves"].double().split(s["k"], 1)
        return (_plain_product(*_plain_quantised(gate / (1 + torch.exp(-gate)) * up), s),)
    total = _plain_sum(s)
    return total.to(DTYPES[s["dtype"]]), _plain_product(*_plain_quantised(_plain_unit(total) * s["weight"]), s)


def _slots(pages, position, page):
    return pages.long()[position // page], position % page


def _plain_prefix(s):
    hk, page = s["kv_heads"], s["page"]
    own = torch.arange(s["most"], device=DEVICE)
    live = own < s["lengths"][:, None]                                                       # [B, T]
    at = s["page_offsets"].long()[:-1, None] + torch.where(live, own, 0) // page
    own_slots = s["page_indices"].long()[at], own.expand_as(live) % page
    shared_slots = _slots(s["prefix_indices"], torch.arange(s["prefix"], device=DEVICE), page)
    q = s["q"].float().unflatten(1, (hk, -1))                                                # [B, HK, G, D]

    def read(cache):
        # [HK, T, D] of the prefix, [B, HK, T, D] of the sequences
        return cache[shared_slots].float().transpose(0, 1).contiguous(), cache[own_slots].float().transpose(1, 2).contiguous()

    (shared_keys, own_keys), (shared_values, own_values) = read(s["key_cache"]), read(s["value_cache"])
    rows = q.transpose(0, 1).flatten(1, 2)                                                   # [HK, B G, D]
    shared = (shared_keys @ rows.transpose(1, 2).contiguous()).transpose(1, 2) * s["scale"]
    shared = shared.unflatten(1, (s["sequences"], -1)).transpose(0, 1)                       # [B, HK, G, T]
    owned = (own_keys @ q.transpose(2, 3).contiguous()).transpose(2, 3) * s["scale"]
    owned = owned.masked_fill(~live[:, None, None], -math.inf)
    peak = torch.maximum(shared.amax(-1, keepdim=True), owned.amax(-1, keepdim=True))
    shared, owned = torch.exp(shared - peak), torch.exp(owned - peak)
    mixed = (shared.transpose(0, 1).flatten(1, 2) @ shared_values).unflatten(1, (s["sequences"], -1)).transpose(0, 1)
    out = (mixed + owned @ own_values) / (shared.sum(-1, keepdim=True) + owned.sum(-1, keepdim=True))
    return out.flatten(1, 2).to(DTYPES[s["dtype"]])


def _plain(s):
    return {"norm": _plain_norm, "norm_backward": _plain_norm_backward, "product": _plain_project, "project": _plain_project,
            "prefix": _plain_prefix}[s["op"]](s)


def run(state):
    return _call(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op in ("norm", "norm_backward"):
        tokens, dim = case["tokens"], case["dim"]
        once = 4 * dim * (2 if case["post"] else 1) + (4 * tokens if case["gated"] else 0)
        if op == "norm":
            return {"bytes": 8 * tokens * dim + once, "flops": tokens * dim * (14 if case["post"] else 9)}
        return {"bytes": 12 * tokens * dim + 2 * once, "flops": tokens * dim * (30 if case["post"] else 18)}
    if op in ("product", "project"):
        m, n, k = case["m"], case["n"], case["k"]
        source = case.get("source")
        rows = {None: m * k, "rows": 2 * m * k, "gated": 4 * m * k, "norm": 6 * m * k}[source]
        return {"bytes": n * k + rows + 2 * m * n + 4 * (n * (2 if case["bias"] else 1) + m), "flops": 2 * m * n * k}
    tokens = sum(_lengths(case))
    rows = case["heads"] * case["dim"]
    return {"bytes": 4 * (case["prefix"] + tokens) * case["kv_heads"] * case["dim"] + 4 * case["sequences"] * rows,
            "flops": 4 * (case["prefix"] * case["sequences"] + tokens) * rows}


# ------------------------------------------------------------------------------------------ exact results
def _exact_total(s):
    x = s["block"].double()
    if s["post"]:
        x = x * s["post_weight"].double() / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[1] + EPS)
    if s["gated"]:
        x = x * s["gate"].double()[:, None]
    return s["residual"].double() * RESIDUAL_SCALE + x * BLOCK_SCALE


def _exact_normed(x, weight):
    return x * weight.double() / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[1] + EPS)


def _exact_norm_backward(s):
    """Differentiated through the definition by hand: of y = w x / n(x) with n = sqrt(mean x^2 + eps)."""
    def through(x, weight, g):
        n = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[1] + EPS)
        along = (g * weight * x).sum(-1, keepdim=True)
        return g * weight / n - x * along / (x.shape[1] * n.pow(3)), (g * x / n).sum(0)

    into, grad_weight = through(s["sum"].double(), s["weight"].double(), s["grad_output"].double())
    into = into + s["grad_sum"].double()
    block = s["block"].double()
    branch = _exact_normed(block, s["post_weight"]) if s["post"] else block
    grad_gate, grad_post = s["gate"], s["post_weight"]
    down = into * BLOCK_SCALE
    if s["gated"]:
        grad_gate = (down * branch).sum(-1)
        down = down * s["gate"].double()[:, None]
    if s["post"]:
        down, grad_post = through(block, s["post_weight"].double(), down)
    return down, into * RESIDUAL_SCALE, grad_gate, grad_post, grad_weight


def _exact_product(s):
    outputs = ()
    if s["op"] == "product":
        whole, scales = s["x"].double(), s["x_scales"].double()[:, None]
    else:
        if s["source"] == "rows":
            x = s["x"].double()
        elif s["source"] == "gated":
            gate, up = s["halves"][:, :s["k"]].double(), s["halves"][:, s["k"]:].double()
            x = gate * torch.sigmoid(gate) * up
        else:
            total = _exact_total(s)
            outputs, x = (total,), _exact_normed(total, s["weight"])
        most = x.abs().max(1, keepdim=True).values
        whole, scales = torch.round(127 * x / most), most / 127        # to even between two
    y = (whole @ s["weight_i8"].double().t().contiguous()) * scales * s["weight_scales"].double()
    return (*outputs, y + s["bias_values"].double() if s["bias"] else y)


def _exact_prefix(case, s):
    hk, page = case["kv_heads"], case["page"]

    def rows(cache, pages, count):
        return cache[pages.long()].flatten(0, 1)[:count].double().transpose(0, 1)             # [HK, T, D]

    shared = [rows(s[name], s["prefix_indices"], case["prefix"]) for name in ("key_cache", "value_cache")]
    offsets, outs = s["page_offsets"].tolist(), []
    for b, count in enumerate(_lengths(case)):
        pages = s["page_indices"][offsets[b]:offsets[b + 1]]
        k, v = (torch.cat((old, rows(s[name], pages, count)), 1) for old, name in zip(shared, ("key_cache", "value_cache")))
        scores = s["q"][b].double().unflatten(0, (hk, -1)) @ k.transpose(1, 2).contiguous() * s["scale"]
        outs.append((torch.softmax(scores, -1) @ v.contiguous()).flatten(0, 1))
    return torch.stack(outs)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        total = _exact_total(s)
        return total, _exact_normed(total, s["weight"])
    if op == "norm_backward":
        return _exact_norm_backward(s)
    return _exact_prefix(case, s) if op == "prefix" else _exact_product(s)
