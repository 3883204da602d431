"""The operators around block-scaled FP8 linear layers, as cases with inputs, one pass and a yardstick.

A checkpoint whose FP8 weights carry one scale for each block of 128 x 128 is served with activations that carry one scale
for each 128 consecutive values of a token.  What a decoder block then calls, and each case is one call of it:

* ``quant``: a token's values in groups of 128 to FP8, each group by its own scale;
* ``norm``: RMSNorm (with the residual added and written) and that quantisation in one pass;
* ``silu``: ``silu(gate) * up`` and that quantisation in one pass;
* ``mm``: the matrix product of such activations with such weights;
* ``rope``: the norm of each query and key head of a qkv projection's result, and the rotation by the token's position.

Sizes are those of this repository's benchmark and tests, or generic.
"""
from __future__ import annotations

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8, FP8_MAX, LEAST = torch.float8_e4m3fn, 448.0, 1e-10      # a group's largest magnitude counts as at least LEAST
GROUP = 128
MOST_FLOPS, MOST_VALUES = 9.6e11, 117_000_000      # of a drawn case: the products' operations, the other operators' values read


# ------------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # a single decode token ahead of a projection: latency
        dict(name="quant, 1 token", kind="quant", tokens=1, hidden=4096, dtype="bf16"),
        # a full prefill batch ahead of a down projection
        dict(name="quant, 4096 tokens", kind="quant", tokens=4096, hidden=14336, dtype="bf16"),
        # a served decode batch between two halves of a block
        dict(name="norm, 32 tokens", kind="norm", tokens=32, hidden=4096, residual=True, dtype="bf16"),
        # a ragged prefill batch
        dict(name="norm, 3333 tokens", kind="norm", tokens=3333, hidden=5120, residual=True, dtype="fp16"),
        # a few decode tokens, then a prefill batch, between gate/up and down projection
        dict(name="silu, 7 tokens", kind="silu", tokens=7, hidden=14336, dtype="bf16"),
        dict(name="silu, 2048 tokens", kind="silu", tokens=2048, hidden=14336, dtype="bf16"),
        # one small layer at one token: what a call costs when there is hardly any work in it
        dict(name="mm, small layer, 1 token", kind="mm", tokens=1, k=2048, n=2048, bias=False, dtype="bf16"),
        # a served decode batch through a gate/up projection
        dict(name="mm, 32 tokens", kind="mm", tokens=32, k=4096, n=28672, bias=False, dtype="bf16"),
        # a ragged prefill chunk; K ends inside a block
        dict(name="mm, 333 tokens", kind="mm", tokens=333, k=2976, n=10240, bias=True, dtype="fp16"),
        # a full prefill batch through a gate/up projection
        dict(name="mm, 4096 tokens", kind="mm", tokens=4096, k=4096, n=28672, bias=False, dtype="bf16"),
        # a served decode batch behind the qkv projection
        dict(name="rope, 32 tokens", kind="rope", tokens=32, heads_q=32, heads_k=8, head_dim=128, rotary=128, halves=True,
             cache="fp32", dtype="bf16"),
        # a ragged prefill batch; a quarter of each head rotated, neighbours in pairs
        dict(name="rope, 5001 tokens", kind="rope", tokens=5001, heads_q=40, heads_k=8, head_dim=128, rotary=32, halves=False,
             cache="fp16", dtype="fp16"),
    ]


def _log(rng, low, high, step=1):
    """A multiple of `step` between `low` and `high`, even over their logarithm."""
    v = low * (high / low) ** rng.random()
    return int(min(high, max(low, round(v / step) * step)))


def draw(rng):
    kind = rng.choice(["mm", "mm", "mm", "quant", "norm", "silu", "rope"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "mm":
        # mostly whole blocks, and layers that end inside one
        k, n = _log(rng, 512, 14336, rng.choice([128, 128, 16])), _log(rng, 512, 28672, rng.choice([128, 128, 16]))
        tokens = _log(rng, 1, max(1, min(8192, int(MOST_FLOPS / (2 * k * n)))))
        return dict(kind=kind, tokens=tokens, k=k, n=n, bias=rng.random() < 0.3, dtype=dtype)
    if kind == "rope":
        heads_k, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        heads_q = heads_k * rng.choice([1, 4, 5, 7])
        tokens = _log(rng, 1, min(8192, MOST_VALUES // ((heads_q + 2 * heads_k) * head_dim)))
        return dict(kind=kind, tokens=tokens, heads_q=heads_q, heads_k=heads_k, head_dim=head_dim,
                    rotary=rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4]), halves=rng.random() < 0.7,
                    cache=rng.choice(["fp32", dtype]), dtype=dtype)
    hidden = _log(rng, 512, 14336, rng.choice([128, 128, 8]))
    tokens = _log(rng, 1, min(8192, MOST_VALUES // (2 * hidden)))
    if kind == "norm":
        return dict(kind=kind, tokens=tokens, hidden=hidden, residual=rng.random() < 0.7, dtype=dtype)
    if kind == "quant":
        dtype = rng.choice([dtype, dtype, "fp32"])
    return dict(kind=kind, tokens=tokens, hidden=hidden, dtype=dtype)


# ------------------------------------------------------------------------------------------------ what a program has ready

def _randn(shape, gen, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _activations(shape, gen, dtype):
    """Values of a layer's input: normal, with a few channels that are much larger than the rest, as trained models have them."""
    x = torch.randn(shape, device="cuda", generator=gen)
    x[:, torch.randint(0, shape[1], (max(1, shape[1] // 256),), device="cuda", generator=gen)] *= 20.0
    return x.to(dtype)


def _blocks(x, rows):
    """FP8 codes of `x` and the scales of its blocks of `rows` x 128."""
    r, c = x.shape
    padded = torch.zeros((-(-r // rows) * rows, -(-c // GROUP) * GROUP), device=x.device)
    padded[:r, :c] = x
    b = padded.view(padded.shape[0] // rows, rows, padded.shape[1] // GROUP, GROUP)
    scale = b.abs().amax(dim=(1, 3)).clamp(min=LEAST) / FP8_MAX
    return (b / scale[:, None, :, None]).reshape(padded.shape)[:r, :c].contiguous().to(FP8), scale


def _columns(scale):
    """The same values, a group's scales of all tokens next to each other: as the quantisers of this package leave them."""
    return scale.t().contiguous().t()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, tokens, dtype = case["kind"], case["tokens"], DTYPES[case["dtype"]]
    if kind == "quant":
        return dict(kind=kind, x=_activations((tokens, case["hidden"]), gen, dtype))
    if kind == "norm":
        hidden = case["hidden"]
        s = dict(kind=kind, x=_activations((tokens, hidden), gen, dtype), weight=_randn((hidden,), gen, dtype, 0.1) + 1,
                 epsilon=1e-5, residual=None, residual_out=None)
        if case["residual"]:
            s["residual"] = _randn((tokens, hidden), gen, dtype, 4.0)
            s["residual_out"] = torch.empty_like(s["residual"])
        return s
    if kind == "silu":
        return dict(kind=kind, x=_randn((tokens, 2 * case["hidden"]), gen, dtype, 2.0))
    if kind == "mm":
        k, n = case["k"], case["n"]
        a, scale_a = _blocks(_activations((tokens, k), gen, torch.float32), 1)
        w, scale_w = _blocks(_randn((n, k), gen, scale=0.02) * (1 + torch.rand((n, 1), device="cuda", generator=gen)), GROUP)
        return dict(kind=kind, a=a, scale_a=_columns(scale_a), w=w.t(), scale_w=scale_w.t(), dtype=dtype,
                    bias=_randn((n,), gen, dtype, 0.1) if case["bias"] else None)
    hq, hk, d, rotary = case["heads_q"], case["heads_k"], case["head_dim"], case["rotary"]
    length = 8192
    angle = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    return dict(kind=kind, qkv=_randn((tokens, (hq + 2 * hk) * d), gen, dtype, 3.0), heads_q=hq, heads_k=hk, head_dim=d,
                epsilon=1e-6, q_weight=_randn((d,), gen, dtype, 0.1) + 1, k_weight=_randn((d,), gen, dtype, 0.1) + 1,
                cache=torch.cat((angle.cos(), angle.sin()), dim=1).to(DTYPES[case["cache"]]), halves=case["halves"],
                positions=torch.randint(0, length, (tokens,), device="cuda", generator=gen))


# ------------------------------------------------------------------------------------------------------------ plain forms

def _grouped(y):
    """Codes and scales of fp32 values in groups of 128; the last group may be shorter."""
    t, h = y.shape
    rest = -h % GROUP
    g = torch.nn.functional.pad(y, (0, rest)).view(t, -1, GROUP)
    scale = g.abs().amax(dim=2).clamp(min=LEAST) / FP8_MAX
    codes = (g / scale[:, :, None]).view(t, -1)[:, :h]
    return codes.to(FP8), scale


def _spread(scale, rows, columns):
    """Scales of blocks as one for each value."""
    return scale.repeat_interleave(rows, dim=0).repeat_interleave(columns, dim=1)


def _plain_mm(s):
    a, w = s["a"], s["w"]
    (m, k), n = a.shape, w.shape[1]
    x = a.float() * _spread(s["scale_a"], 1, GROUP)[:, :k]
    y = w.float() * _spread(s["scale_w"], GROUP, GROUP)[:k, :n]
    out = x @ y
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(s["dtype"])


def _plain_rope(s):
    d, halves, t = s["head_dim"], s["halves"], s["qkv"].shape[0]
    cos, sin = s["cache"][s["positions"]].float().chunk(2, dim=1)
    cos, sin, half = cos[:, None], sin[:, None], cos.shape[1]

    def one(x, weight):
        x = x.float().view(t, -1, d)
        x = x * torch.rsqrt(x.square().mean(dim=2, keepdim=True) + s["epsilon"]) * weight.float()
        turned, kept = x[..., :2 * half], x[..., 2 * half:]
        u, v = (turned[..., :half], turned[..., half:]) if halves else (turned[..., 0::2], turned[..., 1::2])
        u, v = u * cos - v * sin, v * cos + u * sin
        turned = torch.cat((u, v), dim=2) if halves else torch.stack((u, v), dim=3).flatten(2)
        return torch.cat((turned, kept), dim=2).to(s["qkv"].dtype)

    nq, nk = s["heads_q"] * d, s["heads_k"] * d
    return one(s["qkv"][:, :nq], s["q_weight"]), one(s["qkv"][:, nq:nq + nk], s["k_weight"])


def _plain(s):
    kind = s["kind"]
    if kind == "mm":
        return _plain_mm(s)
    if kind == "rope":
        return _plain_rope(s)
    if kind == "quant":
        return _grouped(s["x"].float())
    if kind == "silu":
        gate, up = s["x"].float().chunk(2, dim=1)
        return _grouped(gate / (1 + torch.exp(-gate)) * up)
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    codes, scale = _grouped(x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + s["epsilon"]) * s["weight"].float())
    return (codes, scale) if s["residual"] is None else (codes, scale, x.to(s["x"].dtype))


# -------------------------------------------------------------------------------------------------------------- one pass

def _own(s):
    from vllm_amd import _custom_ops as ops
    kind = s["kind"]
    if kind == "mm":
        return ops.block_scaled_mm(s["a"], s["w"], s["scale_a"], s["scale_w"], s["dtype"], s["bias"])
    if kind == "rope":
        return ops.qk_norm_rope(s["qkv"], s["heads_q"], s["heads_k"], s["head_dim"], s["epsilon"], s["q_weight"], s["k_weight"],
                                s["cache"], s["positions"], s["halves"])
    if kind == "quant":
        return ops.scaled_fp8_group_quant(s["x"])
    if kind == "silu":
        return ops.silu_and_mul_group_quant(s["x"])
    codes, scale = ops.rms_norm_group_quant(s["x"], s["weight"], s["epsilon"], s["residual"], s["residual_out"])
    return (codes, scale) if s["residual"] is None else (codes, scale, s["residual_out"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------ yardsticks

def work(case):
    kind, t = case["kind"], case["tokens"]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind == "mm":
        k, n = case["k"], case["n"]
        gk, gn = -(-k // GROUP), -(-n // GROUP)
        total = t * k + k * n + 4 * (t + gn) * gk + 2 * t * n + (2 * n if case["bias"] else 0)
        return {"bytes": total, "flops": 2 * t * n * k}
    if kind == "rope":
        values, d = t * (case["heads_q"] + case["heads_k"]) * case["head_dim"], case["head_dim"]
        rows = min(t, 8192) * case["rotary"] * (4 if case["cache"] == "fp32" else 2)
        return {"bytes": 4 * values + rows + 8 * t + 4 * d, "flops": 10 * values}
    h = case["hidden"]
    codes = t * h + 4 * t * -(-h // GROUP)
    if kind == "quant":
        return {"bytes": size * t * h + codes, "flops": 3 * t * h}
    if kind == "silu":
        return {"bytes": 4 * t * h + codes, "flops": 8 * t * h}
    return {"bytes": (6 if case["residual"] else 2) * t * h + 2 * h + codes, "flops": 8 * t * h}


# ------------------------------------------------------------------------------------------------------- in 64 bits

def _exact_groups(y):
    """(values a group's codes round, scale) from the definition: a value over its group's largest magnitude, times 448."""
    t, h = y.shape
    scale = torch.empty((t, -(-h // GROUP)), dtype=torch.float64, device=y.device)
    value = torch.empty_like(y)
    for g in range(scale.shape[1]):
        part = y[:, g * GROUP:(g + 1) * GROUP]
        scale[:, g] = part.abs().max(dim=1).values.clamp(min=LEAST) / FP8_MAX
        value[:, g * GROUP:(g + 1) * GROUP] = part / scale[:, g:g + 1]
    return value, scale


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "quant":
        return _exact_groups(s["x"].double())
    if kind == "silu":
        h = case["hidden"]
        gate, up = s["x"][:, :h].double(), s["x"][:, h:].double()
        return _exact_groups(gate * torch.sigmoid(gate) * up)
    if kind == "norm":
        x = s["x"].double()
        if s["residual"] is not None:
            x = x + s["residual"].double()
        rms = ((x ** 2).sum(dim=1, keepdim=True) / case["hidden"] + s["epsilon"]) ** 0.5
        value, scale = _exact_groups(x / rms * s["weight"].double())
        return (value, scale) if s["residual"] is None else (value, scale, x)
    if kind == "mm":
        a, w = s["a"].double(), s["w"].double()
        out = torch.zeros((case["tokens"], case["n"]), dtype=torch.float64, device=a.device)
        for i in range(s["scale_a"].shape[1]):      # block by block of K: product, then the two scales
            rows = slice(i * GROUP, (i + 1) * GROUP)
            columns = s["scale_w"][i].double()[torch.arange(case["n"], device=a.device) // GROUP]
            out += (a[:, rows] @ w[rows]) * s["scale_a"][:, i, None].double() * columns
        return out if s["bias"] is None else out + s["bias"].double()
    d, rotary, t = case["head_dim"], case["rotary"], case["tokens"]
    turn = torch.complex(*(s["cache"][s["positions"], i * rotary // 2:(i + 1) * rotary // 2].double() for i in range(2)))[:, None]
    outs, first = [], 0
    for heads, weight in ((case["heads_q"], s["q_weight"]), (case["heads_k"], s["k_weight"])):
        x = s["qkv"][:, first:first + heads * d].double().reshape(t, heads, d)
        first += heads * d
        x = x / ((x ** 2).sum(dim=2, keepdim=True) / d + s["epsilon"]) ** 0.5 * weight.double()
        real, imag = ((slice(0, rotary // 2), slice(rotary // 2, rotary)) if s["halves"] else (slice(0, rotary, 2), slice(1, rotary, 2)))
        z = torch.complex(x[..., real].contiguous(), x[..., imag].contiguous()) * turn
        x[..., real], x[..., imag] = z.real, z.imag
        outs.append(x)
    return tuple(outs)
